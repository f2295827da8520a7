"""Element offsets past 31 and 32 bits in the feed-forward side of a block.  Rows are
zero but for groups at the start, in the middle, across the boundary and at the end:
what a wrapped offset reads or writes shows in one of them, and the zero rows add
nothing to the weights' gradients."""
import pytest
import torch

from ffn_ref import assert_within, block_norm64, block_norm_bwd64, dropout_mult, gated_ffn64
from helpers import seeded_normal

pytestmark = pytest.mark.gpu

EPS = 1e-5


@pytest.fixture(autouse=True)
def _memory(cuda_device):
    if torch.cuda.get_device_properties(cuda_device).total_memory < 64 << 30:
        pytest.skip("needs 64 GB of device memory")
    yield
    torch.cuda.empty_cache()


def _rows(m, boundary):
    starts = (0, m // 2, boundary - 8, m - 16)
    return torch.cat([torch.arange(s, s + 16) for s in starts])


def _spread(m, cols, at, seed, dev):
    t = torch.zeros(m, cols, dtype=torch.bfloat16, device=dev)
    t[at.to(dev)] = seeded_normal((len(at), cols), seed, dev)
    return t


def test_gated_ffn(cuda_device):
    import teenyformers_b200 as tfb
    dev, m, d, F = cuda_device, 80003, 2048, 14336   # z: 2.3e9 elements
    at = _rows(m, (1 << 31) // (2 * F))
    x, dy = _spread(m, d, at, 1, dev), _spread(m, d, at, 2, dev)
    w1 = (seeded_normal((2 * F, d), 3, dev, torch.float32) / d ** 0.5).bfloat16()
    w2 = (seeded_normal((d, F), 4, dev, torch.float32) / F ** 0.5).bfloat16()
    at = at.to(dev)
    ref = gated_ffn64(x[at], w1, w2, "silu", dy=dy[at])
    y, z = tfb.gated_ffn(x, w1, w2, save=True)
    assert_within("z", z[at], ref["z"])
    assert_within("y", y[at], ref["y"])
    assert torch.count_nonzero(y).item() == torch.count_nonzero(y[at]).item()
    got = dict(zip(("dx", "dw_gate_up", "dw_down"), tfb.gated_ffn_bwd(x, w1, w2, z, dy)))
    got["dx"] = got["dx"][at]
    for name, t in got.items():
        assert_within(name, t, ref[name])
    assert tfb.device_status() == 0


def test_block_norm(cuda_device):
    import teenyformers_b200 as tfb
    dev, cols = cuda_device, 4096
    boundary = (1 << 31) // cols
    rows = boundary + 37
    at = _rows(rows, boundary)
    rng = tfb.dropout_rng(11, 5, dev)
    mult = torch.stack([torch.from_numpy(dropout_mult(cols, 0.1, rng, 6, start=int(r) * cols))
                        for r in at]).to(dev)
    x, f = _spread(rows, cols, at, 1, dev), _spread(rows, cols, at, 2, dev)
    wp, wn = ((1.0 + 0.1 * seeded_normal((cols,), k, dev, torch.float32)).bfloat16() for k in (3, 4))
    idx = at.to(dev)
    kw = dict(p=0.1, rng=rng, site=6)
    y, h = tfb.block_norm(x, f, wp, None, wn, eps=EPS, **kw)
    ry, rh = block_norm64(x[idx], f[idx], wp, None, wn, EPS, 1.0, 1.0, mult)
    assert_within("y", y[idx], ry)
    assert_within("h", h[idx], rh)
    del x, h
    dy, dh = _spread(rows, cols, at, 5, dev), _spread(rows, cols, at, 6, dev)
    got = dict(zip(("dx", "df", "dw_post", "dgate", "dw_pre"),
                   tfb.block_norm_bwd(f, y, dy, dh, wp, None, wn, eps=EPS, **kw)))
    ref = block_norm_bwd64(f[idx], y[idx], dy[idx], dh[idx], wp, None, wn, EPS, 1.0, 1.0, mult)
    for name, want in ref.items():
        assert_within(name, got[name][idx] if name in ("dx", "df") else got[name], want)
    assert tfb.device_status() == 0


def test_dropout(cuda_device):
    import teenyformers_b200 as tfb
    n, run = (1 << 32) + 21, 4096
    x = torch.zeros(n, dtype=torch.bfloat16, device=cuda_device)
    starts = (0, (1 << 31) - 64, (1 << 32) - 2048, n // 8 * 8 - 64)
    vals = seeded_normal((len(starts), run), 3, cuda_device)
    for s, v in zip(starts, vals):
        x[s:s + run] = v[:n - s] if s + run > n else v
    want = [x[s:s + run].clone() for s in starts]
    rng = tfb.dropout_rng(3, 1, cuda_device)
    tfb.dropout(x, 0.25, rng, site=9, out=x)
    for s, v in zip(starts, want):
        mult = torch.from_numpy(dropout_mult(v.numel(), 0.25, rng, 9, start=s)).to(cuda_device)
        # one fp32 product of exact factors, rounded to bf16
        assert torch.equal(x[s:s + run], (v.float() * mult.float()).bfloat16()), s
    assert tfb.device_status() == 0
