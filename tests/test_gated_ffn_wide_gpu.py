"""The gradient product of a short K in whole 256-column tiles (more tiles than half the CTA
pairs, d_model below 1985), ragged in every direction, and with offsets past 31 bits; the
2-norm of the error for all activations."""
import math

import pytest
import torch

from ffn_ref import U, assert_within, gated_ffn64, rel_l2
from helpers import seeded_normal

pytestmark = pytest.mark.gpu

NAMES = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _inputs(m, d, F, dev, seed=0):
    x = seeded_normal((m, d), seed, dev)
    w1 = (seeded_normal((2 * F, d), seed + 1, dev, torch.float32) * (1.28 / math.sqrt(d))).bfloat16()
    w2 = (seeded_normal((d, F), seed + 2, dev, torch.float32) * (1.28 / math.sqrt(F))).bfloat16()
    return x, w1, w2


@pytest.mark.parametrize("m,d,F", [(1030, 520, 2568), (2100, 1032, 1416), (2561, 72, 1032)])
@pytest.mark.parametrize("act", list(NAMES))
def test_wide_tiles(cuda_device, m, d, F, act):
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, d, F, cuda_device, seed=m)
    dy = seeded_normal((m, d), 78, cuda_device)
    ref = gated_ffn64(x, w1, w2, act, dy=dy)
    y, z = tfb.gated_ffn(x, w1, w2, NAMES[act], save=True)
    bufs = [torch.full((t.shape[0] + 2, t.shape[1]), float("nan"), dtype=torch.bfloat16,
                       device=cuda_device) for t in (x, w1, w2)]
    got = tfb.gated_ffn_bwd(x, w1, w2, z, dy, NAMES[act], grads=[b[1:-1] for b in bufs])
    assert_within("y", y, ref["y"])
    for name, t in zip(("dx", "dw_gate_up", "dw_down"), got):
        assert_within(name, t, ref[name])
    for b in bufs:
        assert torch.isnan(b[0]).all() and torch.isnan(b[-1]).all()
    assert tfb.device_status() == 0


@pytest.mark.parametrize("m,d,F", [(1024, 512, 1408), (4096, 1024, 2048), (2048, 2048, 1408)])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
def test_error_is_that_of_two_roundings(cuda_device, m, d, F, act):
    """A rounding's error is at most U / sqrt(3) in the 2-norm, relative, and each result has
    its own and its bf16 operand's."""
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, d, F, cuda_device, seed=5)
    dy = seeded_normal((m, d), 6, cuda_device)
    ref = gated_ffn64(x, w1, w2, act, dy=dy)
    y, z = tfb.gated_ffn(x, w1, w2, NAMES[act], save=True)
    got = dict(zip(("dx", "dw_gate_up", "dw_down"), tfb.gated_ffn_bwd(x, w1, w2, z, dy, NAMES[act])),
               y=y)
    for name, t in got.items():
        assert rel_l2(t, ref[name][0]) <= math.sqrt(2) * U / math.sqrt(3), name


def test_offsets_past_31_bits(cuda_device):
    """z of 2.3e9 elements through the wide tiles' tensor maps; rows are zero but for groups at
    the start, in the middle, across the boundary and at the end."""
    import teenyformers_b200 as tfb
    if torch.cuda.get_device_properties(cuda_device).total_memory < 64 << 30:
        pytest.skip("needs 64 GB of device memory")
    dev, m, d, F = cuda_device, 80003, 1032, 14336
    b = (1 << 31) // (2 * F)
    at = torch.cat([torch.arange(s, s + 16) for s in (0, m // 2, b - 8, m - 16)]).to(dev)
    x, dy = (torch.zeros(m, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    x[at], dy[at] = seeded_normal((64, d), 1, dev), seeded_normal((64, d), 2, dev)
    w1 = (seeded_normal((2 * F, d), 3, dev, torch.float32) / d ** 0.5).bfloat16()
    w2 = (seeded_normal((d, F), 4, dev, torch.float32) / F ** 0.5).bfloat16()
    ref = gated_ffn64(x[at], w1, w2, "gelu", dy=dy[at])
    y, z = tfb.gated_ffn(x, w1, w2, tfb.TF_ACT_GELU, save=True)
    assert_within("z", z[at], ref["z"])
    assert_within("y", y[at], ref["y"])
    got = dict(zip(("dx", "dw_gate_up", "dw_down"),
                   tfb.gated_ffn_bwd(x, w1, w2, z, dy, tfb.TF_ACT_GELU)))
    got["dx"] = got["dx"][at]
    for name, t in got.items():
        assert_within(name, t, ref[name])
    assert tfb.device_status() == 0
    del x, dy, y, z, got
    torch.cuda.empty_cache()
