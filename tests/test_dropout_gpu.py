"""Dropout from a counter-based generator: its mask against host arithmetic of the
published generator, its values, and the calls a user may make of it."""
import numpy as np
import pytest
import torch

from ffn_ref import dropout_mult
from helpers import seeded_normal

pytestmark = pytest.mark.gpu


def _want(x, p, rng, site, residual=None):
    """The multiplier in fp32 is one rounding of 65536 / t; the product and the sum are
    fp32 operations, rounded once more to the type: the kernel's own steps, exactly."""
    mult = torch.from_numpy(dropout_mult(x.numel(), p, rng, site).astype(np.float32)).to(x.device)
    y = torch.where(mult.view(x.shape) > 0, x.float() * mult.view(x.shape), 0.0)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


@pytest.mark.parametrize("n", [1, 7, 8, 9, 64, 1001, 40037, 1 << 20])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
def test_values(cuda_device, n, dtype, with_residual):
    import teenyformers_b200 as tfb
    rng = tfb.dropout_rng(0x123456789ABCDEF0 + n, (1 << 63) + 5, cuda_device)
    x = seeded_normal((n,), n, cuda_device, dtype)
    r = seeded_normal((n,), n + 1, cuda_device, dtype) if with_residual else None
    full = torch.full((n + 16,), float("nan"), dtype=dtype, device=cuda_device)
    for p, site in ((0.1, 0), (0.5, 3), (0.999, 0xFFFFFFFF)):
        y = tfb.dropout(x, p, rng, site=site, residual=r, out=full[:n])
        want = _want(x, p, rng, site, r)
        # x * scale + r may be one fused operation in the kernel: one fp32 rounding less
        tol = 2.0 ** -23 * (want.float().abs() + (r.float().abs() if with_residual else 0))
        if dtype == torch.bfloat16:
            tol = tol + 2.0 ** -7 * want.float().abs() * (1.0 if with_residual else 0.0)
        assert ((y.float() - want.float()).abs() <= tol).all()
        assert torch.equal(y == 0, want == 0) or with_residual
        assert torch.isnan(full[n:]).all()


def test_edges_of_p(cuda_device):
    import teenyformers_b200 as tfb
    rng = tfb.dropout_rng(1, 2, cuda_device)
    x = seeded_normal((1003,), 1, cuda_device)
    r = seeded_normal((1003,), 2, cuda_device)
    assert torch.equal(tfb.dropout(x, 0.0, None), x)
    assert torch.equal(tfb.dropout(x, 0.0, None, residual=r), (x.float() + r.float()).bfloat16())
    assert not tfb.dropout(x, 1.0, rng).any()
    assert torch.equal(tfb.dropout(x, 1.0, rng, residual=r), r)
    assert torch.equal(tfb.dropout(x, 2.0 ** -18, rng), x)     # rounds to 0: nothing dropped
    # what is dropped leaves nothing behind, whatever it held
    bad = torch.full_like(x, float("nan"))
    bad[::2] = float("inf")
    y = tfb.dropout(bad, 0.5, rng)
    kept = torch.from_numpy(dropout_mult(1003, 0.5, rng, 0) > 0).to(x.device)
    assert (y[~kept] == 0).all() and not torch.isfinite(y[kept]).any()


def test_sites_offsets_and_seeds_differ_and_the_rate_holds(cuda_device):
    import teenyformers_b200 as tfb
    n, p = 1 << 20, 0.3
    x = torch.ones(n, device=cuda_device)
    masks = [tfb.dropout(x, p, tfb.dropout_rng(s, o, cuda_device), site=k) > 0
             for s, o, k in ((1, 0, 0), (2, 0, 0), (1, 1, 0), (1, 0, 1), (1, 1 << 32, 0))]
    for i, a in enumerate(masks):
        # 5 standard deviations of a binomial share
        assert abs(float(a.float().mean()) - (1 - p)) <= 5 * (p * (1 - p) / n) ** 0.5
        for b in masks[:i]:
            agree = float((a == b).float().mean())
            q = p * p + (1 - p) * (1 - p)
            assert abs(agree - q) <= 5 * (q * (1 - q) / n) ** 0.5


def test_backward_draws_the_same_mask_in_place_and_in_graphs(cuda_device):
    import teenyformers_b200 as tfb
    op = tfb.DropoutOp(0.25, site=4)
    rng = tfb.dropout_rng(7, 100, cuda_device)
    x = seeded_normal((33, 72), 1, cuda_device)
    y = op.forward(x, rng)
    g = op.backward(torch.ones_like(x), rng)
    assert torch.equal((y != 0), (g != 0) & (x != 0))
    z = x.clone()
    assert torch.equal(tfb.dropout(z, 0.25, rng, site=4, out=z), y)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        out = op.forward(x, rng)
    for off in (100, 101):
        rng[1] = off
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, op.forward(x, rng))
    assert not torch.equal(out, y)


def test_refusals(cuda_device):
    import teenyformers_b200 as tfb
    rng = tfb.dropout_rng(1, 0, cuda_device)
    x = seeded_normal((64,), 1, cuda_device)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(tfb.TfError):
            tfb.dropout(x, p, rng)
    with pytest.raises(ValueError):
        tfb.dropout(x, 0.1, None)
    with pytest.raises(ValueError):
        tfb.dropout(x, 0.1, rng.int())
    with pytest.raises(ValueError):
        tfb.dropout(x, 0.1, rng.cpu())
    with pytest.raises(ValueError):
        tfb.dropout(x.half(), 0.1, rng)
    with pytest.raises(ValueError):
        tfb.dropout(x[::2], 0.1, rng)
    with pytest.raises(ValueError):
        tfb.dropout(x, 0.1, rng, site=-1)
    with pytest.raises(ValueError):
        tfb.dropout(x, 0.1, rng, residual=x[:32])
    with pytest.raises(tfb.TfError):      # 2 bytes off a 16-byte boundary
        tfb.dropout(x[1:33], 0.1, rng)
    assert tfb.dropout(x[:0], 0.1, rng).shape == (0,)
