"""The gated feed-forward block, forward and backward, against its formulas in 64
bits (tests/ffn_ref.py gives the bounds), with the calls a user may make: any
number of tokens, sizes that fill no tile, captured graphs, other streams."""
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


def _guarded(shape, dtype, dev):
    """A tensor with a NaN guard of one more row before and after it, and a check of it."""
    full = torch.full((shape[0] + 2,) + tuple(shape[1:]), float("nan"), dtype=dtype, device=dev)
    def check(name):
        assert torch.isnan(full[0]).all() and torch.isnan(full[-1]).all(), f"{name}: guard written"
    return full[1:-1], check


SIZES = [(1, 8, 8), (1, 64, 128), (2, 520, 1416), (3, 72, 136), (7, 4096, 512), (16, 256, 512),
         (17, 128, 72), (33, 264, 1000), (64, 520, 200), (65, 136, 264), (128, 256, 1024),
         (129, 256, 128), (200, 64, 64), (300, 520, 1416), (513, 1032, 264),
         # few tiles and a long sum: of dx, of the weights' gradients, ragged
         (129, 520, 2776), (5, 8, 5000), (4100, 64, 72), (2056, 8, 8),
         # every product in 256 x 256 tiles, a long K in each
         (1030, 3208, 2568),
         # a deep ring in clusters of one, two and four
         (300, 1032, 2776), (130, 2568, 1032), (50, 4096, 4096), (20, 4096, 4096)]


@pytest.mark.parametrize("m,d,F", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_forward(cuda_device, m, d, F, act):
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, d, F, cuda_device, seed=m + d + F)
    res = seeded_normal((m, d), 77, cuda_device)
    ref = gated_ffn64(x, w1, w2, act)
    y, c0 = _guarded((m, d), torch.bfloat16, cuda_device)
    a, c1 = _guarded((m, F), torch.bfloat16, cuda_device)
    z, c2 = _guarded((m, 2 * F), torch.float32, cuda_device)
    tfb.gated_ffn(x, w1, w2, NAMES[act], out=y, act_out=a)
    assert_within("y", y, ref["y"])
    y2, z2 = tfb.gated_ffn(x, w1, w2, NAMES[act], residual=res, save=True, out=y, act_out=a,
                           z_out=z)
    assert_within("y + residual", y2, gated_ffn64(x, w1, w2, act, residual=res)["y"])
    assert_within("z", z2, ref["z"])
    for c, n in ((c0, "y"), (c1, "a"), (c2, "z")):
        c(n)
    assert tfb.device_status() == 0


@pytest.mark.parametrize("m,d,F", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_backward(cuda_device, m, d, F, act):
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, d, F, cuda_device, seed=m + d + F)
    dy = seeded_normal((m, d), 78, cuda_device)
    ref = gated_ffn64(x, w1, w2, act, dy=dy)
    _, z = tfb.gated_ffn(x, w1, w2, NAMES[act], save=True)
    g = [_guarded(t.shape, torch.bfloat16, cuda_device) for t in (x, w1, w2)]
    got = tfb.gated_ffn_bwd(x, w1, w2, z, dy, NAMES[act], grads=[t for t, _ in g])
    for name, t, (_, check) in zip(("dx", "dw_gate_up", "dw_down"), got, g):
        assert_within(name, t, ref[name])
        check(name)
    assert tfb.device_status() == 0


@pytest.mark.parametrize("m,d,F", [(1024, 512, 1408), (2048, 1024, 2048), (96, 1024, 2048)])
def test_error_is_that_of_two_roundings(cuda_device, m, d, F):
    """Over many values the error is random: a rounding's is at most U / sqrt(3) in the
    2-norm, relative, and each result has its own and its bf16 operand's."""
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, d, F, cuda_device, seed=5)
    dy = seeded_normal((m, d), 6, cuda_device)
    ref = gated_ffn64(x, w1, w2, "silu", dy=dy)
    y, z = tfb.gated_ffn(x, w1, w2, save=True)
    got = dict(zip(("dx", "dw_gate_up", "dw_down"), tfb.gated_ffn_bwd(x, w1, w2, z, dy)), y=y)
    for name, t in got.items():
        assert rel_l2(t, ref[name][0]) <= math.sqrt(2) * U / math.sqrt(3), name


def test_gradients_against_differences(cuda_device):
    """dL/dp of L = sum(dy * y) along a direction, against a central difference of the
    64-bit forward pass on the same weights."""
    import teenyformers_b200 as tfb
    m, d, F, h = 37, 136, 264, 1e-4
    x, w1, w2 = _inputs(m, d, F, cuda_device, seed=9)
    dy = seeded_normal((m, d), 10, cuda_device)
    for act in NAMES:
        _, z = tfb.gated_ffn(x, w1, w2, NAMES[act], save=True)
        grads = tfb.gated_ffn_bwd(x, w1, w2, z, dy, NAMES[act])
        for i, g in enumerate(grads):
            p = [t.double() for t in (x, w1, w2)]
            v = seeded_normal(p[i].shape, 20 + i, cuda_device, torch.float32).double()
            def loss(s):
                q = list(p)
                q[i] = p[i] + s * v
                return float((dy.double() * gated_ffn64(*q, act)["y"][0]).sum())
            want = (loss(h) - loss(-h)) / (2 * h)
            got = float((g.double() * v).sum())
            # N products of a gradient with relative error 2 U and a random v: the errors add
            # as their norms do; 4 standard deviations. The difference's own error is O(h^2).
            tol = 4 * 2 * U / math.sqrt(3) * float((g.double() * v).norm()) + 1e-4 * abs(want)
            assert abs(got - want) <= tol, (act, i, got, want, tol)


@pytest.mark.parametrize("m", [1, 300])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_saturated_and_huge_pre_activations(cuda_device, m, act):
    """g far outside the activation's bend: the value is 0 or g, the slope 0 or 1, with no
    0 * inf on the way.  x picks one column of the weights, so z is known exactly, dz is
    the first column of dw_gate_up (summed over the tokens) and y that of a's products."""
    import teenyformers_b200 as tfb
    g = torch.tensor([0.0, -0.0, 3.0, -3.0, 20.0, -20.0, 90.0, -90.0, 3e4, -3e4, 1e12, -1e12, 1e20,
                      -1e20, 1e30, -1e30], device=cuda_device)
    F, d = g.numel(), 8
    x = torch.zeros((m, d), device=cuda_device, dtype=torch.bfloat16)
    x[:, 0] = 1
    w1 = torch.zeros((2 * F, d), device=cuda_device, dtype=torch.bfloat16)
    w1[:F, 0] = g.bfloat16()
    w1[F:, 0] = 1
    w2 = torch.ones((d, F), device=cuda_device, dtype=torch.bfloat16)
    dy = torch.full((m, d), 0.125, device=cuda_device, dtype=torch.bfloat16)   # da = 1
    y, z = tfb.gated_ffn(x, w1, w2, NAMES[act], save=True)
    assert torch.equal(z[0, :F], w1[:F, 0].float()) and (z[:, F:] == 1).all()
    _, dw1, dw2 = tfb.gated_ffn_bwd(x, w1, w2, z, dy, NAMES[act])
    ref = gated_ffn64(x, w1, w2, act, dy=dy)
    assert torch.isfinite(y).all() and torch.isfinite(dw1).all() and torch.isfinite(dw2).all()
    assert_within("dw_gate_up", dw1, ref["dw_gate_up"])
    a = dw2[0].double() / (m * 0.125)                                            # mean of a
    want = torch.where(g.double() > 8, w1[:F, 0].double(), torch.zeros_like(a))
    far = g.abs() > 8
    assert ((a - want).abs()[far] <= 3 * U * want.abs()[far] + 1e-6).all()


def test_skipped_gradients_and_no_tokens(cuda_device):
    import teenyformers_b200 as tfb
    for m, d, F in ((129, 136, 2776), (4100, 64, 72), (70, 136, 264)):
        x, w1, w2 = _inputs(m, d, F, cuda_device)
        dy = seeded_normal((m, d), 3, cuda_device)
        _, z = tfb.gated_ffn(x, w1, w2, save=True)
        full = tfb.gated_ffn_bwd(x, w1, w2, z, dy)
        for need in [(True, False, False), (False, True, False), (False, False, True),
                     (True, True, False), (False, True, True), (True, False, True)]:
            part = tfb.gated_ffn_bwd(x, w1, w2, z, dy, need=need)
            for on, p, f in zip(need, part, full):
                assert (p is None) if not on else torch.equal(p, f)
    assert tfb.gated_ffn_bwd(x, w1, w2, z, dy, need=(False, False, False)) == (None, None, None)
    e = x[:0]
    y, z = tfb.gated_ffn(e, w1, w2, save=True)
    assert y.shape == (0, 136) and z.shape == (0, 528)
    dx, d1, d2 = tfb.gated_ffn_bwd(e, w1, w2, z, dy[:0])
    assert dx.shape == (0, 136) and not d1.any() and not d2.any()


@pytest.mark.parametrize("m", [1, 16, 100, 300])
def test_repeats_bit_for_bit_and_rows_do_not_mix(cuda_device, m):
    """Two calls give the same bits, and a token's result does not depend on the others in
    the call (its products and sums are the same)."""
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, 520, 1416, cuda_device, seed=2)
    y = tfb.gated_ffn(x, w1, w2)
    assert torch.equal(y, tfb.gated_ffn(x, w1, w2))
    x2 = x.clone()
    x2[1:] = seeded_normal((m - 1, 520), 50, cuda_device) * float("inf") if m > 1 else x[1:]
    y2 = tfb.gated_ffn(x2, w1, w2)
    assert torch.equal(y[0], y2[0])


def test_leading_dims_and_residual_in_place(cuda_device):
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(24, 136, 264, cuda_device)
    y = tfb.gated_ffn(x.view(2, 3, 4, 136), w1, w2)
    assert y.shape == (2, 3, 4, 136) and torch.equal(y.view(24, 136), tfb.gated_ffn(x, w1, w2))
    for m in (24, 200):
        x, w1, w2 = _inputs(m, 136, 264, cuda_device)
        res = seeded_normal((m, 136), 8, cuda_device)
        want = tfb.gated_ffn(x, w1, w2, residual=res)
        tfb.gated_ffn(x, w1, w2, residual=res, out=res)
        assert torch.equal(res, want)


@pytest.mark.parametrize("m", [1, 64, 300])
def test_captured_and_replayed_on_another_stream(cuda_device, m):
    """Forward and backward captured while eager calls on the same tensors live, replayed
    on new inputs, twice, from a stream of its own."""
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(m, 520, 264, cuda_device, seed=1)
    dy = seeded_normal((m, 520), 2, cuda_device)
    def step():
        y, z = tfb.gated_ffn(x, w1, w2, save=True)
        return (y,) + tfb.gated_ffn_bwd(x, w1, w2, z, dy)
    eager = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = step()
    for seed in (1, 31):
        x.copy_(seeded_normal((m, 520), seed, cuda_device))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        s.synchronize()
        want = step()
        for got, w in zip(captured, want):
            assert torch.equal(got, w)
    assert all(torch.isfinite(t).all() for t in eager)
    assert tfb.device_status() == 0


def test_two_calls_at_once(cuda_device):
    """Independent calls on two streams overlap without touching each other."""
    import teenyformers_b200 as tfb
    sets = [(_inputs(m, 520, 1416, cuda_device, seed=m)) for m in (4, 300)]
    want = [tfb.gated_ffn(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(tfb.gated_ffn(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals(cuda_device):
    import teenyformers_b200 as tfb
    x, w1, w2 = _inputs(4, 64, 128, cuda_device)
    with pytest.raises(ValueError):
        tfb.gated_ffn(x, w1[:-8], w2)
    with pytest.raises(ValueError):
        tfb.gated_ffn(x.float(), w1, w2)
    with pytest.raises(ValueError):
        tfb.gated_ffn(x.t().contiguous().t(), w1, w2)
    with pytest.raises(ValueError):
        tfb.gated_ffn(x, w1, w2.cpu())
    with pytest.raises(ValueError):
        tfb.gated_ffn(x, w1, w2, residual=x[:2])
    with pytest.raises(ValueError):
        tfb.gated_ffn(x, w1, w2, out=torch.empty(3, 64, device=cuda_device, dtype=torch.bfloat16))
    with pytest.raises(tfb.TfError):
        tfb.gated_ffn(x, w1, w2, act=7)
    with pytest.raises(tfb.TfError):   # sizes no multiple of 8
        tfb.gated_ffn(*_inputs(4, 60, 128, cuda_device))
    with pytest.raises(tfb.TfError):
        tfb.gated_ffn(*_inputs(4, 64, 100, cuda_device))
    _, z = tfb.gated_ffn(x, w1, w2, save=True)
    with pytest.raises(ValueError):
        tfb.gated_ffn_bwd(x, w1, w2, z.bfloat16(), x)
    with pytest.raises(ValueError):
        tfb.gated_ffn_bwd(x, w1, w2, z[:2], x)
    with pytest.raises(ValueError):
        tfb.gated_ffn_bwd(x, w1, w2, z, x, workspace=torch.empty(16, device=cuda_device))
