"""The norms around a block with its gate, scales and dropout, forward and backward,
against the formulas in 64 bits (tests/ffn_ref.py gives the bounds)."""
import pytest
import torch

from ffn_ref import assert_within, block_norm64, block_norm_bwd64, dropout_mult
from helpers import seeded_normal

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _w(cols, seed, dev):
    return (1.0 + 0.1 * seeded_normal((cols,), seed, dev, torch.float32)).bfloat16()


def _case(rows, cols, gate_rows, post, pre, dev, seed=0):
    x, f = (seeded_normal((rows, cols), seed + i, dev) for i in (1, 2))
    gate = seeded_normal((gate_rows, cols), seed + 3, dev) if gate_rows else None
    return (x, f, _w(cols, seed + 4, dev) if post else None, gate,
            _w(cols, seed + 5, dev) if pre else None)


def _mult(rows, cols, p, rng, site, dev):
    if not p:
        return None
    return torch.from_numpy(dropout_mult(rows * cols, p, rng, site)).to(dev).view(rows, cols)


SHAPES = [(1, 8), (3, 24), (1, 4096), (5, 256), (17, 264), (37, 512), (6, 520), (1037, 1000),
          (12, 1032), (9, 2048), (300, 2056), (4, 4104), (600, 4096), (5, 8192)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("post,pre,gate,p", [(True, True, 1, 0.0), (True, True, 0, 0.1),
                                             (True, False, -1, 0.3), (False, True, 1, 0.2),
                                             (False, False, -1, 0.0), (False, False, 0, 0.5)])
def test_forward_and_backward(cuda_device, rows, cols, post, pre, gate, p):
    import teenyformers_b200 as tfb
    dev = cuda_device
    gate_rows = rows if gate < 0 else gate
    x, f, wp, g, wn = _case(rows, cols, gate_rows, post, pre, dev, seed=rows + cols)
    rng = tfb.dropout_rng(rows * 7919 + cols, 3, dev) if p else None
    kw = dict(eps=EPS, residual_scale=0.75, branch_scale=-1.25, p=p, rng=rng, site=2)
    mult = _mult(rows, cols, p, rng, 2, dev)
    bufs = [torch.full((rows + 2, cols), float("nan"), dtype=torch.bfloat16, device=dev)
            for _ in range(2)]
    y, h = tfb.block_norm(x, f, wp, g, wn, out=bufs[0][1:-1], norm_out=bufs[1][1:-1], **kw)
    ry, rh = block_norm64(x, f, wp, g, wn, EPS, 0.75, -1.25, mult)
    assert_within("y", y, ry)
    if pre:
        assert_within("h", h, rh)
    for b in bufs:
        assert torch.isnan(b[0]).all() and torch.isnan(b[-1]).all()
    dy = seeded_normal((rows, cols), 91, dev)
    dh = seeded_normal((rows, cols), 92, dev) if pre else None
    got = tfb.block_norm_bwd(f, y, dy, dh, wp, g, wn, **kw)
    ref = block_norm_bwd64(f, y, dy, dh, wp, g, wn, EPS, 0.75, -1.25, mult)
    for name, t in zip(("dx", "df", "dw_post", "dgate", "dw_pre"), got):
        assert (t is None) == (name not in ref), name
        if t is not None:
            assert_within(name, t, ref[name])
    again = tfb.block_norm_bwd(f, y, dy, dh, wp, g, wn, **kw)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("rows,cols,gate_rows", [(2400, 264, 2), (2400, 264, 3), (2400, 264, 50),
                                                 (2400, 4096, 2), (2400, 4096, 5), (2400, 4096, 400),
                                                 (2400, 1000, 1200), (2072, 512, 296),
                                                 (3000, 64, 3), (600, 8192, 4)])
def test_gate_rows_shared_by_sequences(cuda_device, rows, cols, gate_rows):
    """Gates of one row for several rows of x: their gradient joins the rows of one team,
    of several, and of teams whose rows end inside another gate's."""
    import teenyformers_b200 as tfb
    x, f, wp, g, wn = _case(rows, cols, gate_rows, True, True, cuda_device)
    y, h = tfb.block_norm(x, f, wp, g, wn, eps=EPS)
    ry, rh = block_norm64(x, f, wp, g, wn, EPS, 1.0, 1.0)
    assert_within("y", y, ry)
    assert_within("h", h, rh)
    dy, dh = (seeded_normal((rows, cols), s, cuda_device) for s in (5, 6))
    got = tfb.block_norm_bwd(f, y, dy, dh, wp, g, wn, eps=EPS)
    ref = block_norm_bwd64(f, y, dy, dh, wp, g, wn, EPS, 1.0, 1.0)
    for name, t in zip(("dx", "df", "dw_post", "dgate", "dw_pre"), got):
        assert_within(name, t, ref[name])


@pytest.mark.parametrize("rows,cols", [(1, 64), (77, 1000), (300, 4096)])
def test_only_the_norm_before_a_block(cuda_device, rows, cols):
    import teenyformers_b200 as tfb
    x = seeded_normal((rows, cols), 1, cuda_device)
    w = _w(cols, 2, cuda_device)
    y, h = tfb.block_norm(x, None, w_pre=w, eps=EPS)
    assert y is x
    assert_within("h", h, block_norm64(x, None, None, None, w, EPS, 1.0, 1.0)[1])
    dh = seeded_normal((rows, cols), 3, cuda_device)
    for dy in (None, seeded_normal((rows, cols), 4, cuda_device)):
        dx, df, dw_post, dgate, dw_pre = tfb.block_norm_bwd(None, x, dy, dh, w_pre=w, eps=EPS,
                                                            branch=False)
        ref = block_norm_bwd64(None, x, dy, dh, None, None, w, EPS, 1.0, 1.0, branch=False)
        assert df is None and dw_post is None and dgate is None
        assert_within("dx", dx, ref["dx"])
        assert_within("dw_pre", dw_pre, ref["dw_pre"])


def test_gradients_against_differences(cuda_device):
    """L = sum(cy y) + sum(ch h): each gradient along a direction against a central
    difference of the 64-bit forward pass."""
    import teenyformers_b200 as tfb
    rows, cols, s = 24, 136, 1e-5
    base = _case(rows, cols, 3, True, True, cuda_device)
    rng = tfb.dropout_rng(3, 4, cuda_device)
    mult = _mult(rows, cols, 0.2, rng, 1, cuda_device)
    kw = dict(eps=EPS, residual_scale=0.5, branch_scale=1.5, p=0.2, rng=rng, site=1)
    cy, ch = (seeded_normal((rows, cols), k, cuda_device) for k in (61, 62))
    y, _ = tfb.block_norm(*base, **kw)
    dx, df, dwp, dg, dwn = tfb.block_norm_bwd(base[1], y, cy, ch, *base[2:], **kw)
    for i, grad in zip(range(5), (dx, df, dwp, dg, dwn)):
        p = [t.double() for t in base]
        v = seeded_normal(p[i].shape, 70 + i, cuda_device, torch.float32).double()
        def loss(t):
            q = list(p)
            q[i] = p[i] + t * v
            (yy, _), (hh, _) = block_norm64(*q, EPS, 0.5, 1.5, mult)
            return float((cy.double() * yy).sum() + (ch.double() * hh).sum())
        want = (loss(s) - loss(-s)) / (2 * s)
        got = float((grad.double() * v).sum())
        # roundings of the gradient and of the saved y (2^-8 each, relative): 4 standard
        # deviations of their random sum, against the norm of the terms
        terms = float((grad.double() * v).norm())
        tol = 4 * 2 * 2.0 ** -8 / 3 ** 0.5 * terms + 1e-4 * abs(want) + 2.0 ** -8 * terms
        assert abs(got - want) <= tol, (i, got, want, tol)


def test_rows_of_zeros_and_loud_rows(cuda_device):
    """A row of zeros has the inverse RMS 1 / sqrt(eps); a row of large values must not
    overflow its sum of squares in fp32."""
    import teenyformers_b200 as tfb
    x, f, wp, g, wn = _case(8, 520, 1, True, True, cuda_device)
    x[0], f[0] = 0, 0
    x[1], f[1] = x[1] * 1e15, f[1] * 1e15
    f[2] = f[2] * 1e-20
    y, h = tfb.block_norm(x, f, wp, g, wn, eps=EPS)
    ry, rh = block_norm64(x, f, wp, g, wn, EPS, 1.0, 1.0)
    assert_within("y", y, ry)
    assert_within("h", h, rh)
    dy, dh = (seeded_normal((8, 520), s, cuda_device) for s in (5, 6))
    got = tfb.block_norm_bwd(f, y, dy, dh, wp, g, wn, eps=EPS)
    ref = block_norm_bwd64(f, y, dy, dh, wp, g, wn, EPS, 1.0, 1.0)
    for name, t in zip(("dx", "df", "dw_post", "dgate", "dw_pre"), got):
        assert_within(name, t, ref[name])


def test_nan_stays_in_its_row(cuda_device):
    import teenyformers_b200 as tfb
    x, f, wp, g, wn = _case(6, 264, 1, True, True, cuda_device)
    y0, h0 = tfb.block_norm(x, f, wp, g, wn)
    f[3, 5] = float("nan")
    y, h = tfb.block_norm(x, f, wp, g, wn)
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(h[keep], h0[keep])
    assert torch.isnan(y[3]).all() and torch.isnan(h[3]).all()


def test_in_place_captured_and_on_another_stream(cuda_device):
    import teenyformers_b200 as tfb
    x, f, wp, g, wn = _case(300, 1000, 3, True, True, cuda_device)
    rng = tfb.dropout_rng(3, 0, cuda_device)
    op = tfb.BlockNormOp(eps=EPS, branch_scale=0.5, p=0.1, site=9)
    dy, dh = (seeded_normal((300, 1000), s, cuda_device) for s in (5, 6))
    def step():
        y, h = op.forward(x, f, wp, g, wn, rng=rng)
        return (y, h) + op.backward(f, y, dy, dh, wp, g, wn, rng=rng)
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    for off in (0, 5):
        rng[1] = off
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    rng[1] = 0
    z = x.clone()
    y, h = tfb.block_norm(z, f, wp, g, wn, eps=EPS, branch_scale=0.5, p=0.1, rng=rng, site=9, out=z)
    assert torch.equal(z, want[0]) and torch.equal(h, want[1])


def test_no_rows(cuda_device):
    import teenyformers_b200 as tfb
    x, f, wp, g, wn = _case(4, 64, 1, True, True, cuda_device)
    y, h = tfb.block_norm(x[:0], f[:0], wp, g, wn)
    assert y.shape == h.shape == (0, 64)
    dx, df, dwp, dg, dwn = tfb.block_norm_bwd(f[:0], y, x[:0], x[:0], wp, g, wn)
    assert dx.shape == (0, 64) and not dwp.any() and not dg.any() and not dwn.any()


def test_refusals(cuda_device):
    import teenyformers_b200 as tfb
    x, f, wp, g, wn = _case(6, 64, 1, True, True, cuda_device)
    with pytest.raises(ValueError):
        tfb.block_norm(x, f[:3], wp, g, wn)
    with pytest.raises(ValueError):
        tfb.block_norm(x, f, wp[:32], g, wn)
    with pytest.raises(ValueError):
        tfb.block_norm(x, f, wp, g.expand(4, 64).contiguous(), wn)   # 4 does not divide 6
    with pytest.raises(ValueError):
        tfb.block_norm(x.float(), f, wp, g, wn)
    with pytest.raises(ValueError):
        tfb.block_norm(x, f, p=0.5)
    with pytest.raises(ValueError):
        tfb.block_norm_bwd(f, x, x, None, wp, g, wn)
    with pytest.raises(ValueError):
        tfb.block_norm_bwd(None, x, x, x, wp, g, wn)
    with pytest.raises(ValueError):
        tfb.block_norm_bwd(None, x, None, None)
    for bad in (dict(eps=-1.0), dict(eps=float("nan")), dict(residual_scale=float("inf")),
                dict(p=2.0, rng=tfb.dropout_rng(1, 1, cuda_device))):
        with pytest.raises(tfb.TfError):
            tfb.block_norm(x, f, wp, g, wn, **bad)
    with pytest.raises(tfb.TfError):
        tfb.block_norm(x, None)                        # neither a branch nor a norm
    for cols in (12, 8200):
        t = torch.zeros((2, cols), dtype=torch.bfloat16, device=cuda_device)
        with pytest.raises(tfb.TfError):
            tfb.block_norm(t, t)
