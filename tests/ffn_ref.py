"""64-bit forms of the feed-forward block, the block norm and dropout, each with
a bound on a kernel's error that follows from its arithmetic:

  u = 2^-8            a bf16 rounding, relative to the value (half of finfo.eps)
  n * 2^-23           a sum of n fp32 terms in any order, relative to the sum of
                      their absolute values (2^-23: accumulation may truncate)

A bound is computed with the same formulas on absolute values.  Everything is
torch float64 on the inputs' device."""
import math

import numpy as np
import torch

U = 2.0 ** -8
ACC = 2.0 ** -23


# ------------------------------------------------------------------ activations
def act64(name, g):
    """act(g), act'(g)"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return (0.5 * g * (1 + t),
            0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g))


LIP, LIP2 = 1.13, 1.0   # largest |act'| and |act''| of the three activations (1.129, 0.80)
ACT = 2.0 ** -18        # relative error of an activation or slope computed with fast fp32 exp


def gated_ffn64(x, w1, w2, name, residual=None, dy=None):
    """{name: (value, bound)} for z and y, and with dy for dx, dw_gate_up, dw_down."""
    x, w1, w2 = x.double(), w1.double(), w2.double()
    m, d = x.shape
    F = w2.shape[1]
    z = x @ w1.t()
    e_z = (d + 2) * ACC * (x.abs() @ w1.abs().t())
    g, u = z[:, :F], z[:, F:]
    e_g, e_u = e_z[:, :F], e_z[:, F:]
    v, s = act64(name, g)
    # an activation's own error is relative to g where it nearly vanishes
    e_v = LIP * e_g + ACT * g.abs().clamp(max=8.0)
    a = v * u
    e_a = u.abs() * e_v + v.abs() * e_u + U * a.abs()
    y = a @ w2.t()
    e_y = e_a @ w2.abs().t() + (F + 2) * ACC * (a.abs() @ w2.abs().t())
    if residual is not None:
        y = y + residual.double()
    out = {"z": (z, e_z), "y": (y, e_y + U * y.abs())}
    if dy is None:
        return out
    dy = dy.double()
    da = dy @ w2
    e_da = (d + 2) * ACC * (dy.abs() @ w2.abs())
    dg, du = da * u * s, da * v
    e_s = LIP2 * e_g + ACT * (1 + g.abs().clamp(max=8.0))
    e_dg = e_da * (u * s).abs() + (da * s).abs() * e_u + (da * u).abs() * e_s + U * dg.abs()
    e_du = e_da * v.abs() + da.abs() * e_v + U * du.abs()
    dz, e_dz = torch.cat([dg, du], 1), torch.cat([e_dg, e_du], 1)
    dx = dz @ w1
    out["dx"] = (dx, e_dz @ w1.abs() + (2 * F + 2) * ACC * (dz.abs() @ w1.abs()) + U * dx.abs())
    dw1 = dz.t() @ x
    out["dw_gate_up"] = (dw1, e_dz.t() @ x.abs() + (m + 2) * ACC * (dz.abs().t() @ x.abs())
                         + U * dw1.abs())
    dw2 = dy.t() @ a
    out["dw_down"] = (dw2, dy.abs().t() @ e_a + (m + 2) * ACC * (dy.abs().t() @ a.abs())
                      + U * dw2.abs())
    return out


# ------------------------------------------------------------------ Philox4x32-10
def philox_words(counter, key):
    """Ten rounds on arrays of four 32-bit counter words (unsigned 64-bit host arithmetic)."""
    c = [np.asarray(w, np.uint64) for w in counter]
    k0, k1 = key
    lo = np.uint64(0xFFFFFFFF)
    sh = np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ np.uint64(k0), b & lo, (a >> sh) ^ c[3] ^ np.uint64(k1), a & lo]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def dropout_mult(n, p, rng, site, start=0):
    """float64 numpy [n]: the multiplier of elements start .. start + n - 1 (start % 8 == 0)."""
    t = int(math.floor((1.0 - p) * 65536.0 + 0.5))
    seed, offset = (int(v) & (2 ** 64 - 1) for v in rng.cpu().tolist())
    g = np.arange(start // 8, start // 8 + (n + 7) // 8, dtype=np.uint64)
    z = np.zeros_like(g)
    words = philox_words([g, z + np.uint64(site), z + np.uint64(offset & 0xFFFFFFFF),
                          z + np.uint64(offset >> 32)], (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    return np.where(halves.reshape(-1)[:n] < t, 65536.0 / t if t else 0.0, 0.0)


# ------------------------------------------------------------------ block norm
def block_norm64(x, f, w_post, gate, w_pre, eps, rs, bs, mult=None):
    """((y, bound), (h, bound) or None); mult: the dropout's multiplier or None."""
    x = x.double()
    rows, cols = x.shape
    k = (cols + 64) * ACC
    if f is None:
        y, ay = x, torch.zeros_like(x)
    else:
        v = f.double()
        if w_post is not None:
            v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * w_post.double()
        if gate is not None:
            v = v * gate.double().repeat_interleave(rows // gate.shape[0], 0)
        if mult is not None:
            v = v * mult
        y = rs * x + bs * v
        ay = (rs * x).abs() + (bs * v).abs()
    h = None
    if w_pre is not None:
        r = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
        hv = y * r * w_pre.double()
        # an error e of y reaches h as r w (e + |y| mean(|y| e) r^2)
        e = k * ay
        h = (hv, U * hv.abs() + k * hv.abs()
             + r * w_pre.double().abs() * (e + y.abs() * (y.abs() * e).mean(1, keepdim=True) * r * r))
    return (y, U * y.abs() + k * ay), h


def block_norm_bwd64(f, y, dy, dh, w_post, gate, w_pre, eps, rs, bs, mult=None, branch=True):
    """{name: (value, bound)} for dx, df, dw_post, dgate, dw_pre (those that exist)."""
    like = dy if dy is not None else dh
    rows, cols = like.shape
    k = 4 * (cols + 64) * ACC
    kr = k + (rows + 2) * ACC
    t = dy.double() if dy is not None else torch.zeros_like(like, dtype=torch.float64)
    at = t.abs()
    out = {}
    if w_pre is not None:
        yd, d = y.double(), dh.double()
        r = 1 / torch.sqrt((yd * yd).mean(1, keepdim=True) + eps)
        q = d * w_pre.double()
        t = t + r * (q - yd * r * r * (q * yd).mean(1, keepdim=True))
        at = at + r * (q.abs() + yd.abs() * r * r * (q * yd).abs().mean(1, keepdim=True))
        out["dw_pre"] = ((d * yd * r).sum(0), (d * yd * r).abs().sum(0))
    out["dx"] = (rs * t, abs(rs) * at)
    if branch:
        mv = bs if mult is None else bs * mult
        t, at = t * mv, at * abs(mv) if mult is None else at * mv.abs()
        n = f.double() if f is not None else None
        r = None
        if w_post is not None:
            r = 1 / torch.sqrt((n * n).mean(1, keepdim=True) + eps)
            n = n * r
        if gate is not None:
            u = n * w_post.double() if w_post is not None else n
            G = gate.shape[0]
            out["dgate"] = ((t * u).reshape(G, rows // G, cols).sum(1),
                            (at * u.abs()).reshape(G, rows // G, cols).sum(1))
            ge = gate.double().repeat_interleave(rows // G, 0)
            t, at = t * ge, at * ge.abs()
        if w_post is not None:
            out["dw_post"] = ((t * n).sum(0), (at * n.abs()).sum(0))
            t, at = t * w_post.double(), at * w_post.double().abs()
            t = r * (t - n * (t * n).mean(1, keepdim=True))
            at = r * (at + n.abs() * (at * n.abs()).mean(1, keepdim=True))
        out["df"] = (t, at)
    return {name: (v, U * v.abs() + (kr if name.startswith(("dw", "dg")) else k) * a)
            for name, (v, a) in out.items()}


def assert_within(name, got, ref):
    """|got - value| <= bound everywhere (both of ref = (value, bound) as got)."""
    value, bound = ref
    got = got.double()
    assert got.shape == value.shape, f"{name}: {tuple(got.shape)} vs {tuple(value.shape)}"
    assert torch.isfinite(got).all(), f"{name}: non-finite values"
    # 1e-30: an exact zero times anything; values below fp32's normal range are flushed
    over = ((got - value).abs() - bound - 1e-30)
    worst = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or float(over.max()) <= 0, (
        f"{name}: off by {float((got - value).abs().flatten()[worst]):.3e} where "
        f"{float(bound.flatten()[worst]):.3e} is allowed (value {float(value.flatten()[worst]):.3e})")


def rel_l2(got, value):
    return float((got.double() - value).norm() / value.norm())
