"""The feed-forward side of a transformer block, as cases that can be timed.

Three operators that a block needs next to its attention:

  gated feed-forward   y = (act(x Wg^T) * (x Wu^T)) Wd^T, serving and training (forward + backward)
  block norm           y = rs x + bs dropout(gate * RMSNorm(f)), h = RMSNorm(y): the norm after a block with
                       its gate and residual scales, and the norm before the next one; forward and backward
  dropout              by a counter-based generator, its mask never stored

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the
framework's own entry points.
"""
import functools
import math

import numpy as np
import torch

own = False

EPS = 1e-5
SITE = 3  # which dropout of a step this is: a small number that a model gives each of its dropouts

# Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011)
M0, M1 = 0xD2511F53, 0xCD9E8D57
W0, W1 = 0x9E3779B9, 0xBB67AE85
U32 = 0xFFFFFFFF


def listed():
    return [
        # one new token of one sequence through the 8B layer's feed-forward block
        {"name": "ffn token", "kind": "ffn", "m": 1, "d": 4096, "d_ff": 14336, "act": "silu", "residual": False},
        # one new token each for a batch of 64 sequences, with the residual stream added
        {"name": "ffn decode batch", "kind": "ffn", "m": 64, "d": 4096, "d_ff": 14336, "act": "silu", "residual": True},
        # a short ragged prompt through a small model whose sizes fill no tile
        {"name": "ffn ragged", "kind": "ffn", "m": 777, "d": 1032, "d_ff": 2776, "act": "gelu_tanh", "residual": True},
        # the prefill of 16384 tokens
        {"name": "ffn prefill", "kind": "ffn", "m": 16384, "d": 4096, "d_ff": 14336, "act": "silu", "residual": False},
        # a training step on the ragged end of a small data set, erf GELU
        {"name": "ffn step ragged", "kind": "ffn_step", "m": 1111, "d": 520, "d_ff": 1416, "act": "gelu"},
        # a training step of the 8B layer's block on 8192 tokens
        {"name": "ffn step", "kind": "ffn_step", "m": 8192, "d": 4096, "d_ff": 14336, "act": "silu"},
        # four decoding sequences: latency
        {"name": "norm decode", "kind": "norm", "rows": 4, "cols": 4096, "gate_rows": 1, "post": True, "pre": True,
         "p": 0.0, "rs": 1.0, "bs": 0.5},
        # prefill of 8 sequences, each with a gate of its own
        {"name": "norm prefill", "kind": "norm", "rows": 16384, "cols": 4096, "gate_rows": 8, "post": True, "pre": True,
         "p": 0.0, "rs": 1.0, "bs": 1.0},
        # the same in training, one gate for all rows and dropout on the branch: its backward pass
        {"name": "norm backward", "kind": "norm_bwd", "rows": 16384, "cols": 4096, "gate_rows": 1, "post": True,
         "pre": True, "p": 0.1, "rs": 1.0, "bs": 1.0},
        # a ragged batch of a small model with a gate for each token and no norm after the sum
        {"name": "norm backward ragged", "kind": "norm_bwd", "rows": 1037, "cols": 1000, "gate_rows": 1037,
         "post": True, "pre": False, "p": 0.0, "rs": 0.75, "bs": 1.25},
        # dropout on a small fp32 tensor with an odd number of elements
        {"name": "dropout odd", "kind": "dropout", "n": 40037, "dtype": "f32", "p": 0.3, "residual": False},
        # dropout on a whole batch's hidden states, added to the residual stream
        {"name": "dropout batch", "kind": "dropout", "n": 16384 * 4096, "dtype": "bf16", "p": 0.1, "residual": True},
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(step, v // step * step)


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "ffn_step", "norm", "norm_bwd", "dropout"])
    if kind in ("ffn", "ffn_step"):
        return {"kind": kind, "m": _log(rng, 1, 16384 if kind == "ffn" else 8192), "d": _log(rng, 64, 4096, 8),
                "d_ff": _log(rng, 64, 14336, 8), "act": rng.choice(["silu", "gelu", "gelu_tanh"]),
                **({"residual": rng.random() < 0.5} if kind == "ffn" else {})}
    if kind in ("norm", "norm_bwd"):
        rows, cols = _log(rng, 1, 16384), _log(rng, 8, 4096, 8)
        gates = [0, 1, rows] + ([2] if rows % 2 == 0 else [])
        post, pre = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        return {"kind": kind, "rows": rows, "cols": cols, "gate_rows": rng.choice(gates), "post": post, "pre": pre,
                "p": rng.choice([0.0, 0.1, 0.25]), "rs": rng.choice([1.0, 0.75]), "bs": rng.choice([1.0, 0.22])}
    return {"kind": kind, "n": _log(rng, 1, 1 << 26), "dtype": rng.choice(["bf16", "f32"]),
            "p": rng.choice([0.05, 0.1, 0.5]), "residual": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    bf16 = torch.bfloat16

    def normal(*shape, scale=1.0, mean=0.0, dtype=bf16):
        return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)

    def rng():
        return torch.randint(-(1 << 62), 1 << 62, (2,), generator=g, device="cuda", dtype=torch.int64)

    s = {"case": case}
    kind = case["kind"]
    if kind in ("ffn", "ffn_step"):
        m, d, f = case["m"], case["d"], case["d_ff"]
        s["x"] = normal(m, d)                                      # what the norm before the block gives
        s["w_gate_up"] = normal(2 * f, d, scale=1.28 / math.sqrt(d))  # [gate; up], 0.02 at d = 4096
        s["w_down"] = normal(d, f, scale=1.28 / math.sqrt(f))
        if kind == "ffn_step":
            s["dy"] = normal(m, d, scale=1e-2)
        else:
            s["residual"] = normal(m, d) if case["residual"] else None
            s["out"] = torch.empty((m, d), dtype=bf16, device="cuda")     # kept by a serving loop
            s["act_buf"] = torch.empty((m, f), dtype=bf16, device="cuda")
        return s
    if kind in ("norm", "norm_bwd"):
        r, c = case["rows"], case["cols"]
        wide = torch.ones(c, device="cuda")
        wide[torch.randperm(c, generator=g, device="cuda")[:max(1, c // 256)]] = 8.0  # a few loud channels
        s["x"] = (normal(r, c, dtype=torch.float32) * wide).to(bf16)
        s["f"] = normal(r, c, scale=0.7)
        s["w_post"] = normal(c, scale=0.05, mean=1.0) if case["post"] else None
        s["w_pre"] = normal(c, scale=0.05, mean=1.0) if case["pre"] else None
        s["gate"] = normal(case["gate_rows"], c, scale=0.4, mean=0.5) if case["gate_rows"] else None
        s["rng"] = rng() if case["p"] else None
        if kind == "norm":
            s["y"], s["h"] = (torch.empty((r, c), dtype=bf16, device="cuda") for _ in range(2))
        else:
            s["dy"], s["dh"] = normal(r, c, scale=1e-2), normal(r, c, scale=1e-2) if case["pre"] else None
            s["y"] = _norm_forward(s)[0].to(bf16)  # the forward's, as a training program keeps it
            del s["x"]
        return s
    dtype = bf16 if case["dtype"] == "bf16" else torch.float32
    s["x"] = normal(case["n"], dtype=dtype)
    s["residual"] = normal(case["n"], dtype=dtype) if case["residual"] else None
    s["rng"] = rng()
    s["out"] = torch.empty_like(s["x"])
    return s


# ------------------------------------------------------------------ plain forms
def _mul_hi_lo(a, m):
    """The two halves of the 64-bit product of 32-bit words, in signed 64-bit integers."""
    low, high = a * (m & 0xFFFF), a * (m >> 16)
    return (high + (low >> 16)) >> 16, (low + ((high & 0xFFFF) << 16)) & U32


def _philox_round(c, k):
    (h0, l0), (h1, l1) = _mul_hi_lo(c[0], M0), _mul_hi_lo(c[2], M1)
    return h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0


def _keep(rng, n, p):
    """Which of n elements stay: element i has 16 bits of the group i // 8's 128, and stays where they are below
    the threshold; and what a kept element is multiplied by."""
    t = int(math.floor((1.0 - p) * 65536.0 + 0.5))
    group = torch.arange((n + 7) // 8, dtype=torch.int64, device=rng.device)
    seed, offset = rng[0], rng[1]
    c = (group, torch.full_like(group, SITE), offset & U32, (offset >> 32) & U32)
    keys = [((seed + r * W0) & U32, (((seed >> 32) & U32) + r * W1) & U32) for r in range(10)]
    words = functools.reduce(_philox_round, keys, c)
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=-1)
    return halves.reshape(-1)[:n] < t, (65536.0 / t if t else 0.0)


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _ffn_plain(s):
    c = s["case"]
    x, w1, w2 = s["x"].float(), s["w_gate_up"].float(), s["w_down"].float()
    gate, up = (x @ w1.t()).chunk(2, dim=-1)
    value, slope = _act(c["act"], gate)
    a = value * up
    y = a @ w2.t()
    if c["kind"] == "ffn":
        return (y + s["residual"].float() if c["residual"] else y).bfloat16()
    dy = s["dy"].float()
    da = dy @ w2
    dz = torch.cat([da * up * slope, da * value], dim=-1)
    return {"y": y.bfloat16(), "dx": (dz @ w1).bfloat16(), "dw_gate_up": (dz.t() @ x).bfloat16(),
            "dw_down": (dy.t() @ a).bfloat16()}


def _rms(v):
    return torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS)


def _rows_of(gate, rows):
    return gate.float().repeat_interleave(rows // gate.shape[0], dim=0)


def _branch_scale(s, rows, cols):
    """What multiplies the (normalised) branch: the gate, the dropout and the branch's scale."""
    c = s["case"]
    v = c["bs"]
    if s["rng"] is not None:
        keep, scale = _keep(s["rng"], rows * cols, c["p"])
        v = v * scale * keep.reshape(rows, cols).float()
    return v


def _norm_forward(s):
    c = s["case"]
    f = s["f"].float()
    n = f * _rms(f) * s["w_post"].float() if c["post"] else f
    if s["gate"] is not None:
        n = n * _rows_of(s["gate"], c["rows"])
    y = c["rs"] * s["x"].float() + _branch_scale(s, c["rows"], c["cols"]) * n
    return y, (y * _rms(y) * s["w_pre"].float() if c["pre"] else None)


def _norm_backward(s):
    c = s["case"]
    f, y, d = s["f"].float(), s["y"].float(), s["dy"].float()
    out = {}
    if c["pre"]:
        r, dh = _rms(y), s["dh"].float()
        t = dh * s["w_pre"].float()
        d = d + r * (t - y * (r * r) * (t * y).mean(dim=-1, keepdim=True))
        out["dw_pre"] = (dh * y * r).sum(dim=0)
    out["dx"] = c["rs"] * d
    d = d * _branch_scale(s, c["rows"], c["cols"])
    r = _rms(f) if c["post"] else None
    n = f * r if c["post"] else f
    if s["gate"] is not None:
        u = n * s["w_post"].float() if c["post"] else n
        out["dgate"] = (d * u).reshape(c["gate_rows"], -1, c["cols"]).sum(dim=1)
        d = d * _rows_of(s["gate"], c["rows"])
    if c["post"]:
        out["dw_post"] = (d * n).sum(dim=0)
        t = d * s["w_post"].float()
        d = r * (t - n * (t * n).mean(dim=-1, keepdim=True))
    out["df"] = d
    return {k: v.bfloat16() for k, v in out.items()}


def _dropout_plain(s):
    keep, scale = _keep(s["rng"], s["case"]["n"], s["case"]["p"])
    y = torch.where(keep, s["x"].float() * scale, 0.0)
    return (y + s["residual"].float() if s["residual"] is not None else y).to(s["x"].dtype)


# ------------------------------------------------------------------ one pass
def _run_own(s):
    import teenyformers_b200 as tfb

    c = s["case"]
    kind = c["kind"]
    if kind in ("ffn", "ffn_step"):
        act = {"silu": tfb.TF_ACT_SILU, "gelu": tfb.TF_ACT_GELU, "gelu_tanh": tfb.TF_ACT_GELU_TANH}[c["act"]]
        if kind == "ffn":
            return tfb.gated_ffn(s["x"], s["w_gate_up"], s["w_down"], act, residual=s["residual"], out=s["out"],
                                 act_out=s["act_buf"])
        y, z = tfb.gated_ffn(s["x"], s["w_gate_up"], s["w_down"], act, save=True)
        dx, dw_gate_up, dw_down = tfb.gated_ffn_bwd(s["x"], s["w_gate_up"], s["w_down"], z, s["dy"], act)
        return {"y": y, "dx": dx, "dw_gate_up": dw_gate_up, "dw_down": dw_down}
    if kind == "norm":
        return tfb.block_norm(s["x"], s["f"], s["w_post"], s["gate"], s["w_pre"], eps=EPS, residual_scale=c["rs"],
                              branch_scale=c["bs"], p=c["p"], rng=s["rng"], site=SITE, out=s["y"], norm_out=s["h"])
    if kind == "norm_bwd":
        dx, df, dw_post, dgate, dw_pre = tfb.block_norm_bwd(
            s["f"], s["y"], s["dy"], s["dh"], s["w_post"], s["gate"], s["w_pre"], eps=EPS, residual_scale=c["rs"],
            branch_scale=c["bs"], p=c["p"], rng=s["rng"], site=SITE)
        return {"dx": dx, "df": df, "dw_post": dw_post, "dgate": dgate, "dw_pre": dw_pre}
    return tfb.dropout(s["x"], c["p"], s["rng"], site=SITE, residual=s["residual"], out=s["out"])


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind in ("ffn", "ffn_step"):
        return _ffn_plain(state)
    if kind == "norm":
        y, h = _norm_forward(state)
        return y.bfloat16(), (h.bfloat16() if h is not None else None)
    return _norm_backward(state) if kind == "norm_bwd" else _dropout_plain(state)


def work(case):
    kind = case["kind"]
    if kind in ("ffn", "ffn_step"):
        m, d, f = case["m"], case["d"], case["d_ff"]
        weights = 3 * f * d * 2
        if kind == "ffn":
            return {"bytes": weights + 2 * m * d * (3 if case["residual"] else 2), "flops": 6 * m * d * f}
        return {"bytes": 2 * weights + 2 * m * d * 4, "flops": 18 * m * d * f}
    if kind in ("norm", "norm_bwd"):
        n, c = case["rows"] * case["cols"], case["cols"]
        vectors = 2 * c * (case["gate_rows"] + case["post"] + case["pre"])
        if kind == "norm":
            return {"bytes": 2 * n * (3 + case["pre"]) + vectors, "flops": 12 * n}
        reads = 2 + 2 * case["pre"] - (0 if case["post"] or case["gate_rows"] else 1)
        return {"bytes": 2 * n * (reads + 2) + 2 * vectors, "flops": 30 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": size * case["n"] * (3 if case["residual"] else 2), "flops": 2 * case["n"]}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_multiplier(rng, shape, p):
    """dropout's multiplier of each element, by 64-bit unsigned host arithmetic."""
    n = int(np.prod(shape))
    t = int(math.floor((1.0 - p) * 65536.0 + 0.5))
    seed, offset = (int(v) & (2 ** 64 - 1) for v in rng.cpu().tolist())
    groups = np.arange((n + 7) // 8, dtype=np.uint64)
    c0, c1 = groups, np.full_like(groups, SITE)
    c2, c3 = np.full_like(groups, offset & U32), np.full_like(groups, offset >> 32)
    k0, k1 = seed & U32, seed >> 32
    for _ in range(10):
        a, b = c0 * np.uint64(M0), c2 * np.uint64(M1)
        c0, c1, c2, c3 = ((b >> np.uint64(32)) ^ c1 ^ np.uint64(k0), b & np.uint64(U32),
                          (a >> np.uint64(32)) ^ c3 ^ np.uint64(k1), a & np.uint64(U32))
        k0, k1 = (k0 + W0) & U32, (k1 + W1) & U32
    words = np.stack([c0, c1, c2, c3], axis=1).astype(np.uint32)
    bits = np.ascontiguousarray(words).astype("<u4").view("<u2").reshape(-1)[:n]
    kept = torch.from_numpy((bits < t)).to(rng.device).reshape(shape)
    return kept.double() * (65536.0 / t if t else 0.0)


def _exact_act(name, g):
    if name == "silu":
        e = 1 / (1 + torch.exp(-g))
        return g * e, e + g * e * (1 - e)
    if name == "gelu":
        phi = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * phi
    a, b = math.sqrt(2 / math.pi), 0.044715
    # 0.5 (1 + tanh v) = 1 / (1 + exp(-2 v))
    e = 1 / (1 + torch.exp(-2 * a * (g + b * g ** 3)))
    return g * e, e + g * e * (1 - e) * 2 * a * (1 + 3 * b * g ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    kind = case["kind"]
    if kind in ("ffn", "ffn_step"):
        f = case["d_ff"]
        wg, wu, wd = s["w_gate_up"][:f], s["w_gate_up"][f:], s["w_down"]
        g, u = torch.matmul(s["x"], wg.T), torch.matmul(s["x"], wu.T)
        v, dv = _exact_act(case["act"], g)
        y = torch.matmul(v * u, wd.T)
        if kind == "ffn":
            return y if s["residual"] is None else s["residual"] + y
        da = torch.matmul(s["dy"], wd)
        dg, du = da * u * dv, da * v
        return {"y": y, "dx": torch.matmul(dg, wg) + torch.matmul(du, wu),
                "dw_gate_up": torch.cat([torch.matmul(dg.T, s["x"]), torch.matmul(du.T, s["x"])]),
                "dw_down": torch.matmul(s["dy"].T, v * u)}
    if kind == "dropout":
        y = s["x"] * _exact_multiplier(s["rng"], (case["n"],), case["p"])
        return y if s["residual"] is None else s["residual"] + y
    rows, cols = case["rows"], case["cols"]
    mult = case["bs"] * (_exact_multiplier(s["rng"], (rows, cols), case["p"]) if s["rng"] is not None else 1.0)
    f = s["f"]
    wp = s["w_post"]
    gate = None if s["gate"] is None else s["gate"][torch.arange(rows, device=f.device) // (rows // case["gate_rows"])]
    rf = 1 / torch.sqrt(f.pow(2).sum(-1, keepdim=True) / cols + EPS) if case["post"] else 1.0
    fn = f * rf
    branch = fn * wp if case["post"] else fn
    gated = branch if gate is None else branch * gate
    if kind == "norm":
        y = case["rs"] * s["x"] + mult * gated
        h = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / cols + EPS) * s["w_pre"] if case["pre"] else None
        return y, h
    total = s["dy"]
    dw_pre = None
    if case["pre"]:
        ry = 1 / torch.sqrt(s["y"].pow(2).sum(-1, keepdim=True) / cols + EPS)
        yn = s["y"] * ry
        q = s["dh"] * s["w_pre"]
        total = total + ry * q - ry * yn * ((q * yn).sum(-1, keepdim=True) / cols)
        dw_pre = (s["dh"] * yn).sum(0)
    dgated = total * mult
    dgate = None
    dbranch = dgated
    if gate is not None:
        dgate = (dgated * branch).view(case["gate_rows"], rows // case["gate_rows"], cols).sum(1)
        dbranch = dgated * gate
    df, dw_post = dbranch, None
    if case["post"]:
        q = dbranch * wp
        df = rf * q - rf * fn * ((q * fn).sum(-1, keepdim=True) / cols)
        dw_post = (dbranch * fn).sum(0)
    return {"dx": case["rs"] * total, "df": df, "dw_post": dw_post, "dgate": dgate, "dw_pre": dw_pre}
