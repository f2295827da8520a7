"""The feed-forward sublayer: the gated feed-forward, the block norms and dropout run
together, as in training and in decoding, against 64-bit autograd."""
import math

import pytest
import torch

from ffn_ref import U, act64, dropout_mult, rel_l2
from helpers import seeded_normal

pytestmark = pytest.mark.gpu


def _weights(d, F, dev, post=True, gate_rows=1, nxt=True, seed=0):
    n = lambda *s, k=0, scale=1.0, mean=0.0: (
        seeded_normal(s, seed + k, dev, torch.float32) * scale + mean).bfloat16()
    w = {"norm": n(d, k=1, scale=0.1, mean=1.0), "w_gate_up": n(2 * F, d, k=2, scale=1.28 / d ** 0.5),
         "w_down": n(d, F, k=3, scale=1.28 / F ** 0.5)}
    if post:
        w["post_norm"] = n(d, k=4, scale=0.1, mean=1.0)
    if gate_rows:
        w["gate"] = n(gate_rows, d, k=5, scale=0.3, mean=0.7)
    if nxt:
        w["next_norm"] = n(d, k=6, scale=0.1, mean=1.0)
    return w


def _norm(v, w):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w


def _forward64(x, w, act, rs, bs, mult):
    h = _norm(x, w["norm"])
    F = w["w_down"].shape[1]
    z = h @ w["w_gate_up"].t()
    f = (act64(act, z[:, :F])[0] * z[:, F:]) @ w["w_down"].t()
    v = _norm(f, w["post_norm"]) if "post_norm" in w else f
    if "gate" in w:
        v = v * w["gate"].repeat_interleave(x.shape[0] // w["gate"].shape[0], 0)
    y = rs * x + bs * (v * mult if mult is not None else v)
    return y, (_norm(y, w["next_norm"]) if "next_norm" in w else None)


@pytest.mark.parametrize("rows,d,F,act,post,gate_rows,nxt,p", [
    (512, 256, 512, "silu", True, 1, True, 0.1),
    (300, 520, 1416, "gelu", True, 4, True, 0.0),
    (1000, 264, 704, "gelu_tanh", False, 0, True, 0.2),
    (256, 136, 264, "silu", True, 256, False, 0.0),
    (257, 128, 256, "silu", False, 0, False, 0.25)])
def test_training_step(cuda_device, rows, d, F, act, post, gate_rows, nxt, p):
    import teenyformers_b200 as tfb
    from teenyformers_b200.ffn import FeedForwardSublayer
    w = _weights(d, F, cuda_device, post, gate_rows, nxt, seed=rows)
    x = seeded_normal((rows, d), 1, cuda_device)
    dy, dhn = (seeded_normal((rows, d), k, cuda_device) for k in (2, 3))
    rng = tfb.dropout_rng(rows, 17, cuda_device)
    layer = FeedForwardSublayer(w, {"silu": 0, "gelu": 1, "gelu_tanh": 2}[act], residual_scale=0.9,
                                branch_scale=1.1, p=p, site=5)
    y, hn, saved = layer.forward(x, rng=rng, train=True)
    dx, grads = layer.backward(saved, dy, dhn if nxt else None, rng=rng)

    w64 = {k: v.double().requires_grad_() for k, v in w.items()}
    x64 = x.double().requires_grad_()
    mult = torch.from_numpy(dropout_mult(rows * d, p, rng, 5)).to(x.device).view(rows, d) if p else None
    y64, h64 = _forward64(x64, w64, act, 0.9, 1.1, mult)
    loss = (y64 * dy.double()).sum() + ((h64 * dhn.double()).sum() if nxt else 0)
    loss.backward()
    # Each value on the way to a result is rounded to bf16 once, an error of at most
    # U / sqrt(3) of its 2-norm, and independent errors add as squares: h, a and f before
    # y and hn and their own; for a gradient those three, y, df, dz, a, dh, the residual's
    # gradient and its own.
    step = U / math.sqrt(3)
    assert rel_l2(y, y64.detach()) <= math.sqrt(4) * step
    if nxt:
        assert rel_l2(hn, h64.detach()) <= math.sqrt(4) * step
    assert set(grads) == set(w)
    assert rel_l2(dx, x64.grad) <= math.sqrt(10) * step
    for k, g in grads.items():
        assert rel_l2(g, w64[k].grad) <= math.sqrt(10) * step, k
    assert tfb.device_status() == 0


def test_decoding_agrees_with_training_forward(cuda_device):
    """Token by token (the few-token kernels) and all at once (the tile or pair kernels)
    give the same values up to two roundings; a caller's own h is used."""
    from teenyformers_b200.ffn import FeedForwardSublayer
    import teenyformers_b200 as tfb
    w = _weights(264, 520, cuda_device)
    layer = FeedForwardSublayer(w)
    x = seeded_normal((300, 264), 9, cuda_device)
    y, hn, _ = layer.forward(x, train=True)
    for i in (0, 7, 299):
        yi, hi = layer.forward(x[i:i + 1].contiguous())
        assert rel_l2(yi, y[i:i + 1].double()) <= 4 * U / math.sqrt(3)
        assert rel_l2(hi, hn[i:i + 1].double()) <= 4 * U / math.sqrt(3)
    _, h = tfb.block_norm(x, None, w_pre=w["norm"])
    y2, hn2 = layer.forward(x, h=h)
    assert torch.equal(y, y2) and torch.equal(hn, hn2)


def test_step_captured_next_to_an_eager_one(cuda_device):
    """A whole training step in a graph, replayed with new inputs and a new dropout offset
    while results of eager steps on the same weights are alive."""
    import teenyformers_b200 as tfb
    from teenyformers_b200.ffn import FeedForwardSublayer
    w = _weights(136, 264, cuda_device)
    layer = FeedForwardSublayer(w, p=0.2, site=1)
    x, dy, dhn = (seeded_normal((200, 136), k, cuda_device) for k in (1, 2, 3))
    rng = tfb.dropout_rng(1, 0, cuda_device)
    def step():
        y, hn, saved = layer.forward(x, rng=rng, train=True)
        dx, g = layer.backward(saved, dy, dhn, rng=rng)
        return [y, hn, dx] + [g[k] for k in sorted(g)]
    eager = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    for off in (0, 1):
        rng[1] = off
        x.copy_(seeded_normal((200, 136), 1 + off, cuda_device))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        if off == 0:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
