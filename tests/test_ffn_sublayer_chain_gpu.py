"""Feed-forward sublayers one behind the other, trained: the norm before the second is
the first one's last, computed once in the forward pass."""
import math

import pytest
import torch

from ffn_ref import U, act64, dropout_mult, rel_l2
from helpers import seeded_normal

pytestmark = pytest.mark.gpu

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _weights(d, F, dev, seed):
    n = lambda *s, k=0, scale=1.0, mean=0.0: (
        seeded_normal(s, seed + k, dev, torch.float32) * scale + mean).bfloat16()
    return {"norm": n(d, k=1, scale=0.1, mean=1.0), "w_gate_up": n(2 * F, d, k=2, scale=1.28 / d ** 0.5),
            "w_down": n(d, F, k=3, scale=1.28 / F ** 0.5), "post_norm": n(d, k=4, scale=0.1, mean=1.0),
            "gate": n(1, d, k=5, scale=0.3, mean=0.7)}


def _norm(v, w):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w


def _sublayer64(x, h, w, act, mult):
    F = w["w_down"].shape[1]
    z = h @ w["w_gate_up"].t()
    f = (act64(act, z[:, :F])[0] * z[:, F:]) @ w["w_down"].t()
    v = _norm(f, w["post_norm"]) * w["gate"]
    return 0.9 * x + 1.1 * (v * mult if mult is not None else v)


@pytest.mark.parametrize("rows,d,F,act,p,last", [(300, 264, 520, "silu", 0.1, True),
                                                 (257, 136, 264, "gelu", 0.0, True),
                                                 (64, 128, 256, "gelu_tanh", 0.0, False)])
def test_two_sublayers(cuda_device, rows, d, F, act, p, last):
    import teenyformers_b200 as tfb
    from teenyformers_b200.ffn import FeedForwardSublayer
    dev = cuda_device
    w1, w2 = _weights(d, F, dev, 10 * rows), _weights(d, F, dev, 10 * rows + 100)
    w1["next_norm"] = w2["norm"]                       # one weight: the norm between the two
    if last:
        w2["next_norm"] = (1.0 + 0.1 * seeded_normal((d,), 7, dev, torch.float32)).bfloat16()
    kw = dict(residual_scale=0.9, branch_scale=1.1, p=p)
    a = FeedForwardSublayer(w1, ACTS[act], site=1, **kw)
    b = FeedForwardSublayer(w2, ACTS[act], site=2, **kw)
    x, dy, dhn = (seeded_normal((rows, d), k, dev) for k in (1, 2, 3))
    rng = tfb.dropout_rng(rows, 17, dev)

    y1, h1, s1 = a.forward(x, rng=rng, train=True)
    y2, h2, s2 = b.forward(y1, h=h1, rng=rng, train=True)
    d1, g2 = b.backward(s2, dy, dhn if last else None, rng=rng)
    dx, g1 = a.backward(s1, d1, rng=rng)               # h1's gradient is in d1

    l1 = {k: v.double().requires_grad_() for k, v in w1.items()}
    l2 = {k: v.double().requires_grad_() for k, v in w2.items()}
    l1["next_norm"] = l2["norm"]
    x64 = x.double().requires_grad_()
    mult = [torch.from_numpy(dropout_mult(rows * d, p, rng, k)).to(dev).view(rows, d) if p else None
            for k in (1, 2)]
    m1 = _sublayer64(x64, _norm(x64, l1["norm"]), l1, act, mult[0])
    m2 = _sublayer64(m1, _norm(m1, l2["norm"]), l2, act, mult[1])
    loss = (m2 * dy.double()).sum()
    if last:
        loss = loss + (_norm(m2, l2["next_norm"]) * dhn.double()).sum()
    loss.backward()

    # Every bf16 value on the way is off by at most U / sqrt(3) of its 2-norm, and independent
    # errors add as squares.  Forward: h, a, f, y of each (8).  A gradient of the second sublayer
    # has at most those and df, dz, a, dh, the residual's gradient and its own (6); one of the
    # first the second's dx (1) and its own six more.
    step = U / math.sqrt(3)
    assert rel_l2(y2, m2.detach()) <= math.sqrt(8) * step
    assert set(g1) == set(w1) - {"next_norm"} and set(g2) == set(w2)
    for k, g in g2.items():                            # norm: the whole gradient of the shared one
        assert rel_l2(g, l2[k].grad) <= math.sqrt(14) * step, k
    for k, g in g1.items():
        assert rel_l2(g, l1[k].grad) <= math.sqrt(21) * step, k
    assert rel_l2(dx, x64.grad) <= math.sqrt(21) * step
    assert tfb.device_status() == 0


def test_a_gradient_of_hn_without_its_norm_is_refused(cuda_device):
    from teenyformers_b200.ffn import FeedForwardSublayer
    w = _weights(64, 128, cuda_device, 1)
    layer = FeedForwardSublayer(w)
    x = seeded_normal((4, 64), 1, cuda_device)
    _, hn, saved = layer.forward(x, train=True)
    assert hn is None
    with pytest.raises(ValueError):
        layer.backward(saved, x, x)
    with pytest.raises(ValueError):
        layer.backward(saved, None, None)
