"""The activations and their slopes one by one, relative to their value: through weights of
one column, for which z, a and dz are exact but for their one rounding."""
import math

import pytest
import torch

from ffn_ref import U

pytestmark = pytest.mark.gpu

NAMES = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
# An fp32 chain around one exponential: __expf is within 2 + 1.2 |x| units of 2^-23 of exp(x) and
# its argument within 2^-23 |x|, |x| <= 72 here (g^2 / 2 at 12; 50 for the tanh form at -8):
# 161 x 2^-23 together, and some ten operations and a polynomial within 16 more.
EXACT = 177 * 2.0 ** -23


def _values(name, n):
    """n bf16 numbers from -12 (tanh form -8, whose slope's factors underflow further down) to 8."""
    lo = -8.0 if name == "gelu_tanh" else -12.0
    g = torch.cat([torch.linspace(lo, 0, n - n // 4), torch.linspace(0, 8, n // 4)])
    return g.bfloat16()


def _exact(name, g):
    """value, slope and the sum of the slope's two terms' absolute values, in forms that keep
    the tail in 64 bits: 1 + erf and 1 + tanh lose it there too."""
    if name == "gelu":
        cdf = torch.exp(torch.special.log_ndtr(g))
        rest = g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    else:
        k = math.sqrt(2 / math.pi)
        v, dv = (g, 1.0) if name == "silu" else (2 * k * (g + 0.044715 * g ** 3),
                                                 2 * k * (1 + 3 * 0.044715 * g * g))
        cdf = torch.sigmoid(v)
        rest = g * cdf * torch.sigmoid(-v) * dv
    return g * cdf, cdf + rest, cdf + rest.abs()


# one token; the pair kernels with a half-wide, a wide and a long gradient product
@pytest.mark.parametrize("m,d", [(1, 512), (2048, 1024), (4096, 1024), (2048, 2048)])
@pytest.mark.parametrize("name", list(NAMES))
def test_value_and_slope(cuda_device, m, d, name):
    import teenyformers_b200 as tfb
    dev = cuda_device
    g = _values(name, d).to(dev)
    x = torch.zeros((m, d), dtype=torch.bfloat16, device=dev)
    rows = sorted({0, m - 1})
    x[rows, 0] = 1
    w1 = torch.zeros((2 * d, d), dtype=torch.bfloat16, device=dev)
    w1[:d, 0], w1[d:, 0] = g, 1
    w2 = torch.eye(d, dtype=torch.bfloat16, device=dev)
    dy = torch.zeros((m, d), dtype=torch.bfloat16, device=dev)
    dy[0] = 1
    y, z = tfb.gated_ffn(x, w1, w2, NAMES[name], save=True)
    assert torch.equal(z[0, :d], g.float()) and (z[0, d:] == 1).all()
    _, dw1, dw2 = tfb.gated_ffn_bwd(x, w1, w2, z, dy, NAMES[name])
    value, slope, parts = _exact(name, g.double())
    tol = (U + EXACT) * value.abs() + 1e-37
    for r in rows:
        assert ((y[r].double() - value).abs() <= tol).all(), "value"
    assert ((dw2[:, :].diagonal().double() - value).abs() <= tol).all(), "a of the backward pass"
    # (dg of token 0, the only one with a gradient; the slope's two terms may cancel)
    err = (dw1[:d, 0].double() - slope).abs()
    assert (err <= U * slope.abs() + EXACT * parts + 1e-37).all(), "slope"
    assert tfb.device_status() == 0
