"""The probability as the caller gives it, in 64 bits: t = floor((1 - p) * 65536 + 1/2) of
these p is another number for p rounded to 32 bits."""
import math

import numpy as np
import pytest
import torch

from ffn_ref import assert_within, block_norm64, block_norm_bwd64, dropout_mult
from helpers import seeded_normal

pytestmark = pytest.mark.gpu

P = [0.2528, 0.3153, 0.5028, 0.5653]


def _t(p):
    return math.floor((1.0 - p) * 65536.0 + 0.5)


def test_these_probabilities_tell_the_two_apart():
    for p in P:
        assert _t(p) != _t(float(np.float32(p)))


@pytest.mark.parametrize("p", P)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dropout(cuda_device, p, dtype):
    import teenyformers_b200 as tfb
    n = 1 << 21                       # one element in 65536 is kept or dropped by t's last unit
    rng = tfb.dropout_rng(5, 6, cuda_device)
    x = torch.ones(n, dtype=dtype, device=cuda_device)
    y = tfb.dropout(x, p, rng, site=3)
    mult = torch.from_numpy(dropout_mult(n, p, rng, 3)).to(cuda_device)
    assert torch.equal(y, mult.float().to(dtype))


@pytest.mark.parametrize("p", P[:2])
def test_block_norm(cuda_device, p):
    import teenyformers_b200 as tfb
    rows, cols = 2048, 512
    rng = tfb.dropout_rng(7, 8, cuda_device)
    x, f, dy = (seeded_normal((rows, cols), k, cuda_device) for k in (1, 2, 3))
    x.zero_()
    mult = torch.from_numpy(dropout_mult(rows * cols, p, rng, 4)).to(cuda_device).view(rows, cols)
    kw = dict(eps=1e-5, p=p, rng=rng, site=4)
    y, _ = tfb.block_norm(x, f, **kw)
    assert torch.equal(y != 0, (mult > 0) & (f != 0))
    assert_within("y", y, block_norm64(x, f, None, None, None, 1e-5, 1.0, 1.0, mult)[0])
    _, df, _, _, _ = tfb.block_norm_bwd(f, y, dy, None, **kw)
    assert torch.equal(df != 0, (mult > 0) & (dy != 0))
    assert_within("df", df, block_norm_bwd64(f, y, dy, None, None, None, None, 1e-5, 1.0, 1.0,
                                             mult)["df"])
