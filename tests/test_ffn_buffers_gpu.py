"""A buffer that a call would not write is refused, not ignored."""
import pytest
import torch

from helpers import seeded_normal

pytestmark = pytest.mark.gpu


def test_buffers_that_would_not_be_written(cuda_device):
    import teenyformers_b200 as tfb
    dev = cuda_device
    x, f = (seeded_normal((6, 64), k, dev) for k in (1, 2))
    w = torch.ones(64, dtype=torch.bfloat16, device=dev)
    buf = torch.empty_like(x)
    with pytest.raises(ValueError):
        tfb.block_norm(x, None, w_pre=w, out=buf)       # y is x
    w1, w2 = (torch.zeros(s, dtype=torch.bfloat16, device=dev) for s in ((256, 64), (64, 128)))
    with pytest.raises(ValueError):
        tfb.gated_ffn(x, w1, w2, z_out=torch.empty((6, 256), device=dev))   # z is not saved


def test_buffers_that_are_written(cuda_device):
    import teenyformers_b200 as tfb
    dev = cuda_device
    x, f = (seeded_normal((6, 64), k, dev) for k in (1, 2))
    w = torch.ones(64, dtype=torch.bfloat16, device=dev)
    y, h = torch.empty_like(x), torch.empty_like(x)
    got = tfb.block_norm(x, f, w_pre=w, out=y, norm_out=h)
    assert got[0] is y and got[1] is h
    _, got = tfb.block_norm(x, None, w_pre=w, norm_out=h)
    assert got is h
    kept = h.clone()
    _, got = tfb.block_norm(x, f, w_post=w, norm_out=h)     # no h: None, and the buffer as it was
    assert got is None and torch.equal(h, kept)
