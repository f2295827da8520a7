"""Gates shared by sequences together with dropout, element by element against 64 bits."""
import pytest
import torch

from ffn_ref import assert_within, block_norm64, block_norm_bwd64, dropout_mult
from helpers import seeded_normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,gate_rows", [(2400, 264, 2), (2400, 1000, 50), (1205, 4096, 5),
                                                 (600, 8192, 4), (37, 64, 37)])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True)])
def test_shared_gate_and_dropout(cuda_device, rows, cols, gate_rows, post, pre):
    import teenyformers_b200 as tfb
    dev, p = cuda_device, 0.2
    x, f, dy, dh = (seeded_normal((rows, cols), k, dev) for k in (1, 2, 3, 4))
    gate = seeded_normal((gate_rows, cols), 5, dev)
    wp, wn = ((1.0 + 0.1 * seeded_normal((cols,), k, dev, torch.float32)).bfloat16() for k in (6, 7))
    wp, wn, dh = wp if post else None, wn if pre else None, dh if pre else None
    rng = tfb.dropout_rng(rows, cols, dev)
    mult = torch.from_numpy(dropout_mult(rows * cols, p, rng, 3)).to(dev).view(rows, cols)
    kw = dict(eps=1e-5, residual_scale=0.75, branch_scale=1.25, p=p, rng=rng, site=3)
    y, h = tfb.block_norm(x, f, wp, gate, wn, **kw)
    ry, rh = block_norm64(x, f, wp, gate, wn, 1e-5, 0.75, 1.25, mult)
    assert_within("y", y, ry)
    if pre:
        assert_within("h", h, rh)
    got = tfb.block_norm_bwd(f, y, dy, dh, wp, gate, wn, **kw)
    ref = block_norm_bwd64(f, y, dy, dh, wp, gate, wn, 1e-5, 0.75, 1.25, mult)
    for name, t in zip(("dx", "df", "dw_post", "dgate", "dw_pre"), got):
        assert (t is None) == (name not in ref)
        if t is not None:
            assert_within(name, t, ref[name])
