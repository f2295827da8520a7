"""Results of the backward pass in the place of inputs that nothing reads any more."""
import pytest
import torch

from helpers import seeded_normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,d,F", [(129, 136, 2776), (300, 520, 264), (4100, 64, 72)])
def test_in_place(cuda_device, m, d, F):
    import teenyformers_b200 as tfb
    dev = cuda_device
    x, dy = (seeded_normal((m, d), k, dev) for k in (1, 2))
    w1, w2 = (seeded_normal((2 * F, d), 3, dev) * 0.1, seeded_normal((d, F), 4, dev) * 0.1)
    _, z = tfb.gated_ffn(x, w1, w2, save=True)
    dx, g1, g2 = tfb.gated_ffn_bwd(x, w1, w2, z, dy)
    for need, pick in (((True, False, True), "x"), ((True, True, False), "dy"),
                       ((True, False, False), "x"), ((True, False, False), "dy")):
        a = {"x": x.clone(), "dy": dy.clone()}
        got = tfb.gated_ffn_bwd(a["x"], w1, w2, z, a["dy"], need=need, grads=(a[pick], None, None))
        assert got[0] is a[pick]
        for on, t, want in zip(need, got, (dx, g1, g2)):
            assert torch.equal(t, want) if on else t is None
    for buf, need in ((x, (True, True, False)), (dy, (True, False, True)), (x, (True, True, True))):
        with pytest.raises(tfb.TfError):
            tfb.gated_ffn_bwd(x, w1, w2, z, dy, need=need, grads=(buf, None, None))
    over = w1.clone()
    got = tfb.gated_ffn_bwd(x, over, w2, z, dy, need=(False, True, True), grads=(None, over, None))
    assert torch.equal(got[1], g1) and torch.equal(got[2], g2)
