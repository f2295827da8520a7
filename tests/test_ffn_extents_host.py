"""Sizes at the edge of 32 bits, refused before a launch (no GPU)."""
import ctypes

from teenyformers_b200 import _capi
from teenyformers_b200._capi import TF_ERR_TOO_LARGE

FAKE = ctypes.c_void_p(0x10000)      # 16-byte aligned, never dereferenced
EDGE = (1 << 31) - 1


def test_extents_whose_tiles_overflow(native_lib):
    """Tiles are counted in 32 bits after rounding an extent up to 256."""
    def fwd(m=4, d=64, F=128):
        return _capi.raw("tf_b200_gated_ffn_fwd_bf16", FAKE, FAKE, FAKE, None, FAKE, None, FAKE, m,
                         d, F, 0, None)
    def bwd(m=4, d=64, F=128):
        at = [ctypes.c_void_p(k << 44) for k in range(1, 10)]
        return _capi.raw("tf_b200_gated_ffn_bwd_bf16", *at, m, d, F, 0, None)
    for m in (EDGE, EDGE - 100, EDGE - 254):
        assert fwd(m=m, d=8, F=8) == TF_ERR_TOO_LARGE
        assert bwd(m=m, d=8, F=8) == TF_ERR_TOO_LARGE
        assert _capi.raw("tf_b200_gated_ffn_bwd_workspace_size", m, 8, 8) == 0
    d = (1 << 31) - 248                   # % 8 == 0
    assert fwd(m=1, d=d, F=8) == bwd(m=1, d=d, F=8) == TF_ERR_TOO_LARGE
    F = (1 << 30) - 120                   # 2 F is 2^31 - 240
    assert fwd(m=1, d=8, F=F) == bwd(m=1, d=8, F=F) == TF_ERR_TOO_LARGE
