"""Sizes at the edge of 32 bits, refused before a launch (no GPU)."""
import ctypes

import pytest
import torch

from teenyformers_b200 import _capi, ops
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


class Shape:
    """What the wrappers ask of a tensor before they allocate: rows past 32 bits need 68 GB."""
    is_cuda = True

    def __init__(self, *shape):
        self.shape = torch.Size(shape)

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()


def test_extents_past_31_bits_are_refused():
    """A C int takes the low 32 bits: 2^32 + 5 rows would be 5, 2^32 + 8 columns 8."""
    assert ctypes.c_int((1 << 32) + 5).value == 5
    for rows in (1 << 31, (1 << 32) + 5):
        with pytest.raises(ValueError):
            ops._norm_shapes(Shape(rows, 8), None, None, None)
        with pytest.raises(ValueError):
            ops._ffn_shapes(Shape(rows, 8), Shape(16, 8), Shape(8, 8))
    wide = (1 << 32) + 8
    with pytest.raises(ValueError):
        ops._norm_shapes(Shape(1, wide), None, None, None)
    for d, F in ((wide, 8), (8, wide)):
        with pytest.raises(ValueError):
            ops._ffn_shapes(Shape(1, d), Shape(2 * F, d), Shape(d, F))
    assert ops._norm_shapes(Shape(1 << 30, 8), None, None, None) == (1 << 30, 8, 1)
    assert ops._ffn_shapes(Shape(3, 5, 8), Shape(32, 8), Shape(8, 16)) == (15, 8, 16)
