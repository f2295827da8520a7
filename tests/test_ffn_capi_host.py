"""Host-side checks of the feed-forward, block-norm and dropout entry points (no
GPU): bad arguments are refused before the device is touched, and the workspace
queries and the generator's host form are what they say."""
import ctypes

import numpy as np
import pytest

from ffn_ref import philox_words
from teenyformers_b200 import _capi
from teenyformers_b200._capi import (TF_ERR_INVALID_ARG, TF_ERR_MISALIGNED, TF_ERR_TOO_LARGE,
                                     TF_ERR_UNSUPPORTED, TF_OK)

FAKE = ctypes.c_void_p(0x10000)      # 16-byte aligned, never dereferenced
ODD = ctypes.c_void_p(0x10002)


def test_philox_known_answers():
    """Known answers published with the generator: zeros, ones, and digits of pi."""
    f = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((f, f, f, f), (f, f), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = philox_words([np.array([c], np.uint64) for c in counter], key)
        assert tuple(int(w[0]) for w in got) == want


def ffn(*, x=FAKE, w1=FAKE, w2=FAKE, r=None, a=FAKE, z=None, y=FAKE, m=4, d=64, F=128, act=0):
    return _capi.raw("tf_b200_gated_ffn_fwd_bf16", x, w1, w2, r, a, z, y, m, d, F, act, None)


def test_gated_ffn_refusals(native_lib):
    assert ffn(m=-1) == TF_ERR_INVALID_ARG
    assert ffn(act=3) == TF_ERR_INVALID_ARG
    assert ffn(act=-1) == TF_ERR_INVALID_ARG
    assert ffn(d=60) == TF_ERR_UNSUPPORTED
    assert ffn(F=100) == TF_ERR_UNSUPPORTED
    assert ffn(F=0) == TF_ERR_UNSUPPORTED
    assert ffn(F=0x7FFFFFF8) == TF_ERR_TOO_LARGE
    assert ffn(m=1 << 30, d=1 << 16) == TF_ERR_TOO_LARGE     # tiles past 31 bits
    assert ffn(d=1 << 24, F=1 << 24) == TF_ERR_TOO_LARGE
    for k in ("x", "w1", "w2", "a", "y"):
        assert ffn(**{k: None}) == TF_ERR_INVALID_ARG
        assert ffn(**{k: ODD}) == TF_ERR_MISALIGNED
    assert ffn(r=ODD) == TF_ERR_MISALIGNED
    assert ffn(z=ODD) == TF_ERR_MISALIGNED
    assert ffn(m=0, x=None) == TF_OK


def ffn_bwd(*, x=FAKE, w1=FAKE, w2=FAKE, z=FAKE, dy=FAKE, dx=FAKE, d1=FAKE, d2=FAKE, ws=FAKE, m=4,
            d=64, F=128, act=0):
    return _capi.raw("tf_b200_gated_ffn_bwd_bf16", x, w1, w2, z, dy, dx, d1, d2, ws, m, d, F, act,
                     None)


def test_gated_ffn_bwd_refusals(native_lib):
    assert ffn_bwd(m=-1) == TF_ERR_INVALID_ARG
    assert ffn_bwd(act=9) == TF_ERR_INVALID_ARG
    assert ffn_bwd(d=4) == TF_ERR_UNSUPPORTED
    for k in ("x", "w1", "w2", "z", "dy", "ws"):
        assert ffn_bwd(**{k: None}) == TF_ERR_INVALID_ARG
    for k in ("x", "w1", "w2", "z", "dy", "dx", "d1", "d2", "ws"):
        assert ffn_bwd(**{k: ODD}) == TF_ERR_MISALIGNED
    assert ffn_bwd(dx=None, d1=None, d2=None) == TF_OK       # nothing asked for
    size = lambda m, d, F: _capi.raw("tf_b200_gated_ffn_bwd_workspace_size", m, d, F)
    up = lambda n: -(-n // 256) * 256
    assert size(7, 64, 128) == up(7 * 128 * 3 * 2)           # dz and a
    assert size(0, 64, 128) == size(5, 64, 100) == size(5, 60, 128) == size(5, 0, 128) == 0
    assert size(1 << 20, 4096, 1 << 16) == (1 << 36) * 6     # no 32-bit overflow
    # few tokens and a long sum for dx: fp32 partial sums besides
    assert size(129, 1032, 2776) >= up(129 * 2776 * 6) + 2 * 129 * 1032 * 4
    # many tokens and small weights: of the weights' gradients
    assert size(8192, 64, 64) > up(8192 * 64 * 6) + 2 * 2 * 64 * 64 * 4


def norm(*, x=FAKE, f=FAKE, wp=FAKE, g=FAKE, wn=FAKE, y=FAKE, h=FAKE, rng=None, rows=6, cols=64,
         gr=1, eps=1e-5, rs=1.0, bs=1.0, p=0.0, site=0):
    return _capi.raw("tf_b200_block_norm_fwd_bf16", x, f, wp, g, wn, y, h, rng, rows, cols, gr, eps,
                     rs, bs, p, site, None)


def test_block_norm_refusals(native_lib):
    nan = float("nan")
    assert norm(rows=-1) == TF_ERR_INVALID_ARG
    assert norm(cols=12) == TF_ERR_UNSUPPORTED
    assert norm(cols=8200) == TF_ERR_UNSUPPORTED
    for gr in (0, -1, 4):
        assert norm(gr=gr) == TF_ERR_INVALID_ARG
    for bad in (dict(eps=-1.0), dict(eps=nan), dict(rs=nan), dict(bs=float("inf")), dict(p=-0.5),
                dict(p=1.5), dict(p=nan), dict(p=0.5)):
        assert norm(**bad) == TF_ERR_INVALID_ARG
    assert norm(p=0.5, rng=ctypes.c_void_p(0x10004)) == TF_ERR_MISALIGNED
    assert norm(p=0.5, rng=FAKE, rows=1 << 30, gr=1, cols=8192) == TF_ERR_TOO_LARGE
    for k in ("x", "y", "h"):
        assert norm(**{k: None}) == TF_ERR_INVALID_ARG
    for k in ("x", "f", "wp", "g", "wn", "y", "h"):
        assert norm(**{k: ODD}) == TF_ERR_MISALIGNED
    assert norm(f=None, wp=None, g=None, wn=None) == TF_ERR_INVALID_ARG
    assert norm(f=None) == TF_ERR_INVALID_ARG                # a gate without a branch
    assert norm(rows=0, x=None) == TF_OK


def norm_bwd(*, f=FAKE, y=FAKE, dy=FAKE, dh=FAKE, wp=FAKE, g=FAKE, wn=FAKE, dx=FAKE, df=FAKE,
             dwp=FAKE, dg=FAKE, dwn=FAKE, rng=None, ws=FAKE, rows=6, cols=64, gr=1, eps=1e-5, rs=1.0,
             bs=1.0, p=0.0, site=0):
    return _capi.raw("tf_b200_block_norm_bwd_bf16", f, y, dy, dh, wp, g, wn, dx, df, dwp, dg, dwn,
                     rng, ws, rows, cols, gr, eps, rs, bs, p, site, None)


def test_block_norm_bwd_refusals(native_lib):
    for k in ("f", "y", "dh", "dx", "df", "dwp", "dg", "dwn", "ws"):
        assert norm_bwd(**{k: None}) == TF_ERR_INVALID_ARG, k
    for k in ("f", "y", "dy", "dh", "wp", "g", "wn", "dx", "df", "dwp", "dg", "dwn", "ws"):
        assert norm_bwd(**{k: ODD}) == TF_ERR_MISALIGNED, k
    assert norm_bwd(dy=None, dh=None, wn=None) == TF_ERR_INVALID_ARG
    assert norm_bwd(wn=None) == TF_ERR_INVALID_ARG           # dh without its norm
    assert norm_bwd(p=0.5) == TF_ERR_INVALID_ARG
    assert norm_bwd(gr=5) == TF_ERR_INVALID_ARG
    size = lambda r, c: _capi.raw("tf_b200_block_norm_bwd_workspace_size", r, c)
    assert size(0, 64) == 0 and size(4, 12) == 0
    assert size(1, 64) == (1 + 1) * 2 * 64 * 4
    # at most 296 CTAs, whatever the rows: two fp32 rows of columns for each and its teams
    assert size(1 << 30, 4096) <= 296 * (1 + 1) * 2 * 4096 * 4
    assert size(1 << 30, 512) <= 296 * (1 + 8) * 2 * 512 * 4


@pytest.mark.parametrize("fn", ["tf_b200_dropout_bf16", "tf_b200_dropout_f32"])
def test_dropout_refusals(native_lib, fn):
    def drop(x=FAKE, r=None, y=FAKE, rng=FAKE, n=64, p=0.5, site=0):
        return _capi.raw(fn, x, r, y, rng, n, p, site, None)
    for p in (-0.1, 1.5, float("nan")):
        assert drop(p=p) == TF_ERR_INVALID_ARG
    assert drop(rng=None) == TF_ERR_INVALID_ARG
    assert drop(rng=ctypes.c_void_p(0x10004)) == TF_ERR_MISALIGNED
    assert drop(x=None) == TF_ERR_INVALID_ARG
    assert drop(y=None) == TF_ERR_INVALID_ARG
    assert drop(x=ODD) == drop(y=ODD) == drop(r=ODD) == TF_ERR_MISALIGNED
    assert drop(n=(1 << 35) + 1) == TF_ERR_TOO_LARGE
    assert drop(n=0, x=None) == TF_OK
