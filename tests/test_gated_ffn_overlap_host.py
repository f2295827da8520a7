"""Results of the backward pass laid over what the launch that writes them still reads (no GPU)."""
import ctypes

from teenyformers_b200 import _capi
from teenyformers_b200._capi import TF_ERR_INVALID_ARG

M, D, F = 4, 64, 128
AT = {k: i << 44 for i, k in enumerate(("x", "w1", "w2", "z", "dy", "dx", "g1", "g2", "ws"), 1)}
BYTES = {"x": M * D * 2, "dy": M * D * 2, "w1": 4 * F * D, "dx": M * D * 2, "g1": 4 * F * D,
         "g2": 2 * F * D}


def bwd(**over):
    a = dict(AT, **over)
    return _capi.raw("tf_b200_gated_ffn_bwd_bf16", *(ctypes.c_void_p(v) for v in a.values()), M, D, F,
                     0, None)


def test_results_over_inputs_that_are_still_read(native_lib):
    # (which result needs the input; only calls that are refused: the addresses are made up)
    for k, needed_by in (("x", "g1"), ("dy", "g2"), ("w1", "dx")):
        for out in ("dx", "g1", "g2"):
            for off in (0, 16, BYTES[k] - 16, 16 - BYTES[out]):
                assert bwd(**{out: AT[k] + off}) == TF_ERR_INVALID_ARG, (k, out, off)
                others = {o: 0 for o in ("dx", "g1", "g2") if o not in (out, needed_by)}
                assert bwd(**{out: AT[k] + off}, **others) == TF_ERR_INVALID_ARG, (k, out, off)
