"""Host-side mirror of teenyformers' attention-path custom ops, over the C ABI.

The reference defines each op as a CustomOp (graph node: name, output-shape
inference) plus a RuntimeOp (activation-input count, param-cache shapes,
forward and backward launch).  The classes here keep those names, argument
meanings and shape rules and launch the sm_100a kernels through
``include/teenyformers_b200.h``; tensors are torch CUDA tensors (torch is the
device-memory / stream plumbing only):

  FlashAttn2Op        src/kernels/flash_attn2.rs:393-429 (non-causal)
  CausalFlashAttn2Op  src/kernels/flash_attn2.rs:539-575
  RopeOp              src/kernels/rope.rs:246-281
  TransposeHeadsOp    src/kernels/transpose_heads.rs:168-203
  MergeHeadsOp        src/kernels/transpose_heads.rs:276-312
  GatedFfnOp          src/layers/ffn.rs:47-56 with src/kernels/swiglu.rs:56-261
  BlockNormOp         src/kernels/fused_add_rmsnorm.rs:53-340, gated and scaled
  DropoutOp           (no counterpart)

Errors: the reference asserts on bad shapes (src/layers/attention.rs:68);
here a bad call raises ValueError (shape) or TfError (status from the C ABI).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _capi
from ._capi import (TF_ACT_GELU, TF_ACT_GELU_TANH, TF_ACT_SILU, TF_ROPE_INTERLEAVED,
                    TF_ROPE_ROTATE_HALF, TfError, call)

__all__ = [
    "FlashAttn2Op", "CausalFlashAttn2Op", "RopeOp", "TransposeHeadsOp", "MergeHeadsOp",
    "flash_attn2_fwd", "flash_attn2_bwd", "rope", "rope_transpose", "transpose_heads",
    "merge_heads", "bwd_workspace", "rmsnorm", "swiglu", "flash_attn2_decode",
    "decode_workspace", "linear", "linear_swiglu", "swiglu_weight_blocks", "rope_table",
    "linear_qkv_rope", "linear_push", "gated_ffn", "gated_ffn_bwd", "block_norm",
    "block_norm_bwd", "dropout", "dropout_rng", "GatedFfnOp", "BlockNormOp", "DropoutOp",
    "TF_ROPE_INTERLEAVED", "TF_ROPE_ROTATE_HALF", "TF_ACT_SILU", "TF_ACT_GELU",
    "TF_ACT_GELU_TANH", "TfError",
]


def _ptr(t: torch.Tensor | None):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _need(cond: bool, msg: str):
    if not cond:
        raise ValueError(msg)


def _as4(x: torch.Tensor) -> torch.Tensor:
    """[BH, S, D] (reference layout) -> [1, BH, S, D]; [B, H, S, D] unchanged."""
    _need(x.dim() in (3, 4), f"expected [BH,S,D] or [B,H,S,D], got {tuple(x.shape)}")
    return x.unsqueeze(0) if x.dim() == 3 else x


# ----------------------------------------------------------------- functional API
def flash_attn2_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float,
                    causal: bool, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None):
    """O, LSE of flash attention.  q [B,Hq,Sq,D] / k,v [B,Hkv,Sk,D] (or 3-D
    [BH,S,D]); bf16 -> tcgen05 kernel, fp32 -> reference-ABI fp32 kernel."""
    q4, k4, v4 = _as4(q), _as4(k), _as4(v)
    B, Hq, Sq, D = q4.shape
    Hkv, Sk = k4.shape[1], k4.shape[2]
    _need(k4.shape == v4.shape and k4.shape[0] == B and k4.shape[3] == D, "k/v shape mismatch")
    for t in (q, k, v):
        _need(t.is_cuda and t.is_contiguous(), "inputs must be contiguous CUDA tensors")
        _need(t.dtype == q.dtype, "q, k, v dtypes differ")
    o = torch.empty_like(q) if out is None else out
    l = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if lse is None else lse
    if q.dtype == torch.bfloat16:
        call("tf_b200_flash_attn2_fwd_bf16", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(l), B, Hq,
             Hkv, Sq, Sk, D, float(softmax_scale), int(bool(causal)), _stream(q))
    elif q.dtype == torch.float32:
        _need(Hq == Hkv, "the fp32 reference-ABI kernels are MHA only")
        call("tf_b200_flash_attn2_fwd_f32", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(l), B * Hq,
             D, Sq, Sk, float(softmax_scale), float("-inf"), int(bool(causal)), _stream(q))
    else:
        raise ValueError(f"unsupported dtype {q.dtype}")
    return o, l


def bwd_workspace(q: torch.Tensor) -> torch.Tensor:
    q4 = _as4(q)
    B, Hq, Sq, _ = q4.shape
    n = _capi.raw("tf_b200_flash_attn2_bwd_workspace_size", B, Hq, Sq)
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=q.device)


def flash_attn2_bwd(q, k, v, o, lse, do, softmax_scale: float, causal: bool,
                    workspace: torch.Tensor | None = None, grads=None):
    """(dQ, dK, dV) of flash attention; same layouts as the forward."""
    q4, k4 = _as4(q), _as4(k)
    B, Hq, Sq, D = q4.shape
    Hkv, Sk = k4.shape[1], k4.shape[2]
    for t in (q, k, v, o, do, lse):
        _need(t.is_cuda and t.is_contiguous(), "inputs must be contiguous CUDA tensors")
    if grads is None:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    else:
        dq, dk, dv = grads
    if q.dtype == torch.bfloat16:
        ws = bwd_workspace(q) if workspace is None else workspace
        call("tf_b200_flash_attn2_bwd_bf16", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(do),
             _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), B, Hq, Hkv, Sq, Sk, D,
             float(softmax_scale), int(bool(causal)), _stream(q))
    elif q.dtype == torch.float32:
        _need(Hq == Hkv, "the fp32 reference-ABI kernels are MHA only")
        call("tf_b200_flash_attn2_bwd_f32", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(do),
             _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv), B * Hq, D, Sq, Sk, float(softmax_scale),
             int(bool(causal)), _stream(q))
    else:
        raise ValueError(f"unsupported dtype {q.dtype}")
    return dq, dk, dv


def decode_workspace(q: torch.Tensor, n_heads_kv: int, cache_capacity: int) -> torch.Tensor | None:
    B, Hq, n_q, D = q.shape
    n = _capi.raw("tf_b200_flash_attn2_decode_workspace_size", B, Hq, n_heads_kv, n_q,
                  cache_capacity, D)
    return torch.empty(int(n), dtype=torch.uint8, device=q.device) if n else None


def flash_attn2_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       cache_seqlens: torch.Tensor, softmax_scale: float,
                       out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                       workspace: torch.Tensor | None = None):
    """KV-cache decode: q [B,Hq,n_q,D], caches [B,Hkv,cap,D], cache_seqlens [B] int32 (device);
    the last n_q cached keys are the new tokens'.  Returns (o, lse)."""
    for t in (q, k_cache, v_cache):
        _need(t.is_cuda and t.is_contiguous() and t.dtype == torch.bfloat16 and t.dim() == 4,
              "q and the caches must be contiguous 4-D bf16 CUDA tensors")
    _need(cache_seqlens.is_cuda and cache_seqlens.dtype == torch.int32 and
          cache_seqlens.is_contiguous(), "cache_seqlens must be a contiguous int32 CUDA tensor")
    B, Hq, n_q, D = q.shape
    _, Hkv, cap, Dk = k_cache.shape
    _need(k_cache.shape == v_cache.shape and k_cache.shape[0] == B and Dk == D,
          "cache shape mismatch")
    _need(cache_seqlens.numel() == B, "cache_seqlens must have one entry per sequence")
    o = torch.empty_like(q) if out is None else out
    l = torch.empty((B, Hq, n_q), dtype=torch.float32, device=q.device) if lse is None else lse
    ws = decode_workspace(q, Hkv, cap) if workspace is None else workspace
    call("tf_b200_flash_attn2_decode_bf16", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(o),
         _ptr(l), _ptr(cache_seqlens), B, Hq, Hkv, n_q, cap, D, float(softmax_scale), _ptr(ws),
         _stream(q))
    return o, l


def rope(x: torch.Tensor, rope_base: float, style: int = TF_ROPE_INTERLEAVED,
         inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """RoPE on [..., S, D] rows (pos = index along S); reference rope.rs:57-140."""
    _need(x.is_cuda and x.is_contiguous() and x.dim() >= 2, "x must be a contiguous CUDA tensor")
    S, D = x.shape[-2], x.shape[-1]
    bh = x.numel() // max(S * D, 1)
    y = torch.empty_like(x) if out is None else out
    fn = {torch.float32: "tf_b200_rope_f32", torch.bfloat16: "tf_b200_rope_bf16"}.get(x.dtype)
    _need(fn is not None, f"unsupported dtype {x.dtype}")
    call(fn, _ptr(x), _ptr(y), bh, S, D, float(math.log(rope_base)), int(style),
         int(bool(inverse)), _stream(x))
    return y


def rope_transpose(x: torch.Tensor, rope_base: float, style: int = TF_ROPE_INTERLEAVED,
                   inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused [B,S,H,D] -> RoPE -> [B,H,S,D]; inverse: [B,H,S,D] -> RoPE^-1 -> [B,S,H,D]."""
    _need(x.is_cuda and x.is_contiguous() and x.dim() == 4 and x.dtype == torch.bfloat16,
          "x must be a contiguous 4-D bf16 CUDA tensor")
    if not inverse:
        B, S, H, D = x.shape
        shape = (B, H, S, D)
    else:
        B, H, S, D = x.shape
        shape = (B, S, H, D)
    y = torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else out
    call("tf_b200_rope_transpose_bf16", _ptr(x), _ptr(y), B, S, H, D,
         float(math.log(rope_base)), int(style), int(bool(inverse)), _stream(x))
    return y


def transpose_heads(x: torch.Tensor, n_heads: int) -> torch.Tensor:
    """[B?, S, H*D] -> [B?, H, S, D], bit-exact (transpose_heads.rs:49-71)."""
    _need(x.is_cuda and x.is_contiguous() and x.dim() in (2, 3), "x must be [S,D] or [B,S,D]")
    x3 = x.unsqueeze(0) if x.dim() == 2 else x
    B, S, DM = x3.shape
    _need(DM % n_heads == 0, "d_model must be divisible by n_heads")
    D = DM // n_heads
    y = torch.empty((B, n_heads, S, D), dtype=x.dtype, device=x.device)
    call("tf_b200_transpose_heads", _ptr(x), _ptr(y), B, S, n_heads, D, x.element_size(),
         _stream(x))
    return y[0] if x.dim() == 2 else y


def merge_heads(x: torch.Tensor) -> torch.Tensor:
    """[B?, H, S, D] -> [B?, S, H*D], bit-exact (transpose_heads.rs:76-96)."""
    _need(x.is_cuda and x.is_contiguous() and x.dim() in (3, 4), "x must be [H,S,D] or [B,H,S,D]")
    x4 = x.unsqueeze(0) if x.dim() == 3 else x
    B, H, S, D = x4.shape
    y = torch.empty((B, S, H * D), dtype=x.dtype, device=x.device)
    call("tf_b200_merge_heads", _ptr(x), _ptr(y), B, S, H, D, x.element_size(), _stream(x))
    return y[0] if x.dim() == 3 else y


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float,
            residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
            residual_out: torch.Tensor | None = None):
    """y = h * rsqrt(mean(h^2) + eps) * weight with h = x (+ residual) over the
    last dim (fused_add_rmsnorm.rs:53-110).  With ``residual`` returns (y, h)."""
    for t in (x, weight) + ((residual,) if residual is not None else ()):
        _need(t.is_cuda and t.is_contiguous() and t.dtype == torch.bfloat16,
              "rmsnorm tensors must be contiguous bf16 CUDA tensors")
    N = x.shape[-1]
    _need(weight.numel() == N, "weight must have the last dim's size")
    rows = x.numel() // max(N, 1)
    y = torch.empty_like(x) if out is None else out
    h = None
    if residual is not None:
        _need(residual.shape == x.shape, "residual shape mismatch")
        h = torch.empty_like(x) if residual_out is None else residual_out
    call("tf_b200_rmsnorm_bf16", _ptr(x), _ptr(residual), _ptr(weight), _ptr(y), _ptr(h), rows,
         N, float(eps), _stream(x))
    return (y, h) if residual is not None else y


def swiglu(z: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """[..., 2*d_ff] = gate || up -> silu(gate) * up (swiglu.rs:56-95)."""
    _need(z.is_cuda and z.is_contiguous() and z.dtype == torch.bfloat16,
          "z must be a contiguous bf16 CUDA tensor")
    d_ff = z.shape[-1] // 2
    rows = z.numel() // max(2 * d_ff, 1)
    y = torch.empty(z.shape[:-1] + (d_ff,), dtype=z.dtype, device=z.device) if out is None else out
    call("tf_b200_swiglu_bf16", _ptr(z), _ptr(y), rows, d_ff, _stream(z))
    return y


def _bf16(*ts):
    for t in ts:
        _need(t.is_cuda and t.is_contiguous() and t.dtype == torch.bfloat16,
              "GEMM tensors must be contiguous bf16 CUDA tensors")


def linear(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None = None,
           heads_seq: int = 0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """x @ weight.T on the tcgen05 GEMM (teeny-core Linear in the block).

    x: [..., k] row-major, or (heads_seq > 0) the attention output
    [B, H, heads_seq, 128], read as the [B * heads_seq, H * 128] matrix that
    merge_heads would build.  weight: [n, k].  Returns [..., n] (or
    [B, heads_seq, n]); with ``residual`` (same shape as the output) returns
    bf16(x @ weight.T) + residual."""
    _bf16(x, weight)
    n, k = weight.shape
    if heads_seq > 0:
        _need(x.dim() == 4 and x.shape[2] == heads_seq and x.shape[1] * x.shape[3] == k,
              "heads-layout x must be [B, H, S, 128] with H * 128 == k")
        lead = (x.shape[0], heads_seq)
        m = x.shape[0] * heads_seq
    else:
        _need(x.shape[-1] == k, "x's last dim must match weight's k")
        lead = tuple(x.shape[:-1])
        m = x.numel() // max(k, 1)
    y = torch.empty(lead + (n,), dtype=x.dtype, device=x.device) if out is None else out
    _bf16(y)
    _need(y.numel() == m * n, "out has the wrong size")
    if residual is not None:
        _bf16(residual)
        _need(residual.numel() == m * n, "residual has the wrong size")
    call("tf_b200_gemm_bf16", _ptr(x), _ptr(weight), _ptr(residual), _ptr(y), m, n, k,
         int(heads_seq), _stream(x))
    return y


def swiglu_weight_blocks(w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """[d_ff, k] gate and up weights -> the [2 d_ff, k] block-interleaved weight
    linear_swiglu reads (128-row blocks: gate 0, up 0, gate 1, up 1, ...)."""
    d_ff, k = w_gate.shape
    _need(w_up.shape == w_gate.shape and d_ff % 128 == 0, "gate/up must be [d_ff, k], d_ff % 128 == 0")
    return torch.stack([w_gate.reshape(d_ff // 128, 128, k), w_up.reshape(d_ff // 128, 128, k)],
                       dim=1).reshape(2 * d_ff, k).contiguous()


def linear_swiglu(x: torch.Tensor, w_gate_up_blocks: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(x @ w_gate.T) * (x @ w_up.T) in one GEMM (ffn.rs:47-56 + swiglu.rs:56-95);
    the weight comes from swiglu_weight_blocks."""
    _bf16(x, w_gate_up_blocks)
    n2, k = w_gate_up_blocks.shape
    d_ff = n2 // 2
    _need(x.shape[-1] == k, "x's last dim must match the weight's k")
    m = x.numel() // max(k, 1)
    y = torch.empty(tuple(x.shape[:-1]) + (d_ff,), dtype=x.dtype, device=x.device) if out is None else out
    _bf16(y)
    _need(y.numel() == m * d_ff, "out has the wrong size")
    call("tf_b200_gemm_swiglu_bf16", _ptr(x), _ptr(w_gate_up_blocks), _ptr(y), m, d_ff, k,
         _stream(x))
    return y


def rope_table(seq_len: int, head_dim: int, rope_base: float, device) -> torch.Tensor:
    """[seq_len, head_dim / 2, 2] fp32 (cos, sin) table for linear_qkv_rope."""
    t = torch.empty((seq_len, head_dim // 2, 2), dtype=torch.float32, device=device)
    call("tf_b200_rope_table_f32", _ptr(t), seq_len, head_dim, float(math.log(rope_base)),
         ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream))
    return t


def linear_qkv_rope(x: torch.Tensor, w_qkv: torch.Tensor, n_heads_q: int, n_heads_kv: int,
                    table: torch.Tensor | None, style: int = TF_ROPE_INTERLEAVED, outs=None):
    """x [B, S, d] @ [Wq; Wk; Wv].T -> (q [B, Hq, S, 128], k, v [B, Hkv, S, 128]) with RoPE
    on q and k (attention.rs:89-123: projections, TransposeHeads, RoPE) in one kernel."""
    _bf16(x, w_qkv)
    B, S, d = x.shape
    D = 128
    _need(w_qkv.shape == ((n_heads_q + 2 * n_heads_kv) * D, d), "w_qkv shape mismatch")
    if outs is None:
        outs = (torch.empty((B, n_heads_q, S, D), dtype=x.dtype, device=x.device),
                torch.empty((B, n_heads_kv, S, D), dtype=x.dtype, device=x.device),
                torch.empty((B, n_heads_kv, S, D), dtype=x.dtype, device=x.device))
    q, k, v = outs
    _bf16(q, k, v)
    if table is not None:
        _need(table.is_cuda and table.dtype == torch.float32 and table.is_contiguous()
              and table.shape[0] >= S and table.numel() // table.shape[0] == D,
              "table must be a contiguous fp32 [>= S, 64, 2] CUDA tensor")
    call("tf_b200_gemm_qkv_rope_bf16", _ptr(x), _ptr(w_qkv), _ptr(q), _ptr(k), _ptr(v),
         _ptr(table), B, S, n_heads_q, n_heads_kv, d, int(style), _stream(x))
    return q, k, v


def linear_push(x: torch.Tensor, weight: torch.Tensor, peer_recv_ptrs, rank: int, world: int,
                heads_seq: int = 0) -> None:
    """Tensor-parallel partial product x @ weight.T whose row slice o is stored
    into rank o's receive buffer peer_recv_ptrs[o] at slot [rank]
    ([world, m / world, n] each): the reduce-scatter half of the all-reduce that
    follows o_proj / down_proj, fused into the GEMM."""
    _bf16(x, weight)
    n, k = weight.shape
    m = (x.shape[0] * heads_seq) if heads_seq > 0 else x.numel() // max(k, 1)
    arr = (ctypes.c_void_p * world)(*[int(p) for p in peer_recv_ptrs])
    call("tf_b200_gemm_push_bf16", _ptr(x), _ptr(weight), arr, m, n, k, int(heads_seq), rank,
         world, _stream(x))


# ----------------------------------------------------------------- feed-forward side of a block
# These wrappers sit on the decode path, where a kernel takes a few microseconds:
# messages are formatted only when they are raised, and the stream and device
# are read without torch's Python objects around them.
def _launch(x: torch.Tensor, name: str, *args) -> None:
    """call(name, *args, stream) on the current stream of x's device, with that
    device current (the library launches on the current device)."""
    index = x.get_device()
    stream = torch._C._cuda_getCurrentRawStream(index)
    fn = getattr(_capi.lib(), name)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        raise TfError(name, rc)


def _addr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _dense(x: torch.Tensor, dtype: torch.dtype, what: str, *ts) -> None:
    index = x.get_device()
    for t in ts:
        if t is not None and (t.dtype != dtype or t.get_device() != index
                              or not t.is_contiguous()):
            raise ValueError(f"{what} tensors must be contiguous {dtype} tensors on {x.device}")


def _buffer(t: torch.Tensor | None, shape, dtype: torch.dtype, x: torch.Tensor,
            name: str) -> torch.Tensor:
    if t is None:
        return x.new_empty(shape, dtype=dtype)
    if (t.shape != shape or t.dtype != dtype or t.get_device() != x.get_device()
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} {tuple(shape)} tensor on {x.device}")
    return t


def _rows(x: torch.Tensor, cols: int) -> int:
    rows = x.numel() // (cols or 1)
    if rows >= 1 << 31 or cols >= 1 << 31:  # (a C int would take the low 32 bits)
        raise ValueError(f"{rows} rows of {cols}: at most 2^31 - 1 each")
    return rows


def _ffn_shapes(x, w_gate_up, w_down):
    _need(x.is_cuda and x.dim() >= 1 and w_gate_up.dim() == 2 and w_down.dim() == 2,
          "x must be a [..., d] CUDA tensor, w_gate_up and w_down matrices")
    d_ff, d = w_down.shape[1], w_down.shape[0]
    _need(x.shape[-1] == d and tuple(w_gate_up.shape) == (2 * d_ff, d),
          "expected x [..., d], w_gate_up [2 * d_ff, d], w_down [d, d_ff]")
    _need(d_ff < 1 << 31, "d_ff must be below 2^31")
    return _rows(x, d), d, d_ff


def gated_ffn(x: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor,
              act: int = TF_ACT_SILU, residual: torch.Tensor | None = None, save: bool = False,
              out: torch.Tensor | None = None, act_out: torch.Tensor | None = None,
              z_out: torch.Tensor | None = None):
    """(act(x Wg^T) * (x Wu^T)) Wd^T (+ residual), the gated feed-forward of a block
    (ffn.rs:47-56 around swiglu.rs:56-95), for any number of tokens.

    x [..., d] bf16; w_gate_up [2 * d_ff, d] = [Wg; Wu] (the layer's layout); w_down
    [d, d_ff]; act TF_ACT_SILU / GELU / GELU_TANH.  ``save`` also returns z
    [..., 2 * d_ff] fp32 = x [Wg; Wu]^T for gated_ffn_bwd.  ``out``, ``act_out``
    ([..., d_ff] scratch) and ``z_out`` (with ``save``) are buffers to use instead of
    new ones."""
    m, d, d_ff = _ffn_shapes(x, w_gate_up, w_down)
    lead = x.shape[:-1]
    _dense(x, torch.bfloat16, "gated_ffn", x, w_gate_up, w_down, residual)
    _need(residual is None or residual.shape == x.shape, "residual must have x's shape")
    _need(save or z_out is None, "z_out is written with save=True only")
    y = torch.empty_like(x) if out is None else _buffer(out, x.shape, torch.bfloat16, x, "out")
    a = _buffer(act_out, lead + (d_ff,), torch.bfloat16, x, "act_out")
    z = _buffer(z_out, lead + (2 * d_ff,), torch.float32, x, "z_out") if save else None
    _launch(x, "tf_b200_gated_ffn_fwd_bf16", x.data_ptr(), w_gate_up.data_ptr(),
            w_down.data_ptr(), _addr(residual), a.data_ptr(), _addr(z), y.data_ptr(), m, d, d_ff,
            int(act))
    return (y, z) if save else y


@functools.lru_cache(maxsize=256)
def _ffn_workspace_size(m: int, d: int, d_ff: int) -> int:  # (of the shape alone)
    return _capi.raw("tf_b200_gated_ffn_bwd_workspace_size", m, d, d_ff)


def gated_ffn_bwd(x: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor, z: torch.Tensor,
                  dy: torch.Tensor, act: int = TF_ACT_SILU, grads=None, need=(True, True, True),
                  workspace: torch.Tensor | None = None):
    """(dx, dw_gate_up, dw_down) of gated_ffn from z (gated_ffn(..., save=True)) and dy;
    a False in ``need`` skips that gradient (None in its place).  The residual's
    gradient is dy itself.  ``grads``: three tensors to write instead of new ones (dx over
    x or dy only where dw_gate_up or dw_down, which read them, is skipped)."""
    m, d, d_ff = _ffn_shapes(x, w_gate_up, w_down)
    _dense(x, torch.bfloat16, "gated_ffn", x, w_gate_up, w_down, dy)
    _dense(x, torch.float32, "z", z)
    _need(dy.shape == x.shape, "dy must have x's shape")
    _need(z.shape == x.shape[:-1] + (2 * d_ff,), "z must be [..., 2 * d_ff]")
    given = (None, None, None) if grads is None else grads
    g = [None if not on else torch.empty_like(like) if t is None
         else _buffer(t, like.shape, torch.bfloat16, x, "a gradient")
         for t, like, on in zip(given, (x, w_gate_up, w_down), need)]
    ws = _workspace(_ffn_workspace_size(m, d, d_ff), workspace, x)
    _launch(x, "tf_b200_gated_ffn_bwd_bf16", x.data_ptr(), w_gate_up.data_ptr(),
            w_down.data_ptr(), z.data_ptr(), dy.data_ptr(), _addr(g[0]), _addr(g[1]), _addr(g[2]),
            ws.data_ptr(), m, d, d_ff, int(act))
    return tuple(g)


def dropout_rng(seed: int, offset: int = 0, device="cuda") -> torch.Tensor:
    """The generator words of the dropouts: an int64 [2] tensor (seed, offset).  Give
    every step another offset (in place, if a graph replays the step) and every
    dropout of a step another ``site``; a backward pass needs its forward's."""
    wrap = lambda v: (int(v) + (1 << 63)) % (1 << 64) - (1 << 63)
    return torch.tensor([wrap(seed), wrap(offset)], dtype=torch.int64, device=device)


def _rng_addr(p: float, rng: torch.Tensor | None, site: int, x: torch.Tensor):
    _need(0 <= site < 1 << 32, "site must be a 32-bit number")
    if not p:
        return None
    if (rng is None or rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous()
            or rng.get_device() != x.get_device()):
        raise ValueError(f"p > 0 needs rng, an int64 [2] tensor (seed, offset) on {x.device}")
    return rng.data_ptr()


def _drop_p(p: float) -> float:
    """p for the C ABI, which takes 32 bits: the multiple of 2^-16 that is drawn, rounded from
    the caller's 64-bit p (p rounded to 32 bits first may give the next one).  It is exact in
    32 bits, and rounds to itself there."""
    p = float(p)
    return 1.0 - math.floor((1.0 - p) * 65536.0 + 0.5) / 65536.0 if 0.0 <= p <= 1.0 else p


def _workspace(n: int, ws: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor:
    if ws is None:
        return x.new_empty(n, dtype=torch.uint8)
    if ws.get_device() != x.get_device() or not ws.is_contiguous() or \
            ws.numel() * ws.element_size() < n:
        raise ValueError(f"workspace must be contiguous and have {n} bytes on {x.device}")
    return ws


_DROPOUT = {torch.float32: "tf_b200_dropout_f32", torch.bfloat16: "tf_b200_dropout_bf16"}


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor | None, site: int = 0,
            residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """dropout(x) (+ residual), bf16 or fp32, the mask drawn from (rng, site) by a
    counter-based generator and never stored.  The backward pass is
    ``dropout(dy, p, rng, site)``.  ``out`` may be x or residual."""
    fn = _DROPOUT.get(x.dtype)
    if fn is None:
        raise ValueError(f"unsupported dtype {x.dtype}")
    _need(x.is_cuda, "x must be a CUDA tensor")
    _dense(x, x.dtype, "dropout", x, residual)
    _need(residual is None or residual.shape == x.shape, "residual must have x's shape")
    y = torch.empty_like(x) if out is None else _buffer(out, x.shape, x.dtype, x, "out")
    _launch(x, fn, x.data_ptr(), _addr(residual), y.data_ptr(), _rng_addr(p, rng, site, x),
            x.numel(), _drop_p(p), int(site))
    return y


def _norm_shapes(x, w_post, gate, w_pre):
    if not x.is_cuda or x.dim() < 1:
        raise ValueError("block_norm tensors must be [..., cols] CUDA tensors")
    cols = x.shape[-1]
    rows = _rows(x, cols)
    if (w_post is not None and w_post.numel() != cols) or (
            w_pre is not None and w_pre.numel() != cols):
        raise ValueError("a norm's weight must have the last dim's size")
    if gate is None:
        return rows, cols, 1
    _need(gate.dim() >= 1 and gate.shape[-1] == cols, "gate must be [gate_rows, cols] or [cols]")
    gate_rows = gate.numel() // (cols or 1)
    _need(gate_rows >= 1 and rows % gate_rows == 0, "the gate's rows must divide x's")
    return rows, cols, gate_rows


@functools.lru_cache(maxsize=256)
def _norm_workspace_size(rows: int, cols: int) -> int:  # (of the shape alone)
    return _capi.raw("tf_b200_block_norm_bwd_workspace_size", rows, cols)


def block_norm(x: torch.Tensor, f: torch.Tensor | None, w_post: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, w_pre: torch.Tensor | None = None,
               eps: float = 1e-5, residual_scale: float = 1.0, branch_scale: float = 1.0,
               p: float = 0.0, rng: torch.Tensor | None = None, site: int = 0,
               out: torch.Tensor | None = None, norm_out: torch.Tensor | None = None):
    """The norms on either side of a block's residual sum, in one pass:

        y = residual_scale * x + branch_scale * dropout(gate * RMSNorm(f) * w_post)
        h = RMSNorm(y) * w_pre

    x (residual stream) and f (the block's output) [..., cols] bf16; w_post, w_pre
    [cols] or None (no norm there); gate [gate_rows, cols] or None, one row for
    every rows / gate_rows consecutive rows.  f None: only the norm before a block
    (y is x, and ``out`` is refused).  Returns (y, h), h None without w_pre, when a
    ``norm_out`` is left as it was.  ``out`` may be x."""
    rows, cols, gate_rows = _norm_shapes(x, w_post, gate, w_pre)
    _dense(x, torch.bfloat16, "block_norm", x, f, w_post, gate, w_pre)
    _need(f is None or f.shape == x.shape, "f must have x's shape")
    _need(f is not None or out is None, "without f, y is x: out is not written")
    y = x if f is None else _buffer(out, x.shape, x.dtype, x, "out")
    h = None if w_pre is None else _buffer(norm_out, x.shape, x.dtype, x, "norm_out")
    _launch(x, "tf_b200_block_norm_fwd_bf16", x.data_ptr(), _addr(f), _addr(w_post), _addr(gate),
            _addr(w_pre), y.data_ptr(), _addr(h), _rng_addr(p, rng, site, x), rows, cols, gate_rows,
            float(eps), float(residual_scale), float(branch_scale), _drop_p(p), int(site))
    return y, h


def block_norm_bwd(f: torch.Tensor | None, y: torch.Tensor | None, dy: torch.Tensor | None,
                   dh: torch.Tensor | None, w_post: torch.Tensor | None = None,
                   gate: torch.Tensor | None = None, w_pre: torch.Tensor | None = None,
                   eps: float = 1e-5, residual_scale: float = 1.0, branch_scale: float = 1.0,
                   p: float = 0.0, rng: torch.Tensor | None = None, site: int = 0,
                   branch: bool = True, workspace: torch.Tensor | None = None):
    """(dx, df, dw_post, dgate, dw_pre) of block_norm from dy (None: zero) and dh (with
    w_pre), the forward's f and y, and its rng, p and site; None in the place of what
    was not there.  ``branch=False``: the forward had f None."""
    like = dy if dy is not None else dh
    _need(like is not None, "dy or dh is needed")
    rows, cols, gate_rows = _norm_shapes(like, w_post, gate, w_pre)
    _dense(like, torch.bfloat16, "block_norm", f, y, dy, dh, w_post, gate, w_pre)
    shape = like.shape
    for t in (f, y, dy, dh):
        if t is not None and t is not like and t.shape != shape:
            raise ValueError("f, y, dy and dh must have one shape")
    if (w_pre is None) != (dh is None):
        raise ValueError("dh belongs to w_pre")
    if w_pre is not None and y is None:
        raise ValueError("w_pre needs the forward's y")
    if f is None:
        _need(w_post is None and gate is None, "w_post and gate need f")
    _need(branch or (f is None and not p), "branch=False takes no f, w_post, gate or dropout")
    dx = torch.empty_like(like)
    df = torch.empty_like(like) if branch else None
    dw_post = None if w_post is None else torch.empty_like(w_post)
    dgate = None if gate is None else torch.empty_like(gate)
    dw_pre = None if w_pre is None else torch.empty_like(w_pre)
    ws = _workspace(_norm_workspace_size(rows, cols), workspace, like)
    _launch(like, "tf_b200_block_norm_bwd_bf16", _addr(f), _addr(y), _addr(dy), _addr(dh),
            _addr(w_post), _addr(gate), _addr(w_pre), dx.data_ptr(), _addr(df), _addr(dw_post),
            _addr(dgate), _addr(dw_pre), _rng_addr(p, rng, site, like), ws.data_ptr(), rows, cols,
            gate_rows, float(eps), float(residual_scale), float(branch_scale), _drop_p(p), int(site))
    return dx, df, dw_post, dgate, dw_pre


# ----------------------------------------------------------------- op classes
class FlashAttn2Op:
    """Bidirectional flash attention (reference FlashAttn2Op).

    Primary input q [BH, Nq, D] (or [B, H, Nq, D]); others k, v [BH, Nk, D].
    Output o has q's shape; param cache l [BH, Nq] (the LSE).
    ``n_kv_heads`` (GQA) is an addition: the reference is MHA only.
    """

    causal = False
    name = "flash_attn2"

    def __init__(self, head_dim: int, softmax_scale: float, n_kv_heads: int | None = None):
        self.head_dim = int(head_dim)
        self.softmax_scale = float(softmax_scale)
        self.n_kv_heads = n_kv_heads

    # CustomOp
    def infer_output_shape(self, input_shapes):
        return tuple(input_shapes[0])

    # RuntimeOp
    def n_activation_inputs(self) -> int:
        return 3

    def param_shapes(self, input_shapes, output_shape=None):
        q = tuple(input_shapes[0])
        return [list(q[:-1])]

    def has_backward(self) -> bool:
        return True

    def forward(self, q, k, v):
        _need(q.shape[-1] == self.head_dim, "head_dim mismatch")
        return flash_attn2_fwd(q, k, v, self.softmax_scale, self.causal)

    def backward(self, q, k, v, o, l, grad_output, workspace=None):
        return flash_attn2_bwd(q, k, v, o, l, grad_output, self.softmax_scale, self.causal,
                               workspace=workspace)


class CausalFlashAttn2Op(FlashAttn2Op):
    """Causal (decoder self-attention) flash attention; key k hidden from query q when k > q."""

    causal = True
    name = "causal_flash_attn2"


class RopeOp:
    """Rotary position embedding on [BH, N_CTX, HEAD_DIM] (reference RopeOp).

    ``style`` is an addition (the reference is interleaved only)."""

    name = "rope"

    def __init__(self, head_dim: int, rope_base: float, style: int = TF_ROPE_INTERLEAVED):
        self.head_dim = int(head_dim)
        self.rope_base = float(rope_base)
        self.style = int(style)

    def infer_output_shape(self, input_shapes):
        return tuple(input_shapes[0])

    def n_activation_inputs(self) -> int:
        return 1

    def param_shapes(self, input_shapes, output_shape=None):
        return []

    def has_backward(self) -> bool:
        return True

    def forward(self, x):
        _need(x.shape[-1] == self.head_dim, "head_dim mismatch")
        return rope(x, self.rope_base, self.style, inverse=False)

    def backward(self, grad_output):
        return rope(grad_output, self.rope_base, self.style, inverse=True)


class TransposeHeadsOp:
    """[S, D] -> [H, S, HEAD_DIM] (reference TransposeHeadsOp); backward = merge."""

    name = "transpose_heads"

    def __init__(self, n_heads: int, head_dim: int):
        self.n_heads = int(n_heads)
        self.head_dim = int(head_dim)

    def infer_output_shape(self, input_shapes):
        s = input_shapes[0][-2]
        lead = tuple(input_shapes[0][:-2])
        return lead + (self.n_heads, s, self.head_dim)

    def n_activation_inputs(self) -> int:
        return 1

    def param_shapes(self, input_shapes, output_shape=None):
        return []

    def has_backward(self) -> bool:
        return True

    def forward(self, x):
        return transpose_heads(x, self.n_heads)

    def backward(self, grad_output):
        return merge_heads(grad_output)


class MergeHeadsOp:
    """[H, S, HEAD_DIM] -> [S, D] (reference MergeHeadsOp); backward = transpose."""

    name = "merge_heads"

    def __init__(self, n_heads: int, head_dim: int):
        self.n_heads = int(n_heads)
        self.head_dim = int(head_dim)

    def infer_output_shape(self, input_shapes):
        shp = tuple(input_shapes[0])
        return shp[:-3] + (shp[-2], self.n_heads * self.head_dim)

    def n_activation_inputs(self) -> int:
        return 1

    def param_shapes(self, input_shapes, output_shape=None):
        return []

    def has_backward(self) -> bool:
        return True

    def forward(self, x):
        return merge_heads(x)

    def backward(self, grad_output):
        return transpose_heads(grad_output, self.n_heads)


class GatedFfnOp:
    """The gated feed-forward of a block (the reference builds it from Linear ->
    SwigluOp -> Linear, src/layers/ffn.rs:47-56): primary input x [..., d]; others
    w_gate_up [2 * d_ff, d], w_down [d, d_ff].  Param cache z [..., 2 * d_ff] fp32
    (written when ``forward`` is asked to save it for the backward)."""

    name = "gated_ffn"

    def __init__(self, d_ff: int, act: int = TF_ACT_SILU):
        self.d_ff = int(d_ff)
        self.act = int(act)

    def infer_output_shape(self, input_shapes):
        return tuple(input_shapes[0])

    def n_activation_inputs(self) -> int:
        return 3

    def param_shapes(self, input_shapes, output_shape=None):
        return [list(input_shapes[0][:-1]) + [2 * self.d_ff]]

    def has_backward(self) -> bool:
        return True

    def forward(self, x, w_gate_up, w_down, residual=None, save=False):
        _need(w_down.shape[-1] == self.d_ff, "d_ff mismatch")
        return gated_ffn(x, w_gate_up, w_down, self.act, residual=residual, save=save)

    def backward(self, x, w_gate_up, w_down, z, grad_output, workspace=None):
        return gated_ffn_bwd(x, w_gate_up, w_down, z, grad_output, self.act, workspace=workspace)


class BlockNormOp:
    """The norms around a block's residual sum (the reference's FusedAddRmsNormOp,
    src/kernels/fused_add_rmsnorm.rs:53-110, with the norm after the block, its
    gate, scales and dropout).  Primary input x, other f; outputs (y, h)."""

    name = "block_norm"

    def __init__(self, eps: float = 1e-5, residual_scale: float = 1.0, branch_scale: float = 1.0,
                 p: float = 0.0, site: int = 0):
        self.eps = float(eps)
        self.residual_scale = float(residual_scale)
        self.branch_scale = float(branch_scale)
        self.p = float(p)
        self.site = int(site)

    def infer_output_shape(self, input_shapes):
        return tuple(input_shapes[0])

    def n_activation_inputs(self) -> int:
        return 2

    def param_shapes(self, input_shapes, output_shape=None):
        return []

    def has_backward(self) -> bool:
        return True

    def _kw(self, rng):
        return dict(eps=self.eps, residual_scale=self.residual_scale,
                    branch_scale=self.branch_scale, p=self.p, rng=rng, site=self.site)

    def forward(self, x, f, w_post=None, gate=None, w_pre=None, rng=None):
        return block_norm(x, f, w_post, gate, w_pre, **self._kw(rng))

    def backward(self, f, y, grad_y, grad_h, w_post=None, gate=None, w_pre=None, rng=None):
        return block_norm_bwd(f, y, grad_y, grad_h, w_post, gate, w_pre, **self._kw(rng))


class DropoutOp:
    """Dropout by a counter-based generator; forward and backward draw the same mask."""

    name = "dropout"

    def __init__(self, p: float, site: int = 0):
        self.p = float(p)
        self.site = int(site)

    def infer_output_shape(self, input_shapes):
        return tuple(input_shapes[0])

    def n_activation_inputs(self) -> int:
        return 1

    def param_shapes(self, input_shapes, output_shape=None):
        return []

    def has_backward(self) -> bool:
        return True

    def forward(self, x, rng, residual=None):
        return dropout(x, self.p, rng, self.site, residual=residual)

    def backward(self, grad_output, rng):
        return dropout(grad_output, self.p, rng, self.site)
