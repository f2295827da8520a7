"""The feed-forward sublayer of a transformer block, for training and serving.

Mirrors the second half of teenyformers' ``LlamaBlock::forward``
(src/layers/llama_block.rs:60-65 with src/layers/ffn.rs:47-56), with what models
put around it: a norm after the block beside the one before it, a gate and
scales on the branch, dropout.

    h  = RMSNorm(x) * norm
    f  = (act(h Wg^T) * (h Wu^T)) Wd^T
    y  = residual_scale x + branch_scale dropout(gate * RMSNorm(f) * post_norm)
    hn = RMSNorm(y) * next_norm                    (what the next block reads)

``post_norm``, ``gate`` and ``next_norm`` are optional.  Sublayers follow one another with
``next_norm`` of one as ``norm`` of the next (one tensor, and one eps):

    y1, h1, s1 = first.forward(x, train=True)
    y2, h2, s2 = second.forward(y1, h=h1, train=True)
    d1, g2 = second.backward(s2, dy2, dh2)     # h1's gradient is in d1, the norm's is g2["norm"]
    dx, g1 = first.backward(s1, d1)

Forward: three launches and a fourth for the first norm, which a caller that has h
(the sublayer before's ``hn``) saves; any number of tokens, from one decoding token
on.  Backward: six, and a seventh where few tiles have their sums split.
"""
from __future__ import annotations

import torch

from . import ops


class FeedForwardSublayer:
    """``weights``: norm [d], w_gate_up [2 * d_ff, d] = [gate; up], w_down [d, d_ff] and,
    optionally, post_norm [d], gate [gate_rows, d] or [d], next_norm [d]; bf16."""

    def __init__(self, weights: dict, act: int = ops.TF_ACT_SILU, eps: float = 1e-5,
                 residual_scale: float = 1.0, branch_scale: float = 1.0, p: float = 0.0,
                 site: int = 0):
        self.w = weights
        self.eps = float(eps)
        self.ffn = ops.GatedFfnOp(weights["w_down"].shape[1], act)
        self.norm = ops.BlockNormOp(eps, residual_scale, branch_scale, p, site)
        # without dropout (evaluation, serving)
        self.norm_eval = ops.BlockNormOp(eps, residual_scale, branch_scale)

    def _around(self):
        return (self.w.get("post_norm"), self.w.get("gate"), self.w.get("next_norm"))

    def forward(self, x: torch.Tensor, h: torch.Tensor | None = None,
                rng: torch.Tensor | None = None, train: bool = False):
        """(y, hn), and with ``train`` what backward needs as a third.  h: RMSNorm(x) *
        norm if the caller has it.  rng (ops.dropout_rng) is needed with dropout."""
        w = self.w
        if h is None:
            _, h = ops.block_norm(x, None, w_pre=w["norm"], eps=self.eps)
        if not train:
            f = self.ffn.forward(h, w["w_gate_up"], w["w_down"])
            return self.norm_eval.forward(x, f, *self._around())
        f, z = self.ffn.forward(h, w["w_gate_up"], w["w_down"], save=True)
        y, hn = self.norm.forward(x, f, *self._around(), rng=rng)
        return y, hn, (x, h, f, y, z)

    def backward(self, saved, dy: torch.Tensor | None, dhn: torch.Tensor | None = None,
                 rng: torch.Tensor | None = None):
        """(dx, gradients by the weights' names) from the gradients of y and hn (None: zero,
        but not both), the forward's third result and its rng.  dx and the norm's gradient
        are of x alone, whoever computed h.  dhn None, where hn was not used or where the
        sublayer that took it has its gradient in dy: no gradient of next_norm."""
        x, h, f, y, z = saved
        w = self.w
        post, gate, nxt = self._around()
        if dhn is None:
            nxt = None
        # (f is not needed for its own gradient without a norm or gate after the block)
        dres, df, dpost, dgate, dnext = self.norm.backward(
            f if post is not None or gate is not None else None, y, dy, dhn, post, gate, nxt,
            rng=rng)
        dh, dw1, dw2 = self.ffn.backward(h, w["w_gate_up"], w["w_down"], z, df)
        dx, _, _, _, dnorm = ops.block_norm_bwd(None, x, dres, dh, w_pre=w["norm"], eps=self.eps,
                                                branch=False)
        grads = {"norm": dnorm, "w_gate_up": dw1, "w_down": dw2, "post_norm": dpost,
                 "gate": dgate, "next_norm": dnext}
        return dx, {k: v for k, v in grads.items() if v is not None}
