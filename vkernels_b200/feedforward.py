"""Dense gated feed-forward in 16 bits: the layers of a mixture-of-experts model that are not routed.

``DenseFeedForward`` is the two projections of one such layer, on the weights as the checkpoint holds them. It stands alone (the
first layers of many models are dense), or as the always-on expert of a ``FusedMoEMxfp4`` whose checkpoint keeps that expert in
bf16 (``FusedMoEMxfp4(..., shared_ffn=ffn)``): its second projection then adds the routed experts' result as its residual, so
that the sum costs no pass of its own.
"""
from __future__ import annotations

import torch

from . import torch_ops as ops


class DenseFeedForward:
    """``act(x W1^T + b1) * (x W3^T + b3) @ W2^T + b2 [+ residual]``, weights in bf16 or fp16.

    ``w13`` ``[2 * ispp, hidden]`` holds the gate rows, then the up rows, ``w2`` is ``[hidden, ispp]``; biases ``[2 * ispp]`` and
    ``[hidden]`` or None, all of one type. The activation is the routed layer's: SwiGLU with its limit, or SiTU.

    Called with gradients enabled and weights or x that require one, the result records them (``backward()``); otherwise it may
    be captured into a CUDA graph."""

    def __init__(self, w13: torch.Tensor, w2: torch.Tensor, *, b13: torch.Tensor | None = None, b2: torch.Tensor | None = None,
                 activation: int = ops.SWIGLU, swiglu_limit: float = 0.0, beta: float = 4.0, linear_beta: float = 25.0):
        ops.require(w13.dim() == 2 and w2.dim() == 2 and w13.shape[0] == 2 * w2.shape[1] and w13.shape[1] == w2.shape[0],
                    f"w13 [2 * ispp, hidden] and w2 [hidden, ispp] expected, got {tuple(w13.shape)} and {tuple(w2.shape)}")
        for name, t in (("w2", w2), ("b13", b13), ("b2", b2)):
            ops.require(t is None or (t.dtype == w13.dtype and t.device == w13.device),
                        f"{name} must have the type and device of w13")
        self.w13, self.w2, self.b13, self.b2 = w13, w2, b13, b2
        self.hidden, self.ispp = w2.shape
        self.kind = dict(activation=activation, swiglu_limit=swiglu_limit, beta=beta, linear_beta=linear_beta)

    def records(self, *inputs: torch.Tensor | None) -> bool:
        """Whether a call with these inputs records itself for ``backward()``."""
        return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*inputs, self.w13, self.w2, self.b13, self.b2))

    def product(self, x: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """The gated projection alone: ``[..., ispp]`` for x ``[..., hidden]``."""
        return ops.gated_linear(x, self.w13, self.b13, out=out, **self.kind)

    def project(self, h: torch.Tensor, residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """The second projection alone: ``[..., hidden]`` for a product h ``[..., ispp]``."""
        return ops.fused_linear(h, self.w2, self.b2, residual=residual, out=out)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                product: torch.Tensor | None = None) -> torch.Tensor:
        """y ``[..., hidden]`` for x ``[..., hidden]``. ``out`` (it may be the residual, or x) and ``product`` (``[..., ispp]``, the
        gated projection's result) are places for the results that the caller keeps; ``product`` is written before the residual and
        the second projection's weights are read, and must not overlap them."""
        if product is not None:
            ops.require_apart("product", product, ("the residual", residual), ("w2", self.w2), ("b2", self.b2))
        if out is not None:
            ops.require_apart("out", out, ("w13", self.w13), ("b13", self.b13))
        return self.project(self.product(x, out=product), residual, out=out)

    __call__ = forward
