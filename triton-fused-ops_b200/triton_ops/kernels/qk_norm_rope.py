"""RMSNorm of each query and key head with the rotary rotation, in one pass.

``fused_qk_norm_rope`` launches ``tfo_qk_norm_rope`` (csrc/qk_rope.cu): every
head of q and k is divided by its root mean square, multiplied by a weight
shared by the heads, and rotated at its token's position. Its gradients come
from ``tfo_qk_norm_rope_backward`` (csrc/qk_rope_backward.cu).

Unlike :func:`~triton_ops.kernels.rmsnorm_rope.fused_rmsnorm_rope`, which norms
a whole hidden row and rounds between the norm and the rotation as its
reference does, everything here stays in fp32 up to one rounding of the result.

``qk_norm_rope_reference`` is the same in plain PyTorch, for tests; the op never
calls it.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from triton_ops import _lib
from triton_ops.kernels._native import NativeKernel
from triton_ops.kernels.rope import (
    _dense_heads,
    _empty_like_heads,
    _size_args,
    _strides,
    _table_args,
    rope_heads_reference,
)
from triton_ops.validation import refuse_tangents, validate_head_weight, validate_rope_heads

fused_qk_norm_rope_kernel = NativeKernel(
    "fused_qk_norm_rope_kernel", "tfo_qk_norm_rope", "per-head RMSNorm + rotation of queries and keys in one pass"
)
fused_qk_norm_rope_backward_kernel = NativeKernel(
    "fused_qk_norm_rope_backward_kernel", "tfo_qk_norm_rope_backward", "gradients of heads and weights, fixed sum order"
)


def _weight_code(w: Optional[torch.Tensor], name: str) -> int:
    return _lib.F32 if w is None else _lib.dtype_code(w.dtype, name)


def _forward(q, k, qw, kw, cos, sin, positions, eps, interleaved):
    q_out, k_out = _empty_like_heads(q), _empty_like_heads(k)
    with _lib.on_device(q):
        _lib.call("tfo_qk_norm_rope", q.data_ptr(), _strides(q), _lib.ptr(k), _strides(k), _lib.ptr(qw), _lib.ptr(kw),
                  *_table_args(cos, sin, positions, q), q_out.data_ptr(), _lib.ptr(k_out),
                  *_size_args(q, k, cos, interleaved), float(eps), _lib.dtype_code(q.dtype, "q"),
                  _weight_code(qw, "q_weight"), _weight_code(kw, "k_weight"), _lib.dtype_code(cos.dtype, "cos"),
                  _lib.stream_of(q))
    return q_out, k_out


class _DifferentiableOnce(torch.autograd.Function):
    """Gradients behind what they depend on, with an error where one of them is differentiated."""

    @staticmethod
    def forward(ctx, gradients, *sources):
        return tuple(g.detach() for g in gradients)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("fused_qk_norm_rope is differentiable once: its gradients cannot be differentiated")


class _FusedQKNormRoPE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        q_out, k_out = _forward(q, k, qw, kw, cos, sin, positions, eps, interleaved)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    def backward(ctx, gq, gk=None):
        with torch.no_grad():
            d = _backward(ctx, gq, gk)
        if torch.is_grad_enabled():  # create_graph
            sealed = iter(_DifferentiableOnce.apply([t for t in d if t is not None], *ctx.saved_tensors[:4], gq, gk))
            d = tuple(None if t is None else next(sealed) for t in d)
        return (*d, None, None, None, None, None)


def _backward(ctx, gq, gk):
    """Gradients of q, k (or None) and the weights that want one."""
    q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
    refuse_tangents(gq, gk)
    gq, gk = _dense_heads(gq), _dense_heads(gk if k is not None else None)
    dq, dk = _empty_like_heads(q), _empty_like_heads(k)
    dqw = torch.empty_like(qw) if qw is not None and ctx.needs_input_grad[2] else None
    dkw = torch.empty_like(kw) if kw is not None and ctx.needs_input_grad[3] else None
    with _lib.on_device(q):
        ws = None
        if dqw is not None or dkw is not None:
            ws = _lib.scratch(_lib.load().tfo_qk_norm_rope_backward_workspace_bytes(q.shape[-1]), q.device)
        _lib.call("tfo_qk_norm_rope_backward", gq.data_ptr(), _strides(gq), _lib.ptr(gk), _strides(gk), q.data_ptr(),
                  _strides(q), _lib.ptr(k), _strides(k), _lib.ptr(qw), _lib.ptr(kw),
                  *_table_args(cos, sin, positions, q), dq.data_ptr(), _lib.ptr(dk), _lib.ptr(dqw), _lib.ptr(dkw),
                  *_size_args(q, k, cos, ctx.interleaved), float(ctx.eps), _lib.dtype_code(q.dtype, "q"),
                  _weight_code(qw, "q_weight"), _weight_code(kw, "k_weight"), _lib.dtype_code(cos.dtype, "cos"),
                  _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.stream_of(q))
    return dq, dk, dqw, dkw


def fused_qk_norm_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    q_weight: Optional[torch.Tensor],
    k_weight: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    *,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMSNorm of each head, then the rotation at its token's position, in one launch for q and k.

    Args:
        q, k, cos, sin, positions, interleaved: as for
            :func:`~triton_ops.kernels.rope.fused_rope`
        q_weight, k_weight: [head_dim], any float dtype, or None for ones
        eps: added to the mean of a head's squares before the square root

    Returns:
        (q, k or None) normed and rotated, contiguous, in q's dtype.
        Differentiable (once, in reverse mode) in q, k and the weights: gradients
        made with ``create_graph`` raise where they are differentiated. A tensor
        with a forward-mode tangent is refused.
    """
    fast = _lib.ext()
    if fast is not None:
        try:
            out = fast.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
        except RuntimeError as exc:
            _lib.raise_ext_error(exc)
        if out is not None:
            return out
    cos, sin, positions = validate_rope_heads(q, k, cos, sin, positions)
    validate_head_weight(q, q_weight, "q_weight")
    if k is not None:
        validate_head_weight(q, k_weight, "k_weight")
    else:
        k_weight = None
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        out = _FusedQKNormRoPE.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
        return out if k is not None else (out, None)
    return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


def qk_norm_rope_reference(
    x: torch.Tensor,
    weight: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> torch.Tensor:
    """PyTorch restatement for one tensor, in x's precision (at least fp32)."""
    wide = x if x.dtype == torch.float64 else x.float()
    y = wide / torch.sqrt(wide.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(wide.dtype)
    return rope_heads_reference(y, cos, sin, positions, interleaved).to(x.dtype)


class FusedQKNormRoPE(torch.nn.Module):
    """Module form: holds the fp32 query and key norm weights (initialised to ones)."""

    def __init__(self, head_dim: int, eps: float = 1e-6, interleaved: bool = False):
        super().__init__()
        self.head_dim = head_dim
        self.eps = eps
        self.interleaved = interleaved
        self.q_weight = torch.nn.Parameter(torch.ones(head_dim))
        self.k_weight = torch.nn.Parameter(torch.ones(head_dim))

    def forward(
        self,
        q: torch.Tensor,
        k: Optional[torch.Tensor],
        cos: torch.Tensor,
        sin: torch.Tensor,
        positions: Optional[torch.Tensor] = None,
    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        return fused_qk_norm_rope(q, k, self.q_weight, self.k_weight, cos, sin, positions, self.eps,
                                  interleaved=self.interleaved)
