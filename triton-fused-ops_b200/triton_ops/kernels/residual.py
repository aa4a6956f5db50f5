"""A block's branch added to the residual stream, with the norms before and after the block, in one pass.

``fused_residual_rmsnorm`` launches ``tfo_residual_rmsnorm``
(csrc/residual_norm.cu): the branch is normed, dropped out, gated and scaled,
added to the stream, and the sum is normed for the next block. Its gradients come
from ``tfo_residual_rmsnorm_backward`` (csrc/residual_norm_backward.cu).

``residual_rmsnorm_reference`` is the same in plain PyTorch, for tests; the op
never calls it.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from triton_ops import _lib
from triton_ops.kernels._native import NativeKernel
from triton_ops.kernels.dropout import Seed, dropout_params, module_seed, split_seed
from triton_ops.validation import refuse_tangents, validate_residual_inputs

fused_residual_rmsnorm_kernel = NativeKernel(
    "fused_residual_rmsnorm_kernel", "tfo_residual_rmsnorm", "branch norm, dropout, gate, residual sum and next norm in one pass"
)
fused_residual_rmsnorm_backward_kernel = NativeKernel(
    "fused_residual_rmsnorm_backward_kernel", "tfo_residual_rmsnorm_backward",
    "gradients of rows and parameters, fixed sum order"
)

_PARAMS = ("branch_weight", "gate", "weight", "shift")  # in the C ABI's order


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """[..., hidden] as [rows, hidden] with innermost stride 1 (a view where there is one)."""
    if t is None:
        return None
    t = t.reshape(-1, t.shape[-1])
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _param_rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """[hidden], or [batch, hidden] of rows that do not share memory; innermost stride 1."""
    if t is None:
        return None
    if t.dim() > 1:
        t = t.reshape(t.shape[0], t.shape[-1])
        if t.shape[0] <= 1 or t.stride(0) <= 0:
            t = t.contiguous()
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _row_param(t: Optional[torch.Tensor], grad: Optional[torch.Tensor], name: str) -> _lib.RowParam:
    if t is None:
        return _lib.RowParam(None, 0, _lib.F32, None)
    own = 0 if t.dim() == 1 else max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)
    return _lib.RowParam(t.data_ptr(), own, _lib.dtype_code(t.dtype, name), _lib.ptr(grad))


def _row_params(params, grads=(None,) * 4):
    return (_lib.RowParam * 4)(*(_row_param(t, g, n) for t, g, n in zip(params, grads, _PARAMS)))


def _per_seq(x: torch.Tensor) -> int:
    """Rows of a sequence: x is [batch, ..., hidden]."""
    return x.shape[1:-1].numel() if x.dim() > 1 else 1


class _FusedResidualRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, bw, gate, w, shift, branch_norm, norm, scale, eps, p, seed, offset):
        need = any(ctx.needs_input_grad)
        rows = x.numel() // x.shape[-1]
        h = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if norm else None
        rstd = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if need else None
        x2, res2, params = _rows(x), _rows(residual), [_param_rows(t) for t in (bw, gate, w, shift)]
        if rows:
            with _lib.on_device(x):
                _lib.call("tfo_residual_rmsnorm", x2.data_ptr(), x2.stride(0), res2.data_ptr(), res2.stride(0),
                          _row_params(params), h.data_ptr(), _lib.ptr(y), _lib.ptr(rstd), rows, _per_seq(x), x.shape[-1],
                          int(branch_norm), scale, eps, ctypes.byref(dropout_params(p, seed, offset)) if p else None,
                          _lib.dtype_code(x.dtype, "x"), _lib.dtype_code(residual.dtype, "residual"), _lib.stream_of(x))
        if need:
            tensor, ctx.value = split_seed(seed)
            ctx.save_for_backward(x, residual, bw, gate, w, shift, rstd, tensor)
            ctx.args = branch_norm, scale, p, offset
            ctx.set_materialize_grads(False)
        return (h, y) if norm else h

    @staticmethod
    def backward(ctx, dh, dy=None):
        with torch.no_grad():
            d = _backward(ctx, dh, dy)
        if torch.is_grad_enabled():  # create_graph
            sealed = iter(_DifferentiableOnce.apply([t for t in d if t is not None], *ctx.saved_tensors[:6], dh, dy))
            d = tuple(None if t is None else next(sealed) for t in d)
        return (*d, *(None,) * 7)


class _DifferentiableOnce(torch.autograd.Function):
    """Gradients behind what they depend on, with an error where one of them is differentiated."""

    @staticmethod
    def forward(ctx, gradients, *sources):
        return tuple(g.detach() for g in gradients)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("fused_residual_rmsnorm is differentiable once: its gradients cannot be differentiated")


def _backward(ctx, dh, dy):
    """Gradients of x, residual and the parameters, where one is wanted."""
    x, residual, *params, rstd, tensor = ctx.saved_tensors
    branch_norm, scale, p, offset = ctx.args
    refuse_tangents(dh, dy)
    wanted = ctx.needs_input_grad
    make = torch.empty if x.numel() and (dh is not None or dy is not None) else torch.zeros
    dx = make(x.shape, dtype=x.dtype, device=x.device) if wanted[0] else None
    dres = make(x.shape, dtype=residual.dtype, device=x.device) if wanted[1] else None
    grads = [make(t.shape, dtype=t.dtype, device=t.device) if t is not None and w else None
             for t, w in zip(params, wanted[2:6])]
    if make is torch.empty:
        x2, res2, dh2, dy2 = _rows(x), _rows(residual), _rows(dh), _rows(dy)
        kept = [_param_rows(t) for t in params]
        row = _row_params(kept, grads)
        sizes = (x2.shape[0], _per_seq(x), x.shape[-1])
        types = (_lib.dtype_code(x.dtype, "x"), _lib.dtype_code(residual.dtype, "residual"))
        given = (_lib.ptr(dh2), 0 if dh2 is None else dh2.stride(0), _lib.ptr(dy2), 0 if dy2 is None else dy2.stride(0),
                 x2.data_ptr(), x2.stride(0), res2.data_ptr(), res2.stride(0), row)
        drop = ctypes.byref(dropout_params(p, ctx.value if tensor is None else tensor, offset)) if p else None
        with _lib.on_device(x):
            size = _lib.load().tfo_residual_rmsnorm_backward_workspace_bytes(*given, _lib.ptr(dx), _lib.ptr(dres), *sizes,
                                                                             *types)
            ws = _lib.scratch(size, x.device)
            _lib.call("tfo_residual_rmsnorm_backward", *given, rstd.data_ptr(), _lib.ptr(dx), _lib.ptr(dres), *sizes,
                      int(branch_norm), scale, drop, *types, _lib.ptr(ws), size, _lib.stream_of(x))
    return (dx, dres, *grads)


def fused_residual_rmsnorm(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    *,
    branch_norm: bool = False,
    branch_weight: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    scale: float = 1.0,
    eps: float = 1e-6,
    dropout_p: float = 0.0,
    seed: Seed = None,
    dropout_offset: int = 0,
    norm: bool = True,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The residual stream over a block's end and the next one's norm, in one launch::

        u = x / sqrt(mean(x^2) + eps) * branch_weight      (x itself without branch_norm)
        h = residual + scale * gate * dropout(u)
        y = h / sqrt(mean(h^2) + eps) * weight + shift

    Args:
        x: [..., hidden], what the block's last projection gave; fp16 / bf16 / fp32
        residual: the stream, shaped like x, in x's dtype or fp32
        weight, gate, branch_weight, shift: [hidden], or for x [batch, ..., hidden]
            a row for each sequence [batch, hidden] ([batch, 1, hidden] too, and
            views such as the parts of one conditioning projection); any float
            dtype. None: ones (a shift: zeros)
        branch_norm: norm the branch before it is added
        scale: a number that the branch is multiplied by
        eps: added to the means of squares
        dropout_p, seed, dropout_offset: dropout of the branch, as
            :func:`~triton_ops.kernels.dropout.fused_dropout` of it drops
        norm: False after the last block: y is then None

    Returns:
        (h in the residual's dtype, y in x's dtype), contiguous; fp32 inside, y made
        of the h before its rounding. Differentiable (once, in reverse mode) in
        the tensors: gradients made with ``create_graph`` raise where they are
        differentiated. A tensor with a forward-mode tangent is refused.
    """
    fast = _lib.ext()
    if fast is not None and (seed is None or type(seed) in (int, torch.Tensor)):
        tensor, value = split_seed(seed)
        try:
            out = fast.residual_rmsnorm(x, residual, branch_weight, gate, weight, shift, branch_norm, norm, scale, eps,
                                        dropout_p, tensor, value, seed is not None, dropout_offset)
        except RuntimeError as exc:
            _lib.raise_ext_error(exc)
        except TypeError:  # an argument of another kind: the checks below say which
            out = None
        if out is not None:
            return out
    params = {"branch_weight": branch_weight, "gate": gate, "weight": weight, "shift": shift}
    validate_residual_inputs(x, residual, params, branch_norm, norm, dropout_p, seed, dropout_offset)
    out = _FusedResidualRMSNorm.apply(x, residual, branch_weight, gate, weight, shift, bool(branch_norm), bool(norm),
                                      float(scale), float(eps), float(dropout_p), seed, dropout_offset)
    return out if norm else (out, None)


def residual_rmsnorm_reference(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    *,
    branch_norm: bool = False,
    branch_weight: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    scale: float = 1.0,
    eps: float = 1e-6,
    keep: Optional[torch.Tensor] = None,
    dropout_p: float = 0.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """PyTorch restatement in x's precision (at least fp32); `keep`: truth values of what dropout keeps."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32

    def param(t, otherwise):
        if t is None:
            return otherwise
        return t.to(wide) if t.dim() == 1 else t.to(wide).reshape(t.shape[0], *(1,) * (x.dim() - 2), t.shape[-1])

    def normed(t):
        return t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps)

    u = x.to(wide)
    if branch_norm:
        u = normed(u) * param(branch_weight, 1.0)
    if keep is not None:
        u = torch.where(keep, u / (1 - dropout_p), 0.0)
    h = residual.to(wide) + scale * param(gate, 1.0) * u
    y = normed(h) * param(weight, 1.0) + param(shift, 0.0)
    return h.to(residual.dtype), y.to(x.dtype)


class FusedResidualRMSNorm(torch.nn.Module):
    """Module form: holds the fp32 norm weights (ones) and, with ``layer_scale``, a gate of its own.

    With ``branch_norm`` a block has norms on both sides. In training with
    ``dropout`` > 0 each call has a seed of its own: drawn from torch's generator
    or, with a ``dropout_seed``, numbered from it, as
    :class:`~triton_ops.kernels.dropout.FusedDropout` does.
    """

    def __init__(self, hidden_dim: int, eps: float = 1e-6, *, branch_norm: bool = False, scale: float = 1.0,
                 layer_scale: Optional[float] = None, dropout: float = 0.0, dropout_seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"the dropout probability must be in 0..1, got {dropout}")
        self.hidden_dim, self.eps, self.branch_norm, self.scale, self.dropout = hidden_dim, eps, branch_norm, scale, dropout
        self.weight = torch.nn.Parameter(torch.ones(hidden_dim))
        self.branch_weight = torch.nn.Parameter(torch.ones(hidden_dim)) if branch_norm else None
        self.gate = torch.nn.Parameter(torch.full((hidden_dim,), float(layer_scale))) if layer_scale is not None else None
        self.seed_given = dropout_seed is not None
        self.register_buffer("seed", torch.tensor([dropout_seed or 0], dtype=torch.int64))

    def forward(
        self,
        x: torch.Tensor,
        residual: torch.Tensor,
        gate: Optional[torch.Tensor] = None,
        shift: Optional[torch.Tensor] = None,
    ) -> Tuple[torch.Tensor, torch.Tensor]:
        """(h, y); `gate` takes the place of the module's own."""
        p = self.dropout if self.training else 0.0
        seed = module_seed(self, x.device) if p > 0 else None
        return fused_residual_rmsnorm(x, residual, self.weight, self.gate if gate is None else gate,
                                      branch_norm=self.branch_norm, branch_weight=self.branch_weight, shift=shift,
                                      scale=self.scale, eps=self.eps, dropout_p=p, seed=seed)
