"""Dropout from a counter-based generator: the mask is made again in the backward pass, never stored.

``fused_dropout`` launches ``tfo_dropout`` (csrc/dropout.cu): what is dropped
depends on the seed, the offset and an element's index alone, so the gradient
is the same call on the output's gradient.
:func:`~triton_ops.kernels.residual.fused_residual_rmsnorm` drops the same
elements of its branch for the same seed.

``dropout_keep_reference`` gives the mask in plain PyTorch, for tests; the op
never calls it.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Union

import torch

from triton_ops import _lib
from triton_ops.kernels._native import NativeKernel
from triton_ops.validation import refuse_tangents, validate_dropout

fused_dropout_kernel = NativeKernel(
    "fused_dropout_kernel", "tfo_dropout", "counter-based dropout with an optional residual sum, its own gradient"
)

Seed = Union[int, torch.Tensor, None]


def split_seed(seed: Seed):
    """(device tensor or None, value modulo 2^64)."""
    if isinstance(seed, torch.Tensor):
        return seed, 0
    return None, 0 if seed is None else seed & (2**64 - 1)


def dropout_params(p: float, seed: Seed, offset: int) -> _lib.DropoutParams:
    tensor, value = split_seed(seed)
    return _lib.DropoutParams(p, _lib.ptr(tensor), value, offset)


def _drop(x, residual, p, seed, offset, dtype):
    """Launches tfo_dropout on contiguous tensors."""
    out = torch.empty(x.shape, dtype=dtype, device=x.device)
    with _lib.on_device(x):
        _lib.call("tfo_dropout", x.data_ptr(), _lib.ptr(residual), out.data_ptr(), x.numel(),
                  ctypes.byref(dropout_params(p, seed, offset)), _lib.dtype_code(x.dtype, "x"), _lib.dtype_code(dtype),
                  _lib.stream_of(x))
    return out


class _FusedDropout(torch.autograd.Function):
    """fused_dropout where a gradient is wanted: the gradient of x is the dropout of the output's gradient."""

    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, dtype):
        tensor, ctx.value = split_seed(seed)
        ctx.save_for_backward(tensor)
        ctx.p, ctx.offset, ctx.dtype = p, offset, x.dtype
        ctx.set_materialize_grads(False)
        return _drop(x.contiguous(), None if residual is None else residual.contiguous(), p, seed, offset, dtype)

    @staticmethod
    def backward(ctx, g):
        if g is None:
            return (None,) * 6
        refuse_tangents(g)
        (tensor,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            # 16-bit gradients of an fp32 one's gradient (a second differentiation) go through fp32
            g_in = g if g.dtype in (ctx.dtype, torch.float32) else g.to(ctx.dtype)
            dx = _FusedDropout.apply(g_in, None, ctx.p, ctx.value if tensor is None else tensor, ctx.offset, ctx.dtype)
        return dx, g if ctx.needs_input_grad[1] else None, None, None, None, None


def fused_dropout(
    x: torch.Tensor,
    p: float,
    seed: Seed = None,
    *,
    offset: int = 0,
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``x / (1 - p)`` where kept and 0 elsewhere, ``+ residual``, in one launch and without a stored mask.

    Args:
        x: any shape, fp16 / bf16 / fp32
        p: probability that an element is dropped, in 0..1 (rounded to a multiple
            of 2^-32)
        seed: an int, or one int64 on x's device (read when the kernel runs, so a
            captured graph can be replayed with another one). The same seed
            drops the same elements; it may be None if p is 0
        offset: tells calls that share a seed apart, in 0..2^64 - 1
        residual: shaped like x, in its type or fp32, or None

    Returns:
        A contiguous tensor in x's dtype (with a residual, in the residual's).
        Element i in the order of a contiguous tensor is dropped when word i % 4 of
        the Philox4x32-10 block of counter (i / 4, offset) is below p 2^32; dropped
        elements are zero whatever they were. Differentiable in x and the
        residual, in reverse mode (a forward-mode tangent is refused).
    """
    fast = _lib.ext()
    if fast is not None:
        try:
            tensor, value = split_seed(seed) if seed is None or type(seed) in (int, torch.Tensor) else (None, None)
            out = None if value is None else fast.dropout(x, residual, p, tensor, value, seed is not None, offset)
        except RuntimeError as exc:
            _lib.raise_ext_error(exc)
        except TypeError:  # an argument of another kind: the checks below say which
            out = None
        if out is not None:
            return out
    validate_dropout(x, p, seed, offset, residual)
    dtype = x.dtype if residual is None else residual.dtype
    return _FusedDropout.apply(x, residual, float(p), seed, offset, dtype)


def module_seed(module: torch.nn.Module, device: torch.device) -> torch.Tensor:
    """The seed of one training call of a module with dropout, on `device` (the backward pass reads it again).

    Drawn from torch's generator of the device or, where the module was given a
    seed, the number in its buffer, which goes up by one on the device. A call in
    a backward pass is a forward pass made again for its activations: torch's
    generators are put back for it, the buffer is not, so that it is refused.
    """
    if not module.seed_given:
        return torch.empty(1, dtype=torch.int64, device=device).random_()
    if torch._C._current_graph_task_id() != -1:
        raise RuntimeError("a dropout module with a seed of its own numbers its calls and cannot make one again in a backward "
                           "pass (activation checkpointing): leave its seed out, so that torch's generators give it")
    mine = module.seed.clone()
    module.seed.add_(1)
    return mine


class FusedDropout(torch.nn.Module):
    """Module form: each training call drops other elements.

    Args:
        p: probability that an element is dropped
        seed: None: every call draws its seed on the device from torch's generator,
            as ``torch.nn.Dropout`` draws its mask: ``torch.manual_seed`` governs it,
            activation checkpointing makes the same mask again, modules and ranks
            with generators of their own are independent. An int: calls are
            numbered from it in a buffer of the module, whatever torch's generators
            do; modules whose numbers meet drop the same elements (seeds further
            apart than there are calls do not), and a call in a backward pass
            (checkpointing) raises

    Calls in evaluation mode return x (plus the residual). A captured training
    step takes another seed with each replay.
    """

    def __init__(self, p: float, seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"the dropout probability must be in 0..1, got {p}")
        self.p = p
        self.seed_given = seed is not None
        self.register_buffer("seed", torch.tensor([seed or 0], dtype=torch.int64))

    def next_seed(self, device: Optional[torch.device] = None) -> torch.Tensor:
        """This call's seed, a tensor of its own on `device` (default: that of the module's buffer)."""
        return module_seed(self, self.seed.device if device is None else device)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.training or self.p == 0:
            return x if residual is None else x + residual
        return fused_dropout(x, self.p, self.next_seed(x.device), residual=residual)


def dropout_keep_reference(shape, p: float, seed: int, offset: int = 0, device="cpu") -> torch.Tensor:
    """PyTorch restatement of what is kept, as truth values."""
    low = 0xFFFFFFFF
    count = math.prod(shape)
    block = torch.arange(-(-count // 4), dtype=torch.int64, device=device)
    words = [block & low, block >> 32, torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)]
    key = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        # products of 32-bit words wrap in int64; their halves are the words below
        even, odd = words[0] * 0xD2511F53, words[2] * 0xCD9E8D57
        words = [((odd >> 32) & low) ^ words[1] ^ key[0], odd & low, ((even >> 32) & low) ^ words[3] ^ key[1], even & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    return (torch.stack(words, dim=-1).flatten()[:count] >= round(p * 2**32)).view(shape)
