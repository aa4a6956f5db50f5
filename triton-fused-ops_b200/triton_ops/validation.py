"""Host-side argument checks for the ops.

Function names, argument order, return values and the exception raised for
each failure follow the reference (triton_ops/validation.py:24-348), so its
tests and callers see the same behaviour:

* tensor not on CUDA            -> DeviceError
* dtype outside the allowed set -> UnsupportedDtypeError
* non-contiguous input          -> ValueError
* incompatible shapes           -> ShapeMismatchError
* unknown activation            -> ValueError

Checks the reference lacks but that guard the native kernels against
out-of-bounds reads (odd head_dim, num_heads * head_dim > hidden, a 4-D RoPE
table shorter than seq_len, tensors on different GPUs) raise
ShapeMismatchError / DeviceError as well.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError

SUPPORTED_DTYPES_FLOAT = [torch.float16, torch.bfloat16, torch.float32]
SUPPORTED_DTYPES_FP8 = [torch.uint8]
if hasattr(torch, "float8_e4m3fn"):
    SUPPORTED_DTYPES_FP8.append(torch.float8_e4m3fn)
if hasattr(torch, "float8_e5m2"):
    SUPPORTED_DTYPES_FP8.append(torch.float8_e5m2)

ACTIVATIONS = ("silu", "gelu", "gelu_tanh")


def _check_cuda(tensor: torch.Tensor, tensor_name: str) -> None:
    if not tensor.is_cuda:
        raise DeviceError(
            f"{tensor_name} must be on CUDA device, got {tensor.device}",
            expected_device="cuda",
            actual_device=str(tensor.device),
            tensor_name=tensor_name,
        )


def _check_same_device(ref: torch.Tensor, tensor: torch.Tensor, tensor_name: str) -> None:
    if tensor.device != ref.device:
        raise DeviceError(
            f"{tensor_name} is on {tensor.device} but the op runs on {ref.device}",
            expected_device=str(ref.device),
            actual_device=str(tensor.device),
            tensor_name=tensor_name,
        )


def _check_dtype(tensor: torch.Tensor, tensor_name: str, supported_dtypes: List[torch.dtype]) -> None:
    if tensor.dtype not in supported_dtypes:
        raise UnsupportedDtypeError(
            f"{tensor_name} has unsupported dtype {tensor.dtype}, supported: {supported_dtypes}",
            dtype=tensor.dtype,
            supported_dtypes=supported_dtypes,
            tensor_name=tensor_name,
        )


def _check_contiguous(tensor: torch.Tensor, tensor_name: str) -> None:
    if not tensor.is_contiguous():
        raise ValueError(f"{tensor_name} must be contiguous")


def validate_rmsnorm_rope_inputs(
    x: torch.Tensor,
    weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    num_heads: Optional[int] = None,
) -> Tuple[int, int, int, int, int]:
    """Checks fused RMSNorm+RoPE inputs.

    x is [batch, seq_len, hidden], weight [hidden], cos/sin [seq_len, head_dim]
    or [1, seq_len, 1, head_dim]. Returns (batch, seq_len, hidden, head_dim,
    num_heads); num_heads defaults to hidden // head_dim.
    """
    for t, n in ((x, "x"), (weight, "weight"), (cos, "cos"), (sin, "sin")):
        _check_cuda(t, n)
    for t, n in ((x, "x"), (weight, "weight"), (cos, "cos"), (sin, "sin")):
        _check_dtype(t, n, SUPPORTED_DTYPES_FLOAT)
    _check_contiguous(x, "x")
    _check_contiguous(weight, "weight")

    if x.dim() != 3:
        raise ShapeMismatchError(
            f"x must be 3D [batch, seq_len, hidden_dim], got {x.dim()}D",
            expected=(None, None, None),
            actual=x.shape,
            tensor_name="x",
        )
    batch_size, seq_len, hidden_dim = x.shape

    if weight.shape != (hidden_dim,):
        raise ShapeMismatchError(
            f"weight shape {weight.shape} doesn't match hidden_dim {hidden_dim}",
            expected=(hidden_dim,),
            actual=weight.shape,
            tensor_name="weight",
        )

    if cos.dim() == 2:
        if cos.shape[0] != seq_len:
            raise ShapeMismatchError(
                f"cos seq_len {cos.shape[0]} doesn't match x seq_len {seq_len}",
                expected=(seq_len, None),
                actual=cos.shape,
                tensor_name="cos",
            )
        head_dim = cos.shape[1]
    elif cos.dim() == 4:
        head_dim = cos.shape[3]
    else:
        raise ShapeMismatchError(f"cos must be 2D or 4D, got {cos.dim()}D", tensor_name="cos")

    if sin.shape != cos.shape:
        raise ShapeMismatchError(
            f"sin shape {sin.shape} doesn't match cos shape {cos.shape}",
            expected=cos.shape,
            actual=sin.shape,
            tensor_name="sin",
        )

    if num_heads is None:
        if head_dim == 0 or hidden_dim % head_dim != 0:
            raise ShapeMismatchError(
                f"hidden_dim {hidden_dim} must be divisible by head_dim {head_dim}",
                tensor_name="x",
            )
        num_heads = hidden_dim // head_dim

    return batch_size, seq_len, hidden_dim, head_dim, num_heads


def check_rmsnorm_rope_kernel_bounds(
    x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, seq_len: int, hidden: int, head_dim: int, num_heads: int
) -> None:
    """Extra checks that keep every kernel access inside the given tensors."""
    for t, n in ((cos, "cos"), (sin, "sin")):
        _check_same_device(x, t, n)
    if head_dim <= 0 or head_dim % 2 != 0:
        raise ShapeMismatchError(f"head_dim must be even and positive, got {head_dim}", tensor_name="cos")
    if num_heads < 0 or num_heads * head_dim > hidden:
        raise ShapeMismatchError(
            f"num_heads {num_heads} x head_dim {head_dim} exceeds hidden_dim {hidden}", tensor_name="x"
        )
    if cos.dim() == 4:
        if cos.shape[0] != 1 or cos.shape[2] != 1 or cos.shape[1] < seq_len:
            raise ShapeMismatchError(
                f"4-D cos/sin must be [1, >=seq_len, 1, head_dim], got {tuple(cos.shape)}",
                expected=(1, seq_len, 1, head_dim),
                actual=cos.shape,
                tensor_name="cos",
            )


def validate_gated_mlp_inputs(
    x: torch.Tensor,
    gate_weight: torch.Tensor,
    up_weight: torch.Tensor,
    activation: str = "silu",
) -> Tuple[int, int, int, int]:
    """Checks gated-MLP inputs; returns (batch, seq_len, hidden, intermediate).

    Accepted activations: "silu", "gelu" (erf form) and "gelu_tanh".
    """
    for t, n in ((x, "x"), (gate_weight, "gate_weight"), (up_weight, "up_weight")):
        _check_cuda(t, n)
    for t, n in ((x, "x"), (gate_weight, "gate_weight"), (up_weight, "up_weight")):
        _check_dtype(t, n, SUPPORTED_DTYPES_FLOAT)
    for t, n in ((x, "x"), (gate_weight, "gate_weight"), (up_weight, "up_weight")):
        _check_contiguous(t, n)

    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be 'silu' or 'gelu' (or 'gelu_tanh'), got '{activation}'")

    if x.dim() != 3:
        raise ShapeMismatchError(f"x must be 3D [batch, seq_len, hidden_dim], got {x.dim()}D", tensor_name="x")
    batch_size, seq_len, hidden_dim = x.shape

    if gate_weight.dim() != 2:
        raise ShapeMismatchError(
            f"gate_weight must be 2D [intermediate_dim, hidden_dim], got {gate_weight.dim()}D",
            tensor_name="gate_weight",
        )
    intermediate_dim, gate_hidden = gate_weight.shape
    if gate_hidden != hidden_dim:
        raise ShapeMismatchError(
            f"gate_weight hidden_dim {gate_hidden} doesn't match x hidden_dim {hidden_dim}",
            expected=(None, hidden_dim),
            actual=gate_weight.shape,
            tensor_name="gate_weight",
        )
    if up_weight.shape != gate_weight.shape:
        raise ShapeMismatchError(
            f"up_weight shape {up_weight.shape} doesn't match gate_weight shape {gate_weight.shape}",
            expected=gate_weight.shape,
            actual=up_weight.shape,
            tensor_name="up_weight",
        )
    _check_same_device(x, gate_weight, "gate_weight")
    _check_same_device(x, up_weight, "up_weight")
    return batch_size, seq_len, hidden_dim, intermediate_dim


def validate_fp8_gemm_inputs(
    a: torch.Tensor,
    b: torch.Tensor,
    a_scale: torch.Tensor,
    b_scale: torch.Tensor,
    output_dtype: torch.dtype = torch.float16,
) -> Tuple[int, int, int]:
    """Checks FP8 GEMM inputs (a [M, K], b [K, N]); returns (M, N, K)."""
    _check_cuda(a, "a")
    _check_cuda(b, "b")
    if a_scale is None or b_scale is None:
        raise ValueError("a_scale and b_scale are required for pre-quantized FP8 operands")
    _check_cuda(a_scale, "a_scale")
    _check_cuda(b_scale, "b_scale")
    _check_contiguous(a, "a")
    _check_contiguous(b, "b")

    if output_dtype not in SUPPORTED_DTYPES_FLOAT:
        raise UnsupportedDtypeError(
            f"output_dtype must be float16, bfloat16, or float32, got {output_dtype}",
            dtype=output_dtype,
            supported_dtypes=list(SUPPORTED_DTYPES_FLOAT),
        )
    if a.dim() != 2:
        raise ShapeMismatchError(f"a must be 2D [M, K], got {a.dim()}D", tensor_name="a")
    if b.dim() != 2:
        raise ShapeMismatchError(f"b must be 2D [K, N], got {b.dim()}D", tensor_name="b")
    M, K_a = a.shape
    K_b, N = b.shape
    if K_a != K_b:
        raise ShapeMismatchError(
            f"Matrix dimensions don't match: a is [{M}, {K_a}], b is [{K_b}, {N}]",
            tensor_name="a, b",
        )
    return M, N, K_a


def validate_fp8_quantize_inputs(tensor: torch.Tensor, scale: Optional[torch.Tensor] = None) -> None:
    """Checks a tensor to be quantized (and its optional scale)."""
    _check_cuda(tensor, "tensor")
    _check_dtype(tensor, "tensor", SUPPORTED_DTYPES_FLOAT)
    _check_contiguous(tensor, "tensor")
    if scale is not None:
        _check_cuda(scale, "scale")


def _check_no_tangent(tensor: torch.Tensor, name: str) -> None:
    """Forward mode: the ops of the query/key path have reverse-mode gradients alone, and a tangent would be lost."""
    if torch.autograd.forward_ad.unpack_dual(tensor).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode tangent: only reverse-mode gradients are there")


def refuse_tangents(*grads: Optional[torch.Tensor]) -> None:
    """The same for the gradients that a backward pass is given."""
    for g in grads:
        if g is not None:
            _check_no_tangent(g, "a gradient")


def check_rope_table(ref: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Checks cos/sin ([rows, rotary_dim] or [1, rows, 1, rotary_dim]) and returns them as 2-D rows of stride 1."""
    for t, n in ((cos, "cos"), (sin, "sin")):
        _check_cuda(t, n)
        _check_dtype(t, n, SUPPORTED_DTYPES_FLOAT)
        _check_same_device(ref, t, n)
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{n} must not require a gradient: the rotary tables have none")
        _check_no_tangent(t, n)
    if cos.dim() == 4 and cos.shape[0] == 1 and cos.shape[2] == 1:
        cos = cos[0, :, 0]
    elif cos.dim() != 2:
        raise ShapeMismatchError(
            f"cos must be [rows, rotary_dim] or [1, rows, 1, rotary_dim], got {tuple(cos.shape)}",
            actual=cos.shape, tensor_name="cos",
        )
    if sin.dim() == 4 and sin.shape[0] == 1 and sin.shape[2] == 1:
        sin = sin[0, :, 0]
    if sin.shape != cos.shape:
        raise ShapeMismatchError(
            f"sin shape {tuple(sin.shape)} doesn't match cos shape {tuple(cos.shape)}",
            expected=cos.shape, actual=sin.shape, tensor_name="sin",
        )
    if sin.dtype != cos.dtype:
        cos, sin = cos.float(), sin.float()
    if cos.stride(1) != 1 or sin.stride() != cos.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin


def _check_heads(t: torch.Tensor, name: str) -> None:
    _check_cuda(t, name)
    _check_dtype(t, name, SUPPORTED_DTYPES_FLOAT)
    if t.dim() not in (3, 4):
        raise ShapeMismatchError(
            f"{name} must be [batch, seq_len, heads, head_dim] or [tokens, heads, head_dim], got {t.dim()}D",
            actual=t.shape, tensor_name=name,
        )
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous heads (innermost stride 1), got strides {t.stride()}")
    _check_no_tangent(t, name)


def validate_rope_heads(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor],
    axes: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Checks query/key heads with their rotary tables and positions.

    Returns (cos, sin, positions) with 2-D tables of stride 1 and positions
    (int32 or int64, or None) expanded to q's token dimensions (after one for the
    axes where a token has `axes` positions).
    """
    _check_heads(q, "q")
    if k is not None:
        _check_heads(k, "k")
        _check_same_device(q, k, "k")
        if k.dtype != q.dtype:
            raise UnsupportedDtypeError(f"k has dtype {k.dtype} but q has {q.dtype}", dtype=k.dtype,
                                        supported_dtypes=[q.dtype], tensor_name="k")
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
            raise ShapeMismatchError(
                f"k shape {tuple(k.shape)} doesn't match q shape {tuple(q.shape)} (all but the heads must agree)",
                expected=q.shape, actual=k.shape, tensor_name="k",
            )
    cos, sin = check_rope_table(q, cos, sin)
    head_dim, rotary_dim = q.shape[-1], cos.shape[1]
    if head_dim < 2 or head_dim > 1024:
        raise ShapeMismatchError(f"head_dim must be in 2..1024, got {head_dim}", tensor_name="q")
    if rotary_dim < 2 or rotary_dim % 2 != 0 or rotary_dim > head_dim:
        raise ShapeMismatchError(
            f"rotary_dim (the tables' width) must be even and at most head_dim {head_dim}, got {rotary_dim}",
            tensor_name="cos",
        )
    if positions is None:
        if cos.shape[0] < q.shape[-3]:
            raise ShapeMismatchError(
                f"the tables have {cos.shape[0]} rows for sequences of {q.shape[-3]} tokens",
                expected=(q.shape[-3], rotary_dim), actual=cos.shape, tensor_name="cos",
            )
        return cos, sin, None
    _check_cuda(positions, "positions")
    _check_dtype(positions, "positions", [torch.int32, torch.int64])
    _check_same_device(q, positions, "positions")
    tokens = tuple(q.shape[:-2]) if axes is None else (axes, *q.shape[:-2])
    if axes is not None and (positions.dim() < 1 or positions.shape[0] != axes):
        raise ShapeMismatchError(
            f"positions of {axes} axes must be {tokens}, got {tuple(positions.shape)}", expected=tokens,
            actual=positions.shape, tensor_name="positions",
        )
    try:
        if axes is not None:  # dimensions that are left out lie behind the axes
            positions = positions.view(axes, *(1,) * (len(tokens) - positions.dim()), *positions.shape[1:])
        positions = positions.expand(tokens)
    except RuntimeError:
        raise ShapeMismatchError(
            f"positions shape {tuple(positions.shape)} doesn't fit the tokens {tokens}",
            expected=tokens, actual=positions.shape, tensor_name="positions",
        ) from None
    if cos.shape[0] == 0 and positions.numel():
        raise ShapeMismatchError("the tables have no rows", actual=cos.shape, tensor_name="cos")
    return cos, sin, positions


def validate_head_weight(q: torch.Tensor, weight: Optional[torch.Tensor], name: str) -> None:
    """Checks a per-head norm weight [head_dim] (None: ones)."""
    if weight is None:
        return
    _check_cuda(weight, name)
    _check_dtype(weight, name, SUPPORTED_DTYPES_FLOAT)
    _check_same_device(q, weight, name)
    if weight.shape != (q.shape[-1],):
        raise ShapeMismatchError(
            f"{name} shape {tuple(weight.shape)} doesn't match head_dim {q.shape[-1]}",
            expected=(q.shape[-1],), actual=weight.shape, tensor_name=name,
        )
    _check_contiguous(weight, name)
    _check_no_tangent(weight, name)


def validate_lora_inputs(
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    adapter_ids: torch.Tensor,
    scaling: Optional[torch.Tensor],
    base: Optional[torch.Tensor],
    out: Optional[torch.Tensor],
) -> Tuple[int, int, int, int, int]:
    """Checks the adapters' inputs; returns (tokens, adapters, rank, in_features, out_features)."""
    named = [(x, "x"), (lora_a, "lora_a"), (lora_b, "lora_b")]
    named += [(t, n) for t, n in ((base, "base"), (out, "out")) if t is not None]
    for t, n in named:
        _check_cuda(t, n)
    for t, n in named:
        _check_dtype(t, n, SUPPORTED_DTYPES_FLOAT if t is x else [x.dtype])
        _check_same_device(x, t, n)
    _check_cuda(adapter_ids, "adapter_ids")
    _check_dtype(adapter_ids, "adapter_ids", [torch.int32, torch.int64])
    _check_same_device(x, adapter_ids, "adapter_ids")
    if x.dim() < 1:
        raise ShapeMismatchError("x must be [..., in_features]", actual=x.shape, tensor_name="x")
    if lora_a.dim() != 3:
        raise ShapeMismatchError(f"lora_a must be 3D [adapters, rank, in_features], got {lora_a.dim()}D",
                                 actual=lora_a.shape, tensor_name="lora_a")
    adapters, rank, k = lora_a.shape
    if x.shape[-1] != k:
        raise ShapeMismatchError(f"lora_a in_features {k} doesn't match x {x.shape[-1]}",
                                 expected=(adapters, rank, x.shape[-1]), actual=lora_a.shape, tensor_name="lora_a")
    if lora_b.dim() != 3 or lora_b.shape[0] != adapters or lora_b.shape[2] != rank:
        raise ShapeMismatchError(f"lora_b must be [{adapters}, out_features, {rank}], got {tuple(lora_b.shape)}",
                                 expected=(adapters, None, rank), actual=lora_b.shape, tensor_name="lora_b")
    n = lora_b.shape[1]
    if not (0 < adapters <= 16384 and 0 < rank <= 256 and k > 0):
        raise ShapeMismatchError(f"need 1..16384 adapters of rank 1..256 and in_features > 0, got {tuple(lora_a.shape)}",
                                 actual=lora_a.shape, tensor_name="lora_a")
    _check_contiguous(lora_a, "lora_a")
    _check_contiguous(lora_b, "lora_b")
    if adapter_ids.shape != x.shape[:-1]:
        raise ShapeMismatchError(f"adapter_ids shape {tuple(adapter_ids.shape)} doesn't match x's rows {tuple(x.shape[:-1])}",
                                 expected=tuple(x.shape[:-1]), actual=adapter_ids.shape, tensor_name="adapter_ids")
    for t, name in ((base, "base"), (out, "out")):
        if t is not None and t.shape != (*x.shape[:-1], n):
            raise ShapeMismatchError(f"{name} shape {tuple(t.shape)} doesn't match {(*x.shape[:-1], n)}",
                                     expected=(*x.shape[:-1], n), actual=t.shape, tensor_name=name)
    if scaling is not None:
        _check_cuda(scaling, "scaling")
        _check_dtype(scaling, "scaling", [torch.float32])
        _check_same_device(x, scaling, "scaling")
        if scaling.shape != (adapters,):
            raise ShapeMismatchError(f"scaling must be [{adapters}], got {tuple(scaling.shape)}", expected=(adapters,),
                                     actual=scaling.shape, tensor_name="scaling")
        _check_contiguous(scaling, "scaling")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, lora_a, lora_b, scaling, base, out)):
        raise ValueError("the adapters of many requests serve and have no gradient: call under torch.no_grad()")
    for t, name in (*named, (scaling, "scaling")):
        if t is not None:
            _check_no_tangent(t, name)
    return x.numel() // k, adapters, rank, k, n


def validate_dropout(x: torch.Tensor, p: float, seed, offset: int, residual: Optional[torch.Tensor]) -> None:
    """Checks a dropout's inputs: x of any shape, a residual of its shape and type (or fp32), probability and seed."""
    _check_cuda(x, "x")
    _check_dtype(x, "x", SUPPORTED_DTYPES_FLOAT)
    _check_no_tangent(x, "x")
    if residual is not None:
        check_residual(x, residual)
    check_dropout_key(x, p, seed, offset)


def check_residual(x: torch.Tensor, residual: torch.Tensor) -> None:
    """Checks the residual stream beside x: its shape, and its type or fp32."""
    _check_cuda(residual, "residual")
    _check_dtype(residual, "residual", [x.dtype, torch.float32])
    _check_same_device(x, residual, "residual")
    if residual.shape != x.shape:
        raise ShapeMismatchError(f"residual shape {tuple(residual.shape)} doesn't match x {tuple(x.shape)}",
                                 expected=x.shape, actual=residual.shape, tensor_name="residual")
    _check_no_tangent(residual, "residual")


def check_dropout_key(x: torch.Tensor, p: float, seed, offset: int) -> None:
    """Checks a dropout's probability, seed (an int, or one int64 beside x) and offset."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the dropout probability must be in 0..1, got {p}")
    if not 0 <= offset < 2**64:
        raise ValueError(f"the dropout offset must be in 0..2^64 - 1, got {offset}")
    if seed is None:
        if p > 0:
            raise ValueError("dropout needs a seed")
    elif isinstance(seed, torch.Tensor):
        _check_cuda(seed, "seed")
        _check_dtype(seed, "seed", [torch.int64])
        _check_same_device(x, seed, "seed")
        if seed.numel() != 1:
            raise ShapeMismatchError(f"seed must hold one number, got {tuple(seed.shape)}", actual=seed.shape,
                                     tensor_name="seed")
    elif isinstance(seed, bool) or not isinstance(seed, int):
        raise TypeError(f"seed must be an int or an int64 tensor, got {type(seed).__name__}")


def validate_residual_inputs(x: torch.Tensor, residual: torch.Tensor, params: dict, branch_norm: bool, norm: bool, p: float,
                             seed, offset: int) -> None:
    """Checks the residual stream's inputs; `params` maps names to [hidden] or [batch, hidden] tensors or None."""
    _check_cuda(x, "x")
    _check_dtype(x, "x", SUPPORTED_DTYPES_FLOAT)
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > 2**24:
        raise ShapeMismatchError(f"x must be [..., hidden] with hidden in 1..2^24, got {tuple(x.shape)}", actual=x.shape,
                                 tensor_name="x")
    if x.numel() // x.shape[-1] >= 2**31:
        raise ShapeMismatchError(f"x must have fewer than 2^31 rows, got {tuple(x.shape)}", actual=x.shape, tensor_name="x")
    _check_no_tangent(x, "x")
    check_residual(x, residual)
    hidden = x.shape[-1]
    for name, t in params.items():
        if t is None:
            continue
        _check_cuda(t, name)
        _check_dtype(t, name, SUPPORTED_DTYPES_FLOAT)
        _check_same_device(x, t, name)
        own = 2 <= t.dim() <= x.dim() and t.shape[0] == x.shape[0] and all(n == 1 for n in t.shape[1:-1])
        if not (t.dim() == 1 or own) or t.shape[-1] != hidden:
            raise ShapeMismatchError(
                f"{name} must be [{hidden}], or [{x.shape[0]}, {hidden}] (a row for each sequence, with or without "
                f"dimensions of 1 between), got {tuple(t.shape)}", expected=(hidden,), actual=t.shape, tensor_name=name)
        _check_no_tangent(t, name)
    if params["branch_weight"] is not None and not branch_norm:
        raise ValueError("branch_weight needs branch_norm=True")
    if not norm and (params["weight"] is not None or params["shift"] is not None):
        raise ValueError("weight and shift need norm=True")
    check_dropout_key(x, p, seed, offset)
