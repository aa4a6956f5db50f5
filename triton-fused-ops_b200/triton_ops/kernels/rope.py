"""Rotary positions: tables scaled for long contexts, and the rotation of query and key heads.

``rope_tables`` makes cos/sin rows for a range of positions or for given ones
(``tfo_rope_tables``, csrc/rope_tables.cu). ``fused_rope`` rotates queries and
keys by such rows in one launch (``tfo_rope``, csrc/qk_rope.cu): whole heads or
their first columns, halves or neighbouring pairs, at given positions, and
differentiable. The tables also serve
:func:`~triton_ops.kernels.rmsnorm_rope.fused_rmsnorm_rope`.

``rope_heads_reference`` is the same rotation in plain PyTorch, for tests; the
op never calls it.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple, Union

import torch

from triton_ops import _lib
from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError
from triton_ops.kernels._native import NativeKernel
from triton_ops.validation import SUPPORTED_DTYPES_FLOAT, refuse_tangents, validate_rope_heads

rope_tables_kernel = NativeKernel(
    "rope_tables_kernel", "tfo_rope_tables", "cos/sin rows of rotary positions, angles reduced exactly"
)
fused_rope_kernel = NativeKernel(
    "fused_rope_kernel", "tfo_rope", "rotation of query and key heads in one pass over both"
)

_SCALING_KINDS = ("linear", "ntk", "yarn", "wavelength")
_POS_CODE = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}


class _Scaling(NamedTuple):
    kind: str
    factor: float
    original_max_position: Optional[int]
    beta_fast: float
    beta_slow: float
    low_freq_factor: float
    high_freq_factor: float
    attention_factor: Optional[float]


class RoPEScaling(_Scaling):
    """How the rotary frequencies ``f_i = base^(-2i / rotary_dim)`` change for a context `factor` times as long.

    Kinds:
        "linear":     ``f_i / factor`` (positions interpolated)
        "ntk":        the base becomes ``base * factor^(rotary_dim / (rotary_dim - 2))``, which
                      keeps the fastest pair and slows the slowest by `factor`
        "yarn":       pairs that turn more than `beta_fast` times over
                      `original_max_position` keep ``f_i``, those that turn less than
                      `beta_slow` times get ``f_i / factor``, linear in the pair's index in
                      between (the border indexes rounded outwards); cos and sin are
                      multiplied by `attention_factor` (default ``0.1 ln(factor) + 1``)
        "wavelength": pairs with a wavelength ``2 pi / f_i`` below
                      ``original_max_position / high_freq_factor`` keep ``f_i``, those above
                      ``original_max_position / low_freq_factor`` get ``f_i / factor``, linear
                      in ``original_max_position / wavelength`` in between

    `attention_factor` multiplies cos and sin for every kind when it is given.
    """

    __slots__ = ()

    def __new__(cls, kind: str, factor: float = 1.0, original_max_position: Optional[int] = None, beta_fast: float = 32.0,
                beta_slow: float = 1.0, low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                attention_factor: Optional[float] = None):
        if kind not in _SCALING_KINDS:
            raise ValueError(f"kind must be one of {_SCALING_KINDS}, got '{kind}'")
        if not 0 < factor < math.inf:
            raise ValueError(f"factor must be positive and finite, got {factor}")
        if kind in ("yarn", "wavelength") and not (original_max_position and original_max_position > 0):
            raise ValueError(f"kind '{kind}' needs original_max_position")
        if kind == "yarn" and not beta_fast > beta_slow > 0:
            raise ValueError("yarn needs beta_fast > beta_slow > 0")
        if kind == "wavelength" and not high_freq_factor > low_freq_factor > 0:
            raise ValueError("wavelength needs high_freq_factor > low_freq_factor > 0")
        return _Scaling.__new__(cls, kind, factor, original_max_position, beta_fast, beta_slow, low_freq_factor,
                                high_freq_factor, attention_factor)

    @classmethod
    def _make(cls, values):
        """Checked too, so that ``_replace`` is."""
        return cls(*values)


@lru_cache(maxsize=64)
def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[RoPEScaling] = None) -> Tuple[tuple, float]:
    """(angle per position of each pair, factor on cos and sin), in double precision on the host."""
    if rotary_dim < 2 or rotary_dim % 2 != 0 or rotary_dim > 512:
        raise ShapeMismatchError(f"rotary_dim must be even and in 2..512, got {rotary_dim}")
    if not (base > 1 and math.isfinite(base)):
        raise ValueError(f"base must be above 1 and finite, got {base}")
    pairs = range(rotary_dim // 2)
    if scaling is None:
        return tuple(base ** (-2 * i / rotary_dim) for i in pairs), 1.0
    s, gain = scaling, 1.0
    if s.kind == "ntk":
        if rotary_dim == 2:
            raise ShapeMismatchError("ntk scaling needs a rotary_dim above 2")
        base = base * s.factor ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2 * i / rotary_dim) for i in pairs]
    if s.kind == "linear":
        freq = [f / s.factor for f in freq]
    elif s.kind == "yarn":
        def index_of(turns: float) -> float:  # of the pair that turns so often over the original context
            return rotary_dim * math.log(s.original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(index_of(s.beta_fast)), 0)
        high = min(math.ceil(index_of(s.beta_slow)), rotary_dim - 1)
        span = max(high - low, 0.001)
        slow = [min(1.0, max(0.0, (i - low) / span)) for i in pairs]
        freq = [f * (1 - w) + f / s.factor * w for f, w in zip(freq, slow)]
        gain = 0.1 * math.log(s.factor) + 1.0 if s.factor > 1 else 1.0
    elif s.kind == "wavelength":
        span = s.high_freq_factor - s.low_freq_factor
        keep = [min(1.0, max(0.0, (s.original_max_position * f / (2 * math.pi) - s.low_freq_factor) / span)) for f in freq]
        freq = [f * w + f / s.factor * (1 - w) for f, w in zip(freq, keep)]
    if s.attention_factor is not None:
        gain = float(s.attention_factor)
    return tuple(freq), gain


@lru_cache(maxsize=64)
def _turns(rotary_dim: int, base: float, scaling: Optional[RoPEScaling]):
    """The frequencies as host arrays of turns per position (what the kernel takes; torch's default device may be another
    one), and the gain."""
    freq, gain = rope_frequencies(rotary_dim, base, scaling)
    values = [f / (2 * math.pi) for f in freq]
    return (ctypes.c_double * len(values))(*values), torch.tensor(values, dtype=torch.float64, device="cpu"), gain


def rope_tables(
    positions: Union[int, torch.Tensor],
    rotary_dim: int,
    base: float = 10000.0,
    scaling: Optional[RoPEScaling] = None,
    *,
    dtype: torch.dtype = torch.float32,
    device: Optional[torch.device] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin rows of rotary positions.

    Args:
        positions: a count n (rows of positions 0 .. n - 1), or an int32 / int64
            CUDA tensor of positions, for example the one position of each
            request in a decode step
        rotary_dim: columns that are rotated (even, at most 512)
        base: of the frequencies ``base^(-2i / rotary_dim)``
        scaling: :class:`RoPEScaling` for a longer context, or None
        dtype: float16, bfloat16 or float32
        device: where the rows are made if `positions` is a count (default: the
            current CUDA device)

    Returns:
        (cos, sin), each [n, rotary_dim] or [*positions.shape, rotary_dim]; the
        two halves of a row are equal.
    """
    if dtype not in SUPPORTED_DTYPES_FLOAT:
        raise UnsupportedDtypeError(f"tables must be float16, bfloat16 or float32, got {dtype}", dtype=dtype,
                                    supported_dtypes=list(SUPPORTED_DTYPES_FLOAT))
    turns, turns_t, gain = _turns(int(rotary_dim), float(base), scaling)
    if isinstance(positions, torch.Tensor):
        fast = _lib.ext()
        if fast is not None:
            try:
                out = fast.rope_tables(positions, turns_t, gain, _lib.dtype_code(dtype))
            except RuntimeError as exc:
                _lib.raise_ext_error(exc)
            if out is not None:
                return out
        if not positions.is_cuda:
            raise DeviceError(f"positions must be on CUDA device, got {positions.device}", expected_device="cuda",
                              actual_device=str(positions.device), tensor_name="positions")
        if positions.dtype not in _POS_CODE:
            raise UnsupportedDtypeError(f"positions must be int32 or int64, got {positions.dtype}",
                                        dtype=positions.dtype, supported_dtypes=list(_POS_CODE), tensor_name="positions")
        positions = positions.contiguous()
        shape, dev, at, code = (*positions.shape, rotary_dim), positions.device, positions.data_ptr(), _POS_CODE[positions.dtype]
    else:
        if positions < 0:
            raise ShapeMismatchError(f"the number of positions must not be negative, got {positions}")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise DeviceError(f"the tables are made on a CUDA device, got {dev}", expected_device="cuda",
                              actual_device=str(dev))
        shape, at, code = (int(positions), rotary_dim), None, _lib.POS_NONE
    cos = torch.empty(shape, dtype=dtype, device=dev)
    sin = torch.empty(shape, dtype=dtype, device=dev)
    with _lib.on_device(cos):
        _lib.call("tfo_rope_tables", at, code, cos.numel() // rotary_dim, turns, rotary_dim // 2, gain, cos.data_ptr(),
                  sin.data_ptr(), _lib.dtype_code(dtype), _lib.stream_of(cos))
    return cos, sin


def _strides(t: Optional[torch.Tensor]):
    """(batch, seq, head) strides of [batch, seq, heads, dim] or [tokens, heads, dim]."""
    if t is None:
        return None
    s = t.stride()
    return (ctypes.c_int64 * 3)(*(s[:3] if t.dim() == 4 else (0, s[0], s[1])))


def _table_args(cos, sin, positions, q):
    if positions is None:
        pos = (None, _lib.POS_NONE, 0, 0)
    else:
        s = positions.stride()
        pos = (positions.data_ptr(), _POS_CODE[positions.dtype], *(s if q.dim() == 4 else (0, s[0])))
    return (cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0], *pos)


def _size_args(q, k, cos, interleaved):
    batch = q.shape[0] if q.dim() == 4 else 1
    return (batch, q.shape[-3], q.shape[-2], 0 if k is None else k.shape[-2], q.shape[-1], cos.shape[1], int(interleaved))


def _empty_like_heads(t):
    return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rotate(q, k, cos, sin, positions, interleaved, inverse):
    """Launches tfo_rope on checked arguments."""
    q_out, k_out = _empty_like_heads(q), _empty_like_heads(k)
    with _lib.on_device(q):
        _lib.call("tfo_rope", q.data_ptr(), _strides(q), _lib.ptr(k), _strides(k), *_table_args(cos, sin, positions, q),
                  q_out.data_ptr(), _lib.ptr(k_out), *_size_args(q, k, cos, interleaved), int(inverse),
                  _lib.dtype_code(q.dtype, "q"), _lib.dtype_code(cos.dtype, "cos"), _lib.stream_of(q))
    return q_out, k_out


def _dense_heads(t):
    return None if t is None else t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


class _FusedRoPE(torch.autograd.Function):
    """fused_rope where a gradient is wanted: the gradient is the rotation by the opposite angle."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved, ctx.inverse, ctx.with_k = interleaved, inverse, k is not None
        q_out, k_out = _rotate(q, k, cos, sin, positions, interleaved, inverse)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    def backward(ctx, dq, dk=None):
        cos, sin, positions = ctx.saved_tensors
        refuse_tangents(dq, dk)
        dq, dk = _dense_heads(dq), _dense_heads(dk if ctx.with_k else None)
        out = _FusedRoPE.apply(dq, dk, cos, sin, positions, ctx.interleaved, not ctx.inverse)
        dq, dk = out if ctx.with_k else (out, None)
        return dq, dk, None, None, None, None, None


def fused_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    *,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotates query and key heads by their tokens' table rows, in one launch.

    Args:
        q: [batch, seq_len, heads, head_dim] or [tokens, heads, head_dim], fp16 /
            bf16 / fp32; views are fine as long as each head is contiguous (for
            example the query columns of a fused projection's output)
        k: the same with its own number of heads, or None
        cos, sin: [rows, rotary_dim] or [1, rows, 1, rotary_dim], any float dtype;
            the first rotary_dim / 2 columns are read. rotary_dim <= head_dim;
            the columns of a head from rotary_dim on are copied
        positions: int32 / int64 table rows of the tokens, broadcastable to
            [batch, seq_len] (or [tokens]); default: each token's index in its
            sequence. A position outside the tables gives NaN in the rotated
            columns and sets ``_lib.ERR_BAD_POSITION`` in the device error word
        interleaved: False pairs column i with i + rotary_dim / 2, True pairs 2i
            with 2i + 1

    Returns:
        (rotated q, rotated k or None), contiguous. Differentiable in q and k, in
        reverse mode (a tensor with a forward-mode tangent is refused).
    """
    fast = _lib.ext()
    if fast is not None:
        try:
            out = fast.rope(q, k, cos, sin, positions, interleaved)
        except RuntimeError as exc:
            _lib.raise_ext_error(exc)
        if out is not None:
            return out
    cos, sin, positions = validate_rope_heads(q, k, cos, sin, positions)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _FusedRoPE.apply(q, k, cos, sin, positions, interleaved, False)
        return out if k is not None else (out, None)
    return _rotate(q, k, cos, sin, positions, interleaved, False)


def rope_heads_reference(
    x: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> torch.Tensor:
    """PyTorch restatement of the rotation of one tensor, in x's precision (at least fp32)."""
    rot = cos.shape[-1]
    wide = x if x.dtype == torch.float64 else x.float()
    at = torch.arange(x.shape[-3], device=x.device) if positions is None else positions.long()
    c, s = (t[at][..., None, : rot // 2].to(wide.dtype) for t in (cos, sin))
    u, v = (wide[..., 0:rot:2], wide[..., 1:rot:2]) if interleaved else (wide[..., : rot // 2], wide[..., rot // 2:rot])
    y = (u * c - v * s, u * s + v * c)
    y = torch.stack(y, dim=-1).flatten(-2) if interleaved else torch.cat(y, dim=-1)
    return torch.cat([y, wide[..., rot:]], dim=-1).to(x.dtype)
