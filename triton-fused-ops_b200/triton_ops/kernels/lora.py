"""Low-rank adapters of many requests beside a shared projection.

``fused_lora`` adds ``scaling[i] * B[i] (A[i] x[t])`` of each row's own adapter
``i`` to the shared projection's output (``tfo_lora``, csrc/lora.cu: one launch
for up to 384 rows, a sort and one launch for more), whatever the order of the
requests. ``FP8LoRALinear`` is
:class:`~triton_ops.kernels.fp8_gemm.FP8Linear` with such adapters.

``lora_reference`` is the same in plain PyTorch, for tests; the op never calls it.
"""

from __future__ import annotations

from typing import Optional

import torch

from triton_ops import _lib
from triton_ops.kernels._native import NativeKernel
from triton_ops.kernels.fp8_gemm import FP8Linear
from triton_ops.validation import validate_lora_inputs

fused_lora_kernel = NativeKernel(
    "fused_lora_kernel", "tfo_lora", "rows grouped by adapter, shrink to the rank and expand onto the output"
)

_IDS_CODE = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}


def _rows(t: Optional[torch.Tensor], width: int) -> Optional[torch.Tensor]:
    """[..., width] as [rows, width] with innermost stride 1 (a view where there is one)."""
    if t is None:
        return None
    t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width <= 1 else t.contiguous()


def fused_lora(
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    adapter_ids: torch.Tensor,
    scaling: Optional[torch.Tensor] = None,
    base: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``base[t] + scaling[i] * lora_b[i] @ (lora_a[i] @ x[t])`` with ``i = adapter_ids[t]`` for every row t.

    Args:
        x: [..., in_features], fp16 / bf16 / fp32
        lora_a: [adapters, rank, in_features] in x's dtype (rank <= 256; an
            adapter of lower rank has zero rows)
        lora_b: [adapters, out_features, rank] in x's dtype
        adapter_ids: int32 / int64 adapter of each row, shaped like x without its
            last dimension; negative: none. An id past the end gives a NaN row
            and sets ``_lib.ERR_BAD_ADAPTER`` in the device error word
        scaling: [adapters] fp32 factors, or None for ones
        base: [..., out_features] in x's dtype that the products are added to
            (the shared projection's output), or None for zeros
        out: where to write, or None for a new tensor. It may be `base` itself
            (rows without an adapter are then left as they are) and must not
            otherwise overlap base, x or the adapters. Rows may be strided, for example the
            query columns of a fused projection's output

    Returns:
        [..., out_features] in x's dtype. Sums are fp32, the result is rounded
        once. Serving only: refuses tensors that ask for a gradient or carry a
        forward-mode tangent.
    """
    fast = _lib.ext()
    if fast is not None and x.dim() == 2:
        try:
            got = fast.lora(x, lora_a, lora_b, adapter_ids, scaling, base, out)
        except RuntimeError as exc:
            _lib.raise_ext_error(exc)
        if got is not None:
            return got
    tokens, adapters, rank, k, n = validate_lora_inputs(x, lora_a, lora_b, adapter_ids, scaling, base, out)
    given = out is not None
    if out is None:
        out = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    if out.numel() == 0:
        return out
    try:
        out2 = out.view(-1, n)
    except RuntimeError:
        out2 = None
    if out2 is None or (n > 1 and out2.stride(1) != 1) or (tokens > 1 and out2.stride(0) < n):
        raise ValueError(f"out must be viewable as distinct rows of innermost stride 1, got strides {out.stride()}")
    if given and not out.is_inference():  # written through its pointer: autograd has to know, if it keeps out
        torch.autograd.graph.increment_version(out)
    x2, base2 = _rows(x, k), out2 if base is out else _rows(base, n)
    ids = adapter_ids.reshape(-1).contiguous()
    dtype = _lib.dtype_code(x.dtype, "x")
    with _lib.on_device(x):
        ws = _lib.scratch(_lib.load().tfo_lora_workspace_bytes(tokens, adapters), x.device)
        _lib.call("tfo_lora", x2.data_ptr(), x2.stride(0), lora_a.data_ptr(), lora_b.data_ptr(), ids.data_ptr(),
                  _IDS_CODE[ids.dtype], _lib.ptr(scaling), _lib.ptr(base2), 0 if base2 is None else base2.stride(0),
                  out2.data_ptr(), out2.stride(0), tokens, adapters, rank, k, n, dtype, _lib.ptr(ws),
                  0 if ws is None else ws.numel(), _lib.stream_of(x))
    return out


def lora_reference(
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    adapter_ids: torch.Tensor,
    scaling: Optional[torch.Tensor] = None,
    base: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """PyTorch restatement, one adapter after the other, in fp32."""
    out = torch.zeros((*x.shape[:-1], lora_b.shape[1]), device=x.device) if base is None else base.float()
    for i in range(lora_a.shape[0]):
        s = 1.0 if scaling is None else scaling[i]
        delta = s * ((x.float() @ lora_a[i].float().t()) @ lora_b[i].float().t())
        out = torch.where((adapter_ids == i)[..., None], out + delta, out)
    return out.to(x.dtype)


class FP8LoRALinear(FP8Linear):
    """:class:`FP8Linear` with low-rank adapters of many requests beside its weight.

    The adapters are buffers: ``lora_a`` [max_adapters, rank, in_features],
    ``lora_b`` [max_adapters, out_features, rank] (zeros until
    :meth:`set_adapter`) and ``scaling`` [max_adapters].
    """

    def __init__(self, in_features: int, out_features: int, max_adapters: int, rank: int, bias: bool = False,
                 adapter_dtype: torch.dtype = torch.float16):
        super().__init__(in_features, out_features, bias)
        self.max_adapters = max_adapters
        self.rank = rank
        self.register_buffer("lora_a", torch.zeros(max_adapters, rank, in_features, dtype=adapter_dtype))
        self.register_buffer("lora_b", torch.zeros(max_adapters, out_features, rank, dtype=adapter_dtype))
        self.register_buffer("scaling", torch.ones(max_adapters, dtype=torch.float32))

    def _apply(self, fn, recurse=True):
        scaling = self.scaling
        super()._apply(fn, recurse)
        if self.scaling.dtype != torch.float32:  # .half() and the like: the factors stay fp32
            self.scaling = scaling.to(self.scaling.device)
        return self

    @torch.no_grad()
    def set_adapter(self, index: int, a: torch.Tensor, b: torch.Tensor, scaling: float = 1.0) -> None:
        """Puts an adapter a [r, in_features], b [out_features, r], r <= rank, into slot `index`."""
        if not 0 <= index < self.max_adapters:
            raise ValueError(f"adapter index must be in 0..{self.max_adapters - 1}, got {index}")
        r = a.shape[0]
        if r > self.rank or a.shape != (r, self.in_features) or b.shape != (self.out_features, r):
            from triton_ops.exceptions import ShapeMismatchError

            raise ShapeMismatchError(
                f"adapter must be a [r, {self.in_features}] and b [{self.out_features}, r] with r <= {self.rank}, "
                f"got {tuple(a.shape)} and {tuple(b.shape)}", tensor_name="a, b",
            )
        self.lora_a[index].zero_()[:r] = a.to(self.lora_a)
        self.lora_b[index].zero_()[:, :r] = b.to(self.lora_b)
        self.scaling[index] = scaling

    def forward(self, x: torch.Tensor, adapter_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        y = super().forward(x)
        if adapter_ids is None:
            return y
        if y.dtype != x.dtype:  # an fp32 bias widened the projection
            return y + fused_lora(x, self.lora_a, self.lora_b, adapter_ids, self.scaling)
        return fused_lora(x, self.lora_a, self.lora_b, adapter_ids, self.scaling, base=y, out=y)
