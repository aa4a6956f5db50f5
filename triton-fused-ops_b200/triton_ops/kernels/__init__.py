"""Op implementations (same module layout and names as the reference's triton_ops.kernels)."""

from triton_ops.kernels.fp8_gemm import FP8Linear, fp8_gemm, fp8_gemm_kernel
from triton_ops.kernels.fp8_quantize import (
    dequantize_fp8,
    dequantize_fp8_kernel,
    quantize_fp8,
    quantize_fp8_kernel,
)
from triton_ops.kernels.gated_mlp import FusedGatedMLP, fused_gated_mlp, fused_gated_mlp_kernel
from triton_ops.kernels.lora import FP8LoRALinear, fused_lora, fused_lora_kernel
from triton_ops.kernels.qk_norm_rope import (
    FusedQKNormRoPE,
    fused_qk_norm_rope,
    fused_qk_norm_rope_backward_kernel,
    fused_qk_norm_rope_kernel,
)
from triton_ops.kernels.rmsnorm_rope import (
    FusedRMSNormRoPE,
    fused_rmsnorm_rope,
    fused_rmsnorm_rope_kernel,
    rmsnorm_kernel,
    rope_kernel,
)
from triton_ops.kernels.rope import (
    RoPEScaling,
    fused_rope,
    fused_rope_kernel,
    rope_tables,
    rope_tables_kernel,
)

__all__ = [
    "fused_rmsnorm_rope",
    "FusedRMSNormRoPE",
    "rmsnorm_kernel",
    "rope_kernel",
    "fused_rmsnorm_rope_kernel",
    "rope_tables",
    "RoPEScaling",
    "fused_rope",
    "rope_tables_kernel",
    "fused_rope_kernel",
    "fused_qk_norm_rope",
    "FusedQKNormRoPE",
    "fused_qk_norm_rope_kernel",
    "fused_qk_norm_rope_backward_kernel",
    "fused_gated_mlp",
    "FusedGatedMLP",
    "fused_gated_mlp_kernel",
    "fp8_gemm",
    "FP8Linear",
    "fp8_gemm_kernel",
    "fused_lora",
    "FP8LoRALinear",
    "fused_lora_kernel",
    "quantize_fp8",
    "dequantize_fp8",
    "quantize_fp8_kernel",
    "dequantize_fp8_kernel",
]
