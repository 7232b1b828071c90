"""sm_100a fused ops behind the reference's kernel-package names.

Mirrors the export list of the reference's ``solution/kernels/__init__.py:3-51``,
and adds (no counterpart there) the operators of preference and policy tuning,
norms of queries and keys with their rotation, positions of several axes, and
projections with several adapters.
"""

from .attention import window_attention

from .chunked_ce import (
    _chunked_cross_entropy_fused_kernel,
    chunk_cross_entropy_triton,
    make_triton_chunked_loss_function,
    patch_soup_chunked_loss,
    fused_linear_cross_entropy,
)
from .multi_lora import multi_lora_linear
from .qk_norm_rope import apply_multi_axis_rope, apply_qk_norm_rope, rope_axes
from .rmsnorm import (
    _rms_norm_fwd_kernel,
    _rms_norm_bwd_dx_kernel,
    FastRMSNormFunction,
    fast_rms_norm,
    patch_qwen2_rmsnorm,
)
from .rope import (
    _fused_rope_2d_fwd_kernel,
    _fused_rope_2d_bwd_kernel,
    FastRoPEFunction,
    FastRoPEQKFunction,
    apply_fast_rope,
    apply_fast_rope_qk,
    patch_qwen2_rope,
)
from .swiglu import (
    _custom_swiglu_fwd_kernel,
    _custom_swiglu_bwd_kernel,
    FastSwiGLUFunction,
    fast_swiglu,
    patch_qwen2_mlp,
    quantize_8bit,
    swiglu_8bit,
)
from .token_logps import head_token_logps
from .tuning_loss import policy_loss, preference_loss

__all__ = [
    "_chunked_cross_entropy_fused_kernel",
    "chunk_cross_entropy_triton",
    "make_triton_chunked_loss_function",
    "patch_soup_chunked_loss",
    "fused_linear_cross_entropy",
    "_rms_norm_fwd_kernel",
    "_rms_norm_bwd_dx_kernel",
    "FastRMSNormFunction",
    "fast_rms_norm",
    "patch_qwen2_rmsnorm",
    "_fused_rope_2d_fwd_kernel",
    "_fused_rope_2d_bwd_kernel",
    "FastRoPEFunction",
    "FastRoPEQKFunction",
    "apply_fast_rope",
    "apply_fast_rope_qk",
    "patch_qwen2_rope",
    "_custom_swiglu_fwd_kernel",
    "_custom_swiglu_bwd_kernel",
    "FastSwiGLUFunction",
    "fast_swiglu",
    "patch_qwen2_mlp",
    "head_token_logps",
    "preference_loss",
    "policy_loss",
    "window_attention",
    "swiglu_8bit",
    "quantize_8bit",
    "apply_qk_norm_rope",
    "apply_multi_axis_rope",
    "rope_axes",
    "multi_lora_linear",
]
