"""Fused SwiGLU forward and recompute-backward on B200 (sm_100a CUDA via the C ABI).

Drop-in for the reference's ``solution/kernels/swiglu.py``: ``FastSwiGLUFunction``,
``fast_swiglu``, ``patch_qwen2_mlp`` and the kernel handles
``_custom_swiglu_fwd_kernel`` / ``_custom_swiglu_bwd_kernel``; arithmetic of
``swiglu.py:20-95`` (sigmoid recomputed from the saved gate in backward).
The MLP patch keeps the reference's selective recompute: gate/up projections
and SwiGLU run under ``torch.utils.checkpoint``, ``down_proj`` outside it
(``swiglu.py:173-221``).
"""

from __future__ import annotations

import torch
import torch.utils.checkpoint

from .. import _lib
from ._shim import LaunchShim


def _rows(t: torch.Tensor, n: int) -> torch.Tensor:
    t2 = t.reshape(-1, n)
    if t2.stride(-1) != 1:
        t2 = t2.contiguous()
    return t2


def swiglu_forward(g2: torch.Tensor, u2: torch.Tensor, out=None) -> torch.Tensor:
    rows, n = g2.shape
    if out is None:
        out = torch.empty((rows, n), dtype=g2.dtype, device=g2.device)
    _lib.call("soup_swiglu_fwd", g2.device, g2.data_ptr(), g2.stride(0), u2.data_ptr(), u2.stride(0),
              out.data_ptr(), out.stride(0), rows, n, _lib.dtype_code(g2.dtype), _lib.stream_of(g2))
    return out


def swiglu_backward(dy2, g2, u2, dg=None, du=None):
    rows, n = g2.shape
    if dg is None:
        dg = torch.empty((rows, n), dtype=g2.dtype, device=g2.device)
    if du is None:
        du = torch.empty((rows, n), dtype=u2.dtype, device=u2.device)
    _lib.call("soup_swiglu_bwd", g2.device, dy2.data_ptr(), dy2.stride(0), g2.data_ptr(),
              g2.stride(0), u2.data_ptr(), u2.stride(0), dg.data_ptr(), dg.stride(0), du.data_ptr(),
              du.stride(0), rows, n, _lib.dtype_code(g2.dtype), _lib.stream_of(g2))
    return dg, du


class FastSwiGLUFunction(torch.autograd.Function):
    """SwiGLU autograd Function (reference: ``swiglu.py:98-165``)."""

    @staticmethod
    def forward(ctx, gate: torch.Tensor, up: torch.Tensor):
        if up.dtype != gate.dtype:
            raise TypeError(f"gate and up dtypes differ: {gate.dtype} vs {up.dtype}")
        orig_shape = gate.shape
        n = orig_shape[-1]
        g2 = _rows(gate, n)
        u2 = _rows(up, n)
        out = swiglu_forward(g2, u2)
        ctx.save_for_backward(g2, u2)
        ctx.orig_shape = orig_shape
        return out.view(orig_shape)

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        g2, u2 = ctx.saved_tensors
        n = g2.shape[1]
        dy2 = _rows(grad_output, n)
        if dy2.dtype != g2.dtype:
            dy2 = dy2.to(g2.dtype)
        dg, du = swiglu_backward(dy2, g2, u2)
        return dg.view(ctx.orig_shape), du.view(ctx.orig_shape)


def fast_swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up (reference: ``swiglu.py:168-170``)."""
    return FastSwiGLUFunction.apply(gate, up)


# ---- SwiGLU with gate and up kept in 8 bits --------------------------------------
Q8_BLOCK = 64  # consecutive columns that share one fp32 scale


def _rows_8bit(t: torch.Tensor, n: int) -> torch.Tensor:
    t2 = t if t.dim() == 2 and t.stride(1) == 1 else _rows(t, n)
    return t2 if t2.shape[0] < 2 or t2.stride(0) >= n else t2.contiguous()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def quantize_8bit(x2: torch.Tensor):
    """(codes int8 [rows, n], scales fp32 [rows, ceil(n / 64)]) of a CUDA tensor
    [..., n]: per 64 consecutive columns scale = absmax / 127 and
    code = round(x * (127 / absmax)); the kept value is code * scale."""
    if x2.dim() == 0 or x2.shape[-1] == 0:
        raise ValueError(f"quantize_8bit: needs rows of columns, got {tuple(x2.shape)}")
    _lib.dtype_code(x2.dtype)
    if not x2.is_cuda:
        raise ValueError("quantize_8bit: the tensor must be on a CUDA device")
    x2 = _rows_8bit(x2.detach(), x2.shape[-1])
    rows, n = x2.shape
    codes = torch.empty(rows, n, dtype=torch.int8, device=x2.device)
    scales = torch.empty(rows, -(-n // Q8_BLOCK), dtype=torch.float32, device=x2.device)
    if rows == 0:
        return codes, scales
    _lib.call("soup_q8_quantize", x2.device, x2.data_ptr(), _ld(x2), codes.data_ptr(), n,
              scales.data_ptr(), scales.shape[1], rows, n, _lib.dtype_code(x2.dtype), _lib.stream_of(x2))
    return codes, scales


def swiglu_8bit_backward(dy2, g_codes, u_codes, g_scales, u_scales, dg, du, h=None) -> None:
    """dg, du (and, when given, h = silu(g) u) at the kept values; every tensor
    [rows, n] (scales [rows, n / 64 rounded up]), the codes of gate and up with
    one row stride, their scales with one row stride."""
    rows, n = dy2.shape
    _lib.call("soup_swiglu_q8_bwd", dy2.device, dy2.data_ptr(), _ld(dy2), g_codes.data_ptr(),
              u_codes.data_ptr(), _ld(g_codes), g_scales.data_ptr(), u_scales.data_ptr(), _ld(g_scales),
              dg.data_ptr(), _ld(dg), du.data_ptr(), _ld(du), _lib.ptr(h), 0 if h is None else _ld(h),
              rows, n, _lib.dtype_code(dy2.dtype), _lib.stream_of(dy2))


class SwiGLU8BitFunction(torch.autograd.Function):
    """silu(gate) * up whose backward reads gate and up from 8-bit codes."""

    @staticmethod
    def forward(ctx, gate: torch.Tensor, up: torch.Tensor):
        n = gate.shape[-1]
        g2, u2 = _rows_8bit(gate, n), _rows_8bit(up, n)
        rows = g2.shape[0]
        blocks = -(-n // Q8_BLOCK)
        dt = _lib.dtype_code(gate.dtype)
        out = torch.empty(*gate.shape, dtype=gate.dtype, device=gate.device)
        # one buffer: the scales of gate, of up, the codes of gate (16-byte aligned), of up
        c0 = -(-8 * rows * blocks // 16) * 16
        c1 = c0 + -(-rows * n // 16) * 16
        kept = torch.empty(c1 + rows * n, dtype=torch.int8, device=gate.device)
        base = kept.data_ptr()
        _lib.call("soup_swiglu_q8_fwd", gate.device, g2.data_ptr(), _ld(g2), u2.data_ptr(), _ld(u2),
                  out.data_ptr(), n, base + c0, base + c1, n, base, base + 4 * rows * blocks, blocks,
                  rows, n, dt, _lib.stream_of(g2))
        ctx.save_for_backward(kept)
        ctx.args = (rows, n, blocks, c0, c1, dt, gate.dtype)
        return out

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy: torch.Tensor):
        # scales and codes are read by address: as they were, whatever a saved-tensor hook returns
        kept = _lib.dense(ctx.saved_tensors[0])
        rows, n, blocks, c0, c1, dt, dtype = ctx.args
        dy2 = _rows_8bit(dy if dy.dtype is dtype else dy.to(dtype), n)
        dg = torch.empty(*dy.shape, dtype=dtype, device=dy.device)
        du = torch.empty(*dy.shape, dtype=dtype, device=dy.device)
        base = kept.data_ptr()
        _lib.call("soup_swiglu_q8_bwd", dy.device, dy2.data_ptr(), _ld(dy2), base + c0, base + c1, n, base,
                  base + 4 * rows * blocks, blocks, dg.data_ptr(), n, du.data_ptr(), n, None, 0, rows, n,
                  dt, _lib.stream_of(dy2))
        return dg, du


def swiglu_8bit(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up, keeping gate and up for the backward as 8-bit codes (1.0625
    bytes an element instead of the dtype's 2 or 4; see :func:`quantize_8bit`).

    The output is that of the exact gate and up; the gradients are SwiGLU's at the
    kept values, each within absmax / 254 of its block of 64 columns. An infinity
    or NaN makes its whole block's gradient NaN. Same shapes and dtypes (fp32, fp16,
    bf16) on one CUDA device.
    """
    if gate.shape != up.shape or gate.dim() == 0 or gate.shape[-1] == 0:
        raise ValueError(f"swiglu_8bit: gate {tuple(gate.shape)} and up {tuple(up.shape)}")
    if gate.dtype != up.dtype:
        raise TypeError(f"swiglu_8bit: gate and up dtypes differ: {gate.dtype} vs {up.dtype}")
    _lib.dtype_code(gate.dtype)
    if not gate.is_cuda or up.device != gate.device:
        raise ValueError("swiglu_8bit: gate and up must be on one CUDA device")
    if gate.numel() == 0:
        return gate * up
    return SwiGLU8BitFunction.apply(gate, up)


#: Keep the MLP's gate and up in 8 bits from forward to backward instead of
#: recomputing them (takes precedence over RECOMPUTE in training): 2.1 bytes per
#: token and intermediate column, no second gate/up GEMM.
#: The QLoRA step's grouped MLPs do so where they run as one Function
#: (``qlora.FUSE_MLP_BACKWARD``, bf16); others recompute, with a warning.
CHECKPOINT_8BIT = False

#: Recompute gate/up + SwiGLU in backward (the reference's selective recompute,
#: ``swiglu.py:197-214``). False keeps the activations instead: more memory
#: (2 x tokens x intermediate bf16 per layer), no second gate/up GEMM pass.
RECOMPUTE = True


def patch_qwen2_mlp():
    """Route ``Qwen2MLP.forward`` on CUDA tensors through the fused SwiGLU.

    Training with grad: gate/up projections + SwiGLU are checkpointed and
    recomputed in backward, ``down_proj`` stays outside the checkpoint
    (``swiglu.py:197-214``). Eval / no-grad: direct call. CPU tensors and
    non-SiLU activations keep the original forward. Errors on CUDA tensors
    propagate (the reference falls back to eager silently).
    """
    try:
        from transformers.models.qwen2 import modeling_qwen2
    except ImportError:
        return
    cls = modeling_qwen2.Qwen2MLP
    if getattr(cls.forward, "_soup_b200", False):
        return
    original_forward = cls.forward

    def forward(self, x):
        act = getattr(getattr(self, "config", None), "hidden_act", "silu")
        if act != "silu" or not x.is_cuda:
            return original_forward(self, x)
        with_grad = self.training and torch.is_grad_enabled() and getattr(x, "requires_grad", False)
        keep8 = CHECKPOINT_8BIT and with_grad
        recompute = RECOMPUTE and with_grad and not keep8
        group = getattr(self.gate_proj, "lora_group", None)
        if (group is not None and group.kind == "gate_up" and group.members[0] is self.gate_proj
                and group.members[1] is self.up_proj and group.usable(x)):
            # gate/up as one GEMM feeding the fused SwiGLU; same recompute policy
            # (without recompute the SwiGLU backward joins down_proj's dX GEMM)
            return group.mlp(x, self.down_proj, recompute, keep8)
        if keep8:
            return self.down_proj(swiglu_8bit(self.gate_proj(x), self.up_proj(x)))
        if not recompute:
            return self.down_proj(fast_swiglu(self.gate_proj(x), self.up_proj(x)))

        def _swiglu_forward(hidden_states):
            return fast_swiglu(self.gate_proj(hidden_states), self.up_proj(hidden_states))

        # the recomputed region has no random ops: skip the RNG state save/restore,
        # which also keeps the step capturable in a CUDA graph
        swiglu_out = torch.utils.checkpoint.checkpoint(_swiglu_forward, x, use_reentrant=False,
                                                       preserve_rng_state=False)
        return self.down_proj(swiglu_out)

    forward._soup_b200 = True
    forward._soup_original = original_forward
    cls.forward = forward


# ---- kernel handles with the reference's launch signatures ---------------------
def _launch_fwd(gate_ptr, up_ptr, out_ptr, stride_g_row, stride_u_row, stride_o_row, N_cols,
                **_triton_only):
    rows = gate_ptr.numel() // max(int(N_cols), 1) if gate_ptr.dim() < 2 else gate_ptr.shape[0]
    _lib.call("soup_swiglu_fwd", gate_ptr.device, gate_ptr.data_ptr(), int(stride_g_row),
              up_ptr.data_ptr(), int(stride_u_row), out_ptr.data_ptr(), int(stride_o_row), rows,
              int(N_cols), _lib.dtype_code(gate_ptr.dtype), _lib.stream_of(gate_ptr))


def _launch_bwd(grad_ptr, gate_ptr, up_ptr, dgate_ptr, dup_ptr, stride_grad_row, stride_g_row,
                stride_u_row, stride_dg_row, stride_du_row, N_cols, **_triton_only):
    rows = gate_ptr.numel() // max(int(N_cols), 1) if gate_ptr.dim() < 2 else gate_ptr.shape[0]
    _lib.call("soup_swiglu_bwd", gate_ptr.device, grad_ptr.data_ptr(), int(stride_grad_row),
              gate_ptr.data_ptr(), int(stride_g_row), up_ptr.data_ptr(), int(stride_u_row),
              dgate_ptr.data_ptr(), int(stride_dg_row), dup_ptr.data_ptr(), int(stride_du_row),
              rows, int(N_cols), _lib.dtype_code(gate_ptr.dtype), _lib.stream_of(gate_ptr))


_custom_swiglu_fwd_kernel = LaunchShim(
    "_custom_swiglu_fwd_kernel",
    ["gate_ptr", "up_ptr", "out_ptr", "stride_g_row", "stride_u_row", "stride_o_row", "N_cols"],
    _launch_fwd)
_custom_swiglu_bwd_kernel = LaunchShim(
    "_custom_swiglu_bwd_kernel",
    ["grad_ptr", "gate_ptr", "up_ptr", "dgate_ptr", "dup_ptr", "stride_grad_row", "stride_g_row",
     "stride_u_row", "stride_dg_row", "stride_du_row", "N_cols"],
    _launch_bwd)
