"""Causal grouped-query flash attention on B200 (tcgen05 kernels via the C ABI).

No counterpart kernel in the reference: its Qwen2 attention runs through torch's
``scaled_dot_product_attention`` (transformers' ``sdpa_attention_forward``,
called from ``Qwen2Attention.forward``). This module provides the same call for
the QLoRA step:

* :func:`attention_forward` / :class:`FlashAttentionFunction` - q [B, H, S, 128],
  k / v [B, Hk, S, 128] bf16 with any b / h / s strides (transformers' transposed
  [B, S, H, D] projections are read in place) -> out [B, S, H, 128] bf16 (the
  layout the o_proj consumes, no transpose copy) and the row log-sum-exp for
  the backward;
* :func:`window_attention` - the same with a sliding window and a few first
  tokens that stay visible (sinks), forward and backward;
* :func:`soup_attention` - an attention function with transformers'
  ``AttentionInterface`` signature, registered under the name ``"soup_b200"``
  by :func:`register`. Calls the kernels have no form for (an attention mask,
  dropout, a head dim other than 128, non-bf16 or CPU tensors) go to
  transformers' SDPA function unchanged; :func:`soup_mask` decides which calls of a
  model need a mask. Layers with a ``sliding_window`` (and,
  optionally, ``config.attention_sink_tokens``) take :func:`window_attention`.
"""

from __future__ import annotations

import functools
import math

import torch

from .. import _lib

HEAD_DIM = 128
INTERFACE_NAME = "soup_b200"


def _strides(t: torch.Tensor):
    return _lib.i64_array([t.stride(0), t.stride(1), t.stride(2)])


def _check(q, k, v, any_stride: bool = False):
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4:
        raise ValueError("attention: q, k, v must be [B, heads, S, D]")
    B, H, S, D = qs
    Hk = ks[1]
    if ks != vs or ks[0] != B or ks[2] != S or ks[3] != D:
        raise ValueError(f"attention: shapes q {tuple(qs)} k {tuple(ks)} v {tuple(vs)}")
    if Hk == 0 or H % Hk:
        raise ValueError("attention: query heads must be a multiple of the KV heads")
    for t in (q, k, v):
        if t.dtype is not torch.bfloat16 or not t.is_cuda or not (any_stride or t.stride(-1) == 1):
            raise ValueError("attention: q, k, v must be bf16 CUDA tensors with a contiguous last dim")
    return B, H, Hk, S, D


def _s_pad(S: int) -> int:
    return -(-S // 128) * 128


def attention_forward(q, k, v, scale: float, causal: bool = True):
    """(out [B, S, H, D] bf16, lse [B, H, S] fp32) of softmax(scale q k^T) v.

    lse is a view of a [B, H, S rounded up to 128] buffer (the layout the
    backward reads)."""
    B, H, Hk, S, D = _check(q, k, v)
    out = torch.empty(B, S, H, D, dtype=torch.bfloat16, device=q.device)
    lse = torch.empty(B, H, _s_pad(S), dtype=torch.float32, device=q.device)
    _lib.call("soup_attention_fwd", q.device, q.data_ptr(), _strides(q), k.data_ptr(), _strides(k),
              v.data_ptr(), _strides(v), B, H, Hk, S, D, float(scale), int(bool(causal)),
              out.data_ptr(), lse.data_ptr(), _lib.stream_of(q))
    return out, lse[..., :S]


def attention_backward(q, k, v, out, lse, dout, scale: float, causal: bool = True):
    """(dq [B, H, S, D], dk, dv [B, Hk, S, D]) as transposed views of contiguous
    [B, S, heads, D] buffers; lse as returned by :func:`attention_forward`."""
    B, H, Hk, S, D = _check(q, k, v)
    if dout.shape != (B, S, H, D):
        raise ValueError(f"attention: dout must be [B, S, H, D], got {tuple(dout.shape)}")
    dout = dout.to(torch.bfloat16).contiguous()
    out = _lib.dense(out)
    base = lse._base if lse._base is not None else lse
    if base.shape != (B, H, _s_pad(S)) or base.dtype != torch.float32 or not base.is_contiguous():
        raise ValueError("attention: lse must come from attention_forward")
    dq = torch.empty(B, S, H, D, dtype=torch.bfloat16, device=q.device)
    dk = torch.empty(B, S, Hk, D, dtype=torch.bfloat16, device=q.device)
    dv = torch.empty(B, S, Hk, D, dtype=torch.bfloat16, device=q.device)
    nbytes = _lib.lib().soup_attention_bwd_workspace_bytes(B, H, S)
    ws = _lib.scratch(q.device, nbytes)
    _lib.call("soup_attention_bwd", q.device, q.data_ptr(), _strides(q), k.data_ptr(), _strides(k),
              v.data_ptr(), _strides(v), out.data_ptr(), dout.data_ptr(), base.data_ptr(), B, H, Hk,
              S, D, float(scale), int(bool(causal)), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
              ws.data_ptr(), nbytes, _lib.stream_of(q))
    return dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2)


class FlashAttentionFunction(torch.autograd.Function):
    """out [B, S, H, D] = attention(q, k, v) with the tcgen05 kernels; backward
    recomputes P from the saved log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, scale: float, causal: bool):
        out, lse = attention_forward(q, k, v, scale, causal)
        # the padded buffer itself: a saved-tensor hook hands a view back without its base
        ctx.save_for_backward(q, k, v, out, lse._base)
        ctx.scale = scale
        ctx.causal = causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = attention_backward(q, k, v, out, _lib.dense(lse), dout, ctx.scale, ctx.causal)
        return dq, dk, dv, None, None


def flash_attention(q, k, v, scale: float, causal: bool = True):
    return FlashAttentionFunction.apply(q, k, v, scale, causal)


def _kernel_layout(t: torch.Tensor):
    """(t, element strides) in a form the tensor maps can read: 16-byte aligned,
    positive strides that are multiples of 8. Dimensions of size 1 take any
    stride; anything else is copied."""
    b, h, s, d = t.shape
    sb, sh, ss, sd = t.stride()
    if b == 1:
        sb = h * s * d
    if h == 1:
        sh = s * d
    if s == 1:
        ss = d
    if sd != 1 or t.data_ptr() % 16 or (sb | sh | ss) % 8 or sb <= 0 or sh <= 0 or ss <= 0:
        t = t.detach().clone(memory_format=torch.contiguous_format)
        sb, sh, ss = h * s * d, s * d, d
    return t, (_lib.c_i64 * 3)(sb, sh, ss)


def _restored(t: torch.Tensor, saved):
    """:func:`_kernel_layout` of a saved tensor. ``saved`` holds its (strides, kernel
    strides) in the forward: a saved-tensor hook may hand it back in another layout."""
    stride, kernel = saved
    return (t, kernel) if t.stride() == stride and t.data_ptr() % 16 == 0 else _kernel_layout(t)


@functools.lru_cache(maxsize=256)
def _window_workspace_bytes(*sizes: int) -> int:
    return _lib.lib().soup_attention_window_bwd_workspace_bytes(*sizes)


class WindowAttentionFunction(torch.autograd.Function):
    """out [B, S, H, D] of :func:`window_attention`; backward recomputes P from the
    saved log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, scale: float, window: int, sinks: int):
        B, H, S, D = q.shape
        Hk = k.shape[1]
        (q, qs), (k, ks), (v, vs) = _kernel_layout(q), _kernel_layout(k), _kernel_layout(v)
        out = torch.empty(B, S, H, D, dtype=torch.bfloat16, device=q.device)
        lse = torch.empty(B, H, _s_pad(S), dtype=torch.float32, device=q.device)
        _lib.call("soup_attention_window_fwd", q.device, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(),
                  vs, B, H, Hk, S, D, scale, window, sinks, out.data_ptr(), lse.data_ptr(),
                  _lib.stream_of(q))
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.args = ((q.stride(), qs), (k.stride(), ks), (v.stride(), vs), scale, window, sinks)
        return out

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        ql, kl, vl, scale, window, sinks = ctx.args
        B, H, S, D = q.shape
        Hk = k.shape[1]
        (q, qs), (k, ks), (v, vs) = _restored(q, ql), _restored(k, kl), _restored(v, vl)
        out, lse = _lib.dense(out), _lib.dense(lse)
        if dout.dtype is not torch.bfloat16 or not dout.is_contiguous():
            dout = dout.to(torch.bfloat16).contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        dev = q.device
        # [B, heads, S, D] over [B, S, heads, D] memory
        dq = torch.empty_strided((B, H, S, D), (S * H * D, D, H * D, 1), dtype=torch.bfloat16, device=dev)
        kv = (S * Hk * D, D, Hk * D, 1)
        dk = torch.empty_strided((B, Hk, S, D), kv, dtype=torch.bfloat16, device=dev)
        dv = torch.empty_strided((B, Hk, S, D), kv, dtype=torch.bfloat16, device=dev)
        nbytes = _window_workspace_bytes(B, H, Hk, S, window, sinks)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.call("soup_attention_window_bwd", dev, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(),
                  vs, out.data_ptr(), dout.data_ptr(), lse.data_ptr(), B, H, Hk, S, D, scale, window,
                  sinks, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), nbytes,
                  _lib.stream_of(q))
        return dq, dk, dv, None, None, None


def window_attention(q, k, v, scale: float, window: int, sinks: int = 0) -> torch.Tensor:
    """out [B, S, H, D] of causal grouped-query attention in which query i sees
    key j iff j <= i and (i - j < window or j < sinks).

    q [B, H, S, 128], k and v [B, Hk, S, 128] bf16 CUDA tensors, H a multiple of
    Hk, any strides (layouts the kernels cannot read in place are copied);
    window >= 1, sinks >= 0, either may exceed S. Time and memory traffic grow
    with S (window + sinks), not with S^2. Differentiable in q, k and v.
    """
    B, H, Hk, S, D = _check(q, k, v, any_stride=True)
    if D != HEAD_DIM:
        raise ValueError(f"window_attention: head dim must be {HEAD_DIM}, got {D}")
    if not q.get_device() == k.get_device() == v.get_device():
        raise ValueError("window_attention: q, k and v must be on one device")
    if B == 0 or H == 0 or S == 0:
        raise ValueError(f"window_attention: empty input, q {tuple(q.shape)} k {tuple(k.shape)}")
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window_attention: window must be >= 1 and sinks >= 0, got {window}, {sinks}")
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("window_attention: scale must be positive and finite")
    return WindowAttentionFunction.apply(q, k, v, float(scale), min(window, S), min(sinks, S))


def _supported(module, query, key, value, attention_mask, dropout) -> bool:
    return (attention_mask is None and not dropout and query.is_cuda
            and query.dtype == key.dtype == value.dtype == torch.bfloat16
            and query.shape[-1] == HEAD_DIM and query.stride(-1) == 1 and key.stride(-1) == 1
            and value.stride(-1) == 1 and query.shape[2] == key.shape[2]
            and all(t.stride(i) % 8 == 0 for t in (query, key, value) for i in range(3))
            and all(t.data_ptr() % 16 == 0 for t in (query, key, value)))


def soup_attention(module, query, key, value, attention_mask, dropout: float = 0.0,
                   scaling=None, is_causal=None, **kwargs):
    """transformers ``AttentionInterface`` function: (attn_output [B, S, H, D], None).

    Causal when the module is (and the query is longer than one token), as
    transformers' SDPA path decides (``integrations/sdpa_attention.py``). Calls
    outside the kernels' form go to transformers' SDPA function.

    A ``sliding_window`` (transformers passes the layer's) limits each query of a
    causal module to its last ``sliding_window`` keys, plus the first
    ``attention_sink_tokens`` of the sequence when the module's config sets that. With
    a cache the queries are the last tokens of the keys; sinks need the whole sequence
    in one call, since a sliding layer's cache drops the first tokens."""
    window = kwargs.get("sliding_window")
    n_q, n_k = query.shape[2], key.shape[2]
    if (attention_mask is None and n_q <= n_k
            and (is_causal if is_causal is not None else getattr(module, "is_causal", True))):
        # no mask came with the call, so causality and the window are this function's to apply
        sinks = int(getattr(getattr(module, "config", None), "attention_sink_tokens", 0) or 0) if window else 0
        if sinks and n_q < n_k and window <= n_k:
            raise ValueError("soup_attention: attention_sink_tokens with a cache longer than the sliding "
                             "window; run the whole sequence in one call (use_cache=False)")
        hides = bool(window) and window < n_k
        if hides and (n_q == n_k and not dropout and query.is_cuda and query.shape[-1] == HEAD_DIM
                      and query.dtype == key.dtype == value.dtype == torch.bfloat16):
            scale = scaling if scaling is not None else query.shape[-1] ** -0.5
            return window_attention(query, key, value, float(scale), window, sinks), None
        if hides or 1 < n_q < n_k:  # SDPA's own causal mask takes the queries for the first tokens
            k_pos = torch.arange(n_k, device=query.device)
            q_pos = k_pos[n_k - n_q:, None]
            attention_mask = k_pos <= q_pos  # [n_q, n_k], one byte a pair
            if hides:
                attention_mask &= (k_pos > q_pos - window) | (k_pos < sinks)
            attention_mask = attention_mask[None, None]
            is_causal = False  # in the mask
    if not _supported(module, query, key, value, attention_mask, dropout):
        from transformers.integrations.sdpa_attention import sdpa_attention_forward

        return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout,
                                      scaling=scaling, is_causal=is_causal, **kwargs)
    causal = is_causal if is_causal is not None else getattr(module, "is_causal", True)
    causal = bool(causal) and query.shape[2] > 1
    scale = scaling if scaling is not None else query.shape[-1] ** -0.5
    return flash_attention(query, key, value, float(scale), causal), None


def _kernels_mask_it(q_length, kv_length, q_offset, kv_offset, attention_mask, local_size, config) -> bool:
    """Whether :func:`soup_attention` without a mask computes this layer type's causal
    attention: the whole sequence in one call, the window (if any) the layer's own, and
    padding, if any, only behind the tokens of each row, where no token looks."""
    if q_length != kv_length or not isinstance(q_offset, int) or q_offset or kv_offset:
        return False
    if local_size is not None and local_size != getattr(config, "sliding_window", None):
        return False  # attention in chunks
    if attention_mask is None:
        return True
    if attention_mask.dim() != 2 or attention_mask.shape[1] != kv_length or (
            attention_mask.is_cuda and torch.cuda.is_current_stream_capturing()):
        return False  # (a capture cannot look at the values)
    kept = attention_mask != 0
    return not bool((kept[:, 1:] & ~kept[:, :-1]).any())


def soup_mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, attention_mask=None, local_size=None,
              allow_is_causal_skip: bool = True, config=None, **kwargs):
    """transformers ``AttentionMaskInterface`` function of ``INTERFACE_NAME``: no mask for
    the calls that :func:`soup_attention` masks itself, else transformers' SDPA mask
    (padding before or between tokens, caches, packed sequences), which takes the call
    to SDPA."""
    from transformers.masking_utils import sdpa_mask

    if allow_is_causal_skip and _kernels_mask_it(q_length, kv_length, q_offset, kv_offset, attention_mask,
                                                 local_size, config):
        return None
    if local_size is not None and getattr(config, "attention_sink_tokens", 0):
        if not (isinstance(q_offset, int) and attention_mask is None and q_offset + q_length <= local_size):
            raise ValueError("soup_attention: attention_sink_tokens need the whole sequence in one call "
                             "(use_cache=False), with no padding before its tokens")
    if attention_mask is not None and attention_mask.is_cuda and torch.cuda.is_current_stream_capturing():
        allow_is_causal_skip = False
    return sdpa_mask(batch_size=batch_size, q_length=q_length, kv_length=kv_length, q_offset=q_offset,
                     kv_offset=kv_offset, attention_mask=attention_mask, local_size=local_size,
                     allow_is_causal_skip=allow_is_causal_skip, config=config, **kwargs)


def register() -> str:
    """Register :func:`soup_attention` and its masks with transformers under ``INTERFACE_NAME``."""
    from transformers import AttentionInterface, AttentionMaskInterface

    AttentionInterface.register(INTERFACE_NAME, soup_attention)
    AttentionMaskInterface.register(INTERFACE_NAME, soup_mask)
    return INTERFACE_NAME
