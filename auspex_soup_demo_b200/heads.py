"""Attention layers whose queries and keys are normalised for each head, and whose
positions may have several axes.

The reference patches transformers' Qwen2 layers, which rotate q and k as they are by
one position (``solution/kernels/rope.py:199-223``). :func:`install_heads` gives the
attention layers of such a model RMS norms of q and k (``q_norm`` / ``k_norm``, weights
[head_dim]) and / or rotary positions of several axes, both in the pass of the rotation
(:func:`.kernels.apply_qk_norm_rope`, :func:`.kernels.apply_multi_axis_rope`).
"""

from __future__ import annotations

import functools
import threading
from typing import Optional, Sequence

import torch


class MultiAxisRotary(torch.nn.Module):
    """In the place of a model's rotary embedding: hands the layers the positions
    [axes, B, S] and the frequencies themselves instead of cos and sin tables. [B, S]
    positions (text) count for every axis."""

    def __init__(self, inner: torch.nn.Module, axes):
        from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

        super().__init__()
        # formed again: model.to(bf16) has cast the embedding's own copy
        init = (inner.compute_default_rope_parameters if inner.rope_type == "default"
                else ROPE_INIT_FUNCTIONS[inner.rope_type])
        inv_freq, factor = init(inner.config, inner.inv_freq.device)
        if factor != 1.0:
            raise ValueError("install_heads: a rotary embedding with a scaling factor has no form with several axes")
        self.register_buffer("inv_freq", inv_freq.to(torch.float32), persistent=False)
        self.axes = axes
        self.positions = {}  # thread -> [axes, B, S] of its call in progress

    def _apply(self, fn, *args, **kwargs):
        inv = self._buffers.pop("inv_freq")  # frequencies stay fp32 under model.to(bf16)
        try:
            super()._apply(fn, *args, **kwargs)
        finally:
            moved = fn(inv)
            self._buffers["inv_freq"] = inv if moved.device == inv.device else inv.to(moved.device)
        return self

    def take_positions(self, body, args, kwargs):
        """Pre-hook of the model's body: positions of several axes go around it, straight to
        :meth:`forward`. The body itself looks for packed sequences in its positions, and has
        a form of that for [B, S] alone; without any it counts 0, 1, 2, ... of each row."""
        me = threading.get_ident()
        self.positions.pop(me, None)
        pos = kwargs.get("position_ids") if len(args) < 3 else args[2]
        if pos is None or pos.dim() != 3:
            return None
        self.positions[me] = pos
        if len(args) >= 3:
            return (*args[:2], None, *args[3:]), kwargs
        return args, {**kwargs, "position_ids": None}

    def forward(self, x, position_ids):
        n = max(self.axes) + 1
        position_ids = self.positions.pop(threading.get_ident(), position_ids)
        if position_ids.dim() == 2:
            position_ids = position_ids.unsqueeze(0).expand(n, *position_ids.shape)
        elif position_ids.shape[0] < n:
            raise ValueError(f"position_ids must be [B, S] or [{n}, B, S], got {tuple(position_ids.shape)}")
        return position_ids, self.inv_freq


def _attention_forward(self, hidden_states, position_embeddings, attention_mask=None, past_key_values=None, **kwargs):
    """transformers' ``Qwen2Attention.forward`` with the heads' norms and axes."""
    from transformers.models.qwen2 import modeling_qwen2 as m

    from .kernels import apply_multi_axis_rope, apply_qk_norm_rope

    lead = hidden_states.shape[:-1]
    shape = (*lead, -1, self.head_dim)
    q = self.q_proj(hidden_states).view(shape).transpose(1, 2)
    k = self.k_proj(hidden_states).view(shape).transpose(1, 2)
    v = self.v_proj(hidden_states).view(shape).transpose(1, 2)
    qw, kw, eps = None, None, 1e-6
    if self.q_norm is not None:
        qw, kw, eps = self.q_norm.weight, self.k_norm.weight, self.q_norm.variance_epsilon
    first, second = position_embeddings
    if self.rope_axes is not None:
        q, k = apply_multi_axis_rope(q, k, first, second, self.rope_axes, qw, kw, eps)
    else:
        q, k = apply_qk_norm_rope(q, k, qw, kw, first, second, eps)
    if past_key_values is not None:
        k, v = past_key_values.update(k, v, self.layer_idx)
    attend = m.ALL_ATTENTION_FUNCTIONS.get_interface(self.config._attn_implementation, m.eager_attention_forward)
    out, weights = attend(self, q, k, v, attention_mask,
                          dropout=0.0 if not self.training else self.attention_dropout, scaling=self.scaling,
                          sliding_window=self.sliding_window, **kwargs)
    return self.o_proj(out.reshape(*lead, -1).contiguous()), weights


def install_heads(model, qk_norm: bool = True, rope_sections: Optional[Sequence[int]] = None,
                  rope_interleaved: bool = False, train_norms: bool = False):
    """Give every attention layer of a Qwen2 causal-LM ``model`` norms of q and k for each
    head (weights 1; trained with ``train_norms``) and / or positions of several axes
    (``rope_sections``: frequencies of each axis, together half the head dim). Its
    ``position_ids`` are then [B, S] or [axes, B, S]; with the latter every row is one
    sequence (a padding mask [B, S] is taken as ever). CUDA models."""
    from transformers.models.qwen2 import modeling_qwen2 as m

    from .kernels import rope_axes

    if not qk_norm and rope_sections is None:
        raise ValueError("install_heads: nothing to install")
    cfg = model.config
    axes = None
    if rope_sections is not None:
        axes = rope_axes(rope_sections, rope_interleaved)
        half = model.model.rotary_emb.inv_freq.numel()
        if len(axes) != half:
            raise ValueError(f"install_heads: sections of {len(axes)} frequencies, the model has {half}")
        rotary = model.model.rotary_emb = MultiAxisRotary(model.model.rotary_emb, axes)
        model.model.register_forward_pre_hook(rotary.take_positions, with_kwargs=True)
    for layer in model.model.layers:
        attn = layer.self_attn
        attn.q_norm = attn.k_norm = None
        if qk_norm:
            w = attn.q_proj.weight if isinstance(attn.q_proj, torch.nn.Linear) else model.get_input_embeddings().weight
            for name in ("q_norm", "k_norm"):
                norm = m.Qwen2RMSNorm(attn.head_dim, eps=cfg.rms_norm_eps).to(device=w.device, dtype=w.dtype)
                norm.weight.requires_grad_(train_norms)
                setattr(attn, name, norm)
        attn.rope_axes = axes
        attn.forward = functools.partial(_attention_forward, attn)  # (a bound method would not unpickle)
    return model
