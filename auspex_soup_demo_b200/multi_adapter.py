"""Linears with several LoRA adapters on one frozen base weight.

The reference trains one adapter (peft LoRA on bitsandbytes linears). Here a model
built with ``build_qwen2_qlora(adapters=n)`` holds n of them in every target linear:
each sequence (or token) of a batch names its adapter, one pass over the base weights
serves them all (:func:`.kernels.multi_lora_linear`), and a training step gives each
adapter the gradients of its own sequences. ``adapter.save_adapter(index=i)`` writes
adapter i as a PEFT directory.
"""

from __future__ import annotations

import functools
import math
import threading
from typing import Optional, Sequence, Union

import torch


class AdapterIds:
    """The adapter ids of the batch that a model is running: [B] or [B, S] integers on the
    model's device, -1 for none. One object is shared by all of a model's linears.

    The ids that hold for a call of the model are those set when it begins, or its
    ``adapter_ids`` argument (:meth:`follow`). Its layers get them as an argument of
    their own, so that a checkpointed layer that runs again in the backward pass takes
    the ids of its forward pass, whatever was set since."""

    def __init__(self, adapters: int):
        self.adapters = adapters
        self.ids: Optional[torch.Tensor] = None
        self._running = {}  # thread -> the ids of its layers in progress

    def set(self, ids: Optional[torch.Tensor]) -> None:
        self.ids = self._checked(ids)

    @staticmethod
    def _checked(ids: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        if ids is not None and (ids.dim() not in (1, 2) or ids.dtype not in (torch.int64, torch.int32)):
            raise ValueError(f"adapter ids must be int64 or int32 [B] or [B, S], got {ids.dtype} {tuple(ids.shape)}")
        return ids

    def current(self) -> torch.Tensor:
        """The ids of the layer in progress (outside one: those that are set)."""
        running = self._running.get(threading.get_ident())
        ids = running[-1] if running else self.ids
        if ids is None:
            raise ValueError("the batch's adapter ids are not set (AdapterIds.set, or the trainer's adapter_ids)")
        return ids

    def follow(self, model) -> None:
        """Hand the layers of a causal-LM ``model`` the ids of each of its calls."""
        model.model.register_forward_pre_hook(self._begin, with_kwargs=True)
        for layer in model.model.layers:
            layer.register_forward_pre_hook(self._enter, with_kwargs=True)
            layer.register_forward_hook(self._leave, always_call=True)

    def _begin(self, body, args, kwargs):
        ids = kwargs.get("adapter_ids")
        return args, {**kwargs, "adapter_ids": self.ids if ids is None else self._checked(ids)}

    def _enter(self, layer, args, kwargs):
        self._running.setdefault(threading.get_ident(), []).append(kwargs.pop("adapter_ids", self.ids))
        return args, kwargs

    def _leave(self, layer, args, output):
        me = threading.get_ident()
        running = self._running.get(me)
        if running:  # (another hook may have raised before _enter)
            running.pop()
            if not running:
                del self._running[me]


class _MultiLoRABase(torch.nn.Module):
    """y = base(x) + scaling[a] * B_a (A_a x), a the adapter of x's sequence.

    ``lora_A`` [adapters, r, in] and ``lora_B`` [out, adapters, r] (adapter i's factors
    are ``lora_A[i]`` and ``lora_B[:, i]``)."""

    def _init_lora(self, linear: torch.nn.Linear, ids: AdapterIds, r: int, alpha: Union[float, Sequence[float]],
                   lora_dtype: torch.dtype):
        self.in_features, self.out_features = linear.in_features, linear.out_features
        n = ids.adapters
        alphas = list(alpha) if isinstance(alpha, (list, tuple)) else [alpha] * n
        if len(alphas) != n:
            raise ValueError(f"{len(alphas)} alphas for {n} adapters")
        self.alphas = alphas
        dev = linear.weight.device
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())
        self.register_buffer("scaling", torch.tensor([a / r for a in alphas], dtype=torch.float32, device=dev))
        self.lora_A = torch.nn.Parameter(torch.empty(n, r, self.in_features, device=dev, dtype=lora_dtype))
        self.lora_B = torch.nn.Parameter(torch.zeros(self.out_features, n, r, device=dev, dtype=lora_dtype))
        for a in self.lora_A:
            torch.nn.init.kaiming_uniform_(a, a=math.sqrt(5))
        self.adapter_ids = ids

    def base_weight(self, dtype) -> torch.Tensor:
        raise NotImplementedError

    def weight_again(self, dtype):
        """What forms the base weight again in the backward pass; None: it is kept."""
        return None

    def _apply(self, fn, *args, **kwargs):
        # model.to(bf16) casts buffers; the scales stay fp32
        scaling = self._buffers.pop("scaling")
        try:
            super()._apply(fn, *args, **kwargs)
        finally:
            dev = self.lora_A.device
            self._buffers["scaling"] = scaling if scaling.device == dev else scaling.to(dev)
        return self

    def forward(self, x):
        from .kernels import multi_lora_linear

        ids = self.adapter_ids.current()
        args = x, self.base_weight(x.dtype), self.lora_A, self.lora_B, ids, self.scaling, self.bias
        again = self.weight_again(x.dtype)
        return multi_lora_linear(*args) if again is None else multi_lora_linear(*args, again)


class MultiLoRANF4Linear(_MultiLoRABase):
    """Several adapters beside a frozen NF4 base linear."""

    def __init__(self, linear: torch.nn.Linear, ids: AdapterIds, r: int = 16, alpha=32,
                 lora_dtype: torch.dtype = torch.float32):
        from .qlora import nf4_quantize

        super().__init__()
        packed, absmax = nf4_quantize(linear.weight)
        self.register_buffer("packed", packed)
        self.register_buffer("absmax", absmax)
        self._init_lora(linear, ids, r, alpha, lora_dtype)

    def base_weight(self, dtype) -> torch.Tensor:
        from .qlora import nf4_dequantize

        return nf4_dequantize(self.packed, self.absmax, (self.out_features, self.in_features), dtype)

    def weight_again(self, dtype):
        from . import qlora

        return None if qlora.KEEP_BASE_WEIGHTS else functools.partial(self.base_weight, dtype)


class MultiLoRADenseLinear(_MultiLoRABase):
    """Several adapters beside a frozen dense base linear."""

    def __init__(self, linear: torch.nn.Linear, ids: AdapterIds, r: int = 16, alpha=32,
                 lora_dtype: torch.dtype = torch.float32):
        super().__init__()
        self.register_buffer("weight", linear.weight.detach().clone())
        self._init_lora(linear, ids, r, alpha, lora_dtype)

    def base_weight(self, dtype) -> torch.Tensor:
        return self.weight.to(dtype)
