"""A frozen projection with the low-rank adapters of many requests beside it.

The reference trains one adapter (peft LoRA over bitsandbytes linears, no reference
kernel; :class:`..qlora.LoRANF4Linear` here). :func:`multi_lora_linear` takes a stack
of adapters and an adapter id for every token or sequence, so that one pass over the
base weights serves requests of different adapters, or trains several adapters at
once: csrc/multi_lora.cu.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _lib

#: adapters x rank of one call, at most.
MAX_RANK_COLUMNS = 4096
MAX_TOKENS = 1 << 21


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """t as [rows, width] operand rows that TMA can read (copied only if they are not)."""
    t = t.reshape(-1, width)
    if t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < width or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _factor(t: torch.Tensor) -> torch.Tensor:
    """A stack of factors as dense bf16."""
    return _lib.dense(t.detach().to(torch.bfloat16))


class MultiLoRAFunction(torch.autograd.Function):
    """See :func:`multi_lora_linear`; ``per``: tokens of one id."""

    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, ids, scaling, bias, per: int):
        k, n = x.shape[-1], weight.shape[0]
        x2, w = _rows(x, k), _rows(weight, k)
        a16, b16 = _factor(lora_a), _factor(lora_b)
        na, r = lora_a.shape[:2]
        t = x2.shape[0]
        dev = x.device
        y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=dev)
        nbytes = _lib.lib().soup_multi_lora_state_bytes(t, na, r)
        state = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.call("soup_multi_lora_fwd", dev, x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), _lib.ptr(bias),
                  a16.data_ptr(), b16.data_ptr(), scaling.data_ptr(), ids.data_ptr(),
                  1 if ids.dtype is torch.int64 else 0, per, t, n, k, na, r, y.data_ptr(), n, state.data_ptr(),
                  nbytes, _lib.stream_of(x))
        need = ctx.needs_input_grad
        if need[0] or need[2] or need[3]:
            # x is needed for lora_a's gradient alone
            ctx.save_for_backward(x2 if need[2] else None, w, a16, b16, ids, scaling, state)
            ctx.per, ctx.shape = per, x.shape
            ctx.dtypes = lora_a.dtype, lora_b.dtype
        return y

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy):
        # a saved-tensor hook may hand them back in another layout
        x2, w, a16, b16, ids, scaling, state = ctx.saved_tensors
        a16, b16, state = _lib.dense(a16), _lib.dense(b16), _lib.dense(state)
        ids, scaling = ids.contiguous(), scaling.contiguous()
        n, k = w.shape
        w = _rows(w, k)
        na, r = a16.shape[:2]
        need_x, _, need_a, need_b = ctx.needs_input_grad[:4]
        dy2 = _rows(dy, n)
        t = dy2.shape[0]
        dev = dy2.device
        x2 = _rows(x2, k) if need_a else None
        dx = torch.empty(ctx.shape, dtype=dy2.dtype, device=dev) if need_x else None

        def grad(need, like, dtype):
            if not need:
                return None
            return torch.empty(like.shape, dtype=torch.bfloat16 if dtype is torch.bfloat16 else torch.float32,
                               device=dev)

        da, db = grad(need_a, a16, ctx.dtypes[0]), grad(need_b, b16, ctx.dtypes[1])
        nbytes, ws = 0, None
        if need_x or need_a:
            nbytes = _lib.lib().soup_multi_lora_bwd_workspace_bytes(t, na, r)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.call("soup_multi_lora_bwd", dev, dy2.data_ptr(), dy2.stride(0), _lib.ptr(x2),
                  k if x2 is None else x2.stride(0), w.data_ptr(), w.stride(0), a16.data_ptr(), b16.data_ptr(),
                  scaling.data_ptr(), ids.data_ptr(), 1 if ids.dtype is torch.int64 else 0, ctx.per, t, n, k, na, r,
                  state.data_ptr(), state.numel(), _lib.ptr(dx), k, _lib.ptr(da),
                  _lib.F32 if da is None else _lib.dtype_code(da.dtype), _lib.ptr(db),
                  _lib.F32 if db is None else _lib.dtype_code(db.dtype), _lib.ptr(ws), nbytes, _lib.stream_of(dy2))
        if da is not None:
            da = da.to(ctx.dtypes[0])
        if db is not None:
            db = db.to(ctx.dtypes[1])
        return dx, None, da, db, None, None, None, None


def multi_lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                      adapter_ids: torch.Tensor, scaling: Union[float, torch.Tensor] = 1.0,
                      bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x W^T + bias`` plus, for each token, ``scaling * B (A x)`` of its own adapter.

    x [..., K] bfloat16; weight [N, K] and bias [N] bfloat16, frozen. lora_a
    [adapters, rank, K] and lora_b [N, adapters, rank] (adapter i's B is
    ``lora_b[:, i]``), bfloat16, or float32 / float16, which are multiplied as
    bfloat16. adapter_ids: int64 or int32, one for each token (shape x.shape[:-1]) or,
    for x [B, S, K], one for each sequence ([B]); an id outside [0, adapters), e.g. -1,
    takes the projection alone. scaling: a number, or float32 [adapters], constant.
    Adapters of smaller ranks are padded with zero rows and columns, whose gradients
    are 0.

    Products accumulate in 32 bits; A x is rounded to bfloat16 before B. Differentiable
    with respect to x, lora_a and lora_b, once; gradients have their leaves' types, and
    adapters without tokens get zeros. K, N and adapters * rank must be multiples of
    8, adapters * rank at most 4096. Tokens of one adapter should follow one another,
    as requests do: the work of the adapters grows with the different ones among 256
    consecutive tokens. Up to 64 tokens (the next tokens of many requests) take a form
    that streams the weight once through all SMs.
    """
    fn = "multi_lora_linear"
    if x.dim() < 1 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError(f"{fn}: x [..., K], weight [N, K], lora_a [adapters, rank, K], lora_b [N, adapters, rank]; got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)}, {tuple(lora_a.shape)}, {tuple(lora_b.shape)}")
    n, k = weight.shape
    na, r, ka = lora_a.shape
    if x.shape[-1] != k or ka != k or tuple(lora_b.shape) != (n, na, r):
        raise ValueError(f"{fn}: x {tuple(x.shape)}, weight {tuple(weight.shape)}, lora_a {tuple(lora_a.shape)} and "
                         f"lora_b {tuple(lora_b.shape)} do not fit together")
    if 0 in (n, k, na, r) or n % 8 or k % 8 or na * r % 8 or na * r > MAX_RANK_COLUMNS:
        raise ValueError(f"{fn}: N, K and adapters * rank must be multiples of 8, adapters * rank at most "
                         f"{MAX_RANK_COLUMNS}; got N {n}, K {k}, {na} adapters of rank {r}")
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise TypeError(f"{fn}: x and weight must be bfloat16, got {x.dtype} and {weight.dtype}")
    for t in (lora_a, lora_b):
        _lib.dtype_code(t.dtype)
    dev = x.device
    if not x.is_cuda or any(t.device != dev for t in (weight, lora_a, lora_b, adapter_ids)):
        raise ValueError(f"{fn}: all tensors must be on one CUDA device")
    if weight.requires_grad:
        raise ValueError(f"{fn}: the weight is frozen; detach it")
    if adapter_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{fn}: adapter_ids must be int64 or int32, got {adapter_ids.dtype}")
    ishape, lead = tuple(adapter_ids.shape), tuple(x.shape[:-1])
    if ishape == lead:
        per = 1
    elif len(lead) == 2 and ishape == lead[:1]:
        per = max(1, lead[1])
    else:
        raise ValueError(f"{fn}: adapter_ids {ishape} for x {tuple(x.shape)}: one for each token, or for each sequence "
                         "of x [B, S, K]")
    if bias is not None:
        if tuple(bias.shape) != (n,) or bias.dtype is not torch.bfloat16 or bias.device != dev:
            raise ValueError(f"{fn}: bias must be bfloat16 [{n}] on {dev}")
        if bias.requires_grad:
            raise ValueError(f"{fn}: the bias is frozen; detach it")
        bias = bias.contiguous()
    if isinstance(scaling, torch.Tensor):
        if tuple(scaling.shape) != (na,) or scaling.dtype is not torch.float32 or scaling.device != dev:
            raise ValueError(f"{fn}: scaling must be a number, or float32 [{na}] on {dev}")
        if scaling.requires_grad:
            raise ValueError(f"{fn}: scaling is a constant; detach it")
        scaling = scaling.contiguous()
    else:
        scaling = torch.full((na,), float(scaling), dtype=torch.float32, device=dev)
    t = x.numel() // k
    if t > MAX_TOKENS:
        raise ValueError(f"{fn}: at most {MAX_TOKENS} tokens, got {t}")
    if t == 0:
        # empty, connected to the states and the factors
        return x.new_zeros(*lead, n) + (x.sum() + lora_a[:, :0].sum() + lora_b[:0].sum()).to(x.dtype)
    return MultiLoRAFunction.apply(x, weight, lora_a, lora_b, adapter_ids.contiguous(), scaling, bias, per)
