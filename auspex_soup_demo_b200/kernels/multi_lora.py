"""A frozen projection with the low-rank adapters of many requests beside it.

The reference trains one adapter (peft LoRA over bitsandbytes linears, no reference
kernel; :class:`..qlora.LoRANF4Linear` here). :func:`multi_lora_linear` takes a stack
of adapters and an adapter id for every token or sequence, so that one pass over the
base weights serves requests of different adapters, or trains several adapters at
once: csrc/multi_lora.cu.
"""

from __future__ import annotations

import functools
from typing import Callable, Optional, Union

import torch

from .. import _lib

#: adapters x rank of one call, at most.
MAX_RANK_COLUMNS = 4096
MAX_TOKENS = 1 << 21


@functools.lru_cache(maxsize=256)
def _state_bytes(tokens: int, adapters: int, rank: int) -> int:
    return _lib.lib().soup_multi_lora_state_bytes(tokens, adapters, rank)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(tokens: int, adapters: int, rank: int) -> int:
    return _lib.lib().soup_multi_lora_bwd_workspace_bytes(tokens, adapters, rank)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """t as [rows, width] operand rows that TMA can read (copied only if they are not)."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    ld, step = t.stride()
    if step != 1 or ld % 8 or ld < width or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _factor(t: torch.Tensor) -> torch.Tensor:
    """A stack of factors as dense bf16."""
    return _lib.dense(t if t.dtype is torch.bfloat16 else t.detach().to(torch.bfloat16))


def _forward(x, weight, lora_a, lora_b, ids, scaling, bias, per: int):
    """(y, x rows, weight rows, bf16 factors, state)"""
    n, k = weight.shape
    x2, w = _rows(x, k), _rows(weight, k)
    a16, b16 = _factor(lora_a), _factor(lora_b)
    na, r = lora_a.shape[0], lora_a.shape[1]
    t = x2.shape[0]
    y = x.new_empty((*x.shape[:-1], n))
    nbytes = _state_bytes(t, na, r)
    state = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.call("soup_multi_lora_fwd", x.device, x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), _lib.ptr(bias),
              a16.data_ptr(), b16.data_ptr(), scaling.data_ptr(), ids.data_ptr(),
              1 if ids.dtype is torch.int64 else 0, per, t, n, k, na, r, y.data_ptr(), n, state.data_ptr(),
              nbytes, _lib.stream_of(x))
    return y, x2, w, a16, b16, state


class MultiLoRAFunction(torch.autograd.Function):
    """See :func:`multi_lora_linear`; ``per``: tokens of one id."""

    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, ids, scaling, bias, per: int, weight_fn):
        y, x2, w, a16, b16, state = _forward(x, weight, lora_a, lora_b, ids, scaling, bias, per)
        # x is needed for lora_a's gradient alone, the weight for x's
        ctx.save_for_backward(x2 if ctx.needs_input_grad[2] else None,
                              w if ctx.needs_input_grad[0] and weight_fn is None else None, a16, b16, ids, scaling, state)
        ctx.meta = per, x.shape, lora_a.dtype, lora_b.dtype, weight.shape, weight_fn
        return y

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dy):
        # a saved-tensor hook may hand them back in another layout
        x2, w, a16, b16, ids, scaling, state = ctx.saved_tensors
        a16, b16, state = _lib.dense(a16), _lib.dense(b16), _lib.dense(state)
        ids, scaling = ids.contiguous(), scaling.contiguous()
        per, shape, a_dtype, b_dtype, (n, k), weight_fn = ctx.meta
        need_x, _, need_a, need_b = ctx.needs_input_grad[:4]
        if need_x and w is None:
            w = weight_fn()
            if w.shape != (n, k) or w.dtype is not torch.bfloat16 or w.device != dy.device:
                raise ValueError(f"multi_lora_linear: weight_fn formed {w.dtype} {tuple(w.shape)} on {w.device}, the "
                                 f"forward's weight was bfloat16 {(n, k)} on {dy.device}")
        if need_x:
            w = _rows(w, k)
        else:
            w = a16.view(-1, k)  # not read
        na, r = a16.shape[0], a16.shape[1]
        dy2 = _rows(dy, n)
        t = dy2.shape[0]
        dev = dy2.device
        x2 = _rows(x2, k) if need_a else None
        dx = dy2.new_empty(shape) if need_x else None

        def grad(need, like, dtype):
            if not need:
                return None
            return torch.empty_like(like) if dtype is torch.bfloat16 else torch.empty_like(like, dtype=torch.float32)

        da, db = grad(need_a, a16, a_dtype), grad(need_b, b16, b_dtype)
        nbytes, ws = 0, None
        if need_x or need_a:
            nbytes = _workspace_bytes(t, na, r)
            ws = dy2.new_empty(nbytes, dtype=torch.uint8)
        _lib.call("soup_multi_lora_bwd", dev, dy2.data_ptr(), dy2.stride(0), _lib.ptr(x2),
                  k if x2 is None else x2.stride(0), w.data_ptr(), w.stride(0), a16.data_ptr(), b16.data_ptr(),
                  scaling.data_ptr(), ids.data_ptr(), 1 if ids.dtype is torch.int64 else 0, per, t, n, k, na, r,
                  state.data_ptr(), state.numel(), _lib.ptr(dx), k, _lib.ptr(da),
                  _lib.F32 if da is None else _lib.dtype_code(da.dtype), _lib.ptr(db),
                  _lib.F32 if db is None else _lib.dtype_code(db.dtype), _lib.ptr(ws), nbytes, _lib.stream_of(dy2))
        if da is not None and da.dtype is not a_dtype:
            da = da.to(a_dtype)
        if db is not None and db.dtype is not b_dtype:
            db = db.to(b_dtype)
        return dx, None, da, db, None, None, None, None, None


def multi_lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                      adapter_ids: torch.Tensor, scaling: Union[float, torch.Tensor] = 1.0,
                      bias: Optional[torch.Tensor] = None,
                      weight_fn: Optional[Callable[[], torch.Tensor]] = None) -> torch.Tensor:
    """``x W^T + bias`` plus, for each token, ``scaling * B (A x)`` of its own adapter.

    x [..., K] bfloat16; weight [N, K] and bias [N] bfloat16, frozen. lora_a
    [adapters, rank, K] and lora_b [N, adapters, rank] (adapter i's B is
    ``lora_b[:, i]``), bfloat16, or float32 / float16, which are multiplied as
    bfloat16. adapter_ids: int64 or int32, one for each token (shape x.shape[:-1]) or,
    for x [B, S, K], one for each sequence ([B]); an id outside [0, adapters), e.g. -1,
    takes the projection alone. scaling: a number, or float32 [adapters], constant.
    Adapters of smaller ranks are padded with zero rows and columns, whose gradients
    are 0. weight_fn: forms the same weight again; the backward pass then calls it, and the
    weight is not kept for it (``qlora.KEEP_BASE_WEIGHTS``).

    Products accumulate in 32 bits; A x is rounded to bfloat16 before B (and B^T dy before
    A and x), which makes the rounding error of the factors' gradients 1.4 times that of
    their type alone. Differentiable
    with respect to x, lora_a and lora_b, once; gradients have their leaves' types, and
    adapters without tokens get zeros. K, N and adapters * rank must be multiples of
    8, adapters * rank at most 4096. Tokens of one adapter should follow one another,
    as requests do: the work of the adapters grows with the different ones among 256
    consecutive tokens. Up to 256 tokens (the next tokens of many requests) take a form
    that streams the weight once through all SMs.

    A token without an adapter may hold anything: it reaches its own row of y and of
    x's gradient alone. Factors, also those that no token takes, have to be finite:
    adapters are multiplied 64 columns at a time, with zeros where a token has another
    adapter; and a row of x or of y's gradient that is not finite reaches the gradients
    of the adapters that share 64 columns with its own.
    """
    fn = "multi_lora_linear"
    xs, ws, sa, sb = x.shape, weight.shape, lora_a.shape, lora_b.shape
    if len(xs) < 1 or len(ws) != 2 or len(sa) != 3 or len(sb) != 3:
        raise ValueError(f"{fn}: x [..., K], weight [N, K], lora_a [adapters, rank, K], lora_b [N, adapters, rank]; got "
                         f"{tuple(xs)}, {tuple(ws)}, {tuple(sa)}, {tuple(sb)}")
    n, k = ws
    na, r, ka = sa
    if xs[-1] != k or ka != k or sb != (n, na, r):
        raise ValueError(f"{fn}: x {tuple(xs)}, weight {tuple(ws)}, lora_a {tuple(sa)} and lora_b {tuple(sb)} do not "
                         "fit together")
    if n == 0 or k == 0 or na * r == 0 or n % 8 or k % 8 or na * r % 8 or na * r > MAX_RANK_COLUMNS:
        raise ValueError(f"{fn}: N, K and adapters * rank must be multiples of 8, adapters * rank at most "
                         f"{MAX_RANK_COLUMNS}; got N {n}, K {k}, {na} adapters of rank {r}")
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise TypeError(f"{fn}: x and weight must be bfloat16, got {x.dtype} and {weight.dtype}")
    _lib.dtype_code(lora_a.dtype)
    _lib.dtype_code(lora_b.dtype)
    dev = x.device
    if not x.is_cuda or weight.device != dev or lora_a.device != dev or lora_b.device != dev or \
            adapter_ids.device != dev:
        raise ValueError(f"{fn}: all tensors must be on one CUDA device")
    if weight.requires_grad:
        raise ValueError(f"{fn}: the weight is frozen; detach it")
    if adapter_ids.dtype is not torch.int64 and adapter_ids.dtype is not torch.int32:
        raise TypeError(f"{fn}: adapter_ids must be int64 or int32, got {adapter_ids.dtype}")
    ishape = adapter_ids.shape
    if ishape == xs[:-1]:
        per = 1
    elif len(xs) == 3 and ishape == xs[:1]:
        per = max(1, xs[1])
    else:
        raise ValueError(f"{fn}: adapter_ids {tuple(ishape)} for x {tuple(xs)}: one for each token, or for each sequence "
                         "of x [B, S, K]")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype is not torch.bfloat16 or bias.device != dev:
            raise ValueError(f"{fn}: bias must be bfloat16 [{n}] on {dev}")
        if bias.requires_grad:
            raise ValueError(f"{fn}: the bias is frozen; detach it")
        bias = bias.contiguous()
    if isinstance(scaling, torch.Tensor):
        if scaling.shape != (na,) or scaling.dtype is not torch.float32 or scaling.device != dev:
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
        return x.new_zeros(*xs[:-1], n) + (x.sum() + lora_a[:, :0].sum() + lora_b[:0].sum()).to(x.dtype)
    ids = adapter_ids.contiguous()
    if _lib.differentiated(x, lora_a, lora_b):
        return MultiLoRAFunction.apply(x, weight, lora_a, lora_b, ids, scaling, bias, per, weight_fn)
    return _forward(x, weight, lora_a, lora_b, ids, scaling, bias, per)[0]
