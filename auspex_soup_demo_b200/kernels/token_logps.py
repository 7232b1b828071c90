"""Per-token log-probabilities of the lm_head on B200 (tcgen05 GEMMs via the C ABI).

No counterpart in the reference, which trains on the summed cross-entropy of
``chunked_ce.py:267-313``. Preference and policy losses need the log-probability
of every answer token, and hand back one gradient weight per token:

    logps[i] = z_i[t_i] - log sum exp z_i,   z_i = hidden_i W^T
    d loss / d z_i = dlogps[i] (onehot(t_i) - softmax(z_i))

:func:`head_token_logps` runs the logits GEMM with the online-softmax epilogue of
the fused cross-entropy; with a gradient to come, the epilogue also stores the
row-shifted exponentials exp(z - c) in bf16, and the backward multiplies them
by the token weights inside the dX (and dW) GEMMs, so the [tokens, vocab]
logits are formed once and never rewritten. Without a gradient (a reference
model's log-probabilities) nothing of size [tokens, vocab] is written.
"""

from __future__ import annotations

import functools
from typing import Any, Tuple

import torch

from .. import _lib
from . import chunked_ce
from .chunked_ce import IGNORE_INDEX, _extract_head_weight, _tma_rows_ok


def _rows_as(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """t as [rows, dim] operand rows of ``dtype`` that TMA can read."""
    t = t.detach()
    if t.dtype is not dtype:
        t = t.to(dtype)
    return t if _tma_rows_ok(t) and t.stride(0) >= t.shape[1] else t.clone(
        memory_format=torch.contiguous_format)


def _operand_dtype(hidden: torch.Tensor, weight: torch.Tensor) -> torch.dtype:
    """bf16 states with a bf16 head are multiplied as they are, everything else
    as fp16 (the reference's arithmetic, ``chunked_ce.py:196-199``)."""
    both = hidden.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16
    return torch.bfloat16 if both else torch.float16


@functools.lru_cache(maxsize=256)
def _state_bytes(n: int, vocab: int, dim: int) -> int:
    return _lib.lib().soup_head_logps_state_bytes(n, vocab, dim)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n: int, vocab: int, dim: int, backward: int) -> int:
    return _lib.lib().soup_head_logps_workspace_bytes(n, vocab, dim, backward)


def _block_rows(n: int, vocab: int, dim: int) -> int:
    """Rows per launch sequence: what CE_WORKSPACE_BYTES holds (0: all)."""
    budget = chunked_ce.CE_WORKSPACE_BYTES
    full = _state_bytes(n, vocab, dim) + _workspace_bytes(n, vocab, dim, 0)
    if budget <= 0 or full <= budget:
        return n
    return min(n, max(256, int(budget // (full / n)) // 256 * 256))


def _forward(h, w, labels, r0, n, ignore_index, logps, ents, state) -> None:
    """Rows [r0, r0 + n); logps and ents: addresses of the first row's results."""
    v, d = w.shape
    nbytes = _workspace_bytes(n, v, d, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    _lib.call("soup_head_logps_fwd", h.device, h.data_ptr() + r0 * h.stride(0) * 2, h.stride(0),
              w.data_ptr(), w.stride(0), _lib.dtype_code(h.dtype), labels.data_ptr() + r0 * 8, n, v, d,
              ignore_index, logps, ents, _lib.ptr(state), 0 if state is None else state.numel(),
              ws.data_ptr(), nbytes, _lib.stream_of(h))


def _new_state(n, v, d, device) -> torch.Tensor:
    return torch.empty(_state_bytes(n, v, d), dtype=torch.uint8, device=device)


class HeadTokenLogpsFunction(torch.autograd.Function):
    """(logps, entropies) of hidden rows against the head; see :func:`head_token_logps`."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index: int, keep: bool):
        d = hidden.shape[-1]
        v = weight.shape[0]
        dt = _operand_dtype(hidden, weight)
        h = _rows_as(hidden.reshape(-1, d), dt)
        w = _rows_as(weight, dt)
        t = labels if labels.dtype is torch.int64 else labels.to(torch.int64)
        t = t.detach().contiguous()
        n = h.shape[0]
        dev = hidden.device
        logps = torch.empty(*labels.shape, dtype=torch.float32, device=dev)
        ents = torch.empty(*labels.shape, dtype=torch.float32, device=dev)
        rb = _block_rows(n, v, d)
        state = _new_state(n, v, d, dev) if keep and rb == n else None
        for r0 in range(0, n, rb):
            _forward(h, w, t, r0, min(rb, n - r0), ignore_index, logps.data_ptr() + 4 * r0,
                     ents.data_ptr() + 4 * r0, state)
        if keep:
            # h is needed for the head's gradient and to run blocks again
            need_h = ctx.needs_input_grad[1] or state is None
            ctx.save_for_backward(weight, t, state, h if need_h else None)
            ctx.hidden_shape, ctx.hidden_dtype = hidden.shape, hidden.dtype
            ctx.operand_dtype, ctx.ignore_index, ctx.block = dt, ignore_index, rb
        ctx.mark_non_differentiable(ents)
        ctx.set_materialize_grads(False)
        return logps, ents

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, dlogps, _dents):
        if dlogps is None:
            return None, None, None, None, None
        weight, t, state, h = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        dt, ignore = ctx.operand_dtype, ctx.ignore_index
        # a saved-tensor hook may hand them back in another layout (the weight's rows: below)
        t = _lib.dense(t)
        state = None if state is None else _lib.dense(state)
        h = None if h is None else _rows_as(h, dt)
        n, (v, d), dev = t.numel(), weight.shape, weight.device
        g = dlogps.to(torch.float32).contiguous()
        wb = _rows_as(weight, torch.bfloat16) if need_h else None
        w = None
        dh = dw = None
        if need_h:
            out_dt = torch.bfloat16 if ctx.hidden_dtype == torch.bfloat16 else torch.float32
            dh = torch.empty(*ctx.hidden_shape, dtype=out_dt, device=dev)
        if need_w:
            one = ctx.block == n and weight.dtype in (torch.bfloat16, torch.float32)
            dw = torch.empty(v, d, dtype=weight.dtype if one else torch.float32, device=dev)
        for r0 in range(0, n, ctx.block):
            r = min(n, r0 + ctx.block) - r0
            st = state
            if st is None:  # more rows than the budget holds: this block's exponentials again
                if w is None:
                    w = _rows_as(weight, dt)
                    st_buf = _new_state(min(n, ctx.block), v, d, dev)
                    lp = torch.empty(min(n, ctx.block), dtype=torch.float32, device=dev)
                st = st_buf
                _forward(h, w, t, r0, r, ignore, lp.data_ptr(), None, st)
            nbytes = _workspace_bytes(r, v, d, 1)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _lib.call("soup_head_logps_bwd", dev, st.data_ptr(), st.numel(),
                      None if h is None else h.data_ptr() + r0 * h.stride(0) * 2,
                      d if h is None else h.stride(0), _lib.dtype_code(dt), _lib.ptr(wb),
                      d if wb is None else wb.stride(0), g.data_ptr() + 4 * r0, r, v, d,
                      None if dh is None else dh.data_ptr() + r0 * d * dh.element_size(),
                      _lib.F32 if dh is None else _lib.dtype_code(dh.dtype), _lib.ptr(dw),
                      _lib.F32 if dw is None else _lib.dtype_code(dw.dtype), 1 if r0 else 0,
                      ws.data_ptr(), nbytes, _lib.stream_of(weight))
        if dh is not None:
            dh = dh.to(ctx.hidden_dtype)
        if dw is not None:
            dw = dw.to(weight.dtype)
        return dh, dw, None, None, None


def head_token_logps(hidden: torch.Tensor, head: Any, labels: torch.Tensor,
                     ignore_index: int = IGNORE_INDEX) -> Tuple[torch.Tensor, torch.Tensor]:
    """(log-probabilities, entropies) of the labels under the lm_head, both fp32
    and shaped like ``labels``; 0 where the label is ``ignore_index``.

    hidden [..., D] CUDA states; head: the weight [V, D] or a module that holds
    it; labels [...] integers. Labels that are neither ``ignore_index`` nor in
    [0, V) give NaN. The log-probabilities are differentiable with respect to
    hidden and, when it requires grad, the head weight; the entropies are not.
    bf16 operands are used as they are, others as fp16 (then the input gradient
    multiplies a bf16 copy of the head). D must be a multiple of 8. The
    exponentials kept for the backward take 2 V bytes a token up to
    ``chunked_ce.CE_WORKSPACE_BYTES``; beyond that the backward forms them again
    block by block.
    """
    weight = head if isinstance(head, torch.Tensor) else _extract_head_weight(head)
    if weight is None:
        raise ValueError("head_token_logps: no weight found in the head")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"head_token_logps: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)}")
    if tuple(labels.shape) != tuple(hidden.shape[:-1]):
        raise ValueError(f"head_token_logps: labels {tuple(labels.shape)} for hidden {tuple(hidden.shape)}")
    if labels.is_floating_point() or labels.is_complex() or labels.dtype == torch.bool:
        raise TypeError("head_token_logps: labels must be integers")
    for t in (hidden, weight):
        _lib.dtype_code(t.dtype)
    if not hidden.is_cuda or weight.device != hidden.device or labels.device != hidden.device:
        raise ValueError("head_token_logps: hidden, head and labels must be on one CUDA device")
    if weight.shape[0] == 0 or weight.shape[1] == 0 or weight.shape[1] % 8:
        raise ValueError("head_token_logps: the head needs rows, and a width that is a multiple of 8")
    if labels.numel() == 0:
        # empty, connected to the states and the head
        z = hidden.sum(-1, dtype=torch.float32) + weight[:0].sum(dtype=torch.float32)
        return z, z.detach().clone()
    keep = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
    return HeadTokenLogpsFunction.apply(hidden, weight, labels, int(ignore_index), keep)
