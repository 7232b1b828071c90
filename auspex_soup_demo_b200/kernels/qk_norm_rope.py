"""Norms of queries and keys for each head and their rotation, in one pass.

No counterpart in the reference, whose ``solution/kernels/rope.py:120-196`` rotates
rows as they are, by tables of one position. Two entry points beside
:func:`.rope.apply_fast_rope_qk`:

* :func:`apply_qk_norm_rope` - RMS norm of every head's row of q and k, then the
  rotation by cos / sin tables;
* :func:`apply_multi_axis_rope` - rotation by positions of several axes (time,
  height, width of image and video tokens), with or without the norms; the angles
  are formed in the kernel, in 64 bits.

Both are one launch forward and one backward (and one that joins the weights'
gradients): csrc/qk_norm_rope.cu.
"""

from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib

MAX_HEAD_DIM = 512
MAX_AXES = 256

# soup_qk_rope: sizes, types, table strides, six tensors' strides, eps
_DESC = struct.Struct("=5q5q3q24qd")
_NONE = (0, 0, 0, 0)
_TABLES, _INT32, _INT64 = 0, 1, 2


@functools.lru_cache(maxsize=64)
def _axes_bytes(axes: Tuple[int, ...]):
    return (ctypes.c_uint8 * len(axes))(*axes)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(b: int, s: int, hq: int, hk: int, d: int) -> int:
    return _lib.lib().soup_qk_norm_rope_bwd_workspace_bytes(b, s, hq, hk, d)


def rope_axes(sections: Sequence[int], interleaved: bool = False) -> Tuple[int, ...]:
    """The axis of each frequency for :func:`apply_multi_axis_rope`.

    sections: frequencies per axis, e.g. (16, 24, 24) for time, height and width of a
    head dim of 128. In blocks, axis j takes the next ``sections[j]`` frequencies.
    ``interleaved``: the axes take turns (0, 1, 2, 0, 1, 2, ...); axis j > 0 has every
    len(sections)-th frequency of the first len(sections) * sections[j], and axis 0
    the rest.
    """
    return _axes(tuple(sections), bool(interleaved))


@functools.lru_cache(maxsize=64)
def _axes(sections: Tuple[int, ...], interleaved: bool) -> Tuple[int, ...]:
    n = len(sections)
    if not n or any(not isinstance(s, int) or s < 0 for s in sections) or sum(sections) == 0:
        raise ValueError(f"rope_axes: sections must be counts of frequencies, got {sections}")
    if not interleaved:
        return tuple(j for j, s in enumerate(sections) for _ in range(s))
    return tuple(i % n if i < n * sections[i % n] else 0 for i in range(sum(sections)))


def _head_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _out_like(t: torch.Tensor):
    """(output in the order of t's axes, its strides), its rows contiguous (of rows that
    overlap, as those of a sliding view do, the axes' order can be another)."""
    out = torch.empty_like(t)
    st = out.stride()
    if st[3] != 1:
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        st = out.stride()
    return out, st


def _source(a: torch.Tensor, c: torch.Tensor, axes):
    """(table dtype code, source, its three strides, axes) for the C calls: a and c are
    tables [B | 1, S, D] or [S, D], or positions [axes, B | 1, S] or [axes, S] and frequencies."""
    st = a.stride()
    wide = len(st) == 3
    if axes is None:
        # only the first half of a table's row is read
        return _lib.dtype_code(a.dtype), _TABLES, (0, st[0] if wide and a.shape[0] > 1 else 0, st[-2]), None
    return (0, _INT64 if a.dtype is torch.int64 else _INT32,
            (st[0], st[1] if wide and a.shape[1] > 1 else 0, st[-1]), _axes_bytes(axes))


def _forward(q, k, qw, kw, eps, a, c, axes, inverse=0):
    (qo, sq), (ko, sk) = _out_like(q), _out_like(k)
    b, hq, s, d = q.shape
    code = _lib.dtype_code(q.dtype)
    tcode, src, ts, ax = _source(a, c, axes)
    desc = _DESC.pack(b, s, d, hq, k.shape[1], code, code if qw is None else _lib.dtype_code(qw.dtype), tcode, src,
                      inverse, *ts, *q.stride(), *sq, *k.stride(), *sk, *_NONE, *_NONE, eps)
    _lib.call("soup_qk_norm_rope", q.device, q.data_ptr(), qo.data_ptr(), k.data_ptr(), ko.data_ptr(),
              0 if qw is None else qw.data_ptr(), 0 if kw is None else kw.data_ptr(), a.data_ptr(), c.data_ptr(), ax,
              desc, _lib.stream_of(q))
    return qo, ko


class QKNormRoPEFunction(torch.autograd.Function):
    """See :func:`apply_qk_norm_rope` and :func:`apply_multi_axis_rope`; ``axes`` None:
    ``a`` and ``c`` are cos and sin tables, else positions and frequencies."""

    @staticmethod
    def forward(ctx, q, k, qw, kw, eps: float, a, c, axes):
        out = _forward(q, k, qw, kw, eps, a, c, axes)
        if qw is None:
            ctx.save_for_backward(a, c)
        else:
            ctx.save_for_backward(a, c, q, k, qw, kw)
        ctx.meta = eps, axes, q.shape, k.shape, q.dtype
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, gq, gk):
        if gq is None and gk is None:
            return (None,) * 8
        eps, axes, qs, ks, dt = ctx.meta
        saved = ctx.saved_tensors
        a, c = saved[0], saved[1]
        # a saved-tensor hook may hand them back in another layout
        if axes is None:
            if a.stride(-1) != 1 or c.stride() != a.stride():
                a, c = a.contiguous(), c.contiguous()
        elif not c.is_contiguous():
            c = c.contiguous()
        dev = a.device
        gq = torch.zeros(qs, dtype=dt, device=dev) if gq is None else _head_rows(gq)
        gk = torch.zeros(ks, dtype=dt, device=dev) if gk is None else _head_rows(gk)
        if len(saved) == 2:
            dq, dk = _forward(gq, gk, None, None, eps, a, c, axes, 1)
            return dq, dk, None, None, None, None, None, None
        q, k = _head_rows(saved[2]), _head_rows(saved[3])
        qw, kw = _lib.dense(saved[4]), _lib.dense(saved[5])
        _, _, need_q, need_k = ctx.needs_input_grad[:4]
        b, hq, s, d = qs
        hk = ks[1]
        (dq, sq), (dk, sk) = _out_like(q), _out_like(k)
        dqw = torch.empty_like(qw) if need_q else None
        dkw = torch.empty_like(kw) if need_k else None
        nbytes, ws = 0, 0
        if need_q or need_k:
            nbytes = _workspace_bytes(b, s, hq, hk, d)
            buf = a.new_empty(nbytes, dtype=torch.uint8)
            ws = buf.data_ptr()
        tcode, src, ts, ax = _source(a, c, axes)
        desc = _DESC.pack(b, s, d, hq, hk, _lib.dtype_code(dt), _lib.dtype_code(qw.dtype), tcode, src, 0, *ts,
                          *q.stride(), *sq, *k.stride(), *sk, *gq.stride(), *gk.stride(), eps)
        _lib.call("soup_qk_norm_rope_bwd", dev, gq.data_ptr(), q.data_ptr(), dq.data_ptr(), gk.data_ptr(),
                  k.data_ptr(), dk.data_ptr(), qw.data_ptr(), kw.data_ptr(), _lib.ptr(dqw), _lib.ptr(dkw),
                  a.data_ptr(), c.data_ptr(), ax, desc, ws, nbytes, _lib.stream_of(q))
        return dq, dk, dqw, dkw, None, None, None, None


def _check(fn: str, q, k, qw, kw, eps):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"{fn}: q and k must be [B, H, S, D], got {tuple(q.shape)} and {tuple(k.shape)}")
    qs, ks = q.shape, k.shape
    if qs[0] != ks[0] or qs[2:] != ks[2:] or q.dtype != k.dtype:
        raise ValueError(f"{fn}: q and k must share batch, seq, head_dim and dtype, got {tuple(qs)} {q.dtype} and "
                         f"{tuple(ks)} {k.dtype}")
    _lib.dtype_code(q.dtype)
    d = qs[3]
    if d % 2 or not 0 < d <= MAX_HEAD_DIM:
        raise ValueError(f"{fn}: head_dim must be even and at most {MAX_HEAD_DIM}, got {d}")
    if (qs[1] == 0) != (ks[1] == 0):
        raise ValueError(f"{fn}: q and k must both have heads, got {qs[1]} and {ks[1]}")
    if not q.is_cuda or k.device != q.device:
        raise ValueError(f"{fn}: q and k must be on one CUDA device")
    if (qw is None) != (kw is None):
        raise ValueError(f"{fn}: norm weights for both q and k, or for neither")
    if qw is not None:
        for w in (qw, kw):
            if tuple(w.shape) != (d,):
                raise ValueError(f"{fn}: norm weights must be [{d}], got {tuple(w.shape)}")
            if w.device != q.device:
                raise ValueError(f"{fn}: norm weights must be on {q.device}")
        if qw.dtype != kw.dtype or qw.dtype not in (q.dtype, torch.float32):
            raise TypeError(f"{fn}: norm weights must both be {q.dtype} or float32, got {qw.dtype} and {kw.dtype}")
        if not eps >= 0.0:
            raise ValueError(f"{fn}: eps must be 0 or more, not {eps}")


def _apply(q, k, qw, kw, eps, a, c, axes):
    if 0 in q.shape or 0 in k.shape:
        # no rows: empty results, connected to what they are made of
        parts = [q, k] if qw is None else [q * qw[0], k * kw[0]]
        return parts[0].clone(), parts[1].clone()
    q, k = _head_rows(q), _head_rows(k)
    if qw is not None:
        qw, kw = qw.contiguous(), kw.contiguous()
    if _lib.differentiated(q, k, qw, kw):
        return QKNormRoPEFunction.apply(q, k, qw, kw, eps, a, c, axes)
    return _forward(q, k, qw, kw, eps, a, c, axes)


def apply_qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor, eps: float = 1e-6
                       ) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head's row of q [B, H, S, D] and k [B, Hk, S, D], then the
    rotate-half rotation, in one launch.

    q_weight, k_weight [D]: the norms' weights, of q's type or float32. cos, sin:
    tables as :func:`.rope.apply_fast_rope_qk` takes them ([B | 1, 1, S, D],
    [B | 1, S, D] or [S, D]; only the first half of a row is read), of float32,
    bfloat16 or float16. q and k may have any strides with a contiguous last
    dimension (others are copied). Arithmetic in 32 bits, one rounding at the end.
    Differentiable with respect to q, k and both weights, once.
    """
    _check("apply_qk_norm_rope", q, k, q_weight, k_weight, eps)
    if q_weight is None:
        raise ValueError("apply_qk_norm_rope: norm weights are needed; apply_fast_rope_qk rotates alone")
    if cos.dim() == 4 and cos.shape[1] == 1:
        cos = cos[:, 0]
    if sin.dim() == 4 and sin.shape[1] == 1:
        sin = sin[:, 0]
    shape = cos.shape
    if sin.shape != shape or len(shape) not in (2, 3) or shape[-2:] != (q.shape[2], q.shape[3]) or \
            (len(shape) == 3 and shape[0] not in (1, q.shape[0])):
        raise ValueError(f"apply_qk_norm_rope: cos and sin must be [B | 1, 1, S, D], [B | 1, S, D] or [S, D], got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    if cos.device != q.device or sin.device != q.device:
        raise ValueError(f"apply_qk_norm_rope: cos and sin must be on {q.device}")
    if cos.dtype != sin.dtype:
        raise TypeError(f"apply_qk_norm_rope: cos and sin must share their type, got {cos.dtype} and {sin.dtype}")
    _lib.dtype_code(cos.dtype)
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("apply_qk_norm_rope: cos and sin are constants; detach them")
    if cos.stride(-1) != 1 or sin.stride() != cos.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    return _apply(q, k, q_weight, k_weight, float(eps), cos, sin, None)


def apply_multi_axis_rope(q: torch.Tensor, k: torch.Tensor, position_ids: torch.Tensor, inv_freq: torch.Tensor,
                          axes: Sequence[int], q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotate q [B, H, S, D] and k [B, Hk, S, D] by positions of several axes, in one
    launch; with weights [D] also normalise every row first, as
    :func:`apply_qk_norm_rope` does.

    position_ids: int64 or int32 [axes, B | 1, S] or [axes, S], any strides, any sign.
    inv_freq: float32 [D / 2]. axes: the axis of each frequency (:func:`rope_axes`).
    Frequency i of a token turns by position_ids[axes[i]] * inv_freq[i], formed in 64
    bits. Differentiable with respect to q, k and the weights, once.
    """
    fn = "apply_multi_axis_rope"
    _check(fn, q, k, q_weight, k_weight, eps)
    b, _, s, d = q.shape
    if position_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{fn}: position_ids must be int64 or int32, got {position_ids.dtype}")
    shape = tuple(position_ids.shape)
    if len(shape) not in (2, 3) or shape[-1] != s or (len(shape) == 3 and shape[1] not in (1, b)) or shape[0] == 0:
        raise ValueError(f"{fn}: position_ids must be [axes, B | 1, S] or [axes, S], got {shape}")
    axes = tuple(axes)
    if len(axes) != d // 2:
        raise ValueError(f"{fn}: {len(axes)} axes for {d // 2} frequencies")
    if min(axes) < 0 or max(axes) >= min(shape[0], MAX_AXES):
        raise ValueError(f"{fn}: axes must be in [0, {min(shape[0], MAX_AXES)})")
    if inv_freq.dtype is not torch.float32 or tuple(inv_freq.shape) != (d // 2,):
        raise ValueError(f"{fn}: inv_freq must be float32 [{d // 2}], got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if position_ids.device != q.device or inv_freq.device != q.device:
        raise ValueError(f"{fn}: position_ids and inv_freq must be on {q.device}")
    if inv_freq.requires_grad:
        raise ValueError(f"{fn}: inv_freq is a constant; detach it")
    return _apply(q, k, q_weight, k_weight, float(eps), position_ids, inv_freq.contiguous(), axes)
