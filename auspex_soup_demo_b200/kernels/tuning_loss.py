"""Losses over per-token log-probabilities: preference pairs and clipped policies.

No counterpart in the reference (it trains on the cross-entropy alone). Both take
the log-probabilities that :func:`.token_logps.head_token_logps` returns, labels
that mark the answer tokens (``ignore_index`` elsewhere, whose values are not
used), and return a differentiable fp32 scalar with detached metrics:

* :func:`preference_loss` - chosen / rejected pairs scored by their log ratio
  to a reference model (sigmoid, hinge or squared form);
* :func:`policy_loss` - importance ratios to the sampling policy, clipped, with
  an optional KL term to a reference model.

One summing kernel, one joining kernel and one elementwise backward each
(csrc/tuning_loss.cu); sums run in 64 bits and in a fixed order.
"""

from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from .. import _lib
from .chunked_ce import IGNORE_INDEX

LOSS_TYPES = {"sigmoid": 0, "hinge": 1, "ipo": 2}
REDUCTIONS = {"token": 0, "sequence": 1}


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """(t, row stride) of a [rows, cols] tensor whose rows are contiguous and do not overlap."""
    n, s = t.shape
    ld, step = t.stride()
    if (s > 1 and step != 1) or (n > 1 and ld < s):
        return t.detach().contiguous(), s
    return t, ld if n > 1 else s


def _labels(labels: torch.Tensor) -> Tuple[torch.Tensor, int]:
    return _rows(labels if labels.dtype is torch.int64 else labels.to(torch.int64))


_INTEGERS = {torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8}


def _check(fn: str, logps: torch.Tensor, labels: torch.Tensor) -> None:
    shape = logps.shape
    if len(shape) != 2 or 0 in shape:
        raise ValueError(f"{fn}: logps must be [sequences, tokens], got {tuple(shape)}")
    if logps.dtype is not torch.float32:
        raise TypeError(f"{fn}: logps must be float32, got {logps.dtype}")
    if labels.shape != shape:
        raise ValueError(f"{fn}: labels {tuple(labels.shape)} for logps {tuple(shape)}")
    if labels.dtype not in _INTEGERS:
        raise TypeError(f"{fn}: labels must be integers, got {labels.dtype}")
    if not logps.is_cuda or labels.device != logps.device:
        raise ValueError(f"{fn}: logps and labels must be on one CUDA device")


def _constant(fn: str, name: str, t: torch.Tensor, shapes, device) -> None:
    if t.shape not in shapes:
        raise ValueError(f"{fn}: {name} has shape {tuple(t.shape)}, expected one of {list(shapes)}")
    if t.dtype is not torch.float32:
        raise TypeError(f"{fn}: {name} must be float32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{fn}: {name} must be on {device}")
    if t.requires_grad:
        raise ValueError(f"{fn}: {name} is a constant of the loss; detach it")


@functools.lru_cache(maxsize=256)
def _workspace_bytes(fn: str, n: int, s: int) -> int:
    """Of the entry point, rounded up to 16 (what follows it in one buffer is aligned)."""
    return -(-getattr(_lib.lib(), fn)(n, s) // 16) * 16


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, ref, labels, beta, smoothing, loss_type: int, ignore_index: int):
        dev = logps.device
        n, s = logps.shape
        p = n // 2
        x, x_ld = _rows(logps)
        lab, lab_ld = _labels(labels)
        mode, r, r_ld = 0, None, 0
        if ref is not None and ref.dim() == 2:
            mode, (r, r_ld) = 1, _rows(ref)
        elif ref is not None:
            mode, r = 2, ref.contiguous()
        loss = torch.empty((), dtype=torch.float32, device=dev)
        chosen, rejected = torch.empty(2, p, dtype=torch.float32, device=dev).unbind(0)
        nbytes = _workspace_bytes("soup_preference_loss_workspace_bytes", p, s)
        ws = torch.empty(nbytes // 4 + n, dtype=torch.float32, device=dev)  # workspace, then coef
        coef = ws.data_ptr() + nbytes
        _lib.call("soup_preference_loss_fwd", dev, x.data_ptr(), x_ld, _lib.ptr(r), r_ld, mode,
                  lab.data_ptr(), lab_ld, p, s, ignore_index, beta, smoothing, loss_type,
                  loss.data_ptr(), chosen.data_ptr(), coef, ws.data_ptr(), nbytes,
                  _lib.stream_of(logps))
        ctx.save_for_backward(ws, lab)
        ctx.args = (nbytes, n, s, ignore_index)
        ctx.mark_non_differentiable(chosen, rejected)
        ctx.set_materialize_grads(False)
        return loss, chosen, rejected

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, grad, _c, _r):
        if grad is None:
            return (None,) * 7
        ws, lab = ctx.saved_tensors
        off, n, s, ignore_index = ctx.args
        # a saved-tensor hook may hand both back in another layout
        ws, (lab, lab_ld) = _lib.dense(ws), _rows(lab)
        out = torch.empty(n, s, dtype=torch.float32, device=ws.device)
        grad = grad.to(torch.float32)
        _lib.call("soup_preference_loss_bwd", ws.device, grad.data_ptr(), ws.data_ptr() + off,
                  lab.data_ptr(), lab_ld, n // 2, s, ignore_index, out.data_ptr(), _lib.stream_of(ws))
        return (out,) + (None,) * 6


def preference_loss(logps: torch.Tensor, ref_logps: Optional[torch.Tensor], labels: torch.Tensor,
                    beta: float = 0.1, label_smoothing: float = 0.0, loss_type: str = "sigmoid",
                    ignore_index: int = IGNORE_INDEX
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, chosen_rewards, rejected_rewards)`` of P preference pairs.

    logps [2P, S] fp32: the chosen answers, then the rejected ones in the same
    order. ref_logps: the reference model's [2P, S] per token, their per-sequence
    sums [2P], or None (no reference). With r = sum over a sequence's labelled
    tokens of (logps - ref_logps) and h = r_chosen - r_rejected, the loss is the
    mean over the pairs of

    * ``"sigmoid"``: -(1 - e) log sigmoid(beta h) - e log sigmoid(-beta h), e the
      label smoothing in [0, 0.5);
    * ``"hinge"``: max(0, 1 - beta h);
    * ``"ipo"``: (h' - 1 / (2 beta))^2 with each r divided by its number of
      labelled tokens.

    The rewards [P] are beta r, detached. A sequence without labelled tokens has
    r = 0 and no gradient.
    """
    fn = "preference_loss"
    _check(fn, logps, labels)
    n, s = logps.shape
    if n % 2:
        raise ValueError(f"{fn}: logps must hold as many chosen as rejected sequences, got {n} rows")
    if loss_type not in LOSS_TYPES:
        raise ValueError(f"{fn}: loss_type must be one of {sorted(LOSS_TYPES)}, not {loss_type!r}")
    if not (math.isfinite(beta) and beta > 0):
        raise ValueError(f"{fn}: beta must be positive and finite")
    if not 0.0 <= label_smoothing < 0.5 or (label_smoothing and loss_type != "sigmoid"):
        raise ValueError(f"{fn}: label_smoothing must be in [0, 0.5) and needs loss_type 'sigmoid'")
    if ref_logps is not None:
        _constant(fn, "ref_logps", ref_logps, ((n, s), (n,)), logps.device)
    return PreferenceLossFunction.apply(logps, ref_logps, labels, float(beta), float(label_smoothing),
                                        LOSS_TYPES[loss_type], int(ignore_index))


class PolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, advantages, labels, old, ref, lo, hi, kl_coef, reduction: int,
                ignore_index: int, keep: bool):
        dev = logps.device
        b, s = logps.shape
        x, x_ld = _rows(logps)
        lab, lab_ld = _labels(labels)
        o, o_ld = (None, 0) if old is None else _rows(old)
        r, r_ld = (None, 0) if ref is None else _rows(ref)
        a, a_ld = _rows(advantages) if advantages.dim() == 2 else (advantages.contiguous(), 0)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        kl, clipped = torch.empty(2, dtype=torch.float32, device=dev).unbind(0)
        nbytes = _workspace_bytes("soup_policy_loss_workspace_bytes", b, s)
        # workspace, each sequence's weight, and (for a backward) each token's gradient
        ws = torch.empty(nbytes // 4 + b + (b * s if keep else 0), dtype=torch.float32, device=dev)
        factor = ws.data_ptr() + nbytes
        _lib.call("soup_policy_loss_fwd", dev, x.data_ptr(), x_ld, _lib.ptr(o), o_ld, _lib.ptr(r), r_ld,
                  a.data_ptr(), a_ld, lab.data_ptr(), lab_ld, b, s, ignore_index, lo, hi, kl_coef,
                  reduction, loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(), factor,
                  factor + 4 * b if keep else None, ws.data_ptr(), nbytes, _lib.stream_of(logps))
        if keep:
            ctx.save_for_backward(ws)
            ctx.args = (nbytes, b, s)
        ctx.mark_non_differentiable(kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, kl, clipped

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, grad, _k, _c):
        if grad is None:
            return (None,) * 11
        ws = _lib.dense(ctx.saved_tensors[0])
        off, b, s = ctx.args
        out = torch.empty(b, s, dtype=torch.float32, device=ws.device)
        grad = grad.to(torch.float32)
        factor = ws.data_ptr() + off
        _lib.call("soup_policy_loss_bwd", ws.device, grad.data_ptr(), factor, factor + 4 * b, b, s,
                  out.data_ptr(), _lib.stream_of(ws))
        return (out,) + (None,) * 10


def policy_loss(logps: torch.Tensor, advantages: torch.Tensor, labels: torch.Tensor,
                old_logps: Optional[torch.Tensor] = None, ref_logps: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                reduction: str = "token", ignore_index: int = IGNORE_INDEX
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, mean_kl, clipped_share)`` of sampled answers.

    logps [B, S] fp32, advantages [B] or [B, S], old_logps [B, S] of the policy
    that sampled the answers (None: this policy; the ratio is then 1 and its
    gradient that of the log-probability). Per labelled token, with
    r = exp(logps - old_logps):

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^d - d - 1),
        d = ref_logps - logps

    (no KL term without ref_logps). ``reduction="token"`` is the mean over all
    labelled tokens, ``"sequence"`` the mean over the batch of each sequence's
    mean (0 for a sequence without labelled tokens). mean_kl (of e^d - d - 1) and
    clipped_share are detached means over the labelled tokens. A labelled token's NaN
    log-probability (a label outside the vocabulary has one) makes the loss NaN.
    """
    fn = "policy_loss"
    _check(fn, logps, labels)
    b, s = logps.shape
    if reduction not in REDUCTIONS:
        raise ValueError(f"{fn}: reduction must be one of {sorted(REDUCTIONS)}, not {reduction!r}")
    if not (0.0 <= clip_low < 1.0 and 0.0 <= clip_high < math.inf):
        raise ValueError(f"{fn}: clip_low must be in [0, 1), clip_high finite and not negative")
    if not 0.0 <= kl_coef < math.inf:
        raise ValueError(f"{fn}: kl_coef must be finite and not negative")
    if kl_coef and ref_logps is None:
        raise ValueError(f"{fn}: kl_coef needs ref_logps")
    _constant(fn, "advantages", advantages, ((b,), (b, s)), logps.device)
    for name, t in (("old_logps", old_logps), ("ref_logps", ref_logps)):
        if t is not None:
            _constant(fn, name, t, ((b, s),), logps.device)
    keep = torch.is_grad_enabled() and logps.requires_grad
    return PolicyLossFunction.apply(logps, advantages, labels, old_logps, ref_logps, float(clip_low),
                                    float(clip_high), float(kl_coef), REDUCTIONS[reduction],
                                    int(ignore_index), keep)
