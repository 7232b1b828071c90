"""AdamW over many tensors in one launch, with states in 8 or in 32 bits.

The counterpart of the HF Trainer's optimiser step for a user of the reference
(``task/task.yaml:10-22`` sets AdamW and its learning rate; there is no reference
kernel). :class:`.qlora.QLoRATrainer` keeps its LoRA factors in one flat buffer
(``soup_adamw_flat``); :class:`MultiTensorAdamW` takes any list of separate
parameters - LoRA factors, norm weights, a trained head - and steps them together
(csrc/adamw_multi.cu): one launch for up to 960 tensors of a type, whose addresses
are launch arguments, plus one pass over the gradients when their norm is clipped.
"""

from __future__ import annotations

import array
import ctypes
import itertools
import math
import operator
from typing import Iterable, Optional

import torch

from . import _lib

#: Elements that share one scale of an 8-bit state.
STATE_BLOCK = 256


_grad = operator.attrgetter("grad")


def _address(a: array.array) -> int:
    return a.buffer_info()[0]


def _addresses(tensors, sizes, code: int, device):
    """Addresses of tensors that are as a launch needs them, or None."""
    try:
        out = _lib.tensor_addresses(tensors, sizes, code, device)
    except (_lib.SoupError, _lib.SoupLibraryError):
        raise
    except Exception:  # a tensor without an address, say a sparse one
        return None
    return None if isinstance(out, int) else out


class _Held:
    """States and launch tables of one parameter group."""

    __slots__ = ("params", "sizes", "by_dtype", "m", "v", "m_scale", "v_scale")


class MultiTensorAdamW(torch.optim.Optimizer):
    """AdamW (``torch.optim.AdamW``'s form, decoupled weight decay) over CUDA tensors.

    params: parameters or parameter groups (``lr``, ``betas``, ``eps`` and
    ``weight_decay`` per group) of float32, bfloat16 or float16, contiguous, all on
    one device; a step refuses those that have become anything else (``p.data = ...``).
    Moments are kept for every parameter from the start:

    * ``state_bits=32``: two fp32 numbers an element;
    * ``state_bits=8``: two e4m3 numbers an element, m and the square root of v, with
      one fp32 scale for 256 elements each. The update uses the moments before they
      are rounded, and a second moment that is not 0 is not rounded to 0.

    ``max_grad_norm``: scale all gradients by min(1, max_grad_norm / (norm + 1e-6)),
    norm over the gradients of all groups; :attr:`grad_norm` then holds the last
    step's norm (a device scalar). Parameters without a gradient are left out of a
    step. The count of steps is one for all tensors and lives on the device, so a
    step can be captured into a CUDA graph (with the learning rates of the capture).
    A gradient that is not finite reaches its own element, as in
    ``torch.optim.AdamW`` (every element, where the norm is clipped).

    The optimiser's steps share their workspace and states: steps of one optimiser
    on several streams have to be ordered by the caller. A backward pass that needs the
    values before a step has to come before it; after it, it raises.
    """

    def __init__(self, params: Iterable, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, state_bits: int = 8, max_grad_norm: Optional[float] = None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits!r}")
        if max_grad_norm is not None and not (0.0 < max_grad_norm < math.inf):
            raise ValueError(f"max_grad_norm must be a positive number, not {max_grad_norm!r}")
        self.state_bits = state_bits
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None
        self._held = []
        self._step = None
        self._squares = []
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # -- set-up -----------------------------------------------------------------
    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_options(group)
            self._held.append(self._hold(group["params"]))
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_options(group) -> None:
        b1, b2 = group["betas"]
        if not (isinstance(group["lr"], (int, float)) and 0.0 <= group["lr"] < math.inf):
            raise ValueError(f"lr must be a number of 0 or more, not {group['lr']!r}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {group['betas']}")
        if not 1e-30 <= group["eps"] < math.inf:
            raise ValueError(f"eps must be at least 1e-30, not {group['eps']!r}")
        if not group["weight_decay"] >= 0.0:
            raise ValueError(f"weight_decay must be 0 or more, not {group['weight_decay']!r}")

    def _hold(self, params) -> _Held:
        held = _Held()
        if self._step is not None:
            dev = self._step.device
        else:
            dev = params[0].device if params else torch.device("cuda", torch.cuda.current_device())
        if len(set(map(id, params))) != len(params):
            raise ValueError("MultiTensorAdamW: a parameter is in the group twice")
        blocks, total = [], 0
        for p in params:
            _lib.dtype_code(p.dtype)
            if not p.is_cuda or p.device != dev:
                raise ValueError(f"MultiTensorAdamW: parameters must be on one CUDA device, got {p.device} and {dev}")
            if not p.is_contiguous():
                raise ValueError("MultiTensorAdamW: parameters must be contiguous")
            blocks.append(total)
            total += -(-p.numel() // STATE_BLOCK)
        if total >= 1 << 31:
            raise ValueError("MultiTensorAdamW: a parameter group has at most 2^39 elements")
        held.params = list(params)
        held.sizes = [p.numel() for p in params]
        by = {}
        for i, p in enumerate(params):
            if p.numel():
                by.setdefault(p.dtype, []).append(i)
        held.by_dtype = [(_lib.dtype_code(d), d, [held.params[i] for i in idx],
                          array.array("q", [held.sizes[i] for i in idx]), array.array("i", [blocks[i] for i in idx]))
                         for d, idx in by.items()]
        eight = self.state_bits == 8
        dt = torch.float8_e4m3fn if eight else torch.float32
        held.m = torch.zeros(total, STATE_BLOCK, dtype=torch.uint8 if eight else dt, device=dev).view(dt)
        held.v = torch.zeros(total, STATE_BLOCK, dtype=torch.uint8 if eight else dt, device=dev).view(dt)
        held.m_scale = torch.zeros(total, dtype=torch.float32, device=dev) if eight else None
        held.v_scale = torch.zeros(total, dtype=torch.float32, device=dev) if eight else None
        if self._step is None and params:
            self._step = torch.zeros((), dtype=torch.float32, device=dev)
            self._coefs = torch.zeros(4, dtype=torch.float32, device=dev)
        if self.max_grad_norm is not None:
            launches = sum(len(h.by_dtype) for h in itertools.chain(self._held, [held]))
            tensors = sum(len(h.params) for h in itertools.chain(self._held, [held]))
            # one workspace of partial sums for the launches of every type of every group
            per = int(_lib.lib().soup_grad_square_workspace_bytes(1))
            need = int(_lib.lib().soup_grad_square_workspace_bytes(max(1, tensors))) + per * launches
            if not self._squares or self._squares[-1].numel() < need:
                # the smaller ones stay: a captured step may write them
                self._squares.append(torch.empty(need, dtype=torch.uint8, device=dev))
            if self.grad_norm is None:
                self.grad_norm = torch.zeros((), dtype=torch.float32, device=dev)
        for i, p in enumerate(params):
            n = -(-p.numel() // STATE_BLOCK)
            st = {"exp_avg": held.m[blocks[i]:blocks[i] + n], "exp_avg_sq": held.v[blocks[i]:blocks[i] + n]}
            if eight:
                st["exp_avg_scale"] = held.m_scale[blocks[i]:blocks[i] + n]
                st["exp_avg_sq_scale"] = held.v_scale[blocks[i]:blocks[i] + n]
            self.state[p] = st
        return held

    # -- states -----------------------------------------------------------------
    def flat_state(self, group: int = 0) -> dict:
        """The states of a parameter group: ``step`` (completed steps), ``m`` and ``v``
        [blocks, 256], each parameter starting at a block of its own, and with 8-bit
        states ``m_scale`` and ``v_scale`` [blocks] (v then holds square roots)."""
        h = self._held[group]
        out = {"step": self._step, "m": h.m, "v": h.v}
        if self.state_bits == 8:
            out.update(m_scale=h.m_scale, v_scale=h.v_scale)
        return out

    def state_dict(self) -> dict:
        """Options and copies of the states of every group, to be given to
        :meth:`load_state_dict` of an optimiser over parameters of the same sizes."""
        return {"state_bits": self.state_bits,
                "param_groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups],
                "sizes": [list(h.sizes) for h in self._held],
                "states": [{k: v.detach().clone() for k, v in self.flat_state(i).items()}
                           for i in range(len(self._held))]}

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        if state_dict["state_bits"] != self.state_bits:
            raise ValueError(f"the state has {state_dict['state_bits']} bits, the optimiser {self.state_bits}")
        if state_dict["sizes"] != [list(h.sizes) for h in self._held]:
            raise ValueError("the state is of parameters of other sizes")
        for g in state_dict["param_groups"]:
            self._check_options(g)
        for i, (g, st) in enumerate(zip(state_dict["param_groups"], state_dict["states"])):
            self.param_groups[i].update(g)
            for name, t in self.flat_state(i).items():
                t.copy_(st[name])

    # -- step -------------------------------------------------------------------
    def _tables(self, held: _Held, device):
        """(dtype code, parameter addresses, gradient addresses, sizes, blocks, gradients,
        parameters) of each type's parameters that have a gradient; the gradients are kept until
        the launch."""
        out = []
        for code, dtype, params, sizes, blocks in held.by_dtype:
            grads = list(map(_grad, params))
            # p.data = ... gives a parameter other memory, under a gradient that stays
            both = _addresses(grads + params, sizes + sizes, code, device)
            if both is None and any(g is None for g in grads):
                keep = [i for i, g in enumerate(grads) if g is not None]
                if not keep:
                    continue
                params, grads = [params[i] for i in keep], [grads[i] for i in keep]
                sizes, blocks = (array.array(t.typecode, [t[i] for i in keep]) for t in (sizes, blocks))
                both = _addresses(grads + params, sizes + sizes, code, device)
            if both is not None:
                grad_ptrs, ptrs = both[:len(grads)], both[len(grads):]
            else:
                if any(g.layout is not torch.strided for g in grads):
                    raise ValueError("MultiTensorAdamW: gradients must be dense")
                if any(g.dtype != dtype or g.device != device or g.numel() != n for g, n in zip(grads, sizes)):
                    raise ValueError(f"MultiTensorAdamW: gradients must be {dtype} on {device} and of their parameters' "
                                     "sizes")
                ptrs = _addresses(params, sizes, code, device)
                if ptrs is None:
                    raise ValueError(f"MultiTensorAdamW: parameters must stay {dtype} on {device}, contiguous and of the "
                                     "sizes that the optimiser was made with")
                grads = [g.detach().contiguous() for g in grads]
                grad_ptrs = array.array("Q", map(torch.Tensor.data_ptr, grads))
            out.append((code, ptrs, grad_ptrs, sizes, blocks, grads, params))
        return out

    def step(self, closure=None):
        """One step over all parameters that have a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._step is None:  # no parameters at all
            return loss
        dev = self._step.device
        tables = [self._tables(h, dev) for h in self._held]
        launches = sum(map(len, tables))
        if not launches:
            return loss
        stream = _lib.stream_of(self._step)
        partials = ctypes.c_int(0)
        squares = None
        if self.max_grad_norm is not None:
            squares, nbytes = self._squares[-1].data_ptr(), self._squares[-1].numel()
            for code, _, g, sizes, *_ in itertools.chain.from_iterable(tables):
                _lib.call("soup_grad_square", dev, _address(g), _address(sizes), len(g), code, squares,
                          nbytes, ctypes.byref(partials), stream)
        done = 0
        for group, held, table in zip(self.param_groups, self._held, tables):
            b1, b2 = group["betas"]
            for code, p, g, sizes, blocks, _, params in table:
                done += 1
                torch.autograd.graph.increment_version(params)  # autograd sees no other sign of the writes
                _lib.call("soup_adamw_multi", dev, _address(p), _address(g), _address(sizes), _address(blocks), len(p),
                          code, self.state_bits, held.m.data_ptr(), held.v.data_ptr(), _lib.ptr(held.m_scale),
                          _lib.ptr(held.v_scale), group["lr"], b1, b2, group["eps"], group["weight_decay"],
                          self.max_grad_norm or 0.0, squares, partials.value, _lib.ptr(self.grad_norm),
                          self._step.data_ptr(), 1 if done == launches else 0, self._coefs.data_ptr(), stream)
        return loss
