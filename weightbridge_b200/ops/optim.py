"""The optimizer step that produces the weights a sync sends: AdamW over many tensors in one
launch, with states in 32 or 8 bits, and the global gradient norm.
"""
from __future__ import annotations

from typing import Any, Callable, Iterable, Mapping

import torch

from ._ext import ext

STATE_BLOCK = 128           # elements that share a scale in the 8-bit states
# Squares below 2^-126 are no normal fp32 numbers: roots below 2^-63 may count as 0, and eps alone must keep the step
# on such gradients small.  From 2^-50 on an update is off by at most 1.5e-5 of lr (beta2 = 0.999; 3e-7 at 0.95).
MIN_EPS = 2.0 ** -50
MAX_BETA1_FP8, MAX_BETA2_FP8 = 0.98, 0.95       # the longest memories that 8-bit moments keep up with


def grad_norm(tensors: Mapping[str, torch.Tensor] | Iterable[torch.Tensor], group: Any = None) -> torch.Tensor:
    """The 2-norm over all ``tensors`` (a dict or an iterable; ``None`` entries are left out) as
    an fp32 scalar on their device, without waiting for it.

    bf16, fp16 and fp32 tensors of one device, each filling its memory without holes (of a DTensor,
    its local tensor).  The sum
    runs in a fixed order: the same inputs give the same bits.  ``group``: a process group over
    which the squares are summed; a tensor that several of its ranks hold counts once per rank.
    Squares are formed, and up to 64 of them added, in 32 bits, all else in 64: gradients above 2.3e18 can
    make the norm infinite, those below 1.1e-19 lose bits of their squares, and below 2.6e-23 they do not count.
    """
    if not isinstance(tensors, (dict, list, tuple)):
        tensors = dict(tensors) if isinstance(tensors, Mapping) else list(tensors)
    norm, buffer = ext().sum_squares(tensors)
    if group is None:
        return norm
    sum_sq = buffer[0]
    torch.distributed.all_reduce(sum_sq, group=group)
    return sum_sq.sqrt().float()


class AdamW:
    """AdamW (decoupled weight decay) over a dict of tensors, one launch per step.

    ``params``: name -> tensor, e.g. ``dict(model.named_parameters())`` or the tensors a layout
    allocates; bf16, fp16 or fp32 on one CUDA device, each filling its memory without holes (any
    order of dimensions).  They are updated in place.  Of an FSDP trainer's DTensors, their local
    tensors (``parallel.fsdp.convert_to_wb`` returns those) with the gradients' local tensors.
    ``states``: ``"fp32"``, or ``"fp8"``: both moments as e4m3 with one fp32 scale per 128 elements, 2.06 bytes a parameter instead of
    8 (the second moment as its root).  Codes are rounded to nearest, 3 to 6 % from their neighbours'
    borders, and a root decays by ``sqrt(beta2)`` a step: it follows because its block's scale moves, and
    only up to ``beta2`` = 0.95 (normal gradients: 5 % too large in the median there, 17 % at 0.97, 40 % and
    more from 0.98 on, and elements whose gradients become small stop), so larger ones are refused.  A
    block whose largest root stands still to a few percent keeps its other roots from decaying.  The
    first moment's rounding adds up to 6 % of it at ``beta1`` = 0.9, 13 % at 0.98 and 18 to 36 % at 0.99:
    above 0.98 it is refused, too.
    ``betas``: (0.9, 0.999), with 8-bit states (0.9, 0.95).  ``eps``: at least 2^-50 (9e-16).
    ``master``: keep fp32 master weights of 16-bit parameters (taken from the parameters now, and by
    ``read_master``: values written into the parameters otherwise do not last);
    without them an update below half a step of the 16-bit type is lost.  ``no_decay``: names
    without weight decay, or a function of the name.

    The states are flat buffers (``states()``); every tensor's slice starts at a multiple of 128
    elements, in the order of ``params``.  The step count lives on the device, so a captured step
    can be replayed (while the optimizer lives); a step runs on the current stream of the parameters'
    device.  Steps of one optimizer follow one another: whoever takes them on several streams orders
    those, and ``step_count``, ``state_dict`` and ``load_state_dict`` behind them.  fp32 arithmetic with the hardware's
    approximate root and reciprocal (relative errors of 2^-23).
    """

    def __init__(self, params: Mapping[str, torch.Tensor], lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] | None = None,
                 eps: float = 1e-8, weight_decay: float = 0.01, *, states: str = "fp32", master: bool = False,
                 no_decay: Iterable[str] | Callable[[str], bool] = ()):
        if states not in ("fp32", "fp8"):
            raise ValueError(f"AdamW: states must be 'fp32' or 'fp8', not {states!r}")
        if betas is None:
            betas = (0.9, MAX_BETA2_FP8 if states == "fp8" else 0.999)
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), not {betas}")
        for k, most in enumerate((MAX_BETA1_FP8, MAX_BETA2_FP8)):
            if states == "fp8" and betas[k] > most:
                raise ValueError(f"AdamW: 8-bit moments do not follow a beta{k + 1} above {most} (given: {betas[k]}): "
                                 "use a smaller one, or states='fp32'")
        if not MIN_EPS <= eps < float("inf") or not 0.0 <= weight_decay < float("inf"):
            raise ValueError("AdamW: eps must be finite and at least 2^-50 (9e-16), and weight_decay finite and not negative")
        self._check_lr(lr)
        self.lr = lr
        self.betas, self.eps, self.weight_decay = tuple(map(float, betas)), float(eps), float(weight_decay)
        self.state_bits = states
        self.names = list(params)
        skip = no_decay if callable(no_decay) else frozenset(no_decay).__contains__
        if not callable(no_decay) and (unknown := frozenset(no_decay) - set(self.names)):
            raise ValueError(f"AdamW: no_decay names {sorted(unknown)[0]!r}, which is not a parameter")
        self._program = ext().AdamWProgram(self.names, list(params.values()), [0.0 if skip(n) else self.weight_decay for n in self.names],
                                           *self.betas, self.eps, states == "fp8", bool(master))

    @staticmethod
    def _check_lr(lr) -> None:
        if not isinstance(lr, torch.Tensor) and not 0.0 <= lr < float("inf"):
            raise ValueError(f"AdamW: lr must be finite and not negative, not {lr}")

    def step(self, grads: Mapping[str, torch.Tensor] | None = None, *, lr: float | torch.Tensor | None = None,
             max_norm: float | None = None, group: Any = None) -> torch.Tensor | None:
        """One update from ``grads`` (name -> tensor of the parameter's type or fp32; default: the
        parameters' ``.grad``).  A parameter without a gradient is left alone in this step.
        The bias correction counts this optimizer's steps, not a parameter's own: one whose first
        gradient comes late takes a smaller first step than lr (betas 0.9 and 0.95: 0.45 of it).

        ``lr``: this step's learning rate (default: ``self.lr``); a one-element tensor on the
        device is read there, so that it can change under a captured step.  ``max_norm``: scale
        the gradients by ``min(1, max_norm / (norm + 1e-6))``; the global norm is returned as a
        device scalar, and a step whose norm is not finite changes nothing, nor the step count.
        ``group``: the ranks whose squares make up the norm (``grad_norm``).  Nothing waits for
        the GPU.
        """
        p = self._program
        lr = self.lr if lr is None else lr
        self._check_lr(lr)
        on_device = lr if isinstance(lr, torch.Tensor) else None
        number = 0.0 if on_device is not None else float(lr)
        if max_norm is None:
            if group is not None:
                raise ValueError("AdamW.step: a group is for the norm: give max_norm, too")
            return p.step(grads, number, on_device, None, 0.0)
        if not max_norm > 0.0:
            raise ValueError(f"AdamW.step: max_norm must be positive, not {max_norm}")
        sum_sq = None                           # the kernels' own, from these gradients
        if group is not None:
            sum_sq = p.grad_sum_sq(grads)
            torch.distributed.all_reduce(sum_sq, group=group)
        return p.step(grads, number, on_device, sum_sq, float(max_norm))

    def states(self) -> dict[str, torch.Tensor]:
        """The flat state buffers: ``exp_avg`` and ``exp_avg_sq`` (fp32), or ``exp_avg`` and
        ``rms`` (e4m3, the root of the second moment) with ``exp_avg_scale`` and ``rms_scale``;
        ``master`` with master weights (the slices of fp32 parameters are not used).  They are the
        optimizer's own, not copies."""
        p = self._program
        if self.state_bits == "fp8":
            out = {"exp_avg": p.exp_avg, "exp_avg_scale": p.exp_avg_scale, "rms": p.second, "rms_scale": p.second_scale}
        else:
            out = {"exp_avg": p.exp_avg, "exp_avg_sq": p.second}
        if p.master is not None:
            out["master"] = p.master
        return out

    def slices(self, flat: torch.Tensor) -> dict[str, torch.Tensor]:
        """Every parameter's slice of a flat buffer of ``states()``, shaped like the parameter."""
        if flat.numel() != self._program.total:
            raise ValueError("AdamW.slices: not a buffer of one value per element")
        return {n: self._program.slice(flat, i) for i, n in enumerate(self.names)}

    @property
    def step_count(self) -> int:
        """How many updates were taken (reads the device)."""
        return self._program.step_count

    def rebind(self, params: Mapping[str, torch.Tensor]) -> None:
        """Go on with the same parameters at new addresses (their memory was released and
        allocated again, e.g. by an engine that shares the GPU).  Waits for the GPU.  A captured
        step follows: from now on its replays update the parameters where they are now, from
        gradients where they were at the capture."""
        if list(params) != self.names:
            raise ValueError("AdamW.rebind: the parameters' names or their order differ")
        self._program.rebind(list(params.values()))

    def read_master(self) -> None:
        """Take the fp32 master weights from the parameters' present values, as the constructor did.
        A step goes on from the master weights and overwrites the parameters, so whoever changes those
        (a checkpoint loaded into them, weights restored before or after ``rebind``) calls this next.
        Waits for the GPU."""
        self._program.read_master()

    def state_dict(self) -> dict:
        """The step count, the names and the state buffers (not copies)."""
        return {"step": self.step_count, "names": list(self.names), **self.states()}

    def load_state_dict(self, saved: Mapping[str, Any]) -> None:
        """Take over the states of ``saved`` (of an optimizer of the same parameters and state
        bits); with master weights, the parameters keep their values until the next step."""
        if list(saved["names"]) != self.names:
            raise ValueError("AdamW.load_state_dict: the parameters' names or their order differ")
        own = self.states()
        for name, buf in own.items():
            src = saved.get(name)
            if src is None or src.shape != buf.shape or src.dtype != buf.dtype:
                raise ValueError(f"AdamW.load_state_dict: {name} is missing or of another size or type")
        if int(saved["step"]) < 0:
            raise ValueError("AdamW.load_state_dict: the step count is negative")
        for name, buf in own.items():
            if buf.data_ptr() != saved[name].data_ptr():
                buf.copy_(saved[name])
        self._program.step_count = int(saved["step"])
