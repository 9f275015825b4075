"""Orthogonalised updates for the weights of (deformable) convolutions.

A weight (outC, C/groups, kh, kw) is a matrix of outC rows.  :func:`newton_schulz`
turns such a matrix towards the nearest one with orthonormal rows (or columns)
by a quintic polynomial of its singular values; :class:`Muon` is the momentum
optimiser whose updates are made that way, one call of the CUDA kernels for all
parameters of a shape.  No reference counterpart.
"""
from __future__ import annotations

from typing import Iterable, List, Sequence, Union

import torch
from torch import Tensor

from .ops import _flags, _ops

#: (a, b, c) of X <- a X + (b S + c S S) X that drives singular values of
#: (0, 1] to about 1 in five steps.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)

Coefficients = Union[Sequence[float], Sequence[Sequence[float]]]


def _flat_coefficients(coefficients: Coefficients) -> List[float]:
    flat: List[float] = []
    for c in coefficients:
        flat.extend(float(v) for v in c) if isinstance(c, (tuple, list)) else flat.append(float(c))
    return flat


def _cuda_only(name: str, op: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise NotImplementedError(f"pytorch_mps_deform_conv2d_b200.{op} runs on CUDA (sm_100a) "
                                  f"tensors only; {name} is on {t.device}")


def _no_grad_only(op: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{op} has no gradient: call it under torch.no_grad() or on "
                                   "detached tensors")


def newton_schulz(update: Tensor, steps: int = 5, coefficients: Coefficients = COEFFICIENTS,
                  eps: float = 1e-7) -> Tensor:
    """Orthogonalises each matrix of ``update`` (..., rows, cols).

    ``steps`` times ``X <- a X + (b S + c S S) X`` with ``S = X X^T`` (of the
    smaller side), from ``X = update / (norm + eps)`` with the Frobenius norm;
    ``coefficients`` is ``(a, b, c)`` or one triple a step (``a`` at most 15 in
    size, ``b`` and ``c`` too or else ``a + b s + c s^2`` for ``s`` in [0, 1]),
    of polynomials that keep singular values of [0, 1] below 2
    (others may end in NaN).  float32, bfloat16 or float16 in and out, any strides; the
    result is contiguous.  float32 keeps fp32 accuracy, or about that of TF32
    in the math mode ``"tf32"`` (:func:`set_math_mode`).  float16 results are
    off by their own rounding; for bfloat16 the matrix is held in float16 between
    the steps, and where it is nearly square so are the later S and polynomials:
    five steps come out 1.7e-3 to 2.0e-3 from the exact answer (in the 2-norm),
    of which 1.66e-3 are the result's own rounding.  A matrix of zeros stays
    zero; NaN or an infinity makes its whole matrix NaN.  Not differentiable.
    """
    _cuda_only("update", "newton_schulz", update)
    _no_grad_only("newton_schulz", update)
    return _ops().newton_schulz.default(update, int(steps), _flat_coefficients(coefficients), float(eps),
                                _flags(None))


def muon_update_(params: Sequence[Tensor], grads: Sequence[Tensor], momenta: Sequence[Tensor], *,
                 lr: float, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Coefficients = COEFFICIENTS, eps: float = 1e-7,
                 adjust: str = "original", groups: int = 1) -> None:
    """One step of :class:`Muon` on lists of tensors, in place.

    ``m <- momentum m + (1 - momentum) g``, ``u = (1 - momentum) g + momentum m``
    (``nesterov``; else ``u = m``), ``p <- (1 - lr weight_decay) p - lr s
    newton_schulz(u)`` with ``s = sqrt(max(1, rows / cols))`` (``adjust
    "original"``) or ``0.2 sqrt(max(rows, cols))`` (``"match_rms"``).  A tensor
    counts as a matrix of ``shape[0]`` rows, or as ``groups`` of
    ``shape[0] / groups``.  Params and grads: one of float32, bfloat16 and
    float16; momenta: float32 whatever the params are.  ``u`` of 16-bit params
    is rounded to float16 (times a power of two) and orthogonalised as a
    bfloat16 matrix.  Params are dense with dimension 0 outermost (contiguous or
    channels-last), on one device.
    """
    if adjust not in ("original", "match_rms"):
        raise ValueError(f"adjust must be 'original' or 'match_rms', got {adjust!r}")
    for name, ts in (("params", params), ("grads", grads), ("momenta", momenta)):
        for t in ts:
            _cuda_only(name, "muon_update_", t)
    with torch.no_grad():
        _ops().muon_update_.default(list(params), list(grads), list(momenta), float(lr), float(momentum),
                            bool(nesterov), float(weight_decay), int(steps),
                            _flat_coefficients(coefficients), float(eps), adjust == "match_rms",
                            int(groups), _flags(None))


class Muon(torch.optim.Optimizer):
    """Momentum optimiser with orthogonalised updates (:func:`muon_update_`).

    For parameters of two dimensions and more -- a
    :class:`DeformConv2d`'s ``weight``, not its ``bias``.  A grouped
    convolution's parameter group takes ``groups=...``, so that each group's
    rows are a matrix of their own.  The state is one float32 momentum a
    parameter, made by its first step, which no CUDA graph can capture.  ``lr``
    and the other settings are read when ``step`` is called: a captured graph
    keeps those of its capture.
    """

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95,
                 nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Coefficients = COEFFICIENTS, eps: float = 1e-7,
                 adjust: str = "original", groups: int = 1):
        if lr < 0.0:
            raise ValueError(f"lr must be non-negative, got {lr}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must be in [0, 1), got {momentum}")
        if weight_decay < 0.0:
            raise ValueError(f"weight_decay must be non-negative, got {weight_decay}")
        if adjust not in ("original", "match_rms"):
            raise ValueError(f"adjust must be 'original' or 'match_rms', got {adjust!r}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, adjust=adjust,
                                      groups=groups))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        for p in group["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError("Muon takes parameters of two dimensions and more; got shape "
                                 f"{tuple(p.shape)} (leave biases to another optimiser)")
            if group["groups"] < 1 or p.shape[0] % group["groups"] != 0:
                self.param_groups.pop()
                raise ValueError(f"{p.shape[0]} rows are not divisible by "
                                 f"groups={group['groups']}")

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # the base class casts states to their parameter's type; the momentum
        # stays float32
        ours = [p for g in self.param_groups for p in g["params"]]
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip(ours, saved):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None:
                fresh = torch.empty_like(p, dtype=torch.float32)
                self.state[p]["momentum_buffer"] = fresh.copy_(m)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not support sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        # every replay would set it to zero again
                        del self.state[p]
                        raise RuntimeError("Muon: make a step before the one that a CUDA graph "
                                           "captures; the momentum does not exist yet")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
                by_device.setdefault(p.device, []).append((p, p.grad, state["momentum_buffer"]))
            for items in by_device.values():
                ps, gs, ms = zip(*items)
                muon_update_(ps, gs, ms, lr=group["lr"], momentum=group["momentum"],
                             nesterov=group["nesterov"], weight_decay=group["weight_decay"],
                             steps=group["steps"], coefficients=group["coefficients"],
                             eps=group["eps"], adjust=group["adjust"], groups=group["groups"])
        return loss
