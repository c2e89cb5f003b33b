"""From tours back to the heat map: log-probabilities of tours and the losses that turn lengths into a gradient.

What ``greedy_decode_device`` / a sampling decoder (``ml4tsp/nar/decoder/sampling.py:21-43``) draws from a heat map,
``two_opt_device`` improves and ``evaluate_tours`` measures is scored here under the heat map (or under the logits that
an autoregressive decoder wrote), with gradients for ``torch.autograd``: ``tour_log_probs`` (csrc/tour_logprobs.hip),
``clipped_policy_loss`` and ``preference_loss`` (csrc/policy_loss.hip).

Everything runs on the current stream of the tensors' device, without host synchronisation, and may be captured into a
graph; results do not change from run to run.  There is no CPU path, no second derivative, no ``torch.func`` transform
and no forward mode: all of them raise.  The autograd nodes are csrc/learning_ext.cpp.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_ROWS = {"node": 0, "step": 1}


def _check_type(x: torch.Tensor, name: str) -> None:
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")


def _same_device(first: torch.Tensor, what: str, *others: Optional[torch.Tensor]) -> torch.device:
    if first.device.type != "cuda" or any(o is not None and o.device != first.device for o in others):
        raise ValueError(f"{what} must live on the same HIP device")
    return first.device


def tour_log_probs(logits: torch.Tensor, tours: torch.Tensor, *, tours_per_map: int = 1,
                   rows: str = "node") -> torch.Tensor:
    """Log-probability of every choice of every tour; differentiable in ``logits``.

    Step ``t = 0 .. N-2`` of a tour chooses ``tours[:, t+1]`` among the nodes it has not visited yet, with the softmax
    of one row of logits over those nodes.  ``logits`` float32 / bfloat16 / float16:

    * ``rows="node"``: heat maps (M, N, N), the row of the node that is left; tours (M * tours_per_map, N+1), tour ``k``
      uses map ``k // tours_per_map``.  For a heat map of positive weights pass its logarithm.
    * ``rows="step"``: what an autoregressive decoder wrote, (T, N-1, N), a row for every step; ``tours_per_map`` is 1.

    Returns (T, N-1) float32; ``.sum(1)`` is a tour's log-likelihood.  Entries of visited nodes are never used, so no
    mask is needed; -inf (or the type's lowest value) marks forbidden edges.  A step without any open finite entry gets
    -inf and no gradient, a tour that is no permutation of ``0 .. N-1`` gets NaN and no gradient, and a step whose
    incoming gradient is 0 contributes nothing.  Asynchronous on the current stream."""
    if logits.dim() == 2 and rows == "node":
        return tour_log_probs(logits.unsqueeze(0), tours, tours_per_map=tours_per_map, rows=rows)
    if tours.dim() == 1:
        tours = tours.unsqueeze(0)
    if rows not in _ROWS:
        raise ValueError(f"rows must be 'node' or 'step', got {rows!r}")
    _check_type(logits, "logits")
    if tours.dtype.is_floating_point or tours.dtype.is_complex or tours.dtype == torch.bool:
        raise TypeError(f"tours must be integers, got {tours.dtype}")
    per = int(tours_per_map)
    if logits.dim() != 3 or tours.dim() != 2 or per < 1 or tours.shape[1] < 2:
        raise ValueError("expected logits (M, N, N) or (T, N-1, N) and tours (T, N+1)")
    T, n = tours.shape[0], tours.shape[1] - 1
    if rows == "step" and per != 1:
        raise ValueError("rows='step' has logits of its own for every tour: tours_per_map must be 1")
    want = (T // per, n, n) if rows == "node" else (T, n - 1, n)
    if tuple(logits.shape) != want or T % per:
        raise ValueError(f"expected logits {want} for {T} tours of {n} nodes, {per} a map, got {tuple(logits.shape)}")
    _same_device(logits, "logits and tours", tours)
    return _lib.learning_ext().tour_log_probs(logits, tours, per, _ROWS[rows])


@dataclass
class PolicyLossResult:
    """Device-resident result of ``clipped_policy_loss``."""
    loss: torch.Tensor              # () float32, differentiable in log_probs
    kl: torch.Tensor                # () float32 average of exp(d) - 1 - d (not multiplied by kl_coef)
    clip_fraction: torch.Tensor     # () float32 share of the steps (tours) whose ratio is clipped


def _step_arrays(log_probs, mask, **others):
    """Checks shared by the losses: (T, S) arrays of one type, a boolean mask."""
    _check_type(log_probs, "log_probs")
    if log_probs.dim() != 2:
        raise ValueError("expected log_probs (T, steps)")
    for name, x in others.items():
        if x is None:
            continue
        if x.dtype != log_probs.dtype:
            raise TypeError(f"{name} must have the type of log_probs, {log_probs.dtype}, got {x.dtype}")
        if x.shape != log_probs.shape:
            raise ValueError(f"{name} must have the shape of log_probs, {tuple(log_probs.shape)}, got {tuple(x.shape)}")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"mask must be boolean, got {mask.dtype}")
        if mask.shape != log_probs.shape:
            raise ValueError(f"mask must have the shape of log_probs, {tuple(log_probs.shape)}, got {tuple(mask.shape)}")


def clipped_policy_loss(log_probs: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor, *,
                        ref_log_probs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                        clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, ratio: str = "step",
                        average: Optional[str] = None) -> PolicyLossResult:
    """Clipped policy loss with a KL term; differentiable in ``log_probs``.

    ``log_probs`` / ``old_log_probs`` / ``ref_log_probs`` (T, S) of one type (float32, bfloat16, float16): the steps of
    ``tour_log_probs`` now, when the tours were drawn, and under a reference.  ``advantages`` (T,) or (T, S).
    ``mask`` (T, S) boolean, True where a step counts (the others' values are not used).

    ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)`` with ``r = exp(log_probs - old_log_probs)`` for every step,
    or with ``ratio="tour"`` of the tour's summed difference (advantages (T,)), plus ``kl_coef`` times
    ``exp(d) - 1 - d``, ``d = ref_log_probs - log_probs`` of every step.  ``average="step"`` (the default for ratios of
    steps): over all steps that count; ``"tour"`` (always for ratios of tours): over a tour's steps, then over the tours
    that have any.  Nothing that counts: loss 0; an advantage of 0 adds 0 however far its ratio has gone.  Steps of -inf
    now and then alike (forbidden edges) give NaN: mask them.
    Asynchronous on the current stream."""
    _step_arrays(log_probs, mask, old_log_probs=old_log_probs, ref_log_probs=ref_log_probs)
    if ratio not in ("step", "tour") or average not in (None, "step", "tour"):
        raise ValueError("ratio and average must be 'step' or 'tour'")
    average = average or ratio
    if ratio == "tour" and average != "tour":
        raise ValueError("ratios of tours are averaged over tours")
    T, S = log_probs.shape
    if tuple(advantages.shape) not in ((T,), (T, S)) or (ratio == "tour" and advantages.dim() != 1):
        raise ValueError("advantages must be (T,), or (T, steps) with ratios of steps")
    if not advantages.dtype.is_floating_point:
        raise TypeError(f"advantages must be floating point, got {advantages.dtype}")
    if not (0.0 <= clip_low < 1.0 and clip_high >= 0.0 and 0.0 <= kl_coef < math.inf):
        raise ValueError("clip_low must be in [0, 1), clip_high and kl_coef >= 0, kl_coef finite")
    if kl_coef and ref_log_probs is None:
        raise ValueError("kl_coef needs ref_log_probs")
    _same_device(log_probs, "log_probs and the other arrays", old_log_probs, advantages, ref_log_probs, mask)
    return PolicyLossResult(*_lib.learning_ext().policy_loss(
        log_probs, old_log_probs, ref_log_probs, advantages, mask, ratio == "tour", average == "tour", clip_low, clip_high,
        kl_coef))


@dataclass
class PreferenceLossResult:
    """Device-resident result of ``preference_loss``."""
    loss: torch.Tensor              # () float32, differentiable in log_probs
    num_pairs: torch.Tensor         # () int64 pairs the loss is the average of


def preference_loss(log_probs: torch.Tensor, lengths: torch.Tensor, *, tours_per_instance: int,
                    ref_log_probs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                    beta: float = 1.0, label_smoothing: float = 0.0, pairs: str = "all",
                    per_step: bool = False) -> PreferenceLossResult:
    """Preference loss over the tours of every instance, the shorter one preferred; differentiable in ``log_probs``.

    ``log_probs`` / ``ref_log_probs`` (T, S) of one type, T = I * tours_per_instance; ``lengths`` (T,) as
    ``evaluate_tours`` gives them; ``mask`` as in ``clipped_policy_loss``.  A tour's score is ``beta`` times the sum
    (``per_step``: mean) over its steps of ``log_probs - ref_log_probs``; over all pairs of tours of one instance whose
    lengths differ (``pairs="best"``: only those with the instance's first shortest tour) the loss is the average of
    ``-(1 - label_smoothing) log sigmoid(s_short - s_long) - label_smoothing log sigmoid(s_long - s_short)``.
    Sampled tours against the same tours after ``two_opt_device``: stack them as an instance's tours.  NaN lengths are
    in no pair; without any pair the loss is 0.  Steps of -inf (forbidden edges) make a tour's score -inf and two such
    tours' pair NaN: mask them, or mark forbidden edges by a finite logit.  Asynchronous on the current stream."""
    _step_arrays(log_probs, mask, ref_log_probs=ref_log_probs)
    per = int(tours_per_instance)
    T = log_probs.shape[0]
    if per < 1 or T % per or tuple(lengths.shape) != (T,):
        raise ValueError("expected log_probs (I * tours_per_instance, steps) and lengths (I * tours_per_instance,)")
    if lengths.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"lengths must be float32 or float64, got {lengths.dtype}")
    if pairs not in ("all", "best"):
        raise ValueError(f"pairs must be 'all' or 'best', got {pairs!r}")
    if not (0.0 < beta < math.inf and 0.0 <= label_smoothing < 0.5):
        raise ValueError("beta must be > 0 and finite and label_smoothing in [0, 0.5)")
    _same_device(log_probs, "log_probs and the other arrays", lengths, ref_log_probs, mask)
    return PreferenceLossResult(*_lib.learning_ext().preference_loss(
        log_probs, ref_log_probs, lengths, mask, per, pairs == "best", bool(per_step), beta, label_smoothing))
