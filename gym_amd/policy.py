"""The policy's end of the VecEnv loop: logits to actions, their scores with gradients, dropout.

The reference leaves all of this to its trainer: VecEnv::step takes finished actions (wrappers/vec_env/base.h:56-63).  Here

    process_logits     penalties for repeated choices, biases, masks and temperature on a batch of logits (differentiable)
    sample_actions     the same rules, one action per row from softmax and its log-probability, in one pass
    action_log_prob    log-probability and entropy of given actions under the same rules (differentiable)
    dropout            from a counter-based generator; the mask is never stored (differentiable)

run in hand-written HIP kernels behind include/gymhip.h.  Rows are environments (or text streams), columns are actions: two of CartPole's
as well as a vocabulary.  Random numbers are a function of (seed, row, step) alone.  With a row's key its env's GLOBAL index, results do not
depend on the GPU count (as the envs' own resets), and an update that passes a rollout's (row, step) pairs again, in any order, finds
the very masks the rollout ran under.

gym_amd.vec_env calls them from VecLogitActions (step(logits)) and VecObservationDropout.


The tensors' checks, the autograd nodes and the calls of the C ABI are C++ (include/gym/hip_policy.h, which C++ trainers include themselves), bound in
csrc/policy_torch.cpp.  Wrong values raise ValueError, wrong Python types TypeError, and what fails or finds no GPU GymhipError.  There are first derivatives in
reverse mode: a second one (create_graph) and tensors with a forward-mode tangent raise RuntimeError.
"""
from __future__ import annotations

import importlib.util
import os
from typing import NamedTuple

import torch

from . import _lib as L


def _load():
    L.load()   # first: the binding's entry for libgymhip.so then resolves to this very library
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "gymhip_policy.so")
    if not os.path.exists(path):
        raise L.GymhipError(f"{path} not found: the policy operators are not built and there is no fallback")
    spec = importlib.util.spec_from_file_location("gymhip_policy", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_ext = _load()


class ActionSample(NamedTuple):
    """actions [N] int32 (what the engine steps; -1 where nothing could be chosen) and their log-probabilities [N] float32."""
    actions: torch.Tensor
    log_prob: torch.Tensor


class LogitRules(_ext.LogitRules):
    """What is done to a row's logits x before anything is chosen or scored.  With c = how often v occurs in the row's history:

        x' = x, or where c > 0: (x / repetition if x > 0 else x * repetition) - frequency * c - presence
        z  = (x' + bias[v]) / temperature, and -inf where the mask does not allow v, whatever x holds there

    mask          int32 [1, words] (all rows), [rows, words], or with mask_rows [lines, words]; bit v % 32 of word v // 32 set = v allowed
                  (pack_action_mask makes it from booleans)
    mask_rows     int32 [rows]: the mask line of each row; negative = everything allowed, past the last line = nothing
    bias          float32 [width], [1, width] or [rows, width]
    history       int32 / int64 [rows, length] of earlier choices; ids outside [0, width) are skipped (any padding of that kind will do)
    history_len   int32 / int64 [rows]: how many of a row's ids count (None = all)
    repetition, presence, frequency, temperature   a number, or float32 [rows].  repetition > 0, temperature >= 0; the penalties act through
                  `history` alone.  Temperature 0 leaves z undivided, and sample_actions then takes the greatest z (lowest v of equal ones).

    The tensors are read when an operator runs, not copied here; values of the tensors are not checked.  They have no gradient: under autograd
    one that requires it is refused by the differentiable operators (sample_actions takes it)."""

    __slots__ = ()


def pack_action_mask(allowed: torch.Tensor) -> torch.Tensor:
    """Booleans [lines, width] (True = allowed) as the int32 words [lines, ceil(width / 32)] that LogitRules takes."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError("pack_action_mask needs a 2-D bool tensor")
    lines, width = allowed.shape
    words = (width + 31) // 32
    bits = torch.nn.functional.pad(allowed, (0, 32 * words - width)).view(lines, words, 32).to(torch.int64)
    return (bits << torch.arange(32, device=allowed.device)).sum(2).to(torch.int32)   # the low 32 bits, bit 31 as the sign


def _rules(rules):
    if rules is not None and not isinstance(rules, LogitRules):
        raise ValueError("rules must be a LogitRules")
    return rules


def process_logits(logits: torch.Tensor, rules: LogitRules | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """z (LogitRules) of logits [rows, width], rounded to float32 and from there to their type.  Differentiable in the logits.  `out` (not
    under autograd) may be the logits themselves, or memory that shares no element with them or the rules' tensors (other columns of the
    same buffer, say).  It changes in place: a backward pass that has saved it raises."""
    if out is None:
        return _ext.process_logits(logits, _rules(rules))
    _ext.process_logits_into(logits, _rules(rules), out)
    return out


def sample_actions(logits: torch.Tensor, rules: LogitRules | None = None, *, seed: int, step=0, rows=0, out: ActionSample | None = None) -> ActionSample:
    """One action per row of logits [rows, width] from softmax(z), and its log-probability (no gradient: score the action with
    action_log_prob for that).  The draw is a function of the row's z and of (seed, row key, step) alone: `rows` is the key of row 0 (row b
    has rows + b) or int64 [rows]; `step` is a number, an int64 device scalar (one for all rows, read when the kernel runs: advance it
    between replays of a captured graph) or int64 [rows].  Keys and steps count modulo 2^48.

    A row with nothing allowed gives action -1 and log-probability -inf, a row with a NaN or +inf among its allowed z -1 and NaN.

    `out`'s tensors must lie neither in the logits nor in each other.  They change in place: a backward pass that has saved them (action_log_prob saves its actions) raises."""
    if out is None:
        return ActionSample(*_ext.sample_actions(logits, _rules(rules), seed, step, rows))
    _ext.sample_actions(logits, _rules(rules), seed, step, rows, *out)
    return ActionSample(*out)


def action_log_prob(logits: torch.Tensor, actions: torch.Tensor, rules: LogitRules | None = None):
    """(log softmax(z)[action], entropy of softmax(z)), float32 [rows] each, for logits [rows, width] and actions int32 / int64 [rows].
    Differentiable in the logits.  An action that is not allowed, or outside [0, width), has -inf, and one of -inf (also where float32 holds
    nothing so low) hands no gradient back through its log-probability; a row with nothing allowed has -inf, entropy 0 and no gradient, one with a NaN or +inf among its allowed z NaN for
    both and in its gradient, whatever the action."""
    return _ext.action_log_prob(logits, actions, _rules(rules))


def dropout(x: torch.Tensor, p: float, *, seed: int, step=0, rows=0) -> torch.Tensor:
    """x [rows, width] with each element 0 with probability p (p to 16 bits: t = round(65536 p)) and multiplied by 65536 / (65536 - t)
    otherwise.  Which ones follows from (seed, row key, step, column) alone (`rows` and `step` as in sample_actions); give every layer a
    seed of its own.  Differentiable in x; the backward pass draws the mask again, so a device `step` must not be advanced before it."""
    return _ext.dropout(x, p, seed, step, rows)
