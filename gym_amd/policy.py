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
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib as L

_TYPES = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}
_INTS = {torch.int32: L.ACT_I32, torch.int64: L.ACT_I64}


class ActionSample(NamedTuple):
    """actions [N] int32 (what the engine steps; -1 where nothing could be chosen) and their log-probabilities [N] float32."""
    actions: torch.Tensor
    log_prob: torch.Tensor


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name, x, *args):
    """The entry point on x's device and its current stream."""
    index = x.device.index
    if index == torch.cuda.current_device():
        rc = getattr(_lib or _load(), name)(*args, _raw_stream(index))
    else:   # kernels go to the current device
        with torch.cuda.device(index):
            rc = getattr(_lib or _load(), name)(*args, _raw_stream(index))
    if rc:
        L.check(rc, name)


_lib = None


def _load():
    global _lib
    _lib = L.load()
    return _lib


def _ready(x, rules=None, what="logits"):
    """x where it is a matrix the kernels take, its rows in order and its columns adjacent (rows may be apart, or all the same one); else a copy."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{what} must be a 2-D tensor [rows, width]")
    if x.dtype not in _TYPES:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise L.GymhipError(f"{what} is on {x.device}: the policy kernels run on the GPU and have no CPU fallback")
    if x.shape[1] > L.POLICY_MAX_WIDTH:
        raise ValueError(f"{what}: at most 2^24 columns, got {x.shape[1]}")
    if rules is not None and not isinstance(rules, LogitRules):
        raise ValueError("rules must be a LogitRules")
    return _rowwise(x)


def _rowwise(x):
    row, column = x.stride()
    return x if (column == 1 or x.shape[1] == 1) and row >= 0 else x.contiguous()


def _empty_like(x):
    """A contiguous matrix of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _side(t, what, device, dtypes, shapes):
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{what} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the logits on {device}")
    if t.requires_grad:
        raise ValueError(f"{what} requires a gradient: only the logits have one")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {' or '.join(str(s) for s in shapes)}")
    return t if t.dim() == 0 or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


_RULES_SIZE = C.sizeof(L.LogitRules)


class LogitRules:
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

    The tensors are read when an operator runs, not copied here; values of the tensors are not checked."""

    __slots__ = ("mask", "mask_rows", "bias", "history", "history_len", "repetition", "presence", "frequency", "temperature")

    def __init__(self, *, mask=None, mask_rows=None, bias=None, history=None, history_len=None, repetition=1.0, presence=0.0, frequency=0.0,
                 temperature=1.0):
        if mask_rows is not None and mask is None:
            raise ValueError("mask_rows without a mask")
        if history_len is not None and history is None:
            raise ValueError("history_len without a history")
        for name, v in (("repetition", repetition), ("presence", presence), ("frequency", frequency), ("temperature", temperature)):
            if isinstance(v, torch.Tensor):
                continue
            v = float(v)
            if not abs(v) < 3e38 or (name == "repetition" and not v > 0.0) or (name == "temperature" and not v >= 0.0):
                raise ValueError(f"{name} must be finite{', and positive' if name == 'repetition' else ', and not negative' if name == 'temperature' else ''}; got {v}")
        self.mask, self.mask_rows, self.bias, self.history, self.history_len = mask, mask_rows, bias, history, history_len
        self.repetition, self.presence, self.frequency, self.temperature = repetition, presence, frequency, temperature

    def _tensors(self):
        return [v for v in (getattr(self, name) for name in self.__slots__) if isinstance(v, torch.Tensor)]

    def _bind(self, logits):
        """(C struct, tensors it points into) for these logits; checks every shape, type and device."""
        rows, width = logits.shape
        dev, c, keep = logits.device, L.LogitRules(_RULES_SIZE), []
        if self.mask is not None:
            words = (width + 31) // 32
            m = self.mask
            if not isinstance(m, torch.Tensor) or m.dim() != 2 or m.shape[1] < words:
                raise ValueError(f"mask must be an int32 tensor [lines, >= {words}] for {width} columns")
            if self.mask_rows is None and m.shape[0] not in (1, rows):
                raise ValueError(f"mask has {m.shape[0]} lines for {rows} rows: one, one per row, or mask_rows")
            if m.shape[0] < 1:
                raise ValueError("mask has no lines")
            m = _side(m, "mask", dev, (torch.int32,), (tuple(m.shape),))
            if m.shape[0] > 1 and m.stride(0) < words:
                m = m.contiguous()   # lines that share storage (an expanded mask)
            c.mask, c.mask_stride, c.mask_lines = m.data_ptr(), m.stride(0), m.shape[0]
            keep.append(m)
            if self.mask_rows is not None:
                t = _side(self.mask_rows, "mask_rows", dev, (torch.int32,), ((rows,),))
                c.mask_rows = t.data_ptr()
                keep.append(t)
        if self.bias is not None:
            t = _side(self.bias, "bias", dev, (torch.float32,), ((width,), (1, width), (rows, width)))
            if t.dim() == 2 and t.stride(0) < 0:
                t = t.contiguous()
            c.bias, c.bias_stride = t.data_ptr(), (t.stride(0) if t.dim() == 2 and t.shape[0] > 1 else 0)
            keep.append(t)
        if self.history is not None:
            h = self.history
            if not isinstance(h, torch.Tensor) or h.dim() != 2 or h.shape[0] != rows:
                raise ValueError(f"history must be an int32 or int64 tensor [{rows}, length]")
            h = _side(h, "history", dev, (torch.int32, torch.int64), (tuple(h.shape),))
            c.history, c.history_dtype, c.history_stride, c.history_cols = h.data_ptr() or None, _INTS[h.dtype], h.stride(0), h.shape[1]
            keep.append(h)
            if self.history_len is not None and c.history:
                t = _side(self.history_len, "history_len", dev, (torch.int32, torch.int64), ((rows,),))
                c.history_len, c.history_len_dtype = t.data_ptr(), _INTS[t.dtype]
                keep.append(t)
        for name in ("repetition", "presence", "frequency", "temperature"):
            v = getattr(self, name)
            if isinstance(v, torch.Tensor):
                t = _side(v, name, dev, (torch.float32,), ((rows,),))
                setattr(c, name + "_rows", t.data_ptr())
                keep.append(t)
            else:
                setattr(c, name, v)
        return c, keep


def pack_action_mask(allowed: torch.Tensor) -> torch.Tensor:
    """Booleans [lines, width] (True = allowed) as the int32 words [lines, ceil(width / 32)] that LogitRules takes."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError("pack_action_mask needs a 2-D bool tensor")
    lines, width = allowed.shape
    words = (width + 31) // 32
    bits = torch.nn.functional.pad(allowed, (0, 32 * words - width)).view(lines, words, 32).to(torch.int64)
    return (bits << torch.arange(32, device=allowed.device)).sum(2).to(torch.int32)   # the low 32 bits, bit 31 as the sign


def _keys(n, device, seed, step, rows):
    """(C struct, tensors it points into)"""
    if type(step) is int and type(rows) is int:
        return L.RandomKeys(_KEYS_SIZE, 0, seed & _U64, rows, step, None, None), ()
    k, keep = L.RandomKeys(_KEYS_SIZE, 0, int(seed) & _U64), []
    if isinstance(rows, torch.Tensor):
        t = _side(rows, "rows", device, (torch.int64,), ((n,),))
        k.rows = t.data_ptr()
        keep.append(t)
    else:
        k.row = int(rows)
    if isinstance(step, torch.Tensor):
        t = _side(step, "step", device, (torch.int64,), ((), (1,), (n,)))
        k.steps, k.steps_per_row = t.data_ptr(), int(t.dim() == 1 and t.shape[0] == n)
        keep.append(t)
    else:
        k.step = int(step)
    return k, keep


_KEYS_SIZE, _U64 = C.sizeof(L.RandomKeys), 0xFFFFFFFFFFFFFFFF


def _save(ctx, rules, bound, *tensors):
    """For the backward pass: the tensors (its pointers are taken from what comes back: hooks may move saved tensors), the C struct of the rules with
    what it points into, and the rules' tensors among the saved ones, so that changing one in place before it raises."""
    ctx.bound = bound
    ctx.save_for_backward(*tensors, *rules._tensors()) if rules is not None else ctx.save_for_backward(*tensors)


def _bind(rules, x):
    """None, or (C struct, the tensors it points into)"""
    return None if rules is None else rules._bind(x)


def _head(x, bound):
    """(logits, type, rows, width, stride, rules) of a C call"""
    n, width = x.shape
    return x.data_ptr(), _TYPES[x.dtype], n, width, x.stride(0), None if bound is None else C.byref(bound[0])


def _once():
    """The gradients' own kernels have no gradient: under create_graph autograd would take them for constants."""
    if torch.is_grad_enabled():
        raise RuntimeError("the policy operators are differentiable once: create_graph is not available")


class _Process(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rules):
        x = _rowwise(logits)
        bound = _bind(rules, x)
        _save(ctx, rules, bound, x)
        out = _empty_like(x)
        _call("gymhip_process_logits", x, *_head(x, bound), out.data_ptr(), out.stride(0))
        return out

    @staticmethod
    def backward(ctx, grad):
        _once()
        x, grad = _rowwise(ctx.saved_tensors[0]), _rowwise(grad)
        out = _empty_like(x)
        _call("gymhip_process_logits_backward", x, *_head(x, ctx.bound), grad.data_ptr(), grad.stride(0), out.data_ptr(), out.stride(0))
        return out, None


def process_logits(logits: torch.Tensor, rules: LogitRules | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """z (LogitRules) of logits [rows, width], rounded once to their type.  Differentiable in the logits.  `out` (not under autograd) may
    be the logits themselves, or memory that does not touch them."""
    x = _ready(logits, rules)
    if out is None:
        if logits.requires_grad and torch.is_grad_enabled():
            return _Process.apply(logits, rules)
        out = _empty_like(x)
    elif torch.is_grad_enabled() and (logits.requires_grad or out.requires_grad):
        raise ValueError("out= is not available under autograd")
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or (out.stride(1) != 1 and out.shape[1] > 1):
        raise ValueError("out must have the logits' shape, type and device, and adjacent columns")
    bound = _bind(rules, x)
    _call("gymhip_process_logits", x, *_head(x, bound), out.data_ptr(), out.stride(0))
    return out


def sample_actions(logits: torch.Tensor, rules: LogitRules | None = None, *, seed: int, step=0, rows=0, out: ActionSample | None = None) -> ActionSample:
    """One action per row of logits [rows, width] from softmax(z), and its log-probability (no gradient: score the action with
    action_log_prob for that).  The draw is a function of the row's z and of (seed, row key, step) alone: `rows` is the key of row 0 (row b
    has rows + b) or int64 [rows]; `step` is a number, an int64 device scalar (one for all rows, read when the kernel runs: advance it
    between replays of a captured graph) or int64 [rows].  Keys and steps count modulo 2^48.

    A row with nothing allowed gives action -1 and log-probability -inf, a row with a NaN or +inf among its allowed z -1 and NaN."""
    x = _ready(logits, rules)
    n, width = x.shape
    device = x.device
    if out is None:
        actions, log_prob = torch.empty(n, dtype=torch.int32, device=device), torch.empty(n, dtype=torch.float32, device=device)
    else:
        actions, log_prob = out
        _side(actions, "out.actions", device, (torch.int32,), ((n,),))
        _side(log_prob, "out.log_prob", device, (torch.float32,), ((n,),))
        if not (actions.is_contiguous() and log_prob.is_contiguous()):
            raise ValueError("out tensors must be contiguous")
    bound = _bind(rules, x)
    k, keep_keys = _keys(n, device, seed, step, rows)
    nbytes = (_lib or _load()).gymhip_sample_workspace_bytes(n, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call("gymhip_sample_actions", x, *_head(x, bound), C.byref(k), actions.data_ptr(), log_prob.data_ptr(),
          ws.data_ptr() if nbytes else None, nbytes)
    return ActionSample(actions, log_prob)


def _score(x, bound, actions):
    n, width = x.shape
    device = x.device
    nbytes = (_lib or _load()).gymhip_action_log_prob_workspace_bytes(n, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    lp, ent = torch.empty(n, dtype=torch.float32, device=device), torch.empty(n, dtype=torch.float32, device=device)
    log_sum = torch.empty(n, 2, dtype=torch.float64, device=device)
    _call("gymhip_action_log_prob", x, *_head(x, bound), actions.data_ptr(), _INTS[actions.dtype], lp.data_ptr(), ent.data_ptr(), log_sum.data_ptr(),
          ws.data_ptr() if nbytes else None, nbytes)
    return lp, ent, log_sum


class _Score(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, rules):
        ctx.set_materialize_grads(False)
        x = _rowwise(logits)
        bound = _bind(rules, x)
        lp, ent, log_sum = _score(x, bound, actions)
        _save(ctx, rules, bound, x, actions, lp, ent, log_sum)
        return lp, ent

    @staticmethod
    def backward(ctx, g_lp, g_ent):
        _once()
        x, actions, lp, ent, log_sum = ctx.saved_tensors[:5]
        x = _rowwise(x)
        out = _empty_like(x)
        g_lp, g_ent = (g if g is None or g.is_contiguous() else g.contiguous() for g in (g_lp, g_ent))
        _call("gymhip_action_log_prob_backward", x, *_head(x, ctx.bound), actions.data_ptr(), _INTS[actions.dtype], lp.data_ptr(), ent.data_ptr(),
              log_sum.data_ptr(), None if g_lp is None else g_lp.data_ptr(), None if g_ent is None else g_ent.data_ptr(),
              out.data_ptr(), out.stride(0))
        return out, None, None


def action_log_prob(logits: torch.Tensor, actions: torch.Tensor, rules: LogitRules | None = None):
    """(log softmax(z)[action], entropy of softmax(z)), float32 [rows] each, for logits [rows, width] and actions int32 / int64 [rows].
    Differentiable in the logits.  An action that is not allowed, or outside [0, width), has -inf and hands no gradient back through its
    log-probability; a row with nothing allowed has -inf, entropy 0 and no gradient."""
    x = _ready(logits, rules)
    actions = _side(actions, "actions", x.device, (torch.int32, torch.int64), ((x.shape[0],),))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Score.apply(logits, actions, rules)
    return _score(x, _bind(rules, x), actions)[:2]


def _drop(x, p, keys):
    n, width = x.shape
    out = _empty_like(x)
    _call("gymhip_dropout", x, x.data_ptr(), _TYPES[x.dtype], n, width, x.stride(0), p, C.byref(keys), out.data_ptr(), out.stride(0))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, keys, *tensors):
        ctx.p, ctx.keys, ctx.tensors = p, keys, tensors   # keys point into the tensors
        if tensors:   # a change in place before the backward pass raises
            ctx.save_for_backward(*tensors)
        return _drop(_rowwise(x), p, keys)

    @staticmethod
    def backward(ctx, grad):
        _once()
        saved = ctx.saved_tensors
        return (_drop(_rowwise(grad), ctx.p, ctx.keys),) + (None,) * (2 + len(saved))


def dropout(x: torch.Tensor, p: float, *, seed: int, step=0, rows=0) -> torch.Tensor:
    """x [rows, width] with each element 0 with probability p (p to 16 bits: t = round(65536 p)) and multiplied by 65536 / (65536 - t)
    otherwise.  Which ones follows from (seed, row key, step, column) alone (`rows` and `step` as in sample_actions); give every layer a
    seed of its own.  Differentiable in x; the backward pass draws the mask again, so a device `step` must not be advanced before it."""
    matrix = _ready(x, None, "x")
    p = float(p)
    if not 0.0 <= p < 1.0 or round(65536 * p) > 65535:
        raise ValueError(f"p must lie in [0, 1) and round to less than 65536 / 65536, got {p}")
    keys, tensors = _keys(matrix.shape[0], matrix.device, seed, step, rows)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, p, keys, *tensors)
    return _drop(matrix, p, keys)
