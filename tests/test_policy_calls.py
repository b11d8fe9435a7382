"""CPU: calls of the policy operators that the documentation allows, or has to refuse, at the edges: empty batches, numbers at the ends of float32,
tensors that carry derivatives, wrappers around envs of unknown offset."""
import ctypes as C
import math

import pytest
import torch

from gym_amd import _lib as L
from gym_amd import policy
from tests.test_policy_host import HERE, fake_venv, keys_struct, process, recorded, refused, rules_struct  # noqa: F401  (recorded is a fixture)


def test_outputs_come_in_pairs():
    x = torch.zeros(2, 4)
    for kw in (dict(log_prob=torch.zeros(2)), dict(actions=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="both actions and log_prob"):
            policy._ext.sample_actions(x, None, 1, 0, 0, **kw)


def test_forward_mode_derivatives_are_refused():
    """A tangent has no requires_grad: it is not to be dropped in silence.  What has no gradient by its definition takes such logits as it takes leaves."""
    import torch.autograd.forward_ad as fwd
    x, a = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int32)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones(2, 4))
        for call in (lambda: policy.process_logits(dual), lambda: policy.process_logits(dual, out=torch.zeros(2, 4)), lambda: policy.action_log_prob(dual, a),
                     lambda: policy.dropout(dual, 0.5, seed=1), lambda: policy.process_logits(x, out=dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        for rules in (policy.LogitRules(bias=fwd.make_dual(torch.zeros(4), torch.ones(4))), policy.LogitRules(temperature=fwd.make_dual(torch.ones(2), torch.ones(2)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                rules._bind(x)
        with pytest.raises(L.GymhipError, match="no CPU fallback"):   # not refused for its tangent
            policy.sample_actions(dual, seed=1)


# ---- empty batches ---------------------------------------------------------------------------------------------------------------------------

def per_row_rules(n, width, device="cpu", lines=None):
    """Every tensor that a rule may have, for n rows; with `lines` a table of masks, else a line a row."""
    words = (width + 31) // 32
    many = dict(history=torch.zeros(n, 3, dtype=torch.int64, device=device), history_len=torch.zeros(n, dtype=torch.int32, device=device), bias=torch.zeros(n, width, device=device))
    for name in ("repetition", "presence", "frequency", "temperature"):
        many[name] = torch.ones(n, device=device)
    many["mask"] = torch.zeros(n if lines is None else lines, words, dtype=torch.int32, device=device)
    if lines is not None:
        many["mask_rows"] = torch.zeros(n, dtype=torch.int32, device=device)
    return policy.LogitRules(**many)


@pytest.mark.parametrize("n, width", [(0, 40), (0, 0), (3, 0)])
@pytest.mark.parametrize("lines", [None, 1, 5])
def test_rules_of_an_empty_batch(n, width, lines):
    per_row_rules(n, width, lines=lines)._bind(torch.zeros(n, width))


def test_rules_of_an_empty_batch_are_checked_all_the_same():
    x = torch.zeros(0, 40)
    for bad in (dict(mask=torch.zeros(0, 1, dtype=torch.int32)), dict(bias=torch.zeros(0, 39)), dict(history=torch.zeros(2, 3, dtype=torch.int32)),
                dict(temperature=torch.ones(1)), dict(mask=torch.zeros(5, 2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            policy.LogitRules(**bad)._bind(x)


def test_abi_no_rows_is_no_work_whatever_the_rules_point_to():
    """The arrays of an empty batch may be null: no pointer of theirs stands for 'none'."""
    lib, k = L.load(), keys_struct()
    for rules in (rules_struct(mask=HERE, mask_lines=0, mask_stride=2), rules_struct(mask=HERE, mask_lines=5, mask_stride=2), rules_struct(mask_rows=HERE),
                  rules_struct(repetition=0.0), rules_struct(history_len=HERE)):
        r = C.byref(rules)
        assert process(rows=0, ptr=None, out=None, rules=rules) == 0
        assert process(rows=2, width=0, stride=0, ptr=None, out=None, out_stride=0, rules=rules) == 0
        assert lib.gymhip_process_logits_backward(None, L.TYPE_F32, 0, 8, 8, r, None, 8, None, 8, None) == 0
        assert lib.gymhip_sample_actions(None, L.TYPE_F32, 0, 8, 8, r, C.byref(k), None, None, None, 0, None) == 0
        assert lib.gymhip_action_log_prob(None, L.TYPE_F32, 0, 8, 8, r, None, L.ACT_I32, None, None, None, None, 0, None) == 0
        assert lib.gymhip_action_log_prob_backward(None, L.TYPE_F32, 0, 8, 8, r, None, L.ACT_I32, None, None, None, None, None, None, 8, None) == 0
    refused(process(rows=0, ptr=None, out=None, rules=rules_struct(struct_size=3)), "struct_size")


# ---- tensors that require a gradient ---------------------------------------------------------------------------------------------------------

def test_rules_that_are_learned():
    """Refused where their gradient would be lost, taken where there is none to lose."""
    x = torch.zeros(3, 40)
    rules = policy.LogitRules(bias=torch.zeros(40, requires_grad=True), temperature=torch.ones(3, requires_grad=True))
    with pytest.raises(ValueError, match="requires a gradient"):
        rules._bind(x)
    with torch.no_grad():
        rules._bind(x)
    with pytest.raises(ValueError, match="requires a gradient"):
        policy.LogitRules(bias=rules.bias)._bind(x)


# ---- where a wrapper's rows stand among all envs -------------------------------------------------------------------------------------------------

def test_wrappers_take_or_ask_for_the_env_offset(recorded, monkeypatch):
    """Ranks around envs of unknown offset would all draw the same: the offset is to be told then."""
    import torch.distributed as dist
    from gym_amd.vec_env import VecEnvWrapper, VecLogitActions, VecObservationDropout

    def unknown():
        venv = fake_venv()
        del type(venv).env_offset
        return VecEnvWrapper(venv)

    def key(make):
        del recorded[:]
        venv = make()
        venv.reset()
        if isinstance(venv, VecLogitActions):
            venv.step(torch.zeros(4, 2))
        return recorded[-1][3]

    assert key(lambda: VecLogitActions(unknown())) == 0 and key(lambda: VecObservationDropout(unknown(), 0.5)) == 0   # one process has all envs
    assert key(lambda: VecLogitActions(unknown(), env_offset=33)) == 33 and key(lambda: VecObservationDropout(unknown(), 0.5, env_offset=34)) == 34
    assert key(lambda: VecLogitActions(fake_venv(), env_offset=0)) == 0   # what is told wins
    # a wrapper that was told tells those around it
    assert key(lambda: VecLogitActions(VecObservationDropout(unknown(), 0.5, env_offset=34))) == 34
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda *a: 2)
    for make in (VecLogitActions, lambda v: VecObservationDropout(v, 0.5)):
        with pytest.raises(ValueError, match="env_offset"):
            make(unknown())
    assert key(lambda: VecLogitActions(unknown(), env_offset=0)) == 0 and key(lambda: VecLogitActions(fake_venv())) == 10
    monkeypatch.setattr(dist, "get_world_size", lambda *a: 1)
    assert key(lambda: VecLogitActions(unknown())) == 0


# ---- outputs that lie between the rows of an input ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows, width, stride, at", [(3, 8, 16, 7), (3, 8, 16, -7), (3, 8, 15, 8), (3, 8, 16, 9), (3, 8, 16, 16), (3, 8, 16, 1), (3, 8, 8, 8), (3, 8, 16, 39), (1, 8, 0, 7), (1, 8, 16, -7)])
def test_outputs_that_share_elements_with_an_input_are_refused(rows, width, stride, at):
    refused(process(rows=rows, width=width, stride=stride, out_stride=stride, out=HERE + 4 * at), "overlaps an input")


# ---- numbers at the ends of float32 ----------------------------------------------------------------------------------------------------------------

def test_numbers_that_float32_does_not_hold():
    for kw in (dict(temperature=1e-50), dict(temperature=7e-46), dict(temperature=1e39), dict(repetition=1e-50), dict(repetition=1e39), dict(presence=-1e39), dict(frequency=1e39)):
        with pytest.raises(ValueError, match=next(iter(kw))):
            policy.LogitRules(**kw)
    top = torch.finfo(torch.float32).max
    policy.LogitRules(temperature=top, repetition=top, presence=-top, frequency=top)._bind(torch.zeros(3, 40))
    policy.LogitRules(temperature=1e-45, repetition=1e-45, presence=1e-50, frequency=-1e-50)._bind(torch.zeros(3, 40))
    policy.LogitRules(temperature=0.0)._bind(torch.zeros(3, 40))


# ---- results that lie in what is still read --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("actions, log_prob, text", [(8, 4096, "actions overlaps"), (4096, 40, "log_prob overlaps"), (4096, 4096, "log_prob overlaps"), (4096, 4100, "log_prob overlaps"),
                                                     (-4, 4096, "actions overlaps")])
def test_drawn_results_in_the_logits_or_in_each_other_are_refused(actions, log_prob, text):
    """Other rows are read after a row's answer is written.  Two rows of 8 float32, 12 apart: 80 bytes of logits."""
    k = keys_struct()
    refused(L.load().gymhip_sample_actions(HERE, L.TYPE_F32, 2, 8, 12, None, C.byref(k), HERE + actions, HERE + log_prob, None, 0, None), text)


@pytest.mark.parametrize("log_prob, entropy, log_sum, text", [(72, 4096, 8192, "log_prob overlaps"), (4096, 0, 8192, "entropy overlaps"), (4096, 8192, 64, "log_sum overlaps"),
                                                              (4096, 4100, 8192, "entropy overlaps"), (4096, 8192, 8184, "log_sum overlaps")])
def test_scores_in_the_logits_or_in_each_other_are_refused(log_prob, entropy, log_sum, text):
    refused(L.load().gymhip_action_log_prob(HERE, L.TYPE_F32, 2, 8, 12, None, HERE, L.ACT_I32, HERE + log_prob, HERE + entropy, HERE + log_sum, None, 0, None), text)
