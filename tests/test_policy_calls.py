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
