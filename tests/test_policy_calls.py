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
