"""CPU: what the policy operators refuse, before anything could reach a GPU, and their host-side helpers."""
import ctypes as C

import numpy as np
import pytest
import torch

from gym_amd import _lib as L
from gym_amd import policy


def rules_struct(**kw):
    r = L.LogitRules(struct_size=C.sizeof(L.LogitRules), repetition=1.0, temperature=1.0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def keys_struct(**kw):
    k = L.RandomKeys(struct_size=C.sizeof(L.RandomKeys))
    for n, v in kw.items():
        setattr(k, n, v)
    return k


HERE = 1 << 20   # a non-null, aligned address that no refused call reads


def refused(rc, text):
    assert rc == 1, rc
    msg = L.load().gymhip_last_error().decode()
    assert text in msg, msg


def process(ptr=HERE, type=L.TYPE_F32, rows=2, width=8, stride=8, rules=None, out=HERE + 4096, out_stride=8):
    return L.load().gymhip_process_logits(ptr, type, rows, width, stride, None if rules is None else C.byref(rules), out, out_stride, None)


@pytest.mark.parametrize("kw, text", [
    (dict(type=7), "type must be"),
    (dict(rows=-1), "out of range"),
    (dict(width=(1 << 24) + 1, stride=1 << 25, out_stride=1 << 25), "out of range"),
    (dict(ptr=None), "logits is null"),
    (dict(out=None), "out is null"),
    (dict(stride=-8), "stride out of range"),
    (dict(stride=1 << 62), "stride out of range"),
    (dict(ptr=HERE + 2), "not aligned"),
    (dict(out=HERE + 4098), "not aligned"),
    (dict(out_stride=7), "rows overlap"),
    (dict(out=HERE + 4), "overlaps an input"),
    (dict(out=HERE, out_stride=9), "overlaps an input"),
    (dict(rules=rules_struct(struct_size=3)), "struct_size"),
    (dict(rules=rules_struct(mask=HERE, mask_lines=0, mask_stride=1)), "mask_lines"),
    (dict(rules=rules_struct(mask=HERE, mask_lines=3, mask_stride=1)), "mask_lines must be 1 or rows"),
    (dict(width=40, stride=40, out_stride=40, out=HERE + 8192, rules=rules_struct(mask=HERE, mask_lines=2, mask_stride=1)), "shorter than"),
    (dict(rules=rules_struct(mask_rows=HERE)), "without a mask"),
    (dict(rules=rules_struct(history_len=HERE)), "without a history"),
    (dict(rules=rules_struct(history=HERE, history_dtype=2, history_cols=4)), "history_dtype"),
    (dict(rules=rules_struct(history=HERE, history_cols=1 << 31)), "history size"),
    (dict(rules=rules_struct(bias=HERE, bias_stride=-1)), "bias_stride"),
    (dict(rules=rules_struct(repetition=0.0)), "repetition"),
    (dict(rules=rules_struct(repetition=float("nan"))), "repetition"),
    (dict(rules=rules_struct(temperature=-0.5)), "temperature"),
    (dict(rules=rules_struct(presence=float("inf"))), "presence"),
])
def test_abi_refuses(kw, text):
    refused(process(**kw), text)


def test_abi_refuses_the_other_entry_points():
    lib = L.load()
    k = keys_struct()
    refused(lib.gymhip_sample_actions(HERE, L.TYPE_F32, 2, 8, 8, None, None, HERE, HERE, None, 0, None), "keys")
    refused(lib.gymhip_sample_actions(HERE, L.TYPE_F32, 2, 8, 8, None, C.byref(keys_struct(struct_size=1)), HERE, HERE, None, 0, None), "keys")
    refused(lib.gymhip_sample_actions(HERE, L.TYPE_F32, 2, 8, 8, None, C.byref(k), None, HERE, None, 0, None), "actions or log_prob is null")
    refused(lib.gymhip_action_log_prob(HERE, L.TYPE_F32, 2, 8, 8, None, HERE, L.ACT_U8, HERE, HERE, HERE, None, 0, None), "action_dtype")
    refused(lib.gymhip_action_log_prob(HERE, L.TYPE_F32, 2, 8, 8, None, None, L.ACT_I32, HERE, HERE, HERE, None, 0, None), "actions is null")
    refused(lib.gymhip_action_log_prob(HERE, L.TYPE_F32, 2, 8, 8, None, HERE, L.ACT_I32, HERE, None, HERE, None, 0, None), "entropy or log_sum is null")
    refused(lib.gymhip_action_log_prob_backward(HERE, L.TYPE_F32, 2, 8, 8, None, HERE, L.ACT_I32, HERE, HERE, HERE, None, None, HERE + 8, 8, None), "overlaps")
    refused(lib.gymhip_process_logits_backward(HERE, L.TYPE_F32, 2, 8, 8, None, HERE + 4096, 8, HERE + 4100, 8, None), "overlaps")
    for p in (-0.1, 1.0, 1.0 - 2.0 ** -18, float("nan")):
        refused(lib.gymhip_dropout(HERE, L.TYPE_F32, 2, 8, 8, p, C.byref(k), HERE, 8, None), "p must lie")
    refused(lib.gymhip_dropout(HERE, L.TYPE_F32, 2, 8, 8, 0.5, None, HERE, 8, None), "keys")


def test_abi_no_rows_is_no_work():
    lib, k = L.load(), keys_struct()
    assert process(rows=0, ptr=None, out=None) == 0
    assert lib.gymhip_sample_actions(None, L.TYPE_F32, 0, 8, 8, None, C.byref(k), None, None, None, lib.gymhip_sample_workspace_bytes(0, 8), None) == 0
    assert lib.gymhip_dropout(None, L.TYPE_BF16, 0, 8, 8, 0.5, C.byref(k), None, 8, None) == 0


@pytest.mark.parametrize("kw, text", [
    (dict(mask_rows=torch.zeros(2, dtype=torch.int32)), "without a mask"),
    (dict(history_len=torch.zeros(2, dtype=torch.int32)), "without a history"),
    (dict(repetition=0.0), "repetition"), (dict(repetition=float("inf")), "repetition"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(presence=float("nan")), "presence"),
])
def test_rules_refuse(kw, text):
    with pytest.raises(ValueError, match=text):
        policy.LogitRules(**kw)


@pytest.mark.parametrize("kw, text", [
    (dict(mask=torch.zeros(2, 1, dtype=torch.int64)), "mask"),
    (dict(mask=torch.zeros(2, 1, dtype=torch.int32)), r"mask must be an int32 tensor \[lines, >= 2\]"),
    (dict(mask=torch.zeros(5, 2, dtype=torch.int32)), "5 lines"),
    (dict(mask=torch.zeros(0, 2, dtype=torch.int32), mask_rows=torch.zeros(3, dtype=torch.int32)), "no lines"),
    (dict(mask=torch.zeros(5, 2, dtype=torch.int32), mask_rows=torch.zeros(2, dtype=torch.int32)), "mask_rows has shape"),
    (dict(mask=torch.zeros(5, 2, dtype=torch.int32), mask_rows=torch.zeros(3, dtype=torch.int64)), "mask_rows must be"),
    (dict(bias=torch.zeros(39)), "bias has shape"), (dict(bias=torch.zeros(40, dtype=torch.float16)), "bias must be"),
    (dict(bias=torch.zeros(40, requires_grad=True)), "requires a gradient"),
    (dict(history=torch.zeros(2, 4, dtype=torch.int32)), "history must be"), (dict(history=torch.zeros(3, 4)), "history must be"),
    (dict(history=torch.zeros(3, 4, dtype=torch.int32), history_len=torch.zeros(4, dtype=torch.int32)), "history_len has shape"),
    (dict(temperature=torch.ones(4)), "temperature has shape"), (dict(repetition=torch.ones(3, dtype=torch.float64)), "repetition must be"),
])
def test_rules_refuse_for_these_logits(kw, text):
    with pytest.raises(ValueError, match=text):
        policy.LogitRules(**kw)._bind(torch.zeros(3, 40))


def test_rules_accept_every_documented_form():
    r = policy.LogitRules(mask=torch.zeros(1, 2, dtype=torch.int32).expand(3, 2), bias=torch.zeros(3, 80)[:, ::2], history=torch.zeros(3, 0, dtype=torch.int64),
                          history_len=torch.zeros(3, dtype=torch.int64), temperature=torch.ones(6)[::2])
    c, keep = r._bind(torch.zeros(3, 40))
    assert c.mask_stride == 2 and c.bias_stride == 40 and not c.history   # copies where the kernels need adjacent words; an empty history is none
    c, keep = policy.LogitRules(bias=torch.zeros(1, 40).expand(3, 40))._bind(torch.zeros(3, 40))
    assert c.bias_stride == 0


def test_no_cpu_fallback_and_shapes():
    with pytest.raises(L.GymhipError, match="no CPU fallback"):
        policy.sample_actions(torch.zeros(2, 4), seed=1)
    with pytest.raises(L.GymhipError, match="no CPU fallback"):
        policy.dropout(torch.zeros(2, 4), 0.5, seed=1)
    with pytest.raises(ValueError, match="2-D"):
        policy.process_logits(torch.zeros(4))
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        policy.action_log_prob(torch.zeros(2, 4, dtype=torch.float64), torch.zeros(2, dtype=torch.int32))


def test_pack_action_mask():
    g = torch.Generator().manual_seed(1)
    for width in (1, 31, 32, 33, 100):
        allowed = torch.rand(5, width, generator=g) < 0.5
        words = policy.pack_action_mask(allowed)
        assert words.dtype == torch.int32 and words.shape == (5, (width + 31) // 32)
        w = words.numpy().view(np.uint32)
        back = (w[:, np.arange(width) // 32] >> (np.arange(width) % 32).astype(np.uint32)) & 1
        assert np.array_equal(back.astype(bool), allowed.numpy())
    with pytest.raises(ValueError):
        policy.pack_action_mask(torch.zeros(2, 3))


def test_struct_layouts_match_ctypes(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prog = tmp_path / "layout.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gymhip.h"\nint main(){printf("%zu %zu %zu %zu %zu %zu\\n",'
                    'sizeof(gymhip_logit_rules), offsetof(gymhip_logit_rules,history), offsetof(gymhip_logit_rules,temperature),'
                    'sizeof(gymhip_random_keys), offsetof(gymhip_random_keys,row), offsetof(gymhip_random_keys,steps));return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(prog), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(L.LogitRules), L.LogitRules.history.offset, L.LogitRules.temperature.offset, C.sizeof(L.RandomKeys),
                   L.RandomKeys.row.offset, L.RandomKeys.steps.offset]


def test_reference_generator_known_answers():
    """The generator's rounds against the published definition, worked by hand for one round of counter (1, 2, 3, 4), key 5 + 6 * 2^32, and
    uniformity of what the operators take from it: 16-bit lanes' mean within 5 standard errors."""
    from tests import policy_reference as R
    a, b = 1 * 0xD2511F53, 3 * 0xCD9E8D57
    one = [(b >> 32) ^ 2 ^ 5, b & R.LOW, (a >> 32) ^ 4 ^ 6, a & R.LOW]
    c, k = [1, 2, 3, 4], [5, 6]
    for r in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & R.LOW, (a >> 32) ^ c[3] ^ k[1], a & R.LOW]
        k = [(k[0] + 0x9E3779B9) & R.LOW, (k[1] + 0xBB67AE85) & R.LOW]
        if r == 0:
            assert c == one
    got = R.words(1, 2 | 4 << 32, 3, 5 | 6 << 32)   # row 2 + 4 * 2^32, step 3
    assert [int(v) for v in got] == c
    keep = R.kept(64, 1000, 0.25, 99)
    rate = keep.double().mean().item()
    assert abs(rate - 0.75) < 5 * (0.25 * 0.75 / 64000) ** 0.5
    u = R.uniforms(4000, 7)
    assert 0 < u.min() and u.max() < 1 and abs(u.mean().item() - 0.5) < 5 * (1 / 12 / 4000) ** 0.5


# ---- the VecEnv wrappers' host side ------------------------------------------------------------------------------------------------------

def fake_venv(n=4, a_space=None, offset=10):
    from gym_amd import spaces
    from gym_amd.vec_env import VecEnv, VecEnvStepReturn

    class Fake(VecEnv):
        env_offset = offset

        def reset(self, index=None):
            return torch.ones(n, 3) if index is None else torch.ones(3)

        def stepAsync(self, actions):
            self.actions = actions

        def stepWait(self):
            return VecEnvStepReturn(torch.ones(n, 3), torch.zeros(n, 1), torch.zeros(n, 1), [])

        def seed(self, s):
            return [s + i for i in range(n)]

    o, a = spaces.cartpole_spaces()
    return Fake(n, o, a_space or a)


@pytest.fixture
def recorded(monkeypatch):
    """Calls of the operators in place of the kernels."""
    calls = []

    def sample(logits, rules=None, *, seed, step=0, rows=0, out=None):
        calls.append(("sample", seed, int(step), rows, rules))
        return policy.ActionSample(torch.zeros(logits.shape[0], dtype=torch.int32), torch.zeros(logits.shape[0]))

    def drop(x, p, *, seed, step=0, rows=0):
        calls.append(("drop", seed, int(step), rows, tuple(x.shape)))
        return x * 2

    monkeypatch.setattr(policy, "sample_actions", sample)
    monkeypatch.setattr(policy, "dropout", drop)
    return calls


@pytest.mark.parametrize("device_step", [False, True])
def test_wrappers_key_their_draws_by_seed_global_row_and_step(recorded, device_step):
    from gym_amd.vec_env import VecLogitActions, VecObservationDropout
    inner = fake_venv()
    venv = VecLogitActions(VecObservationDropout(inner, 0.25, seed=5, device_step=device_step), seed=6, device_step=device_step)
    assert (venv.reset() == 2).all()
    rules = policy.LogitRules(temperature=0.5)
    for t in range(2):
        r = venv.step(torch.zeros(4, 2))
        assert (r.observation == 2).all() and inner.actions is venv.sample.actions
        venv.rules = rules
    assert (venv.reset(3) == 2).all() and venv.reset(3).shape == (3,)
    assert recorded == [("drop", 5, 0, 10, (4, 3)), ("sample", 6, 0, 10, None), ("drop", 5, 1, 10, (4, 3)), ("sample", 6, 1, 10, rules),
                        ("drop", 5, 2, 10, (4, 3)), ("drop", 5, 3 + (1 << 47), 13, (1, 3)), ("drop", 5, 3 + (1 << 47), 13, (1, 3))]
    del recorded[:]
    assert venv.seed(40) == [40, 41, 42, 43]   # the envs' seeds; the draws start again under the new one
    venv.reset()
    venv.venv.training = False
    assert (venv.step(torch.zeros(4, 2)).observation == 1).all() and (venv.reset(0) == 1).all()
    venv.venv.training = True
    venv.step(torch.zeros(4, 2))
    assert recorded == [("drop", 40, 0, 10, (4, 3)), ("sample", 40, 0, 10, rules), ("sample", 40, 1, 10, rules), ("drop", 40, 2, 10, (4, 3))]


def test_wrappers_refuse(recorded):
    from gym_amd import spaces
    from gym_amd.vec_env import VecLogitActions, VecObservationDropout
    with pytest.raises(TypeError, match="Discrete"):
        VecLogitActions(fake_venv(a_space=spaces.makeBoxSpace(3)))
    for p in (-0.1, 1.0, float("nan"), 1.0 - 2.0 ** -18):
        with pytest.raises(ValueError, match="p must lie"):
            VecObservationDropout(fake_venv(), p)
    venv = VecLogitActions(fake_venv())
    venv.reset()
    for shape in ((4, 3), (3, 2), (4,), (4, 2, 1)):
        with pytest.raises(ValueError, match="logits have shape"):
            venv.step(torch.zeros(shape))
    assert recorded == [] and venv.sample is None


def test_wrappers_have_no_cpu_fallback():
    from gym_amd.vec_env import VecLogitActions, VecObservationDropout
    with pytest.raises(L.GymhipError, match="no CPU fallback"):
        VecLogitActions(fake_venv()).step(torch.zeros(4, 2))
    with pytest.raises(L.GymhipError, match="no CPU fallback"):
        VecObservationDropout(fake_venv(), 0.5).reset()


def test_binding_refuses_other_python_types():
    for bad in (lambda: policy.process_logits([1.0]), lambda: policy.sample_actions(torch.zeros(2, 4), seed="a"), lambda: policy.dropout(torch.zeros(2, 4), 0.5, seed=1, step=None),
                lambda: policy.LogitRules(mask=[1]), lambda: policy.LogitRules(temperature="hot")):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(ValueError, match="rules must be"):
        policy.process_logits(torch.zeros(2, 4), {})
    r = policy.LogitRules(temperature=0.5)
    assert r.temperature == 0.5 and r.mask is None and r.repetition == 1.0
    r.temperature = t = torch.ones(3)
    assert r.temperature is t
    r.temperature = -1.0   # assigned later, refused when used
    with pytest.raises(ValueError, match="temperature"):
        r._bind(torch.zeros(3, 4))
