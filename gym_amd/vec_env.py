"""Host-side mirror of the reference's vectorised-env interface for the hot path.

Same names, argument meaning and error behaviour as the C++ templates it stands in for:

    gym::VecEnv<false>                 wrappers/vec_env/base.h:30-79
    gym::VecEnvWrapper<false>          wrappers/vec_env/vec_env_wrapper.h:12-55
    gym::SyncVecEnv<Monitor<ClipRewardEnv<TimeLimit<Env>>>>   wrappers/vec_env/sync_env.h  -> HipVecEnv
    gym::VecNormalize<false, training, normReward, normObs>   wrappers/vec_env/vec_normalize.h -> VecNormalize
    gym::VecFrameStack / VecNormAndPermute                     vec_frame_stack.cpp, vec_atari.cpp -> gym_amd.atari

VecLogitActions (step takes a policy's logits) and VecObservationDropout have no counterpart there: the reference leaves both to its trainer.

The per-env wrappers are not objects here: TimeLimit / ClipReward / Monitor (and VecNormalize) are flags of ONE fused
kernel.  Returned tensors are views of device buffers that the next step overwrites (the reference allocates fresh
tensors every step, sync_env.h:107-112) — clone what you keep.
"""
from __future__ import annotations

import os
import time
from typing import NamedTuple

import numpy as np
import torch

from . import _lib as L
from . import spaces
from .engine import Engine, EngineConfig

_ENV_IDS = {"CartPole": L.ENV_CARTPOLE, "CartPole-v1": L.ENV_CARTPOLE, "MountainCar": L.ENV_MOUNTAINCAR, "MountainCar-v0": L.ENV_MOUNTAINCAR}


class VecEnvStepReturn(NamedTuple):
    """base.h:18-25: observation [N, F] f32, reward [N, 1] f32, done [N, 1] f32 (0/1), info (one map per env)."""
    observation: torch.Tensor
    reward: torch.Tensor
    done: torch.Tensor
    info: "LazyInfos"


class LazyInfos:
    """vector<AnyMap> info (base.h:24) built on demand: N unordered_maps per step are the reference's host bottleneck at
    large N, so maps are materialised only when indexed, and only finished envs have entries:
    info[i]["episode"] = {"r", "l", "t"} (monitor.h:86-97), info[i]["TimeLimit.truncated"] (time_limit.h:32).

    The reference hands out concrete per-step maps (sync_env.h:101,111); this object reads the engine's buffers on first
    use, so it is only valid until the engine steps again.  It is stamped with the engine's step count at creation and
    RAISES if indexed after a later step (a rollout buffer that keeps `step().info` must read it, or call `.materialize()`,
    before the next step)."""

    def __init__(self, venv: "HipVecEnv"):
        self._venv = venv
        self._host = None
        self._stamp = venv._steps_taken
        self._t = time.perf_counter() - venv._t_start

    def __len__(self):
        return self._venv.numEnvs

    def _fetch(self):
        if self._host is None:
            v = self._venv
            if v._steps_taken != self._stamp:
                raise RuntimeError("this step's info was not read before the next step(): the engine's episode records have been "
                                   "overwritten (read info, or call info.materialize(), before stepping again)")
            ln, tr, ret = v.engine.episode_info()
            done = v.engine.done
            self._host = dict(done=done.cpu().numpy() != 0, length=ln.cpu().numpy(), truncated=tr.cpu().numpy() != 0, ret=ret.cpu().numpy(), t=self._t)
        return self._host

    def materialize(self):
        """Copy this step's records to the host now; the object then stays valid across later steps."""
        self._fetch()
        return self

    def done_indices(self):
        return np.nonzero(self._fetch()["done"])[0]

    def __getitem__(self, i):
        h = self._fetch()
        if i < 0 or i >= len(self):
            raise IndexError(i)
        if not h["done"][i]:
            return {}
        d = {}
        v = self._venv
        if v._wrappers & L.WRAP_TIME_LIMIT:
            d["TimeLimit.truncated"] = bool(h["truncated"][i])
        if v._wrappers & L.WRAP_MONITOR:
            d["episode"] = {"r": float(h["ret"][i]), "l": float(h["length"][i]), "t": h["t"]}
        return d


class VecEnv:
    """gym::VecEnv<false> (base.h:30-79)."""

    def __init__(self, numEnvs: int, o_space, a_space):
        self.numEnvs = int(numEnvs)
        self._o_space, self._a_space = o_space, a_space

    def actionSpace(self):
        return self._a_space

    def observationSpace(self):
        return self._o_space

    def nEnvs(self):
        return self.numEnvs

    def reset(self, index=None):
        raise NotImplementedError

    def stepAsync(self, actions):
        raise NotImplementedError

    def stepWait(self) -> VecEnvStepReturn:
        raise NotImplementedError

    def step(self, actions) -> VecEnvStepReturn:   # base.h:60-63
        self.stepAsync(actions)
        return self.stepWait()

    def isWrapper(self):
        return False

    def render(self):
        raise NotImplementedError("rendering is outside the batched engine (SURVEY.md §2 row 35)")

    def seed(self, _seed: int):
        return []


def allreduce_sum(t: torch.Tensor, group=None):
    """SUM all-reduce of a small device tensor in place.  Backend nccl (= RCCL over xGMI): directly on the device tensor,
    ordered on the current stream.  Any other backend (gloo: CPU tests and 1-GPU rehearsals) is staged through the host —
    gloo's own CUDA path deadlocked on repeated calls on the MI355X box."""
    import torch.distributed as dist
    if dist.get_backend(group) == "nccl":
        dist.all_reduce(t, group=group)
    else:
        h = t.cpu()
        dist.all_reduce(h, group=group)
        t.copy_(h)
    return t


def shard_range(n_global: int, rank: int, world: int):
    """GPU g of G owns the contiguous env range [g*N/G, (g+1)*N/G); seeds follow the GLOBAL index."""
    lo = (n_global * rank) // world
    hi = (n_global * (rank + 1)) // world
    return lo, hi


class HipVecEnv(VecEnv):
    """Drop-in for SyncVecEnv over N CartPole / MountainCar envs with their per-env wrapper chain, on one MI355X.

    `n_envs` is the GLOBAL env count; with `world` > 1 this process holds shard `rank` of it (one process per GPU) and
    env i is still seeded `seed + i` with i the global index, so results do not depend on the GPU count.
    """

    def __init__(self, env_id: str, n_envs: int, max_episode_steps: int | None = None, clip_reward: bool = False, monitor: bool = True,
                 lockstep: bool = True, reset_mode: str | None = None, tape_episodes: int | None = None, device: int | None = None,
                 rank: int | None = None, world: int | None = None, process_group=None, auto_reset: bool = True, exchange: str = "moments"):
        if env_id not in _ENV_IDS:
            raise ValueError(f"unknown env id {env_id!r}; the engine implements {sorted(_ENV_IDS)}")
        if exchange not in ("moments", "rows"):
            raise ValueError("exchange must be 'moments' (reduce launch + 2F+6 doubles) or 'rows' (the partial rows themselves, no reduce launch)")
        self._exchange = exchange   # sharded runs with the normaliser on: what the ranks all-reduce per step (gymhip_set_exchange_form)
        self._auto_reset = bool(auto_reset)   # SyncVecEnv(envs, auto_reset) (sync_env.h:28,44): off = finished envs wait for reset(index)
        self.kind = _ENV_IDS[env_id]
        self.rank = int(os.environ.get("RANK", 0)) if rank is None else rank
        self.world = int(os.environ.get("WORLD_SIZE", 1)) if world is None else world
        self.group = process_group
        self.n_global = int(n_envs)
        lo, hi = shard_range(self.n_global, self.rank, self.world)
        o_space, a_space = spaces.cartpole_spaces() if self.kind == L.ENV_CARTPOLE else spaces.mountaincar_spaces()
        super().__init__(hi - lo, o_space, a_space)
        self.env_offset = lo
        self._wrappers = ((L.WRAP_TIME_LIMIT if max_episode_steps else 0) | (L.WRAP_CLIP_REWARD if clip_reward else 0) | (L.WRAP_MONITOR if monitor else 0) |
                          (0 if auto_reset else L.WRAP_NO_AUTO_RESET))
        self._max_steps = int(max_episode_steps or 0)
        self._lockstep = lockstep
        # CartPole's reset source: "mt19937" (default) = every env's std::mt19937 on the device — the reference's own streams, for ever,
        # no host work; "tape" (or a given tape_episodes) = the same streams drawn on the host into a finite tape that is extended on
        # demand; "rng" = stateless counter RNG (same distribution, not the reference's stream)
        if reset_mode is None:
            reset_mode = "tape" if tape_episodes is not None else "mt19937"
        if reset_mode not in ("mt19937", "tape", "rng"):
            raise ValueError(f"reset_mode {reset_mode!r}: expected 'mt19937', 'tape' or 'rng'")
        self._reset_mode = L.RESET_COUNTER_RNG if (reset_mode == "rng" or self.kind != L.ENV_CARTPOLE) else (L.RESET_TAPE if reset_mode == "tape" else L.RESET_MT19937)
        # Host-drawn reset tape: start with at most 256 MiB of rows (16 B each), at least 8 and at most 2048 per env; the tape
        # guard below extends it (same streams, twice the rows) before any env can run out.
        if tape_episodes is None:
            tape_episodes = int(min(2048, max(8, (256 << 20) // (16 * max(1, hi - lo)))))
        self._tape_episodes = int(tape_episodes)
        self._steps_taken = 0
        self._tape_budget = 0      # VecEnv steps that may still be taken before the tape cursors must be looked at again
        self._device = int(os.environ.get("LOCAL_RANK", 0)) if device is None else device
        self._norm = None          # set by VecNormalize before the engine exists
        self._seed = None          # unseeded envs keep default-constructed mt19937 (seed 5489) — identical streams
        self.engine: Engine | None = None
        self._actions = None
        self._t_start = time.perf_counter()

    @staticmethod
    def make(*args, **kw):   # factory idiom of the reference (sync_env.h:62-64)
        return HipVecEnv(*args, **kw)

    # -- engine construction is deferred so that VecNormalize can fuse itself in -------------------------------
    def _ensure_engine(self):
        if self.engine is not None:
            return
        w = self._wrappers
        kw = {}
        if self._norm is not None:
            nm = self._norm
            w |= (L.WRAP_NORM_OBS if nm["norm_obs"] else 0) | (L.WRAP_NORM_REWARD if nm["norm_reward"] else 0) | (L.WRAP_NORM_TRAINING if nm["training"] else 0)
            kw = dict(clip_obs=nm["clip_obs"], clip_reward=nm["clip_reward"], gamma=nm["gamma"], epsilon=nm["epsilon"])
        cfg = EngineConfig(env_kind=self.kind, n_envs=self.numEnvs, precision=L.PRECISION_LOCKSTEP_F64 if self._lockstep else L.PRECISION_F32,
                           reset_mode=self._reset_mode, wrappers=w, max_episode_steps=self._max_steps, env_offset=self.env_offset,
                           seed=self._seed if self._seed is not None else 0, **kw)
        self.engine = Engine(cfg, self._device)
        if self._exchange == "rows" and self._has_norm() and self.world > 1:
            self.engine.set_exchange_form(L.EXCHANGE_ROWS)
        if self._reset_mode == L.RESET_TAPE:
            if self._seed is None:
                # every unseeded reference env draws from the same default stream: one row set, replicated
                self.engine.seed_reset_tape_unseeded(self._tape_episodes)
            else:
                self.engine.seed_reset_tape(self._seed, self._tape_episodes)
            self._tape_budget = self._tape_steps_for(self._tape_episodes)
        elif self._reset_mode == L.RESET_MT19937 and self._seed is not None:
            self.engine.seed(self._seed)   # never seeded = default-constructed generators, as in the reference

    # -- reset-tape guard ------------------------------------------------------------------------------------------
    # An env consumes one tape row per finished episode (and per reset).  No CartPole episode is shorter than 8 steps
    # (enumerated over the corners of the reset box x every action sequence; cartpole.cpp:19-68) or than TimeLimit's bound,
    # so with r rows left for the env that has consumed most, 8 r - 8 further steps cannot exhaust the tape.  When that budget
    # is spent the cursors are looked at again (one 4-byte read-back) and, with less than a quarter of the rows left, the
    # tape is redrawn from the same std::mt19937 streams with twice the rows.  The kernel's wrap-around (error bit 0) is thus
    # never reached; it is still checked and raised.
    def _min_episode_steps(self):
        return max(1, min(8, self._max_steps) if (self._wrappers & L.WRAP_TIME_LIMIT) else 8)

    def _tape_steps_for(self, rows_left):
        return max(0, self._min_episode_steps() * (rows_left - 1))

    def _tape_spend(self, steps):
        if self._reset_mode != L.RESET_TAPE or self.engine is None:
            return
        self._tape_budget -= steps
        if self._tape_budget > 0:
            return
        e = self.engine
        if e.poll_error() & 1:
            raise RuntimeError("reset tape exhausted: an env replayed old reset states (gymhip error bit 0)")
        used = e.tape_cursor_max()
        if self._tape_episodes - used < max(8, self._tape_episodes // 4):
            self._tape_episodes = max(2 * self._tape_episodes, used + 16)
            e.extend_reset_tape(self._tape_episodes)
        self._tape_budget = self._tape_steps_for(self._tape_episodes - used)

    def _has_norm(self):
        return self._norm is not None and (self._norm["norm_obs"] or self._norm["norm_reward"])

    def _allreduce_moments(self):
        if self.world > 1:
            allreduce_sum(self.engine.moments, self.group)   # RCCL: 2F+6 doubles, latency-bound

    # -- VecEnv interface ------------------------------------------------------------------------------------------
    def seed(self, _seed: int):
        """sync_env.h:74-83: env i <- _seed + i; returns the per-env seeds of this shard."""
        self._seed = int(_seed)
        if self.engine is not None:   # mid-run re-seed: every env's generator restarts (env.h:60-63); the tape is redrawn, cursors rewound
            if self._reset_mode == L.RESET_TAPE:
                self.engine.seed_reset_tape(self._seed, self._tape_episodes)
                self._tape_budget = self._tape_steps_for(self._tape_episodes)
            else:
                self.engine.seed(self._seed)
        return [self._seed + self.env_offset + i for i in range(self.numEnvs)] if self.numEnvs <= 1 << 20 else range(
            self._seed + self.env_offset, self._seed + self.env_offset + self.numEnvs)

    def reset(self, index=None):
        if index is not None:
            # sync_env.h:128-139 (+ vec_normalize.h:179-189 when the normaliser is fused in): one env, returns its row
            if self.engine is None:
                raise RuntimeError("reset(index) before reset()")
            if not 0 <= int(index) < self.numEnvs:
                raise IndexError(f"env index {index} out of range [0, {self.numEnvs})")
            self._tape_spend(self._min_episode_steps())   # a reset consumes a tape row, like one shortest-possible episode
            self.engine.reset_index(int(index))
            e = self.engine
            return (e.obs_norm if (self._norm and self._norm["norm_obs"]) else e.obs)[int(index)]
        self._ensure_engine()
        e = self.engine
        self._tape_spend(self._min_episode_steps())
        if self._has_norm() and self.world > 1:   # sharded: the batch moments are all-reduced between the two halves of the call
            e.reset_begin()
            self._allreduce_moments()
            e.reset_finish()
        else:
            e.reset()
        return e.obs_norm if (self._norm and self._norm["norm_obs"]) else e.obs

    def stepAsync(self, actions):
        self._actions = actions   # tensor_adapter.cpp:22-23: decoded to int32 at launch if not already an integer device tensor

    def stepWait(self) -> VecEnvStepReturn:
        if self.engine is None:
            raise RuntimeError("stepWait() before reset()")
        if self._actions is None:
            raise RuntimeError("stepWait() without stepAsync()")
        e = self.engine
        self._tape_spend(1)
        self._steps_taken += 1
        if self._has_norm() and self.world > 1:
            e.step_begin(self._actions)
            self._allreduce_moments()
            e.step_finish()
        else:
            e.step(self._actions)   # single GPU: no exchange, one launch fewer (the normalise kernel folds the partial rows)
        self._actions = None
        obs = e.obs_norm if (self._norm and self._norm["norm_obs"]) else e.obs
        return VecEnvStepReturn(obs, e.reward.view(-1, 1), e.done.view(-1, 1), LazyInfos(self))

    def episode_statistics(self):
        """(episodes, sum of returns, sum of lengths) over ALL shards — Monitor getters in aggregate (monitor.h:104-107)."""
        tot = torch.from_numpy(self.engine.episode_stats()).to(self.engine.device)
        if self.world > 1:
            allreduce_sum(tot, self.group)
        return tot.cpu().numpy()


class VecEnvWrapper(VecEnv):
    """gym::VecEnvWrapper<false> (vec_env_wrapper.h:12-55): forwards everything to `venv`."""

    def __init__(self, venv: VecEnv, o_space=None, a_space=None):
        super().__init__(venv.nEnvs(), o_space or venv.observationSpace(), a_space or venv.actionSpace())
        self.venv = venv

    # isWrapper() is NOT overridden: nothing in the reference overrides base.h:65, a VecEnvWrapper reports false there too

    def reset(self, index=None):
        return self.venv.reset(index)

    def stepAsync(self, actions):
        self.venv.stepAsync(actions)

    def stepWait(self):
        return self.venv.stepWait()

    def seed(self, _seed):
        return self.venv.seed(_seed)


def _env_offset(venv, told=None):
    """The global index of the first env under any wrappers, the random-number key of row 0: as told, else what the VecEnv says of itself.  One that says
    nothing has all envs if it is the only process; of several ranks each would draw the same, so there it must be told."""
    if told is not None:
        return int(told)
    while not hasattr(venv, "env_offset") and hasattr(venv, "venv"):
        venv = venv.venv
    if not hasattr(venv, "env_offset"):
        import torch.distributed as dist
        if dist.is_available() and dist.is_initialized() and dist.get_world_size() > 1:
            raise ValueError(f"{type(venv).__name__} has no env_offset: with {dist.get_world_size()} ranks pass env_offset=, the global index of this rank's first env")
    return int(getattr(venv, "env_offset", 0))


class _Counter:
    """The step number of the random draws: on the host, or (device=True) an int64 scalar on the GPU that the stream itself advances, so that a
    recorded graph draws anew at every replay (one more launch per step)."""

    def __init__(self, device: bool):
        self._on_device, self.value = bool(device), 0

    def restart(self):
        if isinstance(self.value, torch.Tensor):
            self.value.zero_()   # in place: a recorded graph goes on with the same scalar
        else:
            self.value = 0

    def on(self, device):
        """The number to draw with, for tensors on `device`."""
        if device.type == "cuda" and not isinstance(self.value, torch.Tensor) and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a recorded graph would draw the same at every replay: make the wrapper with device_step=True and take a step before recording"
                               if not self._on_device else "take a step before recording")
        if self._on_device and not isinstance(self.value, torch.Tensor):
            self.value = torch.full((), self.value, dtype=torch.int64, device=device)
        return self.value

    def advance(self):
        if isinstance(self.value, torch.Tensor):
            self.value.add_(1)
        else:
            self.value += 1


class VecLogitActions(VecEnvWrapper):
    """step(logits [N, n]) over a VecEnv with a Discrete(n) action space: one action per env from softmax(logits) under `rules`
    (gym_amd.policy.LogitRules; may be assigned between steps) is drawn on the GPU and handed to the engine as it is (int32, no copy).

    The draw of env i at step t follows from (seed, i's GLOBAL index, t) alone: neither the GPU count nor the order of the calls matters.
    seed(s) gives the envs their seeds and the draws a new one, and restarts t.  `sample` holds the last step's actions and log-probabilities
    (new tensors each step); action_log_prob scores them again, with gradients.  An env whose rules leave nothing to choose gets action -1.
    device_step=True keeps t on the GPU, for steps recorded into a graph.  env_offset: the global index of env 0, for a VecEnv that has no such
    attribute (needed with more than one rank)."""

    def __init__(self, venv: VecEnv, rules=None, seed: int = 0, device_step: bool = False, env_offset: int | None = None):
        super().__init__(venv)
        if not isinstance(venv.actionSpace(), spaces.Discrete):
            raise TypeError(f"VecLogitActions needs a Discrete action space, got {venv.actionSpace()!r}")
        self.rules, self.sample, self.env_offset = rules, None, _env_offset(venv, env_offset)
        self._seed, self._step = int(seed), _Counter(device_step)

    def seed(self, _seed):
        self._seed = int(_seed)
        self._step.restart()
        return self.venv.seed(_seed)

    def stepAsync(self, logits):
        from . import policy
        shape = (self.numEnvs, self.actionSpace().n)
        if tuple(logits.shape) != shape:
            raise ValueError(f"logits have shape {tuple(logits.shape)}, expected {shape}")
        self.sample = policy.sample_actions(logits, self.rules, seed=self._seed, step=self._step.on(logits.device), rows=self.env_offset)
        self._step.advance()
        self.venv.stepAsync(self.sample.actions)


class VecObservationDropout(VecEnvWrapper):
    """Every feature of every observation is 0 with probability p, else divided by 1 - p (gym_amd.policy.dropout: p to 16 bits), for float32,
    float16 and bfloat16 observations of any shape.  The observations are new tensors; what the venv returned stays as it was.

    What is dropped for env i in the t-th observation since seed(s) follows from (seed, i's GLOBAL index, t) alone.  reset(index) has masks
    of its own and leaves t as it is.  training = False passes the observations on untouched (t goes on all the same).
    device_step=True keeps t on the GPU, for steps recorded into a graph.  env_offset as for VecLogitActions."""

    def __init__(self, venv: VecEnv, p: float, seed: int = 0, device_step: bool = False, env_offset: int | None = None):
        super().__init__(venv)
        p = float(p)
        if not 0.0 <= p < 1.0 or round(65536 * p) > 65535:
            raise ValueError(f"p must lie in [0, 1) and round to less than 65536 / 65536, got {p}")
        self.p, self.training, self.env_offset = p, True, _env_offset(venv, env_offset)
        self._seed, self._step = int(seed), _Counter(device_step)

    def seed(self, _seed):
        self._seed = int(_seed)
        self._step.restart()
        return self.venv.seed(_seed)

    def _drop(self, obs, rows, step):
        from . import policy
        n = obs.shape[0]
        return policy.dropout(obs.reshape(n, -1), self.p, seed=self._seed, step=step, rows=rows).view(obs.shape)

    def _next(self, obs):
        step = self._step.on(obs.device)
        if self.training:
            obs = self._drop(obs, self.env_offset, step)
        self._step.advance()
        return obs

    def reset(self, index=None):
        if index is None:
            return self._next(self.venv.reset())
        obs = self.venv.reset(index)
        # the number of the next observation, in the upper half of the steps' 48 bits, which the count does not reach
        return self._drop(obs.unsqueeze(0), self.env_offset + int(index), self._step.on(obs.device) + (1 << 47)).squeeze(0) if self.training else obs

    def stepWait(self):
        r = self.venv.stepWait()
        return r._replace(observation=self._next(r.observation))


class Updater:
    """updateable.h:16-31: the observer a learner holds; `subscribe` appends, `notifyOne` tells only the FIRST subscriber."""

    def __init__(self):
        self._updateables = []

    def subscribe(self, sub):
        if sub is None or not callable(getattr(sub, "update", None)):
            raise ValueError("Updater.subscribe needs an object with update(...)")   # the reference asserts a non-null pointer
        self._updateables.append(sub)

    def notifyOne(self, *args):
        if self._updateables:
            self._updateables[0].update(*args)


class VecNormalize(VecEnvWrapper):
    """gym::VecNormalize<false, isTraining, normReward, normObs> (vec_normalize.h:20-232); TrainingVecNormRO =
    VecNormalize(venv) with the defaults (gym_.h:15-16).  Must wrap a HipVecEnv before its first reset: the
    normaliser runs inside the env's own kernels."""

    def __init__(self, venv: HipVecEnv, clip_obs: float = 10.0, clip_reward: float = 10.0, gamma: float = 0.99, epsilon: float = 1e-8,
                 training: bool = True, norm_reward: bool = True, norm_obs: bool = True):
        if not isinstance(venv, HipVecEnv):
            raise TypeError("VecNormalize fuses into a HipVecEnv; got " + type(venv).__name__)
        if venv.engine is not None:
            raise RuntimeError("wrap the HipVecEnv in VecNormalize before its first reset()")
        super().__init__(venv)
        venv._norm = dict(clip_obs=clip_obs, clip_reward=clip_reward, gamma=gamma, epsilon=epsilon, training=training,
                          norm_reward=norm_reward, norm_obs=norm_obs)

    def oldObs(self):
        """vec_normalize.h:94: the un-normalised observations of the last reset/step."""
        return self.venv.engine.obs

    def update(self, state: torch.Tensor | None, reward: torch.Tensor | None):
        """Updateable::update (vec_normalize.h:191-206): a learner pushes rollout tensors — state [T, N, F] (flattened over
        the first two dims, :197) and reward (reshaped to [-1, 1], :204) — into the running statistics."""
        self.venv._ensure_engine()
        self.venv.engine.update_norm_stats(state, reward)

    def get(self):
        """vec_normalize.h:75-77: (obs RMS, return RMS) as dicts of mean / m_Var / m_Count (running_mean_std.h:17-19)."""
        s = self.venv.engine.get_norm_stats()
        F = self.venv.engine.F
        return (dict(mean=s[:F].copy(), m_Var=s[F:2 * F].copy(), m_Count=float(s[2 * F])),
                dict(mean=float(s[2 * F + 1]), m_Var=float(s[2 * F + 2]), m_Count=float(s[2 * F + 3])))

    def save(self, path):
        """vec_normalize.h:79-92: returns.pt + observation.pt in the reference's own archive format (gym_amd/checkpoint.py)."""
        from .checkpoint import save_running_mean_std
        os.makedirs(path, exist_ok=True)
        obs, ret = self.get()
        if self.venv._norm["norm_reward"]:
            save_running_mean_std(os.path.join(path, "returns.pt"), np.float32(ret["mean"]), np.float32(ret["m_Var"]), ret["m_Count"])
        if self.venv._norm["norm_obs"]:
            save_running_mean_std(os.path.join(path, "observation.pt"), obs["mean"], obs["m_Var"], obs["m_Count"])

    def load(self, path):
        """vec_normalize.h:96-108."""
        from .checkpoint import load_running_mean_std
        self.venv._ensure_engine()
        e = self.venv.engine
        s = e.get_norm_stats()
        F = e.F
        if self.venv._norm["norm_reward"]:
            mean, var, cnt = load_running_mean_std(os.path.join(path, "returns.pt"))
            s[2 * F + 1], s[2 * F + 2], s[2 * F + 3] = float(mean), float(var), cnt
        if self.venv._norm["norm_obs"]:
            mean, var, cnt = load_running_mean_std(os.path.join(path, "observation.pt"))
            if mean.shape != (F,):
                raise ValueError(f"observation.pt holds statistics of shape {mean.shape}, this env has {F} features")
            s[:F], s[F:2 * F], s[2 * F] = mean, var, cnt
        e.set_norm_stats(s)


def TrainingVecNormRO(venv: HipVecEnv) -> VecNormalize:
    """gym_.h:15-16."""
    return VecNormalize(venv, training=True, norm_reward=True, norm_obs=True)
