"""GPU: the policy operators where they are used: VecLogitActions and VecObservationDropout around the engine, an update that scores the rollout's
actions again, and the sizes that take the kernels' other paths (long histories, very wide rows, many of them)."""
import math

import pytest
import torch

from tests import policy_reference as R
from tests.test_gpu_policy import TYPES, U, check_sample, check_score, check_values, logits_of, rules_of, score_bounds

pytestmark = pytest.mark.gpu


def mlp(features, actions, seed):
    """Weights of a small policy, float32 on the GPU."""
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * 0.5).cuda() for s in ((features, 16), (16,), (16, actions), (actions,))]


def forward(w, obs, p=0.0, **keys):
    from gym_amd.policy import dropout
    hidden = torch.tanh(obs @ w[0] + w[1])
    return dropout(hidden, p, **keys) @ w[2] + w[3]


@pytest.mark.parametrize("env_id, n", [("CartPole", 1), ("CartPole", 257), ("MountainCar", 100)])
def test_rollout_and_update(env_id, n):
    """A rollout through both wrappers over the normalised engine, every draw and every dropped place checked against its definition; then the update:
    shuffled rows, each under its rollout's own dropout mask, scored with gradients that are checked against the same network in 64 bits."""
    from gym_amd.policy import LogitRules, action_log_prob, pack_action_mask
    from gym_amd.vec_env import HipVecEnv, VecLogitActions, VecNormalize, VecObservationDropout
    T, p_obs, p_hidden = 5, 0.1, 0.25
    norm = VecNormalize(HipVecEnv(env_id, n, max_episode_steps=20))
    noisy = VecObservationDropout(norm, p_obs, seed=21)
    venv = VecLogitActions(noisy, seed=22)
    width = venv.actionSpace().n
    g = torch.Generator().manual_seed(n)
    allowed = torch.rand(n, width, generator=g) < 0.6
    allowed[:, 0] |= ~allowed.any(1)
    if n > 2:
        allowed[2] = False   # nothing to choose: the engine is handed -1
    mask = pack_action_mask(allowed.cuda())
    venv.rules = LogitRules(mask=mask, temperature=0.8)
    w = mlp(venv.observationSpace()._shape[0], width, 3)
    obs = venv.reset()
    roll = []
    for t in range(T):
        raw = norm.venv.engine.obs_norm
        keep = R.kept(n, raw.shape[1], p_obs, 21, 0, t)
        want = torch.where(keep, raw.cpu().double() * (65536 / (65536 - round(65536 * p_obs))), 0.0)
        assert ((obs.cpu().double() - want).abs() <= 2 * U * want.abs() + 1e-44).all()   # the scale and the product, rounded once each
        logits = forward(w, obs, p_hidden, seed=23, step=t)
        want, _ = R.sample(logits, venv.rules, 22, 0, t)
        r = venv.step(logits)
        assert torch.equal(venv.sample.actions.cpu(), want)
        roll.append((obs, venv.sample.actions, venv.sample.log_prob))
        assert r.observation.data_ptr() != norm.venv.engine.obs_norm.data_ptr()
        obs = r.observation
    # ---- the update: all T * n samples in a random order, at two sizes of minibatch
    obs, actions, old = (torch.cat([r[k] for r in roll]) for k in range(3))
    steps = torch.arange(T).repeat_interleave(n).cuda()
    rows = torch.arange(n).repeat(T).cuda()
    perm = torch.randperm(T * n, generator=g).cuda()
    for part in (perm, perm[: max(1, T * n // 3)]):
        leaves = [v.clone().requires_grad_() for v in w]
        rules = LogitRules(mask=mask, mask_rows=rows[part].int(), temperature=0.8)
        logits = forward(leaves, obs[part], p_hidden, seed=23, step=steps[part], rows=rows[part])
        lp, ent = action_log_prob(logits, actions[part], rules)
        # In 64 bits, with masks and rules written out, and beside every value what float32 may be off by: (terms + 2) U of a sum's absolute terms, 4 U for tanh
        # (its slope is at most 1), and errors of what went in.
        keep = R.kept(len(part), 16, p_hidden, 23, rows[part].cpu(), steps[part].cpu()).double() / (1 - p_hidden)
        o = obs[part].cpu().double()
        exact = [v.cpu().double().requires_grad_() for v in w]
        a0, b0, a1, b1 = (v.detach().abs() for v in exact)
        tanh = torch.tanh(o @ exact[0] + exact[1])
        h = tanh * keep
        logits64 = h @ exact[2] + exact[3]
        e_t = (o.shape[1] + 3) * U * (o.abs() @ a0 + b0) + 4 * U
        e_h = (e_t + 2 * U) * keep
        e_z = ((e_h @ a1 + 19 * U * (h.detach().abs() @ a1 + b1)) / 0.8).amax(1)
        assert ((logits.detach().cpu().double() - logits64.detach()).abs() <= 0.8 * e_z[:, None]).all()
        # a log-probability moves by at most 2 e_z with its logits, twice for the rollout's own rounding, and is rounded itself
        fine = torch.isfinite(old[part])
        off = ((lp - old[part]).detach().cpu().double().abs() <= 4 * e_z + 90 * U * (1 + old[part].cpu().double().abs()))
        assert torch.equal(fine, torch.isfinite(lp)) and off[fine.cpu()].all()
        loss = lp[fine].sum() - 0.01 * ent.sum()
        got = torch.autograd.grad(loss, leaves)
        legal = allowed[rows[part].cpu()]
        some = legal.any(1)
        lsm = torch.log_softmax((logits64 / 0.8).masked_fill(~legal, -1e300)[some], 1)
        taken = lsm.gather(1, actions[part].cpu().long()[some][:, None]).sum()
        pl = (lsm.exp() * lsm).masked_fill(~legal[some], 0.0).sum()
        want = torch.autograd.grad(taken + 0.01 * pl, [*exact, logits64, h], retain_graph=True)
        # dlogits = (hot - p + 0.01 p (log p + H)) / 0.8 with p off by 2 e_z of itself: 4 e_z in all, and the kernel's own rounding, far below 200 U
        dl, dh = want[4].abs(), want[5].abs()
        e_l = ((4 * e_z + 200 * U) / 0.8)[:, None] * some[:, None]
        e_dh = e_l * a1.sum(1)[None, :] + 6 * U * (dl @ a1.t())
        dp = dh * keep
        e_dp = e_dh * keep + dp * (2 * e_t + 6 * U)
        N, ha, oa = len(part) + 2, h.detach().abs(), o.abs()
        limits = [oa.t() @ e_dp + N * U * (oa.t() @ dp), e_dp.sum(0) + N * U * dp.sum(0), ha.t() @ e_l.expand_as(dl) + e_h.t() @ dl + N * U * (ha.t() @ dl),
                  e_l.sum(0) + N * U * dl.sum(0)]
        for a, b, lim in zip(got, want, limits):
            assert ((a.cpu().double() - b).abs() <= lim).all(), ((a.cpu().double() - b).abs() / lim).max()


def test_shards_draw_what_the_whole_draws():
    from gym_amd.vec_env import HipVecEnv, VecLogitActions, VecObservationDropout
    n, T = 301, 12
    mk = lambda rank, world: VecLogitActions(VecObservationDropout(HipVecEnv("CartPole", n, max_episode_steps=30, rank=rank, world=world), 0.2, seed=1), seed=2)
    whole, parts = mk(0, 1), [mk(r, 2) for r in range(2)]
    w = torch.randn(4, 2, generator=torch.Generator().manual_seed(0)).cuda()
    for v in (whole, *parts):
        v.seed(9)
    obs, shards = whole.reset(), [v.reset() for v in parts]
    assert torch.equal(obs, torch.cat(shards))
    for t in range(T):
        # elementwise products: the same float32 bits at any batch size
        policy = lambda o: torch.stack([(o[:, 0] * w[0, k] + o[:, 2] * w[2, k]) for k in range(2)], 1)
        obs = whole.step(policy(obs)).observation
        shards = [v.step(policy(o)).observation for v, o in zip(parts, shards)]
        assert torch.equal(whole.sample.actions, torch.cat([v.sample.actions for v in parts])) and torch.equal(obs, torch.cat(shards)), t
    # one env by itself: masks of their own, the count goes on
    one = whole.reset(200)
    assert one.shape == (4,)
    local = 200 - parts[1].venv.venv.env_offset
    assert torch.equal(one, parts[1].reset(local))


def test_recorded_steps_draw_anew():
    """A step recorded once with both wrappers' counts on the device, replayed with eager work between, against the same steps taken eagerly."""
    from gym_amd.policy import LogitRules
    from gym_amd.vec_env import HipVecEnv, VecLogitActions, VecObservationDropout
    n, T = 500, 6

    def make(device_step):
        venv = VecLogitActions(VecObservationDropout(HipVecEnv("CartPole", n, max_episode_steps=50), 0.3, seed=4, device_step=device_step), LogitRules(temperature=1.5), seed=5,
                               device_step=device_step)
        venv.reset()
        return venv

    recorded, eager = make(True), make(False)
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(T, n, 2, generator=g).cuda()
    static = logits[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        recorded.step(static)
    torch.cuda.current_stream().wait_stream(side)
    eager.step(logits[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = recorded.step(static)
        out, actions, lp = r.observation, recorded.sample.actions, recorded.sample.log_prob
    for t in range(1, T):
        static.copy_(logits[t])
        graph.replay()
        if t % 2:
            torch.cuda.synchronize()
        want = eager.step(logits[t])
        assert torch.equal(actions, eager.sample.actions) and torch.equal(lp, eager.sample.log_prob) and torch.equal(out, want.observation), t
    with pytest.raises(RuntimeError, match="device_step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            static.add_(0)
            eager.step(static)
    torch.cuda.synchronize()


# ---- sizes that take other paths -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("length", [65535, 65536, 70000])
@pytest.mark.parametrize("width", [2, 18, 1000, 9001, 140001])
def test_histories_longer_than_16_bits_count(width, length):
    """One id over and over (its count needs more than 16 bits), ids of all columns, and a short one beside them."""
    from gym_amd.policy import LogitRules, process_logits
    n = 3
    x, g = logits_of(n, width, torch.float32, width)
    h = torch.randint(0, width, (n, length), generator=g).int()
    h[0] = width // 2
    rules = LogitRules(history=h.cuda(), history_len=torch.tensor([length, length, 5]).cuda(), repetition=1.2, presence=0.1, frequency=2.0 ** -14, temperature=0.7)
    z, _, _ = R.apply_rules(x, rules)
    check_values(process_logits(x, rules), z, torch.float32)
    check_sample(x, rules, 3)
    check_score(x, torch.tensor([width // 2, 0, width - 1]).cuda(), rules)


@pytest.mark.parametrize("kind", ["none", "temperature", "table", "all"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n, width", [(1, 1 << 20), (2, (1 << 19) + 77), (5, 131073)])
def test_very_wide_rows(n, width, dtype, kind):
    from gym_amd.policy import process_logits
    x, g = logits_of(n, width, dtype, 7)
    rules = rules_of(kind, n, width, g)
    z, _, _ = R.apply_rules(x, rules)
    check_values(process_logits(x, rules), z, dtype)
    s = check_sample(x, rules, 31, rows=1 << 40, step=5)
    check_score(x, s.actions, rules)


def test_the_widest_row():
    x, g = logits_of(1, 1 << 24, torch.bfloat16, 7)
    s = check_sample(x, None, 31)
    check_score(x, s.actions, None)


def test_many_wide_rows():
    """More wide rows than are worth splitting, against the same rows in small batches (draws: equal; scores: their bounds)."""
    from gym_amd.policy import action_log_prob, sample_actions
    x, g = logits_of(1100, 9001, torch.bfloat16, 9)
    whole = sample_actions(x, seed=1, rows=50)
    for lo, hi in ((0, 3), (500, 520), (1097, 1100)):
        part = check_sample(x[lo:hi], None, 1, rows=50 + lo)
        assert torch.equal(part.actions, whole.actions[lo:hi]) and torch.equal(part.log_prob, whole.log_prob[lo:hi])
    check_score(x, whole.actions, None)


@pytest.mark.parametrize("n, width", [(300001, 18), (40000, 100), (20001, 300), (9001, 2100), (4500, 9001)])
def test_rows_do_not_hang_on_how_many_there_are(n, width):
    """More rows than one pass of any grid: the first, middle and last ones alone give the same actions, and those are the definition's."""
    from gym_amd.policy import sample_actions
    x = (torch.randn(n, width, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 3).half()
    g = torch.Generator().manual_seed(2)
    rules = rules_of("all", n, width, g)
    from gym_amd.policy import LogitRules
    whole = sample_actions(x, rules, seed=1)
    for lo in (0, n // 2, n - 5):
        cut = slice(lo, lo + 5)
        some = LogitRules(mask=rules.mask, bias=rules.bias, history=rules.history[cut], history_len=rules.history_len[cut], repetition=rules.repetition[cut],
                          presence=rules.presence[cut], frequency=rules.frequency[cut], temperature=rules.temperature[cut])
        part = check_sample(x[cut], some, 1, rows=lo)
        assert torch.equal(part.actions, whole.actions[cut]) and torch.equal(part.log_prob, whole.log_prob[cut])


@pytest.mark.parametrize("width", [5, 70, 3001, 9001, 140001])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_bias_and_history_behind_the_mask_are_never_seen(dtype, width):
    from gym_amd.policy import LogitRules, pack_action_mask, process_logits
    n = 6
    x, g = logits_of(n, width, dtype, 3)
    allowed = torch.rand(n, width, generator=g) < 0.5
    allowed[:, 0] = True
    allowed[:, width - 2:] = False
    allowed[5] = False
    bias = torch.randn(n, width, generator=g)
    bias[~allowed] = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(int((~allowed).sum())) % 3]
    bias[4, 0] = -math.inf   # in the open: a choice of weight 0
    x[:, width - 2] = math.inf
    rules = LogitRules(mask=pack_action_mask(allowed.cuda()), bias=bias.cuda(), history=torch.full((n, 4), width - 1).cuda(), presence=3.0, temperature=0.5)
    z, _, _ = R.apply_rules(x, rules)
    check_values(process_logits(x, rules), z, dtype)
    s = check_sample(x, rules, 8)
    check_score(x, torch.zeros(n, dtype=torch.int32).cuda(), rules)
    assert (s.actions[:4] >= 0).all() and int(s.actions[5]) == -1


def test_two_streams_at_once():
    """The same wide call (which has a workspace) on two streams at the same time, again and again."""
    from gym_amd.policy import action_log_prob, sample_actions
    xs = [logits_of(4, 200000, torch.bfloat16, k)[0] for k in range(2)]
    want = [sample_actions(x, seed=6) for x in xs]
    scores = [action_log_prob(x, w.actions) for x, w in zip(xs, want)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                a = sample_actions(xs[k], seed=6)
                got[k].append((a, action_log_prob(xs[k], a.actions)))
    torch.cuda.synchronize()
    for k in range(2):
        for a, (lp, ent) in got[k]:
            assert torch.equal(a.actions, want[k].actions) and torch.equal(a.log_prob, want[k].log_prob)
            assert torch.equal(lp, scores[k][0]) and torch.equal(ent, scores[k][1])


def test_padded_batch_leaves_the_rest():
    """Rows of a larger buffer beyond the batch, and columns beyond the width, are neither read into results nor written."""
    from gym_amd.policy import ActionSample, process_logits, sample_actions
    store = torch.full((10, 40), math.nan, device="cuda")
    g = torch.Generator().manual_seed(1)
    store[:6, :33] = torch.randn(6, 33, generator=g).cuda()
    actions, lp = torch.full((10,), 99, dtype=torch.int32, device="cuda"), torch.full((10,), 99.0, device="cuda")
    s = sample_actions(store[:6, :33], seed=1, out=ActionSample(actions[:6], lp[:6]))
    assert torch.equal(s.actions.cpu(), R.sample(store[:6, :33], None, 1)[0]) and (actions[6:] == 99).all() and (lp[6:] == 99).all()
    process_logits(store[:6, :33], out=store[:6, :33])
    assert torch.isnan(store[6:]).all() and torch.isnan(store[:, 33:]).all()


@pytest.mark.parametrize("width", [2, 18, 300, 3001, 20011])
@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 2e-38, 1e30, 2e38])
def test_temperatures_at_the_ends_of_their_type(width, temperature):
    """So low that 1 / T overflows: the greatest logit has all of the weight, and no gradient is NaN.  So high that every choice is as likely."""
    from gym_amd.policy import LogitRules, action_log_prob, sample_actions
    n = 5
    x, g = logits_of(n, width, torch.float32, width)
    best = x.argmax(1)
    for rules in (LogitRules(temperature=temperature), LogitRules(temperature=torch.full((n,), temperature).cuda(), bias=torch.zeros(width).cuda())):
        s = sample_actions(x, rules, seed=1)
        leaf = x.detach().requires_grad_()
        lp, ent = action_log_prob(leaf, best, rules)
        got, = torch.autograd.grad(lp.sum() + ent.sum(), leaf)
        if temperature < 1:
            assert torch.equal(s.actions.long(), best) and (s.log_prob == 0).all() and (lp == 0).all() and (ent == 0).all() and (got == 0).all()
        else:
            flat = math.log(width)
            assert ((lp + flat).abs() <= 64 * U * flat + 1e-6).all() and ((ent - flat).abs() <= 64 * U * flat + 1e-6).all() and torch.isfinite(got).all()
            assert ((s.log_prob + flat).abs() <= 2 * U * flat + 1e-6).all()


def rules_cut(rules, cut):
    """The same rules for some of the rows."""
    from gym_amd.policy import LogitRules
    if rules is None:
        return None
    pick = lambda v: v[cut] if isinstance(v, torch.Tensor) and v.dim() >= 1 and v.shape[0] > 1 else v
    return LogitRules(mask=rules.mask if rules.mask_rows is not None else pick(rules.mask), mask_rows=pick(rules.mask_rows), bias=rules.bias,
                      history=pick(rules.history), history_len=pick(rules.history_len), repetition=pick(rules.repetition), presence=pick(rules.presence),
                      frequency=pick(rules.frequency), temperature=pick(rules.temperature))


@pytest.mark.parametrize("kind", ["none", "temperature", "table", "all"])
@pytest.mark.parametrize("scale", [3.0, 500.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n, width", [(700, 2083), (2600, 5000), (300, 12345), (1100, 33000), (130, 70001)])
def test_many_rows_of_every_length(n, width, dtype, scale, kind):
    """Rows by a wave, by a workgroup or in parts, as their number and length have it; at a scale of 500 most rows are out of the sums' straight range.  A few
    rows of the whole against the definition."""
    from gym_amd.policy import action_log_prob, process_logits, sample_actions
    g = torch.Generator().manual_seed(width)
    x = (torch.randn(n, width, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * scale).to(dtype)
    rules = rules_of(kind, n, width, g)
    s = sample_actions(x, rules, seed=11, rows=5)
    actions = torch.where(s.actions < 0, 0, s.actions)
    leaf = x.detach().requires_grad_()
    lp, ent = action_log_prob(leaf, actions, rules)
    g_lp, g_ent = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    got, = torch.autograd.grad([lp, ent], leaf, [g_lp, g_ent])
    z = process_logits(x, rules)
    for cut in (slice(0, 3), slice(n // 2, n // 2 + 2), slice(n - 3, n)):
        some = rules_cut(rules, cut)
        a, want_lp = R.sample(x[cut], some, 11, rows=5 + cut.start)
        assert torch.equal(s.actions[cut].cpu(), a)
        fine = torch.isfinite(want_lp)
        assert ((s.log_prob[cut].cpu().double() - want_lp)[fine].abs() <= U * want_lp[fine].abs() + 1e-11).all()   # y in double: 3000 x 2^-53 and the logarithm
        check_values(z[cut], R.apply_rules(x[cut], some)[0], dtype)
        r = R.score(x[cut], actions[cut], some)
        e_lp, e_ent, e_g = score_bounds(r, actions[cut], g_lp[cut], g_ent[cut], dtype)
        fine = torch.isfinite(r["log_prob"])
        assert ((lp[cut].detach().cpu().double() - r["log_prob"])[fine].abs() <= e_lp[fine]).all()
        assert ((ent[cut].detach().cpu().double() - r["entropy"]).abs() <= e_ent).all()
        want = R.score_gradient(r, actions[cut], g_lp[cut], g_ent[cut])
        half = torch.finfo(dtype).eps / 2
        assert ((got[cut].cpu().double() - want).abs() <= e_g + half * (want.abs() + e_g) + torch.finfo(dtype).smallest_normal * half * 1.001).all()


@pytest.mark.parametrize("width", [1, 2, 14, 64, 300, 2083, 9001, 140001])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_choice_with_all_of_the_weight_is_certain(dtype, width):
    """One allowed column, under a penalty and a bias that make its y no float: log-probability, entropy and gradient are 0, not 1e-8 beside it."""
    from gym_amd.policy import LogitRules, action_log_prob, pack_action_mask, sample_actions
    n = 6
    x, g = logits_of(n, width, dtype, width, 9.0)
    at = torch.randint(0, width, (n,), generator=g)
    allowed = torch.zeros(n, width, dtype=torch.bool)
    allowed[torch.arange(n), at] = True
    rules = LogitRules(mask=pack_action_mask(allowed.cuda()), bias=torch.randn(width, generator=g).cuda(), history=at[:, None].expand(n, 3).int().cuda(), repetition=1.1,
                       presence=0.3, frequency=0.07, temperature=0.7)
    for r in (rules, LogitRules(mask=rules.mask, history=rules.history, repetition=1.1, temperature=0.7), LogitRules(mask=rules.mask, bias=rules.bias)):
        s = sample_actions(x, r, seed=1)
        leaf = x.detach().requires_grad_()
        lp, ent = action_log_prob(leaf, s.actions, r)
        got, = torch.autograd.grad(lp.sum() + 3 * ent.sum(), leaf)
        assert torch.equal(s.actions.cpu().long(), at) and (s.log_prob == 0).all() and (lp == 0).all() and (ent == 0).all() and (got == 0).all()
