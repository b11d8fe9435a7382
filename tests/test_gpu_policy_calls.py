"""GPU: calls of the policy operators that the documentation allows and that go wrong quietly: outputs written over what autograd has saved, forward-mode
derivatives, temperatures near 0 under a history, empty batches, buffers that share rows, more work than one pass of a grid."""
import math

import pytest
import torch

from tests import policy_reference as R
from tests.test_gpu_policy import TYPES, U, check_sample, check_score, check_values, half_step, logits_of, rules_of, score_bounds

pytestmark = pytest.mark.gpu


# ---- outputs that a caller hands in ------------------------------------------------------------------------------------------------------------

def test_a_reused_out_is_noticed_before_the_backward_pass():
    """Actions and log-probabilities that the next step overwrites are changed in place, for whoever has saved them."""
    from gym_amd.policy import ActionSample, action_log_prob, sample_actions
    n = 6
    x, _ = logits_of(n, 20, torch.float32, 1)
    store = ActionSample(torch.empty(2, n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda"))
    out = ActionSample(store.actions[0], store.log_prob)
    leaf = x.detach().requires_grad_()
    sample_actions(x, seed=1, step=0, out=out)
    lp, _ = action_log_prob(leaf, out.actions)
    ratio = leaf[:, 0] * out.log_prob   # saves the log-probabilities
    torch.autograd.grad(lp.sum() + ratio.sum(), leaf, retain_graph=True)
    before = store.actions._version, out.log_prob._version
    with torch.no_grad():
        sample_actions(x, seed=1, step=1, out=out)
    assert store.actions._version > before[0] and out.log_prob._version > before[1]   # a view's writes count for its base
    for loss in (lp, ratio):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss.sum(), leaf, retain_graph=True)


def test_processed_logits_written_over_saved_ones_are_noticed():
    from gym_amd.policy import LogitRules, action_log_prob, process_logits
    x, _ = logits_of(3, 20, torch.float32, 1)
    weights = torch.ones(3, 20, device="cuda", requires_grad=True)
    leaf = x.clone().requires_grad_()
    lp, _ = action_log_prob(leaf, torch.zeros(3, dtype=torch.int32, device="cuda"))
    other = torch.zeros(3, 20, device="cuda")
    loss = (weights * other).sum()
    with torch.no_grad():
        process_logits(leaf, LogitRules(temperature=0.5), out=leaf)
        process_logits(x, out=other)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(lp.sum(), leaf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, weights)


def test_out_may_be_inference_tensors():
    """They have no version and cannot be saved: writing them is allowed inside inference mode and outside."""
    from gym_amd.policy import ActionSample, process_logits, sample_actions
    x, _ = logits_of(3, 20, torch.float32, 1)
    with torch.inference_mode():
        out = ActionSample(torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda"))
        z = torch.empty(3, 20, device="cuda")
        sample_actions(x, seed=1, out=out)
        process_logits(x, out=z)
    want = sample_actions(x, seed=1)
    sample_actions(x, seed=1, out=out)
    process_logits(x, out=z)
    assert torch.equal(out.actions, want.actions) and torch.equal(out.log_prob, want.log_prob) and torch.equal(z, x)


# ---- derivatives of other kinds ----------------------------------------------------------------------------------------------------------------

def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    from gym_amd.policy import action_log_prob, dropout, process_logits, sample_actions
    x, _ = logits_of(3, 20, torch.float32, 1)
    a = torch.zeros(3, dtype=torch.int32, device="cuda")
    with fwd.dual_level():
        for base in (x, x.detach().requires_grad_()):
            dual = fwd.make_dual(base, torch.ones_like(x))
            for call in (lambda: process_logits(dual), lambda: action_log_prob(dual, a), lambda: dropout(dual, 0.5, seed=1)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
            assert torch.equal(sample_actions(dual, seed=1).actions, sample_actions(x, seed=1).actions)


# ---- temperatures near 0 -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["history", "history and bias"])
@pytest.mark.parametrize("width", [2, 18, 300, 3001, 20011])
@pytest.mark.parametrize("temperature", [1e-45, 1e-41, 4e-39, 1e-38, 1e-30, 1e-9])
def test_temperatures_near_zero_under_a_history(width, temperature, kind):
    """The greatest y is a penalised one that no float32 holds, another logit lies just below it: all of the weight is the former's, whichever way y rounds."""
    from gym_amd.policy import LogitRules, action_log_prob, sample_actions
    n = 40
    g = torch.Generator().manual_seed(width)
    x = -20 * torch.rand(n, width, generator=g) - 1
    best = torch.randint(0, width, (n,), generator=g)
    other = (best + 1 + torch.randint(0, width - 1, (n,), generator=g)) % width
    rows = torch.arange(n)
    x[rows, best] = 5 + torch.rand(n, generator=g)
    y = x[rows, best].double() / float(torch.tensor(1.3)) - float(torch.tensor(0.1))
    below = y.float()
    x[rows, other] = torch.where(below.double() < y, below, torch.nextafter(below, torch.tensor(0.0)))   # the float next below y
    rules = LogitRules(history=best[:, None].cuda(), repetition=1.3, presence=0.1, temperature=temperature)
    if kind != "history":
        rules.bias = torch.zeros(width).cuda()
    gap = (y - x[rows, other].double()) / float(torch.tensor(temperature))   # in units of the exponent; at 1e-9 at least
    sure = gap > 120   # nothing of the other is left in float32
    assert sure.sum() > n // 2
    x, best = x.cuda(), best.cuda()
    s = sample_actions(x, rules, seed=1)
    leaf = x.detach().requires_grad_()
    lp, ent = action_log_prob(leaf, best, rules)
    got, = torch.autograd.grad(lp.sum() + ent.sum(), leaf)
    assert torch.isfinite(lp).all() and torch.isfinite(ent).all() and torch.isfinite(got).all()
    assert torch.equal(s.actions[sure].cpu().long(), best.cpu()[sure]) and (s.log_prob[sure] == 0).all()
    assert (lp[sure] == 0).all() and (ent[sure] == 0).all() and (got[sure] == 0).all()


# ---- empty batches -------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n, width", [(0, 5), (3, 0), (0, 0)])
@pytest.mark.parametrize("lines", [None, 1, 5])
def test_nothing_to_do_under_every_rule(n, width, lines):
    from gym_amd.policy import action_log_prob, process_logits, sample_actions
    from tests.test_policy_calls import per_row_rules
    rules = per_row_rules(n, width, "cuda", lines)
    x = torch.zeros(n, width, device="cuda", requires_grad=True)
    z = process_logits(x, rules)
    assert z.shape == (n, width) and torch.autograd.grad(z.sum(), x)[0].shape == (n, width)
    s = sample_actions(x, rules, seed=1, rows=torch.arange(n).cuda(), step=torch.zeros(n, dtype=torch.int64).cuda())
    assert s.actions.tolist() == [-1] * n and s.log_prob.tolist() == [-math.inf] * n
    lp, ent = action_log_prob(x, torch.zeros(n, dtype=torch.int32, device="cuda"), rules)
    assert lp.tolist() == [-math.inf] * n and ent.tolist() == [0.0] * n
    assert torch.autograd.grad(ent.sum(), x)[0].shape == (n, width)


# ---- rules that are learned ----------------------------------------------------------------------------------------------------------------------

def test_learned_rules_are_taken_where_no_gradient_is_lost():
    from gym_amd.policy import ActionSample, LogitRules, action_log_prob, process_logits, sample_actions
    x, g = logits_of(4, 30, torch.float32, 3)
    bias, hot = torch.randn(30, generator=g).cuda().requires_grad_(), torch.full((4,), 0.7).cuda().requires_grad_()
    learned, fixed = LogitRules(bias=bias, temperature=hot), LogitRules(bias=bias.detach(), temperature=hot.detach())
    a = torch.arange(4).cuda()
    want = sample_actions(x, fixed, seed=1)
    got = sample_actions(x, learned, seed=1)   # a draw has no gradient, under autograd or not
    assert torch.equal(got.actions, want.actions) and torch.equal(got.log_prob, want.log_prob) and not got.log_prob.requires_grad
    with torch.no_grad():
        assert torch.equal(process_logits(x, learned), process_logits(x, fixed))
        assert torch.equal(action_log_prob(x, a, learned)[0], action_log_prob(x, a, fixed)[0])
    for call in (lambda: process_logits(x, learned), lambda: action_log_prob(x, a, learned), lambda: process_logits(x.clone().requires_grad_(), learned),
                 lambda: sample_actions(x, seed=1, out=ActionSample(want.actions, want.log_prob.clone().requires_grad_()))):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()


# ---- outputs that lie between the rows of an input -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("width", [1, 5, 64, 1000, 9001])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logits_and_results_in_one_buffer(dtype, width):
    """[logits | results] as the two halves of each of a buffer's rows, in either order: they share no element."""
    from gym_amd.policy import process_logits
    n = 5
    x, g = logits_of(n, width, dtype, width)
    rules = rules_of("all", n, width, g)
    want = process_logits(x, rules)
    for first, second in ((0, width), (width, 0), (0, width + 3), (width + 3, 1)):
        both = torch.full((n, 2 * width + 5), 7.0, dtype=dtype, device="cuda")
        both[:, first:first + width] = x
        out = both[:, second:second + width]
        process_logits(both[:, first:first + width], rules, out=out)
        assert torch.equal(out, want) and torch.equal(both[:, first:first + width], x)
        rest = torch.ones(2 * width + 5, dtype=torch.bool, device="cuda")
        rest[first:first + width] = False
        rest[second:second + width] = False
        assert (both[:, rest] == 7).all()


# ---- temperatures up to the greatest float32 ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("width", [2, 18, 300, 9001])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_temperatures_up_to_the_greatest_float32(dtype, width):
    from gym_amd.policy import LogitRules, process_logits
    n = 4
    x, g = logits_of(n, width, dtype, width, 1e4 if dtype == torch.float16 else 1e37)
    bias = (torch.randn(width, generator=g) * 1e37).cuda()
    for temperature in (3.05e38, torch.finfo(torch.float32).max, torch.tensor([1.0, 2.9e38, 3.2e38, torch.finfo(torch.float32).max]).cuda()):
        for rules in (LogitRules(temperature=temperature), LogitRules(temperature=temperature, bias=bias)):
            z, slope, _ = R.apply_rules(x, rules)
            leaf = x.detach().requires_grad_()
            out = process_logits(leaf, rules)
            check_values(out, z, dtype)
            check_sample(x, rules, 5)


# ---- more work than one pass of a grid ---------------------------------------------------------------------------------------------------------------

def shared_rows(n, width, dtype, temperature=True, history=1, scale=3.0):
    """n rows that share their logits in memory, told apart by their histories and temperatures; and the rules."""
    from gym_amd.policy import LogitRules
    x = logits_of(1, width, dtype, width, scale)[0].expand(n, width)
    g = torch.Generator(device="cuda").manual_seed(n)
    t = 0.5 + torch.rand(n, generator=g, device="cuda") if temperature else 1.0
    if not history:
        return x, LogitRules(temperature=t)
    h = torch.randint(0, width, (n, history), generator=g, device="cuda", dtype=torch.int32)
    return x, LogitRules(temperature=t, history=h, repetition=1.3, presence=0.5)


def cut_of(rules, cut):
    from gym_amd.policy import LogitRules
    pick = lambda v: v[cut] if isinstance(v, torch.Tensor) else v
    return LogitRules(history=pick(rules.history), repetition=rules.repetition, presence=rules.presence, temperature=pick(rules.temperature))


def cuts_of(n, trip):
    """Rows of the first trip of the grid's loop, around its end, and of the last."""
    return [slice(0, 3), slice(trip - 2, trip + 3), slice(n - 3, n)]


# (rows, width, type, ids a row, rows of one trip): a row a lane, a wave's vector, a wave's strip, a workgroup's strip, parts
SCORED = [((1 << 24) + 301, 2, torch.float32, 0, 1 << 24), ((1 << 24) + 301, 2, torch.float32, 1, 1 << 24), ((1 << 18) + 9, 200, torch.float32, 1, 1 << 18),
          ((1 << 18) + 9, 300, torch.float32, 0, 1 << 18), ((1 << 18) + 9, 300, torch.float32, 2, 1 << 18), (65541, 4100, torch.bfloat16, 3, 65536),
          (65541, 8200, torch.bfloat16, 3, 65536)]


@pytest.mark.parametrize("n, width, dtype, history, trip", SCORED)
def test_scores_of_more_rows_than_one_trip(n, width, dtype, history, trip):
    from gym_amd.policy import action_log_prob
    x, rules = shared_rows(n, width, dtype, history=history)
    actions = torch.randint(0, width, (n,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        lp, ent = action_log_prob(x, actions, rules)
    for cut in cuts_of(n, trip):
        r = R.score(x[cut], actions[cut], cut_of(rules, cut))
        ones = torch.ones(cut.stop - cut.start)
        e_lp, e_ent, _ = score_bounds(r, actions[cut], ones, ones, dtype)
        assert ((lp[cut].cpu().double() - r["log_prob"]).abs() <= e_lp).all() and ((ent[cut].cpu().double() - r["entropy"]).abs() <= e_ent).all()


# a wave's strip, a workgroup's, parts whose joins are more than one trip, and parts that are themselves
DRAWN = [((1 << 18) + 9, 300, torch.float32, 0, 1 << 18), ((1 << 18) + 9, 300, torch.float32, 2, 1 << 18), (65541, 4100, torch.bfloat16, 3, 65536),
         (65541, 8200, torch.bfloat16, 3, 65536), ((1 << 19) + 5, 8200, torch.bfloat16, 3, 1 << 19)]


@pytest.mark.parametrize("n, width, dtype, history, trip", DRAWN)
def test_draws_of_more_rows_than_one_trip(n, width, dtype, history, trip):
    from gym_amd.policy import sample_actions
    x, rules = shared_rows(n, width, dtype, history=history)
    if isinstance(rules.temperature, torch.Tensor):
        rules.temperature[1::4] = 0.0
    s = sample_actions(x, rules, seed=5, rows=7)
    for cut in cuts_of(n, trip):
        a, lp = R.sample(x[cut], cut_of(rules, cut), 5, rows=7 + cut.start)
        assert torch.equal(s.actions[cut].cpu(), a)
        assert ((s.log_prob[cut].cpu().double() - lp).abs() <= U * lp.abs() + 1e-12).all()


# (rows, width, type, ids, rows of one trip): 256 rows a tile, and rows of two tiles, each
TILED = [((1 << 24) + 301, 3, torch.float16, 0, 1 << 24), ((1 << 24) + 301, 3, torch.float16, 1, 1 << 24), (32771, 8200, torch.bfloat16, 0, 32768), (32771, 8200, torch.bfloat16, 2, 32768)]


@pytest.mark.parametrize("n, width, dtype, history, trip", TILED)
def test_rules_and_gradients_of_more_tiles_than_one_trip(n, width, dtype, history, trip):
    from gym_amd.policy import action_log_prob, process_logits
    x, rules = shared_rows(n, width, dtype, history=history)
    up = logits_of(1, width, dtype, 5)[0].expand(n, width)
    leaf = x.detach().requires_grad_()
    z = process_logits(leaf, rules)
    got, = torch.autograd.grad(z, leaf, up)
    for cut in cuts_of(n, trip):
        want, slope, _ = R.apply_rules(x[cut], cut_of(rules, cut))
        check_values(z[cut], want, dtype, "z")
        check_values(got[cut], up[cut].cpu().double() * slope, dtype, "gradient")
    del z, got
    actions = torch.randint(0, width, (n,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(1))
    g_lp, g_ent = torch.ones(n, device="cuda"), torch.full((n,), 0.3, device="cuda")
    got, = torch.autograd.grad(action_log_prob(leaf, actions, rules), leaf, [g_lp, g_ent])
    for cut in cuts_of(n, trip):
        r = R.score(x[cut], actions[cut], cut_of(rules, cut))
        e_g = score_bounds(r, actions[cut], g_lp[cut], g_ent[cut], dtype)[2]
        want = R.score_gradient(r, actions[cut], g_lp[cut], g_ent[cut])
        lim = e_g + half_step(dtype) * (want.abs() + e_g) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 1.001
        assert ((got[cut].cpu().double() - want).abs() <= lim).all()


@pytest.mark.parametrize("n, width, dtype, trip", [((1 << 24) + 301, 1, torch.float32, 1 << 24), (32771, 4093, torch.float16, 32768)])
def test_dropout_of_more_blocks_than_one_trip(n, width, dtype, trip):
    from gym_amd.policy import dropout
    x = logits_of(1, width, dtype, 5)[0].expand(n, width)
    y = dropout(x, 0.25, seed=3, rows=9)
    for cut in cuts_of(n, trip):
        keep = R.kept(cut.stop - cut.start, width, 0.25, 3, rows=9 + cut.start)
        want = torch.where(keep, x[cut].cpu().double() * (4 / 3), 0.0)
        assert ((y[cut].cpu().double() - want).abs() <= (half_step(dtype) + 2 * U) * want.abs()).all()


# ---- results that lie in what is still read ------------------------------------------------------------------------------------------------------

def test_drawn_results_in_the_logits_or_in_each_other_are_refused():
    from gym_amd._lib import GymhipError
    from gym_amd.policy import ActionSample, sample_actions
    x, _ = logits_of(6, 1, torch.float32, 1)
    store = torch.zeros(40, device="cuda")
    actions = torch.zeros(6, dtype=torch.int32, device="cuda")
    for a, lp in ((actions, x[:, 0]), (x[:, 0].view(torch.int32), store[:6]), (store[:6].view(torch.int32), store[5:11])):
        with pytest.raises(GymhipError, match="overlaps"):
            sample_actions(x, seed=1, out=ActionSample(a, lp))
    # side by side in one buffer is apart
    got = sample_actions(x, seed=1, out=ActionSample(store[:6].view(torch.int32), store[6:12]))
    assert got.actions.tolist() == [0] * 6 and got.log_prob.tolist() == [0.0] * 6 and (store[12:] == 0).all()


# ---- masks of the type's lowest value, penalised ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("width", [1, 2, 18, 300, 3001, 9001, 70001])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_lowest_values_under_penalties(dtype, width):
    """A logit of the type's lowest value that has been chosen before: its y lies below every float32.  Alone in a row it is certain, among its like as likely."""
    from gym_amd.policy import LogitRules, pack_action_mask, process_logits
    n = 5
    low = torch.finfo(dtype).min
    x, g = logits_of(n, width, dtype, width)
    x[:4] = low
    x[4, :max(1, width // 2)] = low
    allowed = torch.ones(n, width, dtype=torch.bool)
    one = torch.randint(0, width, (4,), generator=g)
    allowed[0] = allowed[2] = False
    allowed[0, one[0]] = True
    allowed[2, one] = True
    h = torch.full((n, width + 4), -1)
    h[:, :4] = one
    h[1, :width] = torch.arange(width)
    h[4, :max(1, width // 2)] = torch.arange(max(1, width // 2))
    x[0, ~allowed[0].cuda()] = math.inf
    for rules in (LogitRules(mask=pack_action_mask(allowed.cuda()), history=h.cuda(), repetition=1.3),
                  LogitRules(mask=pack_action_mask(allowed.cuda()), history=h.cuda(), repetition=1.3, bias=torch.zeros(width).cuda()),
                  LogitRules(mask=pack_action_mask(allowed.cuda()), history=h.int().cuda(), repetition=4.0, frequency=1e37)):
        z, _, _ = R.apply_rules(x, rules)
        check_values(process_logits(x, rules), z, dtype)
        s = check_sample(x, rules, 3)
        assert (s.actions >= 0).all() and int(s.actions[0]) == int(one[0])
        lp, _ = check_score(x, s.actions, rules, grad=False)
        assert float(lp[0]) == 0.0 and torch.isfinite(lp).all()
        check_score(x, s.actions, rules)


@pytest.mark.parametrize("width", [1, 2, 18, 300, 3001, 9001, 70001])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_highest_values_under_penalties(dtype, width):
    """A penalty that raises the type's greatest value above every float32 makes it the one choice, not an infinity."""
    from gym_amd.policy import LogitRules, action_log_prob
    n = 3
    x, g = logits_of(n, width, dtype, width)
    at = torch.randint(0, width, (n,), generator=g)
    x[torch.arange(n), at.cuda()] = torch.finfo(dtype).max
    x[2] = torch.finfo(dtype).max
    for bias in (None, torch.zeros(width).cuda()):
        rules = LogitRules(history=at[:, None].cuda(), repetition=0.5, bias=bias)
        s = check_sample(x, rules, 3)
        assert torch.equal(s.actions.cpu().long(), at) and (s.log_prob == 0).all()
        check_score(x, s.actions, rules)
        # another action's log-probability may lie below every float32 (-max / 0.5 and its like): -inf is what it rounds to
        other = torch.zeros(n, dtype=torch.int32).cuda()
        want = R.score(x, other, rules)["log_prob"]
        lp = action_log_prob(x, other, rules)[0].cpu().double()
        far = want < -torch.finfo(torch.float32).max * (1 + U)
        assert (lp[far] == -math.inf).all() and ((lp - want)[~far].abs() <= 4 * U * want[~far].abs()).all()
