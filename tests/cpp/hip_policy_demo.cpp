// gym/hip_policy.h as a C++ trainer uses it: actions from logits, their scores with gradients, dropout; checked against libtorch's own float64 on the CPU.
// Scores are float32 sums of 37 terms against (y - max) of at most about 30: off by at most (4 x 30 + 66) 2^-24 = 1.1e-5 in the worst case, a
// tenth of that as a rule.  Prints one line per check; exit code 0 if all hold.
#include <cstdio>
#include <cstdlib>

#include "gym/hip_policy.h"

using namespace gym::policy;

static int failures = 0;
static void check(bool ok, const char* what) {
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", what);
    failures += !ok;
}
template <typename E, typename F>
static bool throws(F f) {
    try { f(); } catch (const E&) { return true; }
    return false;
}

int main() {
    torch::manual_seed(1);
    const int64_t n = 100, width = 37;
    const auto cpu = torch::randn({n, width}, torch::kFloat64) * 3;
    const auto x = cpu.to(torch::kCUDA, torch::kFloat32);
    const auto exact = x.cpu().to(torch::kFloat64);

    LogitRules rules;
    rules.mask = torch::full({1, 2}, -1, torch::kInt32).to(torch::kCUDA);
    rules.mask.index_put_({0, 0}, 0x7FFFFFF0);   // columns 0 to 3 and 31 are not allowed
    rules.temperature = torch::full({n}, 0.5, torch::kFloat32).to(torch::kCUDA);
    auto z = exact / 0.5;
    for (int64_t v : {0, 1, 2, 3, 31}) z.index_put_({torch::indexing::Slice(), v}, -INFINITY);

    Keys keys;
    keys.seed = 7;
    keys.step = 3;
    auto [actions, log_prob] = sampleActions(x, &rules, keys);
    const auto a = actions.cpu().to(torch::kInt64);
    const auto lp = torch::log_softmax(z, 1);
    check(((a >= 4) & (a < width) & (a != 31)).all().item<bool>(), "actions are allowed ones");
    check(torch::allclose(log_prob.cpu().to(torch::kFloat64), lp.gather(1, a.unsqueeze(1)).squeeze(1), 1e-6, 1e-6), "their log-probabilities");
    auto [again, same] = sampleActions(x, &rules, keys);
    check(torch::equal(again, actions) && torch::equal(same, log_prob), "the same keys draw the same");
    keys.row = 1;
    LogitRules later = rules;
    later.temperature = 0.5;
    const auto moved = std::get<0>(sampleActions(x.slice(0, 1), &later, keys));
    check(torch::equal(moved, actions.slice(0, 1)), "a row's draw follows its key");

    auto leaf = x.clone().requires_grad_();
    auto [score, entropy] = actionLogProb(leaf, actions, &rules);
    (score.sum() + 0.5 * entropy.sum()).backward();
    auto ref = exact.clone().requires_grad_();
    auto open = (ref / 0.5).masked_fill(torch::isinf(z), -1e300);
    auto l = torch::log_softmax(open, 1);
    const auto h = -(l.exp() * l.masked_fill(torch::isinf(z), 0.0)).sum(1);
    (l.gather(1, a.unsqueeze(1)).sum() + 0.5 * h.sum()).backward();
    check(torch::allclose(score.detach().cpu().to(torch::kFloat64), lp.gather(1, a.unsqueeze(1)).squeeze(1), 1.2e-5, 1.2e-5), "scores");
    check(torch::allclose(entropy.detach().cpu().to(torch::kFloat64), h.detach(), 1.2e-5, 1.2e-5), "entropies");
    check(torch::allclose(leaf.grad().cpu().to(torch::kFloat64), ref.grad(), 1e-4, 4e-5), "their gradient");

    check(torch::allclose(processLogits(x, &rules).cpu().to(torch::kFloat64), z, 1e-6, 1e-6), "processed logits");
    auto d = x.clone().requires_grad_();
    auto y = dropout(d, 0.25, keys);
    y.sum().backward();
    check(torch::equal(d.grad() * x, y.detach()), "dropout's gradient has its mask");

    check(throws<std::invalid_argument>([&] { processLogits(x.flatten()); }), "one dimension is refused");
    check(throws<std::invalid_argument>([&] { dropout(x, 1.0, keys); }), "p = 1 is refused");
    check(throws<Error>([&] { processLogits(x.cpu()); }), "the CPU is refused");
    check(throws<std::runtime_error>([&] {
        auto t = x.clone().requires_grad_();
        torch::autograd::grad({std::get<1>(actionLogProb(t, actions)).sum()}, {t}, {}, true, true);
    }), "a second derivative is refused");
    return failures ? EXIT_FAILURE : EXIT_SUCCESS;
}
