// gym/hip_policy.h: what a C++ trainer's calls are refused for before anything could reach a GPU.  Runs on the CPU.  One line per check; exit code 0 if all hold.
#include <cstdio>
#include <cstdlib>

#include "gym/hip_policy.h"

using namespace gym::policy;

static int failures = 0;
template <typename E, typename F>
static void refused(const char* what, const char* text, F f) {
    bool ok = false;
    try { f(); } catch (const E& e) { ok = std::string(e.what()).find(text) != std::string::npos; } catch (const std::exception&) {}
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", what);
    failures += !ok;
}

int main() {
    const auto x = torch::zeros({2, 4});
    using Wrong = std::invalid_argument;
    refused<Wrong>("a tensor that is none, as a temperature", "undefined tensor", [&] { LogitRules r; r.temperature = at::Tensor(); });
    refused<Wrong>("a tensor that is none, as a repetition", "undefined tensor", [&] { PerRow p{at::Tensor()}; });
    refused<Wrong>("one of two outputs", "both actions and log_prob", [&] { sampleActions(x, nullptr, Keys{}, at::Tensor(), torch::zeros({2})); });
    refused<Wrong>("a temperature that float32 does not hold", "temperature", [&] { LogitRules r; r.temperature = 1e-50; gym::policy::detail::Bound(r, x); });
    refused<Error>("the CPU", "no CPU fallback", [&] { processLogits(x); });
    return failures ? EXIT_FAILURE : EXIT_SUCCESS;
}
