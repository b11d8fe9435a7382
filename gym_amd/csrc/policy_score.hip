// policy_score.hip — log-probability and entropy of given actions under the ruled logits: one pass over the logits with a running maximum.
//
// With y the logit after penalties and bias, d = y - max y, t = d log2 e / T and w = 2^t:  S = sum w, D = sum w t,
// log_prob = d_a / T - ln S, entropy = ln 2 (log2 S - D / S).  t and w are float32 (their errors are relative to d, not to y); a lane adds up
// at most 32 of them before it goes on in double.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

// A running (m, S, D) over any set of columns; S and D against m.
struct Run {
    double m, s, d;
    int bad;
};

// S and D of r against another base m >= r.m.
__device__ inline void rebase(Run& r, double m, double k2) {
    if (r.m == m || r.s == 0) { r.m = m; return; }
    const double t = (r.m - m) * k2;
    const double e = (double)__builtin_amdgcn_exp2f((float)t);
    // against the new base every t moves by the same amount
    r.d = e == 0 ? 0.0 : e * (r.d + t * r.s);
    r.s = e * r.s;
    r.m = m;
}

// C columns' y added to a run.  NaN and +inf only mark it.
template <int C, typename Y>
__device__ inline void add_cols(Run& run, const Y* y, double k2) {
    Y m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < C; j++) {
        bad = bad || y[j] != y[j];
        m = y[j] > m ? y[j] : m;
    }
    if (bad || m == INFINITY) run.bad = 1;
    if (!(m < INFINITY)) return;
    if ((double)m > run.m) rebase(run, (double)m, k2);
    const double base = run.m > -INFINITY ? run.m : 0.0;
    const float k = (float)k2;
    float s = 0, d = 0;
#pragma unroll
    for (int j = 0; j < C; j++) {
        float t = (float)(y[j] - (Y)base) * k;
        t = t > -200.f ? t : -200.f;   // 2^-200 is 0 in float32; keeps 0 * inf out
        const float w = __builtin_amdgcn_exp2f(t);
        s += w;
        d = __builtin_fmaf(w, t, d);
    }
    run.s += (double)s;
    run.d += (double)d;
}

// One lane's NV vectors of a tile added to its run: all loads first.  Logits without rules are summed 32 at a time, ruled ones by the vector
// (their y are doubles, and 32 of them more registers than there are).
template <typename E, bool RULES, int NV, int C>
__device__ inline void add_tile(Run& run, const Row& w, const typename E::T* x, int64_t v0, int step, int64_t width, const Rules& r, int64_t b, int64_t lo,
                                uint32_t* counts, const uint32_t* mine, double k2) {
    Raw<E, C> raw[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) raw[k].load(x, v0 + k * step, NV == 1 || v0 + k * step < width ? width : v0 + k * step);
    if constexpr (RULES) {
        if (counts && r.hist) count_ids(r, b, 1, b + 1, width, lo, kBlock * C * NV, counts);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t at = v0 + k * step;
            double y[C];
            if (at < width) ruled_cols(w, raw[k], at, width, mine ? mine + k * step : nullptr, y);
            else
#pragma unroll
                for (int j = 0; j < C; j++) y[j] = -INFINITY;
            add_cols<C>(run, y, k2);
        }
    } else {
        float y[NV * C];
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < C; j++) y[k * C + j] = raw[k].get(j);
        add_cols<NV * C>(run, y, k2);
    }
}

// The group's run from its lanes'.
template <int G>
__device__ inline void join(Run& run, double k2, double* lds) {
    const double m = group_reduce<G>(run.m, Max<double>(), lds);
    run.bad = group_reduce<G>(run.bad, Max<int>(), (int*)lds);
    if (m > -INFINITY) rebase(run, m, k2);
    run.s = group_reduce<G>(run.s, Sum<double>(), lds);
    run.d = group_reduce<G>(run.d, Sum<double>(), lds);
}

__device__ inline void finish(const Run& run, const Row& w, double ya, int64_t b, float* log_prob, float* entropy, double* log_sum) {
    if (run.bad) {
        log_prob[b] = NAN;
        entropy[b] = NAN;
        log_sum[2 * b] = 0;
        log_sum[2 * b + 1] = NAN;
        return;
    }
    const bool empty = run.m == -INFINITY;
    const double ls = empty ? 0.0 : log(run.s);
    log_prob[b] = empty ? -INFINITY : (float)((ya - run.m) / w.temp - ls);
    entropy[b] = empty ? 0.f : (float)(ls - kLn2 * (run.d / run.s));
    log_sum[2 * b] = empty ? 0.0 : run.m;   // apart: beside a mask of the type's lowest value the sum of the two would lose log S
    log_sum[2 * b + 1] = empty ? -INFINITY : ls;
}

__device__ inline int64_t action_of(const void* actions, int act64, int64_t b) {
    return act64 ? ((const int64_t*)actions)[b] : (int64_t)((const int32_t*)actions)[b];
}

// y of one column, -inf outside the row or where it is not allowed.
template <typename E>
__device__ inline double y_at(const Row& w, const typename E::T* x, int64_t width, int64_t v, const uint32_t* count) {
    if (v < 0 || v >= width) return -INFINITY;
    const bool ok = !w.nothing && (!w.mask || ((w.mask[v >> 5] >> (v & 31)) & 1u));
    return ruled(w, (float)x[v], count ? *count : 0u, ok, v);
}

template <typename E, bool RULES, int G, int NV, int C>
__global__ void __launch_bounds__(kBlock) score_rows_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r,
                                                            const void* actions, int act64, float* log_prob, float* entropy, double* log_sum) {
    constexpr int per = kBlock / G, cap = G * C * NV;
    __shared__ __align__(16) uint32_t counts[RULES ? per * cap : 4];
    __shared__ double lds[kBlock / kWave];
    const int lane = (int)threadIdx.x & (G - 1);
    const int group = G >= kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : (int)threadIdx.x / G;
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        if (RULES && r.hist) count_ids(r, band * per, per, rows, width, 0, cap, counts);
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const uint32_t* mine = RULES && r.hist ? counts + group * cap : nullptr;
        const double k2 = kLog2e / w.temp;
        Run run{-INFINITY, 0, 0, 0};
        add_tile<E, RULES, NV, C>(run, w, x, lane * C, G * C, width, r, b, 0, nullptr, mine ? mine + lane * C : nullptr, k2);
        join<G>(run, k2, lds);
        if (lane == 0 && own < rows) {
            const int64_t a = action_of(actions, act64, b);
            finish(run, w, y_at<E>(w, x, width, a, mine && a >= 0 && a < width ? mine + a : nullptr), b, log_prob, entropy, log_sum);
        }
    }
}

// Wider rows: one workgroup goes along a row, or where there are few rows along one of its `splits` parts; parts are joined by a second launch.
struct Part {
    Run run;
    double ya;
};
constexpr int kNv = 4;

template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock) score_wide_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int64_t cuts,
                                                            int splits, int64_t each, const void* actions, int act64, float* log_prob, float* entropy,
                                                            double* log_sum, Part* parts) {
    constexpr int cap = kBlock * E::kVec * kNv;
    __shared__ __align__(16) uint32_t counts[RULES ? cap : 4];
    __shared__ double lds[kBlock / kWave];
    __shared__ double the_ya;
    for (int64_t i = blockIdx.x; i < rows * splits; i += gridDim.x) {
        const int64_t b = splits == 1 ? i : i / splits;
        const int part = splits == 1 ? 0 : (int)(i - b * splits);
        const int64_t c0 = part * each, c1 = c0 + each < cuts ? c0 + each : cuts;
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const double k2 = kLog2e / w.temp;
        const int64_t a = action_of(actions, act64, b);
        Run run{-INFINITY, 0, 0, 0};
        if (threadIdx.x == 0) the_ya = -INFINITY;
        for (int64_t c = c0; c < c1; c++) {
            const int64_t lo = c * cap;
            const uint32_t* mine = RULES && r.hist ? counts : nullptr;
            add_tile<E, RULES, kNv, E::kVec>(run, w, x, lo + threadIdx.x * E::kVec, kBlock * E::kVec, width, r, b, lo, counts,
                                             mine ? mine + threadIdx.x * E::kVec : nullptr, k2);
            if (threadIdx.x == 0 && a >= lo && a < lo + cap) the_ya = y_at<E>(w, x, width, a, mine && a < width ? mine + (a - lo) : nullptr);
        }
        join<kBlock>(run, k2, lds);
        if (threadIdx.x == 0) {
            if (splits == 1) finish(run, w, the_ya, b, log_prob, entropy, log_sum);
            else parts[i] = Part{run, the_ya};
        }
        __syncthreads();
    }
}

// One wave per row joins its at most 64 parts.
__global__ void __launch_bounds__(kBlock) score_join_kernel(int64_t rows, int64_t width, int64_t cap, Rules r, int splits, int64_t each, const void* actions,
                                                            int act64, const Part* parts, float* log_prob, float* entropy, double* log_sum) {
    const int lane = (int)threadIdx.x & (kWave - 1);
    for (int64_t band = blockIdx.x; band * (kBlock / kWave) < rows; band += gridDim.x) {
        const int64_t own = band * (kBlock / kWave) + threadIdx.x / kWave;
        const int64_t b = own < rows ? own : rows - 1;
        const Row w = row_of<false>(r, b);
        Run run{-INFINITY, 0, 0, 0};
        if (lane < splits) run = parts[b * splits + lane].run;
        join<kWave>(run, kLog2e / w.temp, nullptr);
        if (lane == 0 && own < rows) {
            const int64_t a = action_of(actions, act64, b);
            finish(run, w, a >= 0 && a < width ? parts[b * splits + a / cap / each].ya : -INFINITY, b, log_prob, entropy, log_sum);
        }
    }
}

int64_t cuts_of(int vec, int64_t width) {
    const int64_t cap = (int64_t)kBlock * vec * kNv;
    return (width + cap - 1) / cap;
}
bool is_wide(int vec, int64_t width) { return width > (int64_t)kBlock * vec * kNv; }
// As many parts as bring 1024 workgroups, 64 at most, none without a tile.
void split(int vec, int64_t rows, int64_t width, int* splits, int64_t* each) {
    const int64_t cuts = cuts_of(vec, width);
    int64_t n = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    n = n > cuts ? cuts : n;
    n = n > 64 ? 64 : n;
    *each = (cuts + n - 1) / n;
    *splits = (int)((cuts + *each - 1) / *each);
}
size_t parts_bytes(int vec, int64_t rows, int64_t width) {
    if (!is_wide(vec, width)) return 0;
    int splits;
    int64_t each;
    split(vec, rows, width, &splits, &each);
    return splits == 1 ? 0 : sizeof(Part) * (size_t)rows * (size_t)splits;
}

template <typename E, bool RULES, int G, int NV, int C>
void launch_rows(const void* x, int64_t rows, int64_t width, int64_t stride, const Rules& r, const void* actions, int act64, float* lp, float* ent, double* ls,
                 hipStream_t s) {
    constexpr int per = kBlock / G;
    hipLaunchKernelGGL((score_rows_kernel<E, RULES, G, NV, C>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, (const typename E::T*)x, rows, width,
                       stride, r, actions, act64, lp, ent, ls);
}

template <typename E, bool RULES>
void launch(const void* x, int64_t rows, int64_t width, int64_t stride, const Rules& r, const void* actions, int act64, float* lp, float* ent, double* ls,
            void* ws, hipStream_t s) {
    constexpr int v = E::kVec;
    if (width <= 2) return launch_rows<E, RULES, 1, 1, 2>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 4) return launch_rows<E, RULES, 1, 1, 4>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= v) return launch_rows<E, RULES, 1, 1, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 2 * v) return launch_rows<E, RULES, 2, 1, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 4 * v) return launch_rows<E, RULES, 4, 1, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 8 * v) return launch_rows<E, RULES, 8, 1, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 16 * v) return launch_rows<E, RULES, 16, 1, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 64 * v) return launch_rows<E, RULES, 64, 1, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (width <= 64 * v * 4) return launch_rows<E, RULES, 64, 4, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    if (!is_wide(v, width)) return launch_rows<E, RULES, kBlock, kNv, v>(x, rows, width, stride, r, actions, act64, lp, ent, ls, s);
    int splits;
    int64_t each;
    split(v, rows, width, &splits, &each);
    const int64_t cuts = cuts_of(v, width);
    hipLaunchKernelGGL((score_wide_kernel<E, RULES>), dim3(grid_for(rows * splits)), dim3(kBlock), 0, s, (const typename E::T*)x, rows, width, stride, r, cuts,
                       splits, each, actions, act64, lp, ent, ls, (Part*)ws);
    if (splits > 1)
        hipLaunchKernelGGL(score_join_kernel, dim3(grid_for((rows + 3) / 4)), dim3(kBlock), 0, s, rows, width, (int64_t)kBlock * v * kNv, r, splits, each, actions,
                           act64, (const Part*)ws, lp, ent, ls);
}

}  // namespace
}  // namespace policy
}  // namespace gymhip

using namespace gymhip;
using namespace gymhip::policy;

extern "C" {

size_t gymhip_action_log_prob_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0 || width > GYMHIP_POLICY_MAX_WIDTH) return 0;
    const size_t a = parts_bytes(F32::kVec, rows, width), b = parts_bytes(F16::kVec, rows, width);
    return a > b ? a : b;
}

int gymhip_action_log_prob(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules,
                           const void* actions, int action_dtype, float* log_prob, float* entropy, double* log_sum, void* workspace,
                           size_t workspace_bytes, void* stream) {
    Rules r;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (int rc = check_actions(actions, action_dtype, rows)) return rc;
    if (rows && (!log_prob || !entropy || !log_sum)) return fail(GYMHIP_EINVAL, "log_prob, entropy or log_sum is null");
    if (int rc = check_workspace(workspace, workspace_bytes, gymhip_action_log_prob_workspace_bytes(rows, width))) return rc;
    if (!rows) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        with_bool(!r.plain(), [&](auto ruled_) {
            launch<E, decltype(ruled_)::value>(logits, rows, width, stride, r, actions, (int)(action_dtype == GYMHIP_ACT_I64), log_prob, entropy, log_sum, workspace,
                                               (hipStream_t)stream);
        });
    });
}

}  // extern "C"
