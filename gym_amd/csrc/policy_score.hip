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

// N columns' y added to a run.  NaN and +inf only mark it.
template <int N, typename Y>
__device__ inline void add_cols(Run& run, const Y* y, double k2) {
    Y m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < N; j++) {
        bad = bad || y[j] != y[j];
        m = y[j] > m ? y[j] : m;
    }
    if (bad || m == INFINITY) run.bad = 1;
    if (!(m > -INFINITY && m < INFINITY)) return;
    if ((double)m > run.m) rebase(run, (double)m, k2);
    const float k = (float)k2;
    float s = 0, d = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        // y - m where m is a float too is exact to a half step as a float; against an earlier base, which may not be one, it is taken in double
        const float gap = sizeof(Y) == 4 && N > 8 ? (float)(y[j] - m) : (float)((double)y[j] - run.m);
        float t = gap * k;
        t = t > -200.f ? t : -200.f;   // 2^-200 is 0 in float32; keeps 0 * inf out
        const float w = __builtin_amdgcn_exp2f(t);
        s += w;
        d = __builtin_fmaf(w, t, d);
    }
    if (sizeof(Y) == 4 && N > 8) {   // against the columns' own maximum: brought to the run's
        Run more{(double)m, (double)s, (double)d, 0};
        rebase(more, run.m, k2);
        run.s += more.s;
        run.d += more.d;
    } else {
        run.s += (double)s;
        run.d += (double)d;
    }
}

// A lane's columns: nv vectors from `at` on, `step` columns apart, added to its run; `place` is the first's place in the counts.  Logits without
// rules (NV vectors) are loaded first, all of them, and summed together; else it goes a vector at a time, the next one's load under way, in double
// where a bias, or a count in any of the wave's lanes, makes y differ from the logits.  count() makes the counts while the first load is under
// way.
template <typename E, bool RULES, int NV, int C, typename Count>
__device__ inline void add_columns(Run& run, const Row& w, const typename E::T* x, int64_t first, int step, int nv, int64_t width, const Counts& counts, int place,
                                   double k2, Count count) {
    if constexpr (RULES) {
        Vector<E, C> next;
        next.load(w, x, first, width);
        count();
#pragma unroll 1
        for (int k = 0; k < nv; k++) {
            const int64_t at = first + k * step;
            Vector<E, C> v = next;
            if (k + 1 < nv) next.load(w, x, at + step, width);
            if (at >= width) continue;
            if constexpr (NV == 1) {   // narrow rows: all columns alike
                double y[C];
                ruled_cols(w, v.raw, v.bits, at, width, counts, place, counts.words != nullptr, y);
                add_cols<C>(run, y, k2);
            } else {
                // the few columns with a count are left out of the straight pass, and each is added by itself by the lane that owns it
                uint32_t apart = counts.words ? counts.which<C>(place + k * step) & v.bits : 0u;
                const Raw<E, C> whole = v.raw;
                if (w.masked || __any(apart)) v.raw.keep(v.bits & ~apart);
                if (w.biased) {
                    float f[C];
                    double y[C];
                    bias_cols<C>(w, at, width, f);
#pragma unroll
                    for (int j = 0; j < C; j++) y[j] = (double)v.raw.get(j) + (double)f[j];
                    if (w.masked) {   // whatever the bias is there
#pragma unroll
                        for (int j = 0; j < C; j++) y[j] = v.bits >> j & 1 ? y[j] : -INFINITY;
                    }
                    add_cols<C>(run, y, k2);
                } else {
                    float y[C];
#pragma unroll
                    for (int j = 0; j < C; j++) y[j] = v.raw.get(j);
                    add_cols<C>(run, y, k2);
                }
                while (apart) {
                    const int j = __ffs((int)apart) - 1;
                    apart &= apart - 1;
                    const double y = ruled(w, whole.pick(j), counts.at(place + k * step + j), true, at + j);
                    add_cols<1>(run, &y, k2);
                }
            }
        }
    } else {
        Raw<E, C> raw[NV];
        uint32_t bits[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) raw[k].load(x, first + k * step, NV == 1 || first + k * step < width ? width : 0);
        if (w.masked) {
#pragma unroll
            for (int k = 0; k < NV; k++) bits[k] = allowed_bits(w, first + k * step, width);
        }
        float y[NV * C];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (w.masked) raw[k].keep(bits[k]);
#pragma unroll
            for (int j = 0; j < C; j++) y[k * C + j] = raw[k].get(j);
        }
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
__device__ inline double y_at(const Row& w, const typename E::T* x, int64_t width, int64_t v, uint32_t count) {
    if (v < 0 || v >= width) return -INFINITY;
    return ruled(w, (float)x[v], count, allowed(w, v), v);
}

// Rows in the registers of G lanes, of NV vectors each at most (nv: as many as the row has).
template <typename E, bool RULES, int G, int NV, int C>
__global__ void __launch_bounds__(kBlock) score_rows_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int nv, bool half,
                                                            const void* actions, int act64, float* log_prob, float* entropy, double* log_sum) {
    constexpr int per = kBlock / G;
    __shared__ __align__(16) uint32_t words[!RULES ? 4 : NV > 1 ? counts_words<E>() : kBlock * C];
    __shared__ double lds[kBlock / kWave];
    const int cap = G * C * nv;
    const int lane = (int)threadIdx.x & (G - 1);
    const int group = G >= kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : (int)threadIdx.x / G;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, per * cap, NV > 1 && half, NV > 1};
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;   // lanes without a row follow the last one: every exchange has all its lanes
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const double k2 = w.k2;
        Run run{-INFINITY, 0, 0, 0};
        add_columns<E, RULES, NV, C>(run, w, x, lane * C, G * C, nv, width, counts, group * cap + lane * C, k2, [&] {
            if (hist) count_ids(r, band * per, per, rows, width, 0, counts);
        });
        join<G>(run, k2, lds);
        if (lane == 0 && own < rows) {
            const int64_t a = action_of(actions, act64, b);
            finish(run, w, y_at<E>(w, x, width, a, hist && a >= 0 && a < width ? counts.at(group * cap + (int)a) : 0u), b, log_prob, entropy, log_sum);
        }
    }
}

// Wider rows: one workgroup goes along a row tile by tile, or where there are few rows along one of its `splits` parts; parts are joined by a second
// launch.
struct Part {
    Run run;
    double ya;
};

template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock) score_wide_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int nv, bool half,
                                                            int64_t cuts, int splits, int64_t each, const void* actions, int act64, float* log_prob,
                                                            float* entropy, double* log_sum, Part* parts) {
    constexpr int C = E::kVec;
    __shared__ __align__(16) uint32_t words[RULES ? counts_words<E>() : 4];
    __shared__ double lds[kBlock / kWave];
    __shared__ double the_ya;
    const int cap = kBlock * C * nv, place = (int)threadIdx.x * C;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, cap, half, true};
    for (int64_t i = blockIdx.x; i < rows * splits; i += gridDim.x) {
        const int64_t b = splits == 1 ? i : i / splits;
        const int part = splits == 1 ? 0 : (int)(i - b * splits);
        const int64_t c0 = part * each, c1 = c0 + each < cuts ? c0 + each : cuts;
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const double k2 = w.k2;
        const int64_t a = action_of(actions, act64, b);
        Run run{-INFINITY, 0, 0, 0};
        if (threadIdx.x == 0) the_ya = -INFINITY;
        for (int64_t c = c0; c < c1; c++) {
            const int64_t lo = c * cap;
            add_columns<E, RULES, kTile, C>(run, w, x, lo + place, kBlock * C, nv, width, counts, place, k2, [&] {
                if (hist) count_ids(r, b, 1, rows, width, lo, counts);
            });
            if (threadIdx.x == 0 && a >= lo && a < lo + cap) the_ya = y_at<E>(w, x, width, a, hist && a < width ? counts.at((int)(a - lo)) : 0u);
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
        join<kWave>(run, w.k2, nullptr);
        if (lane == 0 && own < rows) {
            const int64_t a = action_of(actions, act64, b);
            finish(run, w, a >= 0 && a < width ? parts[b * splits + a / cap / each].ya : -INFINITY, b, log_prob, entropy, log_sum);
        }
    }
}

// Tiles of nv vectors a lane: half as many where the counts take 32 bits.  (Without rules kTile: their loop over vectors is unrolled.)
int tile_vectors(const Rules& r) { return r.hist && !half_counts(r) ? kTile / 2 : kTile; }

// As many parts as bring 1024 workgroups, 64 at most, none without a tile.
struct Split {
    int64_t cuts, each;
    int splits;
};
Split split_of(int vec, int nv, int64_t rows, int64_t width) {
    const int64_t cap = (int64_t)kBlock * vec * nv;
    Split s;
    s.cuts = (width + cap - 1) / cap;
    int64_t n = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    n = n > s.cuts ? s.cuts : n;
    n = n > 64 ? 64 : n;
    s.each = (s.cuts + n - 1) / n;
    s.splits = (int)((s.cuts + s.each - 1) / s.each);
    return s;
}
// For any type and rules.
size_t parts_bytes(int64_t rows, int64_t width) {
    size_t most = 0;
    for (const int vec : {F32::kVec, F16::kVec})
        for (const int nv : {kTile / 2, kTile}) {
            const Split s = split_of(vec, nv, rows, width);
            const size_t bytes = s.splits > 1 ? sizeof(Part) * (size_t)rows * (size_t)s.splits : 0;
            if (width > (int64_t)kBlock * vec * nv && bytes > most) most = bytes;
        }
    return most;
}

template <typename E, bool RULES>
struct Launch {
    const typename E::T* x;
    int64_t rows, width, stride;
    const Rules& r;
    const void* actions;
    int act64;
    float *lp, *ent;
    double* ls;
    void* ws;
    hipStream_t s;

    template <int G, int NV, int C>
    void in_registers() const {
        constexpr int per = kBlock / G;
        hipLaunchKernelGGL((score_rows_kernel<E, RULES, G, NV, C>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, x, rows, width, stride, r,
                           (int)((width + G * C - 1) / (G * C)), half_counts(r), actions, act64, lp, ent, ls);
    }
    void wide(int nv) const {
        const Split p = split_of(E::kVec, nv, rows, width);
        hipLaunchKernelGGL((score_wide_kernel<E, RULES>), dim3(grid_for(rows * p.splits)), dim3(kBlock), 0, s, x, rows, width, stride, r, nv, half_counts(r),
                           p.cuts, p.splits, p.each, actions, act64, lp, ent, ls, (Part*)ws);
        if (p.splits > 1)
            hipLaunchKernelGGL(score_join_kernel, dim3(grid_for((rows + 3) / 4)), dim3(kBlock), 0, s, rows, width, (int64_t)kBlock * E::kVec * nv, r, p.splits,
                               p.each, actions, act64, (const Part*)ws, lp, ent, ls);
    }
    void operator()() const {
        constexpr int v = E::kVec;
        const int most = tile_vectors(r);
        // few columns: a row per lane, as wide as the row; then as few lanes as hold it, a 16-byte vector each; then several vectors
        if (width <= 2) in_registers<1, 1, 2>();
        else if (width <= 4) in_registers<1, 1, 4>();
        else if (width <= v) in_registers<1, 1, v>();
        else if (width <= 2 * v) in_registers<2, 1, v>();
        else if (width <= 4 * v) in_registers<4, 1, v>();
        else if (width <= 8 * v) in_registers<8, 1, v>();
        else if (width <= 16 * v) in_registers<16, 1, v>();
        else if (width <= 32 * v) in_registers<32, 1, v>();
        else if (width <= 64 * v) in_registers<64, 1, v>();
        else if (width <= 64 * v * most) in_registers<64, kTile, v>();
        else if (width <= (int64_t)kBlock * v * most) in_registers<kBlock, kTile, v>();
        else wide(most);
    }
};

}  // namespace
}  // namespace policy
}  // namespace gymhip

using namespace gymhip;
using namespace gymhip::policy;

extern "C" {

size_t gymhip_action_log_prob_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0 || width > GYMHIP_POLICY_MAX_WIDTH) return 0;
    return parts_bytes(rows, width);
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
            Launch<E, decltype(ruled_)::value>{(const typename E::T*)logits, rows, width, stride, r, actions, (int)(action_dtype == GYMHIP_ACT_I64), log_prob, entropy,
                                               log_sum, workspace, (hipStream_t)stream}();
        });
    });
}

}  // extern "C"
