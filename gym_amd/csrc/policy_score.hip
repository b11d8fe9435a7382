// policy_score.hip — log-probability and entropy of given actions under the ruled logits: one pass over the logits with a running maximum.
//
// With y the logit after penalties and bias, m the greatest y so far, t = (y - m) log2 e / T and w = 2^t:  S = sum w, D = sum w t,
// log_prob = (y_a - m) / T - ln S, entropy = ln 2 (log2 S - D / S).  t and w are float32 (their errors are relative to y - m, not to y).  Longer
// rows: a lane adds up the 4 or 8 columns of a vector (or one counted column) in float32 and goes on in double.  Rows in registers: a lane's 2 to 8 columns and then up to 64
// lanes in pairs, 512 terms at most, all in float32, 13 roundings deep.  m is the same for a wave, so that the sums hardly ever have to be brought to a new one: a few times in
// a row, by the logarithm of its length.  8,192 x 32,768 bf16: 14.6 vector instructions a column all told, the vector unit 79 % busy beside 3.9 of the 4.9 TB/s a copy reaches.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

// A running (m, S, D) over any set of columns, S and D against m.  A NaN or +inf among them makes S NaN; m = -inf: nothing yet.
struct Run {
    double m, s, d;
};

// S and D of r against another base m > r.m.
__device__ inline void rebase(Run& r, double m, double k2) {
    if (r.m > -INFINITY && r.m < m) {
        double t = (r.m - m) * k2;
        t = t > -200 ? t : -200;   // 0 at float32's precision
        const double e = exp2_double(t, 1.0);
        r.d = e * __builtin_fma(t, r.s, r.d);   // against the new base every t moves by the same amount
        r.s = e * r.s;
    }
    r.m = m;
}

// w = 2^t and w t of one column added to s and d.  A NaN gets through by w; where w is 0 (2^-200 is, in float32) t is kept finite.
__device__ inline void add_term(float t, float& s, float& d) {
    const float w = __builtin_amdgcn_exp2f(t);
    s += w;
    d = __builtin_fmaf(w, __builtin_fmaxf(t, -200.f), d);
}

// N columns' y of every lane of the wave added to the lanes' runs, whose m is the wave's.  Floats are taken from m's nearest float, and what that is off by is
// added where t is made: m may be the y of a penalty, and the column that holds it has t = 0.  Both by the same factor: a temperature's reciprocal that passes float32 is
// cut off (`finite`), and if the one were and the other not, t could rise above 0.  LOGITS: no y is anything but a logit, m is a float.
template <int N, bool LOGITS, typename Y>
__device__ inline void add_cols(Run& run, const Y* y, double k2) {
    Y top = y[0];
#pragma unroll
    for (int j = 1; j < N; j++) top = __builtin_elementwise_max(top, y[j]);
    if constexpr (LOGITS) {
        const float m = (float)run.m;
        if (__any(!(top <= m))) rebase(run, (double)group_reduce<kWave>(__builtin_fmaxf(top, m), Max<float>(), (float*)nullptr), k2);
    } else {
        if (__any(!((double)top <= run.m))) rebase(run, group_reduce<kWave>(__builtin_fmax((double)top, run.m), Max<double>(), (double*)nullptr), k2);
    }
    if (run.m == -INFINITY) {
        bool nan = false;
#pragma unroll
        for (int j = 0; j < N; j++) nan = nan || y[j] != y[j];
        if (nan) run.s = NAN;
        return;
    }
    // (below all floats, where a penalty has taken the type's lowest value: no float but -inf is under it, and -inf less -inf must not come up)
    const float k = finite(k2), m = __builtin_fmaxf((float)run.m, -3.4028235e38f);
    const float off = LOGITS || m == (float)INFINITY || run.m == (double)m ? 0.f : finite(((double)m - run.m) * __builtin_fmin(k2, 3e38));
    float s = 0, d = 0;
#pragma unroll
    for (int j = 0; j < N; j++) add_term(sizeof(Y) == 4 ? __builtin_fmaf((float)y[j] - m, k, off) : (float)(y[j] - run.m) * k, s, d);
    run.s += (double)s;
    run.d += (double)d;
}

// A lane's columns: nv vectors from `first` on, `step` columns apart, added to its run, one at a time with the next one's load under way; `place` is the first's
// place in the counts.  count() makes the counts while the first load is under way.
template <typename E, bool RULES, typename Count>
__device__ inline void add_columns(Run& run, const Row& w, const typename E::T* x, int64_t first, int step, int nv, int64_t width, const Counts& counts, int place,
                                   double k2, Count count) {
    constexpr int C = E::kVec;
    Vector<E, C> next;
    next.load(w, x, first, width);
    count();
#pragma unroll 1
    for (int k = 0; k < nv; k++) {
        const int64_t at = first + (int64_t)k * step;
        Vector<E, C> v = next;
        if (k + 1 < nv) next.load(w, x, at + step, width);
        // the few columns with a count are left out of the straight pass, and each is added by itself by the lane that owns it
        uint32_t apart = RULES && counts.words ? counts.which<C>(place + k * step) & v.bits : 0u;
        const Raw<E, C> whole = v.raw;
        if (w.masked || (RULES && __any(apart))) v.raw.keep(v.bits & ~apart);
        if (RULES && w.biased) {
            float f[C];
            double y[C];
            bias_cols<C>(w, at, width, f);
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = (double)v.raw.get(j) + (double)f[j];
            if (w.masked) {   // whatever the bias is there
#pragma unroll
                for (int j = 0; j < C; j++) y[j] = v.bits >> j & 1 ? y[j] : -INFINITY;
            }
            add_cols<C, false>(run, y, k2);
        } else {
            float y[C];
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = v.raw.get(j);
            add_cols<C, !RULES>(run, y, k2);
        }
        if constexpr (RULES) {
            while (__any(apart)) {   // lanes without one add nothing
                const int j = __ffs((int)apart) - 1;
                const double y = apart ? ruled(w, whole.pick(j < 0 ? 0 : j), counts.at(place + k * step + (j < 0 ? 0 : j)), true, at + j) : -(double)INFINITY;
                apart &= apart - 1;
                add_cols<1, false>(run, &y, k2);
            }
        }
    }
}

// The group's run from its lanes': the waves', each against its m, and for a workgroup these.
template <int G>
__device__ inline void join(Run& run, double k2, Run* lds) {
    run.s = group_reduce<kWave>(run.s, Sum<double>(), (double*)nullptr);
    run.d = group_reduce<kWave>(run.d, Sum<double>(), (double*)nullptr);
    if (G == kWave) return;
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = run;
    __syncthreads();
    double m = lds[0].m;
    for (int i = 1; i < kBlock / kWave; i++) m = __builtin_fmax(m, lds[i].m);
    run = Run{m, 0, 0};
    for (int i = 0; i < kBlock / kWave; i++) {
        Run one = lds[i];
        rebase(one, m, k2);
        run.s += one.s;
        run.d += one.d;
    }
}

__device__ inline void finish(const Run& run, const Row& w, double ya, int64_t b, float* log_prob, float* entropy, double* log_sum) {
    if (run.s != run.s) {
        log_prob[b] = NAN;
        entropy[b] = NAN;
        log_sum[2 * b] = 0;
        log_sum[2 * b + 1] = NAN;
        return;
    }
    const bool empty = run.m == -INFINITY;
    const double l2 = empty ? 0.0 : log2_double(run.s), ls = l2 * kLn2;
    double inv = empty ? 0.0 : __builtin_amdgcn_rcp(run.s);   // and a Newton step: 1e-14 of it
    inv = __builtin_fma(__builtin_fma(-run.s, inv, 1.0), inv, inv);
    log_prob[b] = empty ? -INFINITY : (float)(((ya - run.m) * w.k2 - l2) * kLn2);
    entropy[b] = empty ? 0.f : (float)((l2 - run.d * inv) * kLn2);
    log_sum[2 * b] = empty ? 0.0 : run.m;   // apart: beside a mask of the type's lowest value the sum of the two would lose log S
    log_sum[2 * b + 1] = empty ? -INFINITY : ls;
}

__device__ inline int64_t action_of(const void* actions, int act64, int64_t b) {
    return act64 ? ((const int64_t*)actions)[b] : (int64_t)((const int32_t*)actions)[b];
}

// The run of a group whose lanes hold all of its columns, C each: the greatest first, the sums against it.
template <int G, int C, typename Y>
__device__ inline Run run_of(const Y* y, double k2) {
    Y m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < C; j++) {
        bad = bad || !(y[j] < (Y)INFINITY);
        m = __builtin_elementwise_max(m, y[j]);
    }
    m = group_reduce<G>(bad ? (Y)INFINITY : m, Max<Y>(), (Y*)nullptr);
    if (m == (Y)INFINITY) return Run{(double)m, NAN, 0};
    if (m == -(Y)INFINITY) return Run{(double)m, 0, 0};
    const float k = finite(k2);
    float s = 0, d = 0;
#pragma unroll
    for (int j = 0; j < C; j++) add_term((float)(y[j] - m) * k, s, d);
    return Run{(double)m, (double)group_reduce<G>(s, Sum<float>(), (float*)nullptr), (double)group_reduce<G>(d, Sum<float>(), (float*)nullptr)};
}

// The action of a row and its logit, read early: both are on their way while the row is summed.
template <typename E>
struct Chosen {
    int64_t a;
    float x;
    bool inside, open;
    __device__ Chosen(const Row& w, const typename E::T* row, int64_t width, const void* actions, int act64, int64_t b) {
        a = action_of(actions, act64, b);
        inside = a >= 0 && a < width;
        x = inside ? (float)row[a] : 0.f;
        open = inside && allowed(w, a);
    }
    __device__ double y(const Row& w, uint32_t count) const { return open ? ruled(w, x, count, true, a) : -INFINITY; }
};

// Rows in the registers of G <= 64 lanes, a vector each.  Where several lanes share a row bound by the vector unit, by what it takes to join and finish it (1,048,576 x 18 f32:
// 59 us, 81 % busy); of 2 to 4 columns by the launch and the memory (1,048,576 x 3: 12 us, 27 %, 3.4 TB/s, of which 24 bytes a row are the results).
template <typename E, bool RULES, int G, int C>
__global__ void __launch_bounds__(kBlock) score_rows_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, const void* actions,
                                                            int act64, float* log_prob, float* entropy, double* log_sum) {
    constexpr int per = kBlock / G, cap = G * C;
    __shared__ __align__(16) uint32_t words[RULES ? per * cap : 4];
    const int lane = (int)threadIdx.x & (G - 1);
    const int group = G >= kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : (int)threadIdx.x / G;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, per * cap, false, false};
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;   // lanes without a row follow the last one: every exchange has all its lanes
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        Vector<E, C> v;
        v.load(w, x, lane * C, width);
        const Chosen<E> chosen(w, x, width, actions, act64, b);
        Run run;
        if (RULES && (hist || w.biased)) {
            if (hist) count_ids(r, band * per, per, rows, width, 0, counts);
            double y[C];
            ruled_cols(w, v.raw, v.bits, lane * C, width, counts, group * cap + lane * C, hist, y);
            run = run_of<G, C>(y, w.k2);
        } else {
            if (w.masked) v.raw.keep(v.bits);
            float y[C];
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = v.raw.get(j);
            run = run_of<G, C>(y, w.k2);
        }
        if (lane == 0 && own < rows) finish(run, w, chosen.y(w, hist && chosen.inside ? counts.at(group * cap + (int)chosen.a) : 0u), b, log_prob, entropy, log_sum);
    }
}

// Longer rows, by a wave each (G = 64) or a workgroup; under a history nv vectors are a tile, which holds the row.
template <typename E, bool RULES, int G>
__global__ void __launch_bounds__(kBlock) score_strips_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int nv, bool half,
                                                              const void* actions, int act64, float* log_prob, float* entropy, double* log_sum) {
    constexpr int C = E::kVec, per = kBlock / G;
    __shared__ __align__(16) uint32_t words[RULES ? strip_words<G>() : 4];
    __shared__ Run lds[kBlock / kWave];
    const int cap = G * C * nv;
    const int lane = (int)threadIdx.x & (G - 1), group = G == kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : 0;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, per * cap, half, true};
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const Chosen<E> chosen(w, x, width, actions, act64, b);
        Run run{-INFINITY, 0, 0};
        add_columns<E, RULES>(run, w, x, lane * C, G * C, nv, width, counts, group * cap + lane * C, w.k2, [&] {
            if (hist) count_ids(r, band * per, per, rows, width, 0, counts);
        });
        join<G>(run, w.k2, lds);
        if (lane == 0 && own < rows) finish(run, w, chosen.y(w, hist && chosen.inside ? counts.at(group * cap + (int)chosen.a) : 0u), b, log_prob, entropy, log_sum);
    }
}

// Wider rows: one workgroup goes along a row tile by tile, or where there are few rows along one of its `splits` parts; parts are joined by a second
// launch.  (Launch bounds under rules: registers for four waves a SIMD; 512 x 131,072 bf16 under all rules 168 -> 118 us.)
struct Part {
    Run run;
    double ya;
};

template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock, RULES ? 4 : 1) score_wide_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int nv, bool half,
                                                            int64_t cuts, int splits, int64_t each, const void* actions, int act64, float* log_prob,
                                                            float* entropy, double* log_sum, Part* parts) {
    constexpr int C = E::kVec;
    __shared__ __align__(16) uint32_t words[RULES ? strip_words<kBlock>() : 4];
    __shared__ Run lds[kBlock / kWave];
    const int cap = kBlock * C * nv, place = (int)threadIdx.x * C;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, cap, half, true};
    for (int64_t i = blockIdx.x; i < rows * splits; i += gridDim.x) {
        const Cut at_part(i, (uint32_t)splits, rows);
        const int64_t b = at_part.row;
        const int part = (int)at_part.cut;
        const int64_t c0 = part * each, c1 = c0 + each < cuts ? c0 + each : cuts;
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const Chosen<E> chosen(w, x, width, actions, act64, b);
        Run run{-INFINITY, 0, 0};
        double ya = chosen.y(w, 0u);
        if (hist) {
            for (int64_t c = c0; c < c1; c++) {
                const int64_t lo = c * cap;
                add_columns<E, RULES>(run, w, x, lo + place, kBlock * C, nv, width, counts, place, w.k2, [&] { count_ids<false>(r, b, 1, rows, width, lo, counts); });
                if (chosen.inside && chosen.a >= lo && chosen.a < lo + cap) ya = chosen.y(w, counts.at((int)(chosen.a - lo)));
            }
        } else {
            add_columns<E, RULES>(run, w, x, c0 * cap + place, kBlock * C, (int)(c1 - c0) * nv, width, counts, place, w.k2, [] {});
        }
        join<kBlock>(run, w.k2, lds);
        if (threadIdx.x == 0) {
            if (splits == 1) finish(run, w, ya, b, log_prob, entropy, log_sum);
            else parts[b * splits + part] = Part{run, ya};
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
        Run run{-INFINITY, 0, 0};
        if (lane < splits) run = parts[b * splits + lane].run;
        rebase(run, group_reduce<kWave>(run.m, Max<double>(), (double*)nullptr), w.k2);
        join<kWave>(run, w.k2, nullptr);
        if (lane == 0 && own < rows) {
            const int64_t a = action_of(actions, act64, b);
            finish(run, w, a >= 0 && a < width ? parts[b * splits + a / cap / each].ya : -INFINITY, b, log_prob, entropy, log_sum);
        }
    }
}

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
        for (const int nv : {4096 / (kBlock * vec), 8192 / (kBlock * vec)}) {
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

    template <int G, int C>
    void in_registers() const {
        constexpr int per = kBlock / G;
        hipLaunchKernelGGL((score_rows_kernel<E, RULES, G, C>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, x, rows, width, stride, r, actions, act64, lp,
                           ent, ls);
    }
    template <int G>
    void strips(int64_t nv) const {
        constexpr int per = kBlock / G;
        hipLaunchKernelGGL((score_strips_kernel<E, RULES, G>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, x, rows, width, stride, r, (int)nv,
                           half_counts(r), actions, act64, lp, ent, ls);
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
        const int most = strip_vectors<E>(r, kBlock), wave_most = strip_vectors<E>(r, kWave);
        const auto need = [&](int g) { return (width + g * v - 1) / (g * v); };   // vectors a lane
        // few columns: a row per lane, as wide as the row; then as few lanes as hold it, a 16-byte vector each; then several vectors: by a wave a row where
        // there are rows enough (bf16 8192 x 2,083: 14 us, by a workgroup a row 30; f32 4096 x 8,192: 22 and 27; f32 1024 x 8,192: 15 and 10), by a workgroup,
        // and in parts where few rows are long (f32 64 x 32,768: 12 us, unsplit 20)
        int g = 1;
        while (g < kWave && width > g * v) g *= 2;
        g = lanes_for(r, rows, g);
        if (width <= kWave * v && g <= kWave) {
            if (g == 1 && width <= 2) in_registers<1, 2>();
            else if (g == 1 && width <= 4) in_registers<1, 4>();
            else if (g == 1) in_registers<1, v>();
            else if (g == 2) in_registers<2, v>();
            else if (g == 4) in_registers<4, v>();
            else if (g == 8) in_registers<8, v>();
            else if (g == 16) in_registers<16, v>();
            else if (g == 32) in_registers<32, v>();
            else in_registers<64, v>();
        }
        else if (need(kWave) <= (r.hist ? wave_most : 32) && (need(kWave) <= 4 || rows >= 128 * need(kWave)) && (g <= kWave || rows >= 128 * need(kWave)))
            strips<kWave>(need(kWave));
        else if (need(kBlock) <= most || (!r.hist && (need(kBlock) <= 8 || rows >= 1024))) strips<kBlock>(need(kBlock));
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
    if (int rc = check_results(logits, type, rows, width, stride, {{"log_prob", log_prob, rows * 4}, {"entropy", entropy, rows * 4}, {"log_sum", log_sum, rows * 16}})) return rc;
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
