// policy_sample.hip — one action per row from softmax of the ruled logits, and its log-probability.
//
// The action is the least column whose running sum of exp(y / T) passes u times the whole sum.  Everything that decides it is in double: two
// neighbouring columns of a flat row of 2^17 lie 8e-6 of the sum apart, about what float32 sums of them are off by, and the same logits are to
// give the same action however the row is laid out and split: they do but for levels within about 1e-13 of the sum of a border (the weights' 4e-14).  Doubles run at the rate of floats here (30e12 a second, measured), the
// exponential is the 14 instructions of exp2_double, and a double's range lets one pass do without the maximum.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

// A weight: 2^(d k2), d = y - base; never 0, for it stops at 2^-1000: what cannot be chosen (a masked column, one behind the row's end) weighs that much, and walk and
// find_part tell it by its size.
__device__ inline double weight(double d, const Heat& c) { return exp2_double(__builtin_fmax(d, c.least), c.k2); }

// Where a lane stands in its row: `at` its first column, `step` the columns from one of its vectors to the next, `place` its first column's place in
// the counts.
struct Place {
    int64_t at, width;
    int step, place;
    Counts counts;   // words null: no history
};

// f(y) for the y of vector k: floats where they are the logits themselves, else (under a bias, or where a lane of the wave has a count) doubles.
template <typename E, bool RULES, int C, typename F>
__device__ inline void with_y(const Row& w, const Place& p, int k, Vector<E, C> v, F f) {
    if constexpr (RULES) {
        const bool counted = p.counts.any<C>(p.place + k * p.step);
        if (counted || w.biased) {
            double y[C];
            ruled_cols(w, v.raw, v.bits, p.at + k * p.step, p.width, p.counts, p.place + k * p.step, counted, y);
            f(y);
            return;
        }
    }
    if (w.masked) v.raw.keep(v.bits);
    float y[C];
#pragma unroll
    for (int j = 0; j < C; j++) y[j] = v.raw.get(j);
    f(y);
}

// A vector's weights e against `base`, and their sum.
template <int C, typename Y>
__device__ inline double weigh(const Y* y, double base, const Heat& c, double* e) {
    double s = 0;
#pragma unroll
    for (int j = 0; j < C; j++) s += e[j] = weight((double)y[j] - base, c);
    return s;
}
// The same against 0.  A double holds 2^-900 .. 2^900 at full precision, so nothing has to be known of the greatest y beforehand: this is all there
// is to do where no y is above `most` nor a NaN and the row's sum is above kLeastSum.  The level is 2^-53 of that at least, beside which a double does not see the weights
// of 2^-1000: in one lane's running sum they are nothing.  *beyond: the wave's lanes that have such a y (as a lane mask: one
// vector instruction a column).
constexpr double kLeastSum = 0x1p-800;
template <int C, typename Y>
__device__ inline double weigh_0(const Y* y, const Heat& c, double* e, uint64_t* beyond) {
    double s = 0;
#pragma unroll
    for (int j = 0; j < C; j++) {
        *beyond |= __ballot(!(y[j] <= (Y)c.most));
        s += e[j] = weight((double)y[j], c);
    }
    return s;
}
// The sum of vector k's weights against 0, in no order of columns: the few columns with a count are left out of the straight pass, which then is no
// dearer than one without a history, and each is gone through by itself afterwards by the lane that owns it.
template <typename E, bool RULES>
__device__ inline double weigh_apart(const Row& w, const Place& p, int k, Vector<E, E::kVec> v, const Heat& c, uint64_t* beyond) {
    constexpr int C = E::kVec;
    double e[C];
    if constexpr (!RULES) {
        double s = 0;
        with_y<E, false, C>(w, p, k, v, [&](const auto* y) { s = weigh_0<C>(y, c, e, beyond); });
        return s;
    } else {
        const int64_t at = p.at + k * p.step;
        const int place = p.place + k * p.step;
        uint32_t apart = p.counts.words ? p.counts.which<C>(place) & v.bits : 0u;
        const Raw<E, C> whole = v.raw;
        if (w.masked || __any(apart)) v.raw.keep(v.bits & ~apart);
        double s;
        if (w.biased) {
            float f[C];
            double y[C];
            bias_cols<C>(w, at, p.width, f);
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = (double)v.raw.get(j) + (double)f[j];
            s = weigh_0<C>(y, c, e, beyond);
        } else {
            float y[C];
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = v.raw.get(j);
            s = weigh_0<C>(y, c, e, beyond);
        }
        while (apart) {
            const int j = __ffs((int)apart) - 1;
            apart &= apart - 1;
            const double y = ruled(w, whole.pick(j), p.counts.at(place + j), true, at + j);
            s += weigh_0<1>(&y, c, e, beyond);
        }
        return s;
    }
}
__device__ inline bool mine_in(uint64_t lanes) { return lanes >> (threadIdx.x & (kWave - 1)) & 1; }

// The sum of a group's weights against `base`; bad: a NaN or +inf is among its y.
struct Mass {
    double base, sum;
    bool bad;
};

// The greatest y of a group's columns (nv vectors a lane), whatever it is (-inf: there is none at all), the sum against it, and the first column that
// holds it: for greedy rows, and the rare ones out of weigh_0's range.
template <typename E, bool RULES, int G, int C>
__device__ inline Mass sum_against_max(const typename E::T* x, const Row& w, const Place& p, int nv, const Heat& c, double* lds, long long* first) {
    double m = -INFINITY, sum = 0;
    int best = 0;
    bool bad = false;
#pragma unroll 1
    for (int k = 0; k < nv; k++) {
        Vector<E, C> v;
        v.load(w, x, p.at + k * p.step, p.width);
        with_y<E, RULES, C>(w, p, k, v, [&](const auto* y) {
            auto top = y[0];
            bool nan = top != top;
#pragma unroll
            for (int j = 1; j < C; j++) {
                nan = nan || y[j] != y[j];
                top = y[j] > top || top != top ? y[j] : top;
            }
            if (nan || top == INFINITY) bad = true;
            if (nan || !(top > -INFINITY && top < INFINITY)) return;
            if ((double)top > m) {   // never from -inf with a sum
                sum = sum > 0 ? sum * weight(m - (double)top, c) : 0.0;
                m = (double)top;
                best = k;
            }
            double e[C];
            sum += weigh<C>(y, m, c, e);
        });
    }
    const double top = group_reduce<G>(m, Max<double>(), lds);
    sum = m > -INFINITY ? sum * weight(m - top, c) : 0.0;
    Mass mass;
    mass.base = top;
    mass.sum = group_reduce<G>(sum, Sum<double>(), lds);
    mass.bad = group_reduce<G>((int)bad, Max<int>(), (int*)lds) != 0;
    long long at = p.width;
    if (__any(w.greedy)) {   // each lane's first greatest, of which its vector is known
        Vector<E, C> v;
        v.load(w, x, p.at + best * p.step, p.width);
        with_y<E, RULES, C>(w, p, best, v, [&](const auto* y) {
#pragma unroll
            for (int j = C - 1; j >= 0; j--)
                if ((double)y[j] == top) at = p.at + best * p.step + j;
        });
    }
    *first = group_reduce<G>(at, Min<long long>(), (long long*)lds);
    return mass;
}

// The column (0 = the first of the lanes' vectors) of W lanes' vectors that the running sum passes `level` in: e[] a lane's weights, s their sum.  The lanes' running sums are
// added up in different orders, so one may pass the level by a last bit in a lane, or a column, that adds nothing.  Hence what weighs at most `tiny`, 2^-80 of the whole, is
// not chosen: columns up to `tiny`, and lanes up to twice C of those (a lane with more has a column with more, whatever its sum's rounding).
// Should rounding leave the level above all sums, the last column that counts is taken.
template <int W, int C>
__device__ inline int walk(const double* e, double s, double before, double level, double tiny) {
    const int self = (int)(threadIdx.x & (kWave - 1)), lane = self & (W - 1);
    const double upto = running_sum<W>(s, lane);
    int first = self;
    if (W > 1) {
        const uint64_t group = W == 64 ? ~0ull : ((1ull << W) - 1) << (self & ~(W - 1));
        const uint64_t any = __ballot(s > tiny * (2 * C)) & group, hits = __ballot(before + upto > level) & any;
        first = hits ? __ffsll((unsigned long long)hits) - 1 : any ? 63 - __clzll((long long)any) : self;
    }
    // every lane walks its own vector; the chosen lane's answer counts
    double acc = before + (upto - s);
    int at = C;
#pragma unroll
    for (int j = 0; j < C; j++) {
        acc += e[j];
        at = at == C && acc > level && (W == 1 || e[j] > tiny) ? j : at;   // (a lane by itself adds in the columns' order, see kLeastSum)
    }
    if (__any(at == C)) {
        int last = 0;
#pragma unroll
        for (int j = 0; j < C; j++) last = e[j] > tiny ? j : last;
        at = at == C ? last : at;
    }
    if (W > 1) at = __shfl(at, first);
    return (first & (W - 1)) * C + at;
}

// A row's answer, by one lane: `at` its chosen column unless there is none, and where the lane has them that column's weight and logit.  The logarithm of a weight by itself and the sum's
// differ by 1e-16 of y: a column that is all of the sum has probability 1 for certain, and none has more.
template <typename E>
__device__ inline void answer(const Row& w, const typename E::T* x, const Mass& mass, int64_t at, uint32_t count, const Heat& c, int64_t b,
                              int32_t* actions, float* log_prob, const double* chosen, const float* logit) {
    const bool none = mass.bad || mass.base == -INFINITY;
    actions[b] = none ? -1 : (int32_t)at;
    float lp = mass.bad ? NAN : -INFINITY;
    if (!none) {
        const double y = ruled(w, logit ? *logit : (float)x[at], count, true, at) - mass.base;
        const double share = chosen ? *chosen : weight(y, c);
        lp = share >= mass.sum ? 0.0f : (float)__builtin_fmin((y * c.k2 - log2_double(mass.sum)) * kLn2, 0.0);
    }
    log_prob[b] = lp;
}

// (Launch bounds under rules: registers for four waves a SIMD; 512 x 131,072 bf16 under all rules 177 -> 158 us, f32 1,000,000 x 18 after 300 ids 464 -> 360.)

// Rows of at most G * C columns, G <= 64: one vector a lane, kBlock / G rows per workgroup.
template <typename E, bool RULES, int G, int C>
__global__ void __launch_bounds__(kBlock, RULES ? 4 : 1) sample_vectors_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                                int32_t* actions, float* log_prob) {
    constexpr int per = kBlock / G, cap = G * C;
    __shared__ __align__(16) uint32_t words[RULES ? per * cap : 4];
    const int lane = (int)threadIdx.x & (G - 1);
    const int group = G == kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : (int)threadIdx.x / G;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, per * cap, false, false};
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;   // lanes without a row follow the last one: every exchange has all its lanes
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const Place p{lane * C, width, G * C, group * cap + lane * C, counts};
        Vector<E, C> v;
        v.load(w, x, p.at, width);
        if (hist) count_ids(r, band * per, per, rows, width, 0, counts);
        const Heat c = w;
        double s = 0, e[C];
        uint64_t beyond = 0;
        with_y<E, RULES, C>(w, p, 0, v, [&](const auto* y) { s = weigh_0<C>(y, c, e, &beyond); });
        Mass mass{0.0, group_reduce<G>(w.greedy || mine_in(beyond) ? (double)NAN : s, Sum<double>(), (double*)nullptr), false};
        const bool whole = mass.sum > kLeastSum;
        long long first = 0;
        if (__any(!whole)) {   // the same for all lanes that exchange
            const Mass other = sum_against_max<E, RULES, G, C>(x, w, p, 1, c, nullptr, &first);
            if (!whole) {
                mass = other;
                const double base = mass.base > -INFINITY ? mass.base : 0.0;
                with_y<E, RULES, C>(w, p, 0, v, [&](const auto* y) { s = weigh<C>(y, base, c, e); });
            }
        }
        int64_t at = walk<G, C>(e, s, 0.0, row_uniform(keys, b) * mass.sum, mass.sum * 0x1p-80);
        if (w.greedy) at = first;
        double chosen = e[0];
        float logit = v.raw.get(0);
#pragma unroll
        for (int j = 1; j < C; j++) {
            chosen = at == j ? e[j] : chosen;
            logit = at == j ? v.raw.get(j) : logit;
        }
        if (lane == 0 && own < rows)
            answer<E>(w, x, mass, at, hist && at < width ? words[group * cap + at] : 0u, c, b, actions, log_prob, G == 1 ? &chosen : nullptr, G == 1 ? &logit : nullptr);
    }
}

// Where the running sum of n parts passes `level`, 64 parts at a time, by each wave for itself: the part, or the last one should rounding leave the level
// above all sums (*past); *before: what comes before it.  Parts of at most `tiny` are not chosen (see walk).
template <typename F>
__device__ inline int64_t find_part(int64_t n, double level, double tiny, F part_sum, double* before, bool* past) {
    const int lane = (int)threadIdx.x & (kWave - 1);
    int64_t last = 0;
    double run = 0;
    for (int64_t c0 = 0; c0 < n; c0 += kWave) {
        const double e = c0 + lane < n ? part_sum(c0 + lane) : 0.0;
        const double upto = running_sum<kWave>(e, lane);
        const uint64_t some = __ballot(e > tiny), hits = __ballot(run + upto > level) & some;
        if (hits) {
            const int at = __ffsll((unsigned long long)hits) - 1;
            *before = run + __shfl(upto - e, at);
            *past = false;
            return c0 + at;
        }
        if (some) last = c0 + 63 - __clzll((long long)some);
        run += __shfl(upto, kWave - 1);
    }
    *before = 0;
    *past = true;
    return last;
}

// Vectors a lane in a strip of a wave without a history, at most (a workgroup's: a quarter), and where which is taken.  Rows of a wave each are done in fewer
// instructions, a workgroup a row has four times the waves for few rows, parts and a join sixteen times.  Measured, us, wave / workgroup / parts:
// bf16 8192 x 2,083: 26 / 48 / -; f32 8192 x 4,097: 38 / 72 / 117; f32 512 x 16,384: 34 / 14 / 20; bf16 64 x 32,768: 44 / 14.5 / 12.8.
constexpr int kLong = 256;

// A strip of a row: the columns of G = 64 or kBlock lanes, nv vectors each, gone through one vector at a time with the next one's load
// under way: few registers, so that many waves are there to wait for memory and for the workgroup's barriers.
template <typename E, typename F>
__device__ inline void each_vector(const Row& w, const typename E::T* x, const Place& p, int nv, Vector<E, E::kVec> next, F f) {
#pragma unroll 1
    for (int k = 0; k < nv; k++) {
        const Vector<E, E::kVec> v = next;
        if (k + 1 < nv) next.load(w, x, p.at + (k + 1) * p.step, p.width);
        f(k, v);
    }
}

// sums[k * waves + wave]: the sum of each wave's k-th vectors against `base`.  v0: this lane's first vector.
template <typename E, bool RULES, int G>
__device__ inline void strip_sums(const typename E::T* x, const Vector<E, E::kVec>& v0, const Row& w, const Place& p, int nv, const Heat& c, double base,
                                  double* sums) {
    constexpr int C = E::kVec, M = G / kWave;
    const int wave = G > kWave ? (int)threadIdx.x / kWave : 0;
    group_sync<G>();
    each_vector<E>(w, x, p, nv, v0, [&](int k, const Vector<E, C>& v) {
        double s = 0, e[C];
        with_y<E, RULES, C>(w, p, k, v, [&](const auto* y) { s = weigh<C>(y, base, c, e); });
        s = group_reduce<kWave>(s, Sum<double>(), (double*)nullptr);
        if ((threadIdx.x & (kWave - 1)) == 0) sums[k * M + wave] = s;
    });
    group_sync<G>();
}

// The sum of a strip.  KEEP: and against 0 what strip_sums would leave, *kept; else that pass is still to be made.
template <typename E, bool RULES, int G, bool KEEP>
__device__ inline Mass sum_strip(const typename E::T* x, const Vector<E, E::kVec>& v0, const Row& w, const Place& p, int nv, const Heat& c, double* lds,
                                 long long* first, double* sums, bool* kept) {
    constexpr int C = E::kVec, M = G / kWave;
    if (KEEP) *kept = false;
    if (!w.greedy) {   // one row's: all lanes alike
        double sum = 0;
        uint64_t beyond = 0;
        if constexpr (KEEP) {
            const int wave = G > kWave ? (int)threadIdx.x / kWave : 0;
            group_sync<G>();
            each_vector<E>(w, x, p, nv, v0, [&](int k, const Vector<E, C>& v) {
                double s = weigh_apart<E, RULES>(w, p, k, v, c, &beyond);
                s = group_reduce<kWave>(mine_in(beyond) ? (double)NAN : s, Sum<double>(), (double*)nullptr);
                if ((threadIdx.x & (kWave - 1)) == 0) sums[k * M + wave] = s;
                sum += s;
            });
            if (G > kWave) sum = group_reduce<G>((threadIdx.x & (kWave - 1)) == 0 ? sum : 0.0, Sum<double>(), lds);
            group_sync<G>();
        } else {
            each_vector<E>(w, x, p, nv, v0, [&](int k, const Vector<E, C>& v) { sum += weigh_apart<E, RULES>(w, p, k, v, c, &beyond); });
            sum = group_reduce<G>(mine_in(beyond) ? (double)NAN : sum, Sum<double>(), lds);
        }
        if (sum > kLeastSum) {
            if (KEEP) *kept = true;
            return Mass{0.0, sum, false};
        }
    }
    return sum_against_max<E, RULES, G, C>(x, w, p, nv, c, lds, first);
}

// The column of a strip (0 = its first) that the running sum passes `level` in; sums as strip_sums left them for the same base, which is finite, and
// `sum` the strip's.
template <typename E, bool RULES, int G>
__device__ inline int locate(const typename E::T* x, const Row& w, const Place& p, int nv, const Heat& c, double base, double sum, double level,
                             const double* sums, int* lds_at) {
    constexpr int C = E::kVec, M = G / kWave;
    const int wave = G > kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave) : 0;
    const double tiny = sum * 0x1p-80;
    double before;
    bool past;
    // (a wave's 64 vectors with more than this have a lane with more than walk's 2 C tiny; one of at most 256 such parts has)
    const int part = __builtin_amdgcn_readfirstlane((int)find_part(nv * M, level, tiny * (256 * C), [&](int64_t i) { return sums[i]; }, &before, &past));   // (vector, wave)
    if (past) level = INFINITY;
    const int k = part / M, at_wave = part - k * M;
    int column = 0;
    if (wave == at_wave) {
        Vector<E, C> v;
        v.load(w, x, p.at + k * p.step, p.width);
        double s = 0, e[C];
        with_y<E, RULES, C>(w, p, k, v, [&](const auto* y) { s = weigh<C>(y, base, c, e); });
        column = (k * G + at_wave * kWave) * C + walk<kWave, C>(e, s, before, level, tiny);
        if (G > kWave && (threadIdx.x & (kWave - 1)) == 0) *lds_at = column;
    }
    if (G > kWave) {
        __syncthreads();
        column = *lds_at;
        __syncthreads();
    }
    return column;
}

// Rows of one strip: by a wave each (G = 64), or a workgroup.
template <typename E, bool RULES, int G>
__global__ void __launch_bounds__(kBlock, RULES ? 4 : 1) sample_strips_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                               int nv, bool half, int32_t* actions, float* log_prob) {
    constexpr int C = E::kVec, per = kBlock / G;
    __shared__ __align__(16) uint32_t words[RULES ? strip_words<G>() : 4];
    __shared__ double lds[kBlock / kWave];
    __shared__ double few[per][RULES ? 8192 / (kWave * E::kVec) : kLong];   // sums of vectors; of many, where there are no counts, in their place
    __shared__ int lds_at;
    const int cap = G * C * nv;
    const int lane = (int)threadIdx.x & (G - 1), group = G == kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : 0;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, per * cap, half, true};
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const Place p{lane * C, width, G * C, group * cap + lane * C, counts};
        Vector<E, C> v;
        v.load(w, x, p.at, width);
        if (hist) count_ids(r, band * per, per, rows, width, 0, counts);
        const Heat c = w;
        double* const sums = RULES && !hist ? (double*)words + group * kLong : few[group];
        long long first = 0;
        bool kept;
        const Mass mass = sum_strip<E, RULES, G, true>(x, v, w, p, nv, c, lds, &first, sums, &kept);
        int64_t at = first;
        if (!w.greedy && !mass.bad && mass.base > -INFINITY) {   // the group's lanes alike
            if (!kept) strip_sums<E, RULES, G>(x, v, w, p, nv, c, mass.base, sums);
            at = locate<E, RULES, G>(x, w, p, nv, c, mass.base, mass.sum, row_uniform(keys, b) * mass.sum, sums, &lds_at);
        }
        if (lane == 0 && own < rows) answer<E>(w, x, mass, at, hist && at < width ? counts.at(group * cap + (int)at) : 0u, c, b, actions, log_prob, nullptr, nullptr);
    }
}

// Wider rows: one workgroup per strip leaves the sum of the strip's weights, against which base, and where in a greedy row that base (its
// greatest y) is first; then one workgroup per row joins them, finds the strip that the level falls into and goes through that strip once more.
struct Part {
    double base, sum;   // an empty part: -inf, 0;  one with a NaN or +inf: sum NaN
    long long first;
};

template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock, RULES ? 4 : 1) sample_parts_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int nv, bool half,
                                                              int64_t cuts, Part* parts) {
    constexpr int C = E::kVec;
    __shared__ __align__(16) uint32_t words[RULES ? strip_words<kBlock>() : 4];
    __shared__ double lds[kBlock / kWave];
    const int cap = kBlock * C * nv, place = (int)threadIdx.x * C;
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, cap, half, true};
    for (int64_t i = blockIdx.x; i < rows * cuts; i += gridDim.x) {
        const Cut at_cut(i, (uint32_t)cuts, rows);
        const int64_t b = at_cut.row, lo = (int64_t)at_cut.cut * cap;
        const Row w = row_of<RULES>(r, b);
        const Place p{lo + place, width, kBlock * C, place, counts};
        const typename E::T* x = x0 + b * stride;
        Vector<E, C> v;
        v.load(w, x, p.at, width);
        if (hist) count_ids<false>(r, b, 1, rows, width, lo, counts);
        long long first = 0;
        const Mass mass = sum_strip<E, RULES, kBlock, false>(x, v, w, p, nv, w, lds, &first, nullptr, nullptr);
        if (threadIdx.x == 0) parts[b * cuts + at_cut.cut] = Part{mass.base, mass.bad ? (double)NAN : mass.base == -INFINITY ? 0.0 : mass.sum, first};
    }
}

// Every wave of a row's workgroup finds the strip by itself, 64 parts at a time: that takes no barrier.
template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock, RULES ? 4 : 1) sample_join_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys, int nv,
                                                             bool half, int64_t cuts, const Part* parts, int32_t* actions, float* log_prob) {
    constexpr int C = E::kVec;
    __shared__ __align__(16) uint32_t words[RULES ? strip_words<kBlock>() : 4];
    __shared__ double sums[8192 / (kWave * E::kVec)];
    __shared__ int lds_at;
    const int cap = kBlock * C * nv, place = (int)threadIdx.x * C, lane = (int)threadIdx.x & (kWave - 1);
    const bool hist = RULES && r.hist;
    const Counts counts{hist ? words : nullptr, cap, cap, half, true};
    double* const none = nullptr;
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Part* parts_b = parts + b * cuts;
        const Row w = row_of<RULES>(r, b);
        const Heat scale = w;
        const typename E::T* x = x0 + b * stride;
        const double u = row_uniform(keys, b);
        double m = -INFINITY;
        int bad = 0;
        for (int64_t c = lane; c < cuts; c += kWave) {
            m = parts_b[c].base > m ? parts_b[c].base : m;
            bad |= parts_b[c].sum != parts_b[c].sum;
        }
        m = group_reduce<kWave>(m, Max<double>(), none);
        bad = group_reduce<kWave>(bad, Max<int>(), (int*)none);
        const bool any = !bad && m > -INFINITY;   // the same for the whole workgroup, as is what hangs on it
        // a part's sum against m
        auto share = [&](int64_t c) { return parts_b[c].sum > 0 ? parts_b[c].sum * weight(parts_b[c].base - m, scale) : 0.0; };
        double sum = 0;
        long long first = width;
        if (any)
            for (int64_t c = lane; c < cuts; c += kWave) {
                sum += share(c);
                if (parts_b[c].base == m && parts_b[c].first < first) first = parts_b[c].first;
            }
        const Mass mass{m, group_reduce<kWave>(sum, Sum<double>(), none), bad != 0};
        int64_t at = 0;
        if (any && w.greedy) {
            at = group_reduce<kWave>(first, Min<long long>(), (long long*)none);
            if (hist) count_ids<false>(r, b, 1, rows, width, at / cap * cap, counts);
        } else if (any) {
            const double level = u * mass.sum, tiny = mass.sum * 0x1p-80;
            double before;
            bool past;
            const int64_t c = find_part(cuts, level, tiny, share, &before, &past);
            const double base = parts_b[c].base;
            const double target = past ? INFINITY : (level - before) / weight(base - m, scale);
            const int64_t lo = c * cap;
            const Place p{lo + place, width, kBlock * C, place, counts};
            Vector<E, C> v;
            v.load(w, x, p.at, width);
            if (hist) count_ids<false>(r, b, 1, rows, width, lo, counts);
            strip_sums<E, RULES, kBlock>(x, v, w, p, nv, scale, base, sums);
            at = lo + locate<E, RULES, kBlock>(x, w, p, nv, scale, base, parts_b[c].sum, target, sums, &lds_at);
        }
        if (threadIdx.x == 0) answer<E>(w, x, mass, at, any && hist ? counts.at((int)(at % cap)) : 0u, scale, b, actions, log_prob, nullptr, nullptr);
        __syncthreads();
    }
}

// (Without a history the wide form's strips could be longer; of twice or four times the columns the parts take 5 us less of 512 x 131,072 bf16, and the join,
// which goes through one strip once more, 10 to 15 us more.)
int64_t cuts_of(int vec, int nv, int64_t width) {
    const int64_t cap = (int64_t)kBlock * vec * nv;
    return (width + cap - 1) / cap;
}
// The wide form's: as many as still make workgroups enough to fill the chip.
int wide_nv(int vec, int most, int64_t rows, int64_t width) {
    int nv = most;
    while (nv > 1 && rows * cuts_of(vec, nv, width) < 1024) nv /= 2;
    return nv;
}

// For any type and rules.
size_t parts_bytes(int64_t rows, int64_t width) {
    size_t most = 0;
    for (const int vec : {F32::kVec, F16::kVec})
        for (const int nv : {4096 / (kBlock * vec), 8192 / (kBlock * vec)}) {
            const size_t bytes = sizeof(Part) * (size_t)rows * (size_t)cuts_of(vec, wide_nv(vec, nv, rows, width), width);
            if (width > (int64_t)kBlock * vec * nv && bytes > most) most = bytes;
        }
    return most;
}

template <typename E, bool RULES>
struct Launch {
    const typename E::T* x;
    int64_t rows, width, stride;
    const Rules& r;
    const Keys& k;
    int32_t* actions;
    float* log_prob;
    void* ws;
    hipStream_t s;

    template <int G, int C>
    void vectors() const {
        constexpr int per = kBlock / G;
        hipLaunchKernelGGL((sample_vectors_kernel<E, RULES, G, C>), dim3(grid_for((rows + per - 1) / per, 4096)), dim3(kBlock), 0, s, x, rows, width, stride, r, k,
                           actions, log_prob);
    }
    template <int G>
    void strips(int nv) const {
        constexpr int per = kBlock / G;
        hipLaunchKernelGGL((sample_strips_kernel<E, RULES, G>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, x, rows, width, stride, r, k, nv,
                           half_counts(r), actions, log_prob);
    }
    void wide(int nv) const {
        const int64_t cuts = cuts_of(E::kVec, nv, width);
        hipLaunchKernelGGL((sample_parts_kernel<E, RULES>), dim3(grid_for(rows * cuts, 1 << 20)), dim3(kBlock), 0, s, x, rows, width, stride, r, nv, half_counts(r), cuts,
                           (Part*)ws);
        hipLaunchKernelGGL((sample_join_kernel<E, RULES>), dim3(grid_for(rows)), dim3(kBlock), 0, s, x, rows, width, stride, r, k, nv, half_counts(r), cuts,
                           (const Part*)ws, actions, log_prob);
    }
    void operator()() const {
        constexpr int v = E::kVec;
        const int most = strip_vectors<E>(r, kBlock), wave_most = strip_vectors<E>(r, kWave);
        const auto need = [&](int g) { return (int)((width + g * v - 1) / (g * v)); };   // vectors a lane
        // few columns: a row per lane, as wide as the row; then as few lanes as hold it, a 16-byte vector each; then strips (kLong has the figures), of a wave
        // where they are short or there are rows enough, of a workgroup up to 8 vectors a lane or where there are rows enough, else parts
        int g = 1;
        while (g < kWave && width > g * v) g *= 2;
        g = lanes_for(r, rows, g);
        if (width <= kWave * v && g <= kWave) {
            if (g == 1 && width <= 2) vectors<1, 2>();
            else if (g == 1 && width <= 4) vectors<1, 4>();
            else if (g == 1) vectors<1, v>();
            else if (g == 2) vectors<2, v>();
            else if (g == 4) vectors<4, v>();
            else if (g == 8) vectors<8, v>();
            else if (g == 16) vectors<16, v>();
            else if (g == 32) vectors<32, v>();
            else vectors<64, v>();
        }
        else if (need(kWave) <= (r.hist ? wave_most : kLong) && (need(kWave) <= 4 || rows >= 128 * need(kWave)) && (g <= kWave || rows >= 128 * need(kWave)))
            strips<kWave>(need(kWave));
        else if (need(kBlock) <= most || (!r.hist && need(kBlock) <= kLong / 4 && (need(kBlock) <= 8 || rows >= 16 * need(kBlock)))) strips<kBlock>(need(kBlock));
        else wide(wide_nv(v, most, rows, width));
    }
};

}  // namespace
}  // namespace policy
}  // namespace gymhip

using namespace gymhip;
using namespace gymhip::policy;

extern "C" {

size_t gymhip_sample_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0 || width > GYMHIP_POLICY_MAX_WIDTH) return 0;
    return parts_bytes(rows, width);
}

int gymhip_sample_actions(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules,
                          const gymhip_random_keys* keys, int32_t* actions, float* log_prob, void* workspace, size_t workspace_bytes, void* stream) {
    Rules r;
    Keys k;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (int rc = check_keys(keys, &k)) return rc;
    if (rows && (!actions || !log_prob)) return fail(GYMHIP_EINVAL, "actions or log_prob is null");
    if (int rc = check_workspace(workspace, workspace_bytes, gymhip_sample_workspace_bytes(rows, width))) return rc;
    if (int rc = check_results(logits, type, rows, width, stride, {{"actions", actions, rows * 4}, {"log_prob", log_prob, rows * 4}})) return rc;
    if (!rows) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        with_bool(!r.plain(), [&](auto ruled_) {
            Launch<E, decltype(ruled_)::value>{(const typename E::T*)logits, rows, width, stride, r, k, actions, log_prob, workspace, (hipStream_t)stream}();
        });
    });
}

}  // extern "C"
