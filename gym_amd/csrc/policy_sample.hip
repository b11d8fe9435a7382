// policy_sample.hip — one action per row from softmax of the ruled logits, and its log-probability.
//
// The action is the least column whose running sum of exp((y - max y) / T) passes u times the whole sum.  Everything that decides it is in
// double: two neighbouring columns of a flat row of 2^17 lie 8e-6 of the sum apart, less than float32 sums of them are off by, and the same
// logits must give the same action however the row is laid out and split.  Doubles run at the rate of floats here, and the exponential is
// the 16 instructions of exp2_double.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

constexpr double kTiny = 0x1p-900;   // weights below count as none

// A weight against a finite base; NaN does not come here unmarked (see Tile::load).
__device__ inline double weight(double y, double base, double k2) {
    const double t = (y - base) * k2;
    return exp2_double(t > kLeast ? t : kLeast);
}

// One lane's share of a row's tile: NV vectors of C columns, `step` columns apart.  A vector is kept as it lies in memory, and gives its y
// (float where y is the logit itself) each time it is gone through.
template <typename E, bool RULES, int NV, int C>
struct Tile {
    using Y = typename std::conditional<RULES, double, float>::type;
    Raw<E, C> raw[NV];

    __device__ void load(const typename E::T* x, int64_t v0, int step, int64_t width) {
#pragma unroll
        for (int k = 0; k < NV; k++) raw[k].load(x, v0 + k * step, NV == 1 || v0 + k * step < width ? width : v0 + k * step);
    }
    __device__ void get(int k, const Row& w, int64_t at, int64_t width, const uint32_t* counts, Y* y) const {
        if constexpr (RULES) {
            if (at < width) ruled_cols(w, raw[k], at, width, counts, y);
            else
#pragma unroll
                for (int j = 0; j < C; j++) y[j] = -INFINITY;
        } else {
#pragma unroll
            for (int j = 0; j < C; j++) y[j] = raw[k].get(j);
        }
    }
};

// What a tile comes to: its greatest y, and the sum of its weights against that; `bad` where a NaN or +inf is among its y.
// In s[k] the sums of this lane's vectors, against m.  Each vector is summed against its own maximum first, so that one pass over it does.
template <typename E, bool RULES, int G, int NV, int C>
__device__ inline void sum_tile(const Tile<E, RULES, NV, C>& tile, const Row& w, int64_t v0, int step, int64_t width, const uint32_t* counts, double k2,
                                double* lds, double* s, double* m_out, double* sum_out, bool* bad_out) {
    using Y = typename Tile<E, RULES, NV, C>::Y;
    Y m[NV], top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        Y y[C];
        tile.get(k, w, v0 + k * step, width, counts ? counts + k * step : nullptr, y);
        m[k] = -INFINITY;
#pragma unroll
        for (int j = 0; j < C; j++) {
            bad = bad || y[j] != y[j];
            m[k] = y[j] > m[k] ? y[j] : m[k];
        }
        bad = bad || m[k] == INFINITY;
        const double base = m[k] > -INFINITY && m[k] < INFINITY ? (double)m[k] : 0.0;
        s[k] = 0;
#pragma unroll
        for (int j = 0; j < C; j++) s[k] += weight((double)y[j], base, k2);
        top = m[k] > top ? m[k] : top;
    }
    top = group_reduce<G>(top, Max<Y>(), (Y*)lds);
    const double base = top > -INFINITY && top < INFINITY ? (double)top : 0.0;
    double sum = 0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        if (!(NV == 1 && G == 1)) s[k] = m[k] > -INFINITY ? s[k] * weight((double)m[k], base, k2) : 0.0;
        sum += s[k];
    }
    *sum_out = group_reduce<G>(sum, Sum<double>(), lds);
    *m_out = (double)top;
    *bad_out = group_reduce<G>((int)bad, Max<int>(), (int*)lds) != 0;
}

// Which column of a group's tile (0 = its first) the running sum passes `level` in; s[] as sum_tile leaves it, against `base`.  Columns are in
// order of (vector k, lane, element).  If rounding leaves the level above the last sum, the last column with any weight is taken.
template <typename E, bool RULES, int G, int NV, int C>
__device__ inline int locate(const Tile<E, RULES, NV, C>& tile, const Row& w, int64_t v0, int step, int64_t width, const uint32_t* counts, const double* s,
                             double base, double k2, double level, double* lds, int* lds_at) {
    constexpr int W = G < kWave ? G : kWave;           // lanes that exchange
    constexpr int M = G > kWave ? kBlock / kWave : 1;  // waves that share the tile
    const int lane = (int)threadIdx.x & (W - 1), wave = G > kWave ? (int)threadIdx.x / kWave : 0;
    double sums[NV * M];
    if (G > kWave) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const double t = group_reduce<kWave>(s[k], Sum<double>(), lds);
            if (lane == 0) lds[k * M + wave] = t;
        }
        if (threadIdx.x == 0) *lds_at = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV * M; i++) sums[i] = lds[i];
    } else {
#pragma unroll
        for (int k = 0; k < NV; k++) sums[k] = group_reduce<W>(s[k], Sum<double>(), lds);
    }
    // the part (vector, wave) that holds the level, and what comes before it
    int part = -1, some = 0;
    double before = 0;
#pragma unroll
    for (int i = 0; i < NV * M; i++) {
        if (part < 0 && before + sums[i] > level) part = i;
        if (part < 0) before += sums[i];
        if (sums[i] > kTiny) some = i;
    }
    if (part < 0) {
        part = some;
        before = 0;
        level = INFINITY;
    }
    const int kk = NV == 1 ? 0 : __builtin_amdgcn_readfirstlane(part / M), ww = part - kk * M;   // NV > 1 has one row in a wave
    int column = 0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        if (NV > 1 && kk != k) continue;
        const double upto = running_sum<W>(s[k], lane);
        const int self = (int)(threadIdx.x & (kWave - 1));
        const uint64_t group = W == 64 ? ~0ull : ((1ull << W) - 1) << (self & ~(W - 1));
        const uint64_t hits = __ballot(s[k] > 0 && before + upto > level) & group, any = __ballot(s[k] > kTiny) & group;
        const int first = hits ? __ffsll((unsigned long long)hits) - 1 : any ? 63 - __clzll((long long)any) : self;
        // every lane walks its own vector; the chosen lane's answer counts
        typename Tile<E, RULES, NV, C>::Y y[C];
        tile.get(k, w, v0 + k * step, width, counts ? counts + k * step : nullptr, y);
        double acc = before + (upto - s[k]);
        int at = -1, last = 0;
#pragma unroll
        for (int j = 0; j < C; j++) {
            const double e = weight((double)y[j], base, k2);
            acc += e;
            if (e > kTiny) {
                last = j;
                if (at < 0 && acc > level) at = j;
            }
        }
        if (at < 0) at = last;
        if (W > 1) at = __shfl(at, first);
        column = (k * G + (G > kWave ? ww * kWave : 0) + (first & (W - 1))) * C + at;
    }
    if (G > kWave) {
        if (wave == ww && lane == 0) *lds_at = column;
        __syncthreads();
        column = *lds_at;
    }
    return column;
}

// The first column of the row where the tile holds m, or `none`.
template <typename E, bool RULES, int G, int NV, int C>
__device__ inline int64_t first_of(const Tile<E, RULES, NV, C>& tile, const Row& w, double m, int64_t v0, int step, int64_t width, const uint32_t* counts,
                                   long long* lds) {
    long long at = width;
#pragma unroll
    for (int k = NV - 1; k >= 0; k--) {
        typename Tile<E, RULES, NV, C>::Y y[C];
        tile.get(k, w, v0 + k * step, width, counts ? counts + k * step : nullptr, y);
#pragma unroll
        for (int j = C - 1; j >= 0; j--)
            if ((double)y[j] == m) at = v0 + k * step + j;
    }
    return group_reduce<G>(at, Min<long long>(), lds);
}

__device__ inline float log_prob_of(double y, double m, double k2, double sum) { return (float)(((y - m) * k2 - log2_double(sum)) * kLn2); }

// A row in G lanes' registers: rows of at most G * C * NV columns, kBlock / G of them per workgroup.
template <typename E, bool RULES, int G, int NV, int C>
__global__ void __launch_bounds__(kBlock) sample_rows_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                             int32_t* actions, float* log_prob) {
    constexpr int per = kBlock / G, cap = G * C * NV, step = G * C;
    __shared__ __align__(16) uint32_t counts[RULES ? per * cap : 4];
    __shared__ double lds[NV * (kBlock / kWave)];
    __shared__ long long lds_first[kBlock / kWave];
    __shared__ int lds_at;
    const int lane = (int)threadIdx.x & (G - 1);
    const int group = G >= kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / G) : (int)threadIdx.x / G;
    for (int64_t band = blockIdx.x; band * per < rows; band += gridDim.x) {
        if (RULES && r.hist) count_ids(r, band * per, per, rows, width, 0, cap, counts);
        const int64_t own = band * per + group;
        const int64_t b = own < rows ? own : rows - 1;   // lanes without a row follow the last one: every exchange has all its lanes
        const Row w = row_of<RULES>(r, b);
        const typename E::T* x = x0 + b * stride;
        const int64_t v0 = lane * C;
        const uint32_t* mine = RULES && r.hist ? counts + group * cap : nullptr;
        const uint32_t* here = mine ? mine + v0 : nullptr;
        Tile<E, RULES, NV, C> tile;
        tile.load(x, v0, step, width);
        const double u = row_uniform(keys, b);
        const double k2 = kLog2e / w.temp;
        double s[NV], m, sum;
        bool bad;
        sum_tile<E, RULES, G, NV, C>(tile, w, v0, step, width, here, k2, lds, s, &m, &sum, &bad);
        const double base = m > -INFINITY && m < INFINITY ? m : 0.0;
        int64_t at = locate<E, RULES, G, NV, C>(tile, w, v0, step, width, here, s, base, k2, u * sum, lds, &lds_at);
        if (G > kWave ? w.greedy : __any(w.greedy)) {   // the same for all lanes that exchange
            const int64_t first = first_of<E, RULES, G, NV, C>(tile, w, m, v0, step, width, here, lds_first);
            if (w.greedy) at = first;
        }
        if (lane == 0 && own < rows) {
            float lp = bad ? NAN : -INFINITY;
            if (bad || m == -INFINITY) at = -1;
            else lp = log_prob_of(ruled(w, (float)x[at], mine ? mine[at] : 0u, true, at), m, k2, sum);
            actions[b] = (int32_t)at;
            log_prob[b] = lp;
        }
    }
}

// Wider rows: one workgroup per tile leaves the tile's greatest y, the sum of its weights against that, and where it is first; then one
// workgroup per row joins them, finds the tile that the level falls into and goes through that tile once more.
struct Part {
    double m, s;
    long long first;
};

template <typename E, bool RULES, int NV>
__global__ void __launch_bounds__(kBlock) sample_parts_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, int64_t cuts,
                                                              Part* parts) {
    constexpr int C = E::kVec, cap = kBlock * C * NV, step = kBlock * C;
    __shared__ __align__(16) uint32_t counts[RULES ? cap : 4];
    __shared__ double lds[kBlock / kWave];
    __shared__ long long lds_first[kBlock / kWave];
    for (int64_t i = blockIdx.x; i < rows * cuts; i += gridDim.x) {
        const int64_t b = i / cuts, lo = (i - b * cuts) * cap;
        const int64_t v0 = lo + threadIdx.x * C;
        Tile<E, RULES, NV, C> tile;
        tile.load(x0 + b * stride, v0, step, width);
        if (RULES && r.hist) count_ids(r, b, 1, rows, width, lo, cap, counts);
        const uint32_t* here = RULES && r.hist ? counts + threadIdx.x * C : nullptr;
        const Row w = row_of<RULES>(r, b);
        double s[NV], m, sum;
        bool bad;
        sum_tile<E, RULES, kBlock, NV, C>(tile, w, v0, step, width, here, kLog2e / w.temp, lds, s, &m, &sum, &bad);
        const int64_t first = w.greedy ? first_of<E, RULES, kBlock, NV, C>(tile, w, m, v0, step, width, here, lds_first) : 0;
        if (threadIdx.x == 0) parts[i] = Part{m, bad ? (double)NAN : m == -INFINITY ? 0.0 : sum, first};
    }
}

template <typename E, bool RULES, int NV>
__global__ void __launch_bounds__(kBlock) sample_join_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                             int64_t cuts, const Part* parts, int32_t* actions, float* log_prob) {
    constexpr int C = E::kVec, cap = kBlock * C * NV, step = kBlock * C;
    __shared__ __align__(16) uint32_t counts[RULES ? cap : 4];
    __shared__ double lds[NV * (kBlock / kWave)];
    __shared__ long long lds_first[kBlock / kWave];
    __shared__ int lds_at;
    __shared__ double before_part;
    __shared__ int the_part;
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Part* p = parts + b * cuts;
        const Row w = row_of<RULES>(r, b);
        const double k2 = kLog2e / w.temp;
        double m = -INFINITY;
        int bad = 0;
        for (int64_t c = threadIdx.x; c < cuts; c += kBlock) {
            m = p[c].m > m ? p[c].m : m;
            bad |= p[c].s != p[c].s;
        }
        m = group_reduce<kBlock>(m, Max<double>(), lds);
        bad = group_reduce<kBlock>(bad, Max<int>(), (int*)lds);
        if (bad || m == -INFINITY) {   // the same for the whole workgroup
            if (threadIdx.x == 0) {
                actions[b] = -1;
                log_prob[b] = bad ? NAN : -INFINITY;
            }
            continue;
        }
        auto share = [&](int64_t c) { return c < cuts && p[c].s > 0 ? p[c].s * weight(p[c].m, m, k2) : 0.0; };
        double sum = 0;
        long long first = width;
        for (int64_t c = threadIdx.x; c < cuts; c += kBlock) {
            sum += share(c);
            if (p[c].m == m && p[c].first < first) first = p[c].first;
        }
        sum = group_reduce<kBlock>(sum, Sum<double>(), lds);
        int64_t at;
        if (w.greedy) {
            at = group_reduce<kBlock>(first, Min<long long>(), lds_first);
            if (RULES && r.hist) count_ids(r, b, 1, rows, width, at / cap * cap, cap, counts);
        } else {
            const double level = row_uniform(keys, b) * sum;
            if (threadIdx.x == 0) the_part = -1;
            double run = 0;
            int last = 0;   // the last part with any weight, should rounding leave the level above all sums
            for (int64_t c0 = 0; c0 < cuts; c0 += kBlock) {
                const int64_t c = c0 + threadIdx.x;
                const double e = share(c);
                const int lane = (int)threadIdx.x & (kWave - 1), wave = (int)threadIdx.x / kWave;
                const double upto = running_sum<kWave>(e, lane);
                __syncthreads();
                if (lane == kWave - 1) lds[wave] = upto;
                __syncthreads();
                double front = run;
                for (int i = 0; i < kBlock / kWave; i++) {
                    if (i < wave) front += lds[i];
                    run += lds[i];
                }
                const long long hit = e > 0 && front + upto > level ? (long long)c : (long long)cuts;
                const long long least = group_reduce<kBlock>(hit, Min<long long>(), lds_first);
                if (least < cuts) {
                    if (c == least) {
                        the_part = (int)c;
                        before_part = front + (upto - e);
                    }
                    break;
                }
                const long long most = group_reduce<kBlock>(e > 0 ? (long long)c : -1ll, Max<long long>(), lds_first);
                if (most >= 0) last = (int)most;
            }
            __syncthreads();
            const bool over = the_part < 0;
            const int c = over ? last : the_part;
            const double top = p[c].m;
            const double target = over ? INFINITY : (level - before_part) / weight(top, m, k2);
            const int64_t lo = (int64_t)c * cap, v0 = lo + threadIdx.x * C;
            Tile<E, RULES, NV, C> tile;
            tile.load(x0 + b * stride, v0, step, width);
            if (RULES && r.hist) count_ids(r, b, 1, rows, width, lo, cap, counts);
            const uint32_t* here = RULES && r.hist ? counts + threadIdx.x * C : nullptr;
            double s[NV], tile_m, tile_sum;
            bool tile_bad;
            sum_tile<E, RULES, kBlock, NV, C>(tile, w, v0, step, width, here, k2, lds, s, &tile_m, &tile_sum, &tile_bad);
            at = lo + locate<E, RULES, kBlock, NV, C>(tile, w, v0, step, width, here, s, top, k2, target, lds, &lds_at);
        }
        if (threadIdx.x == 0) {
            const uint32_t n = RULES && r.hist ? counts[at % cap] : 0u;
            actions[b] = (int32_t)at;
            log_prob[b] = log_prob_of(ruled(w, (float)x0[b * stride + at], n, true, at), m, k2, sum);
        }
        __syncthreads();
    }
}

// Tiles along a row of the wide form: NV = 4 vectors a lane where that still makes enough workgroups, else 1.
int64_t cuts_of(int vec, int nv, int64_t width) {
    const int64_t cap = (int64_t)kBlock * vec * nv;
    return (width + cap - 1) / cap;
}
bool is_wide(int vec, int64_t width) { return width > (int64_t)kBlock * vec * 4; }
int wide_nv(int vec, int64_t rows, int64_t width) { return rows * cuts_of(vec, 4, width) < 1024 ? 1 : 4; }

size_t parts_bytes(int vec, int64_t rows, int64_t width) {
    if (!is_wide(vec, width)) return 0;
    return sizeof(Part) * (size_t)rows * (size_t)cuts_of(vec, wide_nv(vec, rows, width), width);
}

template <typename E, bool RULES, int G, int NV, int C>
void launch_rows(const void* x, int64_t rows, int64_t width, int64_t stride, const Rules& r, const Keys& k, int32_t* actions, float* log_prob, hipStream_t s) {
    constexpr int per = kBlock / G;
    hipLaunchKernelGGL((sample_rows_kernel<E, RULES, G, NV, C>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, (const typename E::T*)x, rows,
                       width, stride, r, k, actions, log_prob);
}

template <typename E, bool RULES, int NV>
void launch_wide(const void* x, int64_t rows, int64_t width, int64_t stride, const Rules& r, const Keys& k, int32_t* actions, float* log_prob, void* ws,
                 hipStream_t s) {
    const int64_t cuts = cuts_of(E::kVec, NV, width);
    hipLaunchKernelGGL((sample_parts_kernel<E, RULES, NV>), dim3(grid_for(rows * cuts)), dim3(kBlock), 0, s, (const typename E::T*)x, rows, width, stride, r,
                       cuts, (Part*)ws);
    hipLaunchKernelGGL((sample_join_kernel<E, RULES, NV>), dim3(grid_for(rows)), dim3(kBlock), 0, s, (const typename E::T*)x, rows, width, stride, r, k, cuts,
                       (const Part*)ws, actions, log_prob);
}

template <typename E, bool RULES>
void launch(const void* x, int64_t rows, int64_t width, int64_t stride, const Rules& r, const Keys& k, int32_t* actions, float* log_prob, void* ws,
            hipStream_t s) {
    constexpr int v = E::kVec;
    // few columns: a row per lane, as wide as the row; then as few lanes as hold it, a 16-byte vector each
    if (width <= 2) launch_rows<E, RULES, 1, 1, 2>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 4) launch_rows<E, RULES, 1, 1, 4>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= v) launch_rows<E, RULES, 1, 1, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 2 * v) launch_rows<E, RULES, 2, 1, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 4 * v) launch_rows<E, RULES, 4, 1, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 8 * v) launch_rows<E, RULES, 8, 1, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 16 * v) launch_rows<E, RULES, 16, 1, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 64 * v) launch_rows<E, RULES, 64, 1, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 64 * v * 4) launch_rows<E, RULES, 64, 4, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (!is_wide(v, width)) launch_rows<E, RULES, kBlock, 4, v>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (wide_nv(v, rows, width) == 1) launch_wide<E, RULES, 1>(x, rows, width, stride, r, k, actions, log_prob, ws, s);
    else launch_wide<E, RULES, 4>(x, rows, width, stride, r, k, actions, log_prob, ws, s);
}

}  // namespace
}  // namespace policy
}  // namespace gymhip

using namespace gymhip;
using namespace gymhip::policy;

extern "C" {

size_t gymhip_sample_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0 || width > GYMHIP_POLICY_MAX_WIDTH) return 0;
    const size_t a = parts_bytes(F32::kVec, rows, width), b = parts_bytes(F16::kVec, rows, width);
    return a > b ? a : b;
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
    if (!rows) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        with_bool(!r.plain(), [&](auto ruled_) {
            launch<E, decltype(ruled_)::value>(logits, rows, width, stride, r, k, actions, log_prob, workspace, (hipStream_t)stream);
        });
    });
}

}  // extern "C"
