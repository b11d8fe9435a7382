// policy_sample.hip — one action per row from softmax of the ruled logits, and its log-probability.
//
// The action is the least column whose running sum of exp((y - max y) / T) passes u times the whole sum.  Everything that decides it is in
// double: two neighbouring columns of a flat row of 2^17 lie 8e-6 of the sum apart, less than float32 sums of them are off by, and the same
// logits must give the same action however the row is laid out and split.  Doubles run at the rate of floats here, and the exponential is
// the 18 instructions of exp2_double.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

constexpr double kTiny = 0x1p-900;   // weights below count as none

struct Choice {
    int64_t at;   // the action's column, or -1
    float log_prob;
};

__device__ inline double weight(double y, double base, double k) {
    const double t = (y - base) * k;
    return exp2_double(t > kLeast ? t : kLeast);   // -inf - base and its NaN cannot occur: base is finite
}

// Which column of a group's tile the running sum passes `level` in; s[] are the sums of this lane's vectors.  Columns are in order of
// (vector k, lane, element).  If rounding leaves the level above the last sum, the last column with any weight is taken.
template <typename E, bool RULES, int G, int NV>
__device__ inline int64_t locate(const Tile<E, RULES, NV>& tile, const double* s, double base, double k2, double level, double* lds, int* lds_at) {
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
        for (int k = 0; k < NV; k++) sums[k] = group_reduce<G>(s[k], Sum<double>(), lds);
    }
    // the part (vector, wave) that holds the level, and what comes before it
    int part = -1;
    double before = 0;
#pragma unroll
    for (int i = 0; i < NV * M; i++) {
        const bool here = part < 0 && before + sums[i] > level;
        if (here) part = i;
        if (part < 0) before += sums[i];
    }
    if (part < 0) {
        before = 0;
#pragma unroll
        for (int i = 0; i < NV * M; i++)
            if (sums[i] > kTiny) part = i;
        if (part < 0) part = 0;
        level = INFINITY;
    }
    const int kk = part / M, ww = part - kk * M;
    double sk = s[0];
    typename Tile<E, RULES, NV>::Y y[E::kVec];
#pragma unroll
    for (int j = 0; j < E::kVec; j++) y[j] = tile.y[0][j];
#pragma unroll
    for (int k = 1; k < NV; k++)
        if (kk == k) {
            sk = s[k];
#pragma unroll
            for (int j = 0; j < E::kVec; j++) y[j] = tile.y[k][j];
        }
    double upto = sk;
#pragma unroll
    for (int d = 1; d < W; d <<= 1) {
        const double o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    const uint64_t group = W == 64 ? ~0ull : ((1ull << W) - 1) << ((int)(threadIdx.x & (kWave - 1)) & ~(W - 1));
    const uint64_t hits = __ballot(sk > 0 && before + upto > level) & group, some = __ballot(sk > kTiny) & group;
    const int first = hits ? __ffsll((unsigned long long)hits) - 1 : some ? 63 - __clzll((long long)some) : (int)(threadIdx.x & (kWave - 1));
    // every lane walks its own vector; the chosen lane's answer counts
    double acc = before + (upto - sk);
    int at = -1, last = 0;
#pragma unroll
    for (int j = 0; j < E::kVec; j++) {
        const double e = weight((double)y[j], base, k2);
        acc += e;
        if (e > kTiny) {
            last = j;
            if (at < 0 && acc > level) at = j;
        }
    }
    if (at < 0) at = last;
    at = __shfl(at, first);
    int column = (kk * G + (ww * kWave) * (G > kWave) + (first & (W - 1))) * E::kVec + at;
    if (G > kWave) {
        if (wave == ww && lane == 0) *lds_at = column;
        __syncthreads();
        column = *lds_at;
    }
    return column;
}

// The first column where the tile holds m, or `none`.
template <typename E, bool RULES, int G, int NV>
__device__ inline int64_t first_of(const Tile<E, RULES, NV>& tile, double m, int64_t v0, int64_t step, int64_t none, long long* lds) {
    long long at = none;
#pragma unroll
    for (int k = NV - 1; k >= 0; k--)
#pragma unroll
        for (int j = E::kVec - 1; j >= 0; j--)
            if ((double)tile.y[k][j] == m) at = v0 + k * step + j;
    return group_reduce<G>(at, Min<long long>(), lds);
}

__device__ inline float log_prob_of(const Row& w, double y, double m, double sum) { return (float)((y - m) / (double)w.temp - log(sum)); }

// A row in G lanes' registers: rows of at most G * kVec * NV columns, kBlock / G of them per workgroup.
template <typename E, bool RULES, int G, int NV>
__global__ void __launch_bounds__(kBlock) sample_rows_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                             int32_t* actions, float* log_prob) {
    constexpr int per = kBlock / G, cap = G * E::kVec * NV;
    __shared__ uint32_t counts[RULES ? per * cap : 1];
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
        const int64_t v0 = lane * E::kVec, step = (int64_t)G * E::kVec;
        const uint32_t* mine = RULES && r.hist ? counts + group * cap : nullptr;
        Tile<E, RULES, NV> tile;
        bool bad;
        tile.load(w, x, v0, step, width, mine ? mine + v0 : nullptr, &bad);
        using Y = typename Tile<E, RULES, NV>::Y;
        const double m = (double)group_reduce<G>(tile.max(), Max<Y>(), (Y*)lds);
        const int poison = group_reduce<G>((int)bad, Max<int>(), (int*)lds) | (m == INFINITY);
        const double base = m > -INFINITY && m < INFINITY ? m : 0.0;
        const double k2 = kLog2e / (double)w.temp;
        double s[NV], sum = 0;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            s[k] = 0;
#pragma unroll
            for (int j = 0; j < E::kVec; j++) s[k] += weight((double)tile.y[k][j], base, k2);
            sum += s[k];
        }
        sum = group_reduce<G>(sum, Sum<double>(), lds);
        int64_t at = locate<E, RULES, G, NV>(tile, s, base, k2, row_uniform(keys, b) * sum, lds, &lds_at);
        if (__syncthreads_or(w.greedy)) {
            const int64_t first = first_of<E, RULES, G, NV>(tile, m, v0, step, width, lds_first);
            if (w.greedy) at = first;
        }
        if (lane == 0 && own < rows) {
            float lp = poison ? NAN : -INFINITY;
            if (poison || m == -INFINITY) at = -1;
            else lp = log_prob_of(w, ruled(w, (float)x[at], mine ? mine[at] : 0u, true, at), m, sum);
            actions[b] = (int32_t)at;
            log_prob[b] = lp;
        }
        __syncthreads();
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
    constexpr int cap = kBlock * E::kVec * NV;
    __shared__ uint32_t counts[RULES ? cap : 1];
    __shared__ double lds[kBlock / kWave];
    __shared__ long long lds_first[kBlock / kWave];
    for (int64_t i = blockIdx.x; i < rows * cuts; i += gridDim.x) {
        const int64_t b = i / cuts, lo = (i - b * cuts) * cap;
        if (RULES && r.hist) count_ids(r, b, 1, rows, width, lo, cap, counts);
        const Row w = row_of<RULES>(r, b);
        const int64_t v0 = lo + threadIdx.x * E::kVec, step = (int64_t)kBlock * E::kVec;
        Tile<E, RULES, NV> tile;
        bool bad;
        tile.load(w, x0 + b * stride, v0, step, width, RULES && r.hist ? counts + threadIdx.x * E::kVec : nullptr, &bad);
        using Y = typename Tile<E, RULES, NV>::Y;
        const double m = (double)group_reduce<kBlock>(tile.max(), Max<Y>(), (Y*)lds);
        const int poison = group_reduce<kBlock>((int)bad, Max<int>(), (int*)lds) | (m == INFINITY);
        const double base = m > -INFINITY && m < INFINITY ? m : 0.0;
        const double k2 = kLog2e / (double)w.temp;
        double sum = 0;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < E::kVec; j++) sum += weight((double)tile.y[k][j], base, k2);
        sum = group_reduce<kBlock>(sum, Sum<double>(), lds);
        const int64_t first = w.greedy ? first_of<E, RULES, kBlock, NV>(tile, m, v0, step, width, lds_first) : 0;
        if (threadIdx.x == 0) parts[i] = Part{m, poison ? (double)NAN : m == -INFINITY ? 0.0 : sum, first};
        __syncthreads();
    }
}

template <typename E, bool RULES, int NV>
__global__ void __launch_bounds__(kBlock) sample_join_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                             int64_t cuts, const Part* parts, int32_t* actions, float* log_prob) {
    constexpr int cap = kBlock * E::kVec * NV;
    __shared__ uint32_t counts[RULES ? cap : 1];
    __shared__ double lds[NV * (kBlock / kWave)];
    __shared__ long long lds_first[kBlock / kWave];
    __shared__ int lds_at;
    __shared__ double before_part;
    __shared__ int the_part;
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Part* p = parts + b * cuts;
        const Row w = row_of<RULES>(r, b);
        const double k2 = kLog2e / (double)w.temp;
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
                double upto = e;
                const int lane = (int)threadIdx.x & (kWave - 1), wave = (int)threadIdx.x / kWave;
                for (int d = 1; d < kWave; d <<= 1) {
                    const double o = __shfl_up(upto, d);
                    if (lane >= d) upto += o;
                }
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
                if (most >= 0) {
                    last = (int)most;
                }
            }
            __syncthreads();
            const bool over = the_part < 0;
            const int c = over ? last : the_part;
            const double target = over ? INFINITY : (level - before_part) / weight(p[c].m, m, k2);
            const int64_t lo = (int64_t)c * cap;
            if (RULES && r.hist) count_ids(r, b, 1, rows, width, lo, cap, counts);
            Tile<E, RULES, NV> tile;
            bool nan;
            const int64_t v0 = lo + threadIdx.x * E::kVec, step = (int64_t)kBlock * E::kVec;
            tile.load(w, x0 + b * stride, v0, step, width, RULES && r.hist ? counts + threadIdx.x * E::kVec : nullptr, &nan);
            double s[NV];
#pragma unroll
            for (int k = 0; k < NV; k++) {
                s[k] = 0;
#pragma unroll
                for (int j = 0; j < E::kVec; j++) s[k] += weight((double)tile.y[k][j], p[c].m, k2);
            }
            at = lo + locate<E, RULES, kBlock, NV>(tile, s, p[c].m, k2, target, lds, &lds_at);
        }
        if (threadIdx.x == 0) {
            const uint32_t n = RULES && r.hist ? counts[at % cap] : 0u;
            actions[b] = (int32_t)at;
            log_prob[b] = log_prob_of(w, ruled(w, (float)x0[b * stride + at], n, true, at), m, sum);
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

template <typename E, bool RULES, int G, int NV>
void launch_rows(const void* x, int64_t rows, int64_t width, int64_t stride, const Rules& r, const Keys& k, int32_t* actions, float* log_prob, hipStream_t s) {
    constexpr int per = kBlock / G;
    hipLaunchKernelGGL((sample_rows_kernel<E, RULES, G, NV>), dim3(grid_for((rows + per - 1) / per)), dim3(kBlock), 0, s, (const typename E::T*)x, rows, width,
                       stride, r, k, actions, log_prob);
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
    if (width <= v) launch_rows<E, RULES, 1, 1>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 4 * v) launch_rows<E, RULES, 4, 1>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 16 * v) launch_rows<E, RULES, 16, 1>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 64 * v) launch_rows<E, RULES, 64, 1>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (width <= 64 * v * 4) launch_rows<E, RULES, 64, 4>(x, rows, width, stride, r, k, actions, log_prob, s);
    else if (!is_wide(v, width)) launch_rows<E, RULES, kBlock, 4>(x, rows, width, stride, r, k, actions, log_prob, s);
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
