// policy_common.h — what the policy kernels (policy_*.hip) share: element types, the counter-based generator, the rules on logits, reductions
// over groups of lanes, and the host-side checks of the entry points.  Formulas: include/gymhip.h.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/gymhip.h"
#include "gymhip_internal.h"

namespace gymhip {
namespace policy {

constexpr int kBlock = 256;
constexpr int kWave = 64;

// ---- element types: kVec elements are 16 bytes; loads widen to float, stores round once, to nearest even -------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct F32 {
    using T = float;
    static constexpr int kVec = 4;
    __device__ static float widen(uint32_t word, int) { return __uint_as_float(word); }
    __device__ static uint32_t narrow(const float* v) { return __float_as_uint(v[0]); }
};
struct F16 {
    using T = _Float16;
    static constexpr int kVec = 8;
    __device__ static float widen(uint32_t word, int half) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(half ? word >> 16 : word)); }
    __device__ static uint32_t narrow(const float* v) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[0]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16;
    }
};
struct BF16 {
    using T = __bf16;
    static constexpr int kVec = 8;
    __device__ static float widen(uint32_t word, int half) { return __uint_as_float(half ? word & 0xFFFF0000u : word << 16); }
    __device__ static uint32_t narrow(const float* v) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[0]) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[1]) << 16;
    }
};

// kVec columns from v0 on, as floats.  The address has the element's alignment only (odd strides, odd starts); the hardware takes 16-byte
// accesses at any such address, so a row needs no aligned middle of its own.  Columns past the row's end read as `absent`, unread.
template <typename E>
__device__ inline void load_cols(const typename E::T* row, int64_t v0, int64_t width, float* out, float absent) {
    using T = typename E::T;
    if (v0 + E::kVec <= width) {
        struct __attribute__((packed, aligned(sizeof(T)))) U { u32x4 w; };
        const u32x4 w = ((const U*)(row + v0))->w;
#pragma unroll
        for (int j = 0; j < E::kVec; j++) out[j] = E::kVec == 4 ? E::widen(w[j], 0) : E::widen(w[j / 2], j & 1);
    } else {
#pragma unroll
        for (int j = 0; j < E::kVec; j++) out[j] = v0 + j < width ? (float)row[v0 + j] : absent;
    }
}

template <typename E>
__device__ inline void store_cols(typename E::T* row, int64_t v0, int64_t width, const float* v) {
    using T = typename E::T;
    if (v0 + E::kVec <= width) {
        struct __attribute__((packed, aligned(sizeof(T)))) U { u32x4 w; };
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = E::narrow(v + (E::kVec == 4 ? j : 2 * j));
        ((U*)(row + v0))->w = w;
    } else {
#pragma unroll
        for (int j = 0; j < E::kVec; j++)
            if (v0 + j < width) row[v0 + j] = (T)v[j];
    }
}

// ---- random numbers ------------------------------------------------------------------------------------------------------------------
struct Keys {
    uint64_t seed;
    int64_t row, step;
    const int64_t *rows, *steps;
    int steps_per_row;
};

// Philox4x32 (Salmon, Moraes, Dror, Shaw: Parallel Random Numbers: As Easy as 1, 2, 3; SC 2011).  7 rounds are the fewest that the
// paper's statistical batteries pass.
__device__ inline uint4 philox7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint64_t seed) {
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 7; r++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// The generator's words for a row's block: the counter is (block, row key, step) with 48 bits for each of the latter two.
__device__ inline uint4 row_words(const Keys& k, int64_t b, uint32_t block) {
    const uint64_t row = k.rows ? (uint64_t)k.rows[b] : (uint64_t)k.row + (uint64_t)b;
    const uint64_t step = k.steps ? (uint64_t)k.steps[k.steps_per_row ? b : 0] : (uint64_t)k.step;
    return philox7(block, (uint32_t)row, (uint32_t)step, ((uint32_t)(row >> 32) & 0xFFFFu) | ((uint32_t)(step >> 32) << 16), k.seed);
}

// The draw's u: 52 random bits and a half, so that every value is exact in a double and neither 0 nor 1 occurs.
__device__ inline double row_uniform(const Keys& k, int64_t b) {
    const uint4 w = row_words(k, b, 0xFFFFFFFFu);   // a block that no column has
    return ((double)(((uint64_t)w.x << 20) | (w.y >> 12)) + 0.5) * 0x1p-52;
}

// ---- rules ---------------------------------------------------------------------------------------------------------------------------
struct Rules {
    const uint32_t* mask;
    int64_t mask_stride, mask_lines;
    const int32_t* mask_rows;
    const float* bias;
    int64_t bias_stride;
    const void* hist;
    int64_t hist_stride;
    const void* hist_len;
    uint32_t hist_cols;
    int hist64, len64;
    const float *rep_rows, *pres_rows, *freq_rows, *temp_rows;
    float rep, pres, freq, temp;
    __host__ __device__ bool plain() const { return !mask && !bias && !hist; }   // temperature alone
};

// One row's share of them.
struct Row {
    const uint32_t* mask;   // its line, or null where everything is allowed
    const float* bias;
    float rep, pres, freq, temp;
    bool greedy, nothing;   // nothing: its line lies behind the mask's last one
};

template <bool RULES>
__device__ inline Row row_of(const Rules& r, int64_t b) {
    Row w;
    const float t = r.temp_rows ? r.temp_rows[b] : r.temp;
    w.greedy = !(t > 0.f);
    w.temp = w.greedy ? 1.f : t;
    w.mask = nullptr;
    w.bias = nullptr;
    w.nothing = false;
    w.rep = w.pres = w.freq = 0.f;
    if (RULES) {
        if (r.mask) {
            const int64_t line = r.mask_rows ? r.mask_rows[b] : (r.mask_lines == 1 ? 0 : b);
            w.nothing = line >= r.mask_lines;
            if (line >= 0 && !w.nothing) w.mask = r.mask + line * r.mask_stride;
        }
        if (r.bias) w.bias = r.bias + b * r.bias_stride;
        if (r.hist) {
            w.rep = r.rep_rows ? r.rep_rows[b] : r.rep;
            w.pres = r.pres_rows ? r.pres_rows[b] : r.pres;
            w.freq = r.freq_rows ? r.freq_rows[b] : r.freq;
        }
    }
    return w;
}

// The mask's bits of kVec (4 or 8) columns from v0 on, v0 a multiple of kVec and < width.
__device__ inline uint32_t allowed_bits(const Row& w, int64_t v0) {
    if (w.nothing) return 0u;
    return w.mask ? w.mask[v0 >> 5] >> (v0 & 31) : 0xFFu;
}

// y: the logit after penalties and bias, before the temperature.  In double: what is compared and summed must be the formula's value even
// where a bias or a penalty cancels most of the logit.
__device__ inline double penalised(const Row& w, float xf, uint32_t count) {
    double x = xf;
    if (count) {
        x = x > 0 ? x / (double)w.rep : x * (double)w.rep;
        x = x - (double)w.freq * (double)count - (double)w.pres;
    }
    return x;
}
__device__ inline double ruled(const Row& w, float xf, uint32_t count, bool ok, int64_t v) {
    if (!ok) return -INFINITY;
    const double x = penalised(w, xf, count);
    return w.bias ? x + (double)w.bias[v] : x;
}

// How often each id of columns [lo, lo + cap) occurs in the histories of rows [b0, b0 + n): counts[row - b0][id - lo], by the whole workgroup.
// The rows' ids are read as one run of n * hist_cols places (adjacent rows' ids are adjacent in memory); integer LDS atomics, so their
// order is free.  Every thread of the workgroup comes here; counts may be read after it returns.
__device__ inline void count_ids(const Rules& r, int64_t b0, int n, int64_t rows, int64_t width, int64_t lo, int cap, uint32_t* counts) {
    __syncthreads();
    for (int i = threadIdx.x; i < n * cap; i += kBlock) counts[i] = 0;
    __syncthreads();
    const uint32_t cols = r.hist_cols;
    const int64_t hi = lo + cap < width ? lo + cap : width;
    for (uint64_t i = threadIdx.x; i < (uint64_t)n * cols; i += kBlock) {
        uint32_t q = 0, c = (uint32_t)i;
        if (n > 1) {
            if ((uint64_t)n * cols <= 0xFFFFFFFFull) { q = (uint32_t)i / cols; c = (uint32_t)i - q * cols; }
            else { q = (uint32_t)(i / cols); c = (uint32_t)(i - (uint64_t)q * cols); }
        }
        const int64_t b = b0 + q;
        if (b >= rows) break;
        if (r.hist_len) {
            const int64_t len = r.len64 ? ((const int64_t*)r.hist_len)[b] : (int64_t)((const int32_t*)r.hist_len)[b];
            if ((int64_t)c >= len) continue;
        }
        const int64_t at = b * r.hist_stride + c;
        const int64_t id = r.hist64 ? ((const int64_t*)r.hist)[at] : (int64_t)((const int32_t*)r.hist)[at];
        if (id >= lo && id < hi) atomicAdd(&counts[q * cap + (int)(id - lo)], 1u);
    }
    __syncthreads();
}

// ---- reductions over G lanes: G <= 64 adjacent lanes of a wave by exchange, G = kBlock through LDS as well ---------------------------------
template <int G, typename V, typename Op>
__device__ inline V group_reduce(V v, Op op, V* lds) {
#pragma unroll
    for (int s = 1; s < (G < kWave ? G : kWave); s <<= 1) v = op(v, __shfl_xor(v, s));
    if (G > kWave) {
        __syncthreads();
        if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < kBlock / kWave; i++) v = op(v, lds[i]);
    }
    return v;
}

template <typename V> struct Max { __device__ V operator()(V a, V b) const { return a > b ? a : b; } };   // of values without NaN
template <typename V> struct Min { __device__ V operator()(V a, V b) const { return a < b ? a : b; } };
template <typename V> struct Sum { __device__ V operator()(V a, V b) const { return a + b; } };

// 2^t in double to 2e-14 of its value, for -1000 <= t <= 1000: t = n + f, |f| <= 1/2, and a polynomial of degree 9 through the Chebyshev nodes
// for 2^f.  18 instructions, all at the double (= single) rate.
__device__ inline double exp2_double(double t) {
    const double shifted = t + 0x1.8p52;                                     // n in the low word
    const double f = t - (shifted - 0x1.8p52);
    double p = 0x1.b6571de2f2351p-24;
    p = __builtin_fma(p, f, 0x1.63ef969a64d3cp-20);
    p = __builtin_fma(p, f, 0x1.ffcb76789860fp-17);
    p = __builtin_fma(p, f, 0x1.43088e257f341p-13);
    p = __builtin_fma(p, f, 0x1.5d87fe908f88ap-10);
    p = __builtin_fma(p, f, 0x1.3b2ab72b175eep-7);
    p = __builtin_fma(p, f, 0x1.c6b08d7044119p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff8149f2p-3);
    p = __builtin_fma(p, f, 0x1.62e42fefa39f7p-1);
    p = __builtin_fma(p, f, 0x1.000000000003dp+0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(shifted) << 20), __double2loint(p));
}
// Below 2^-1000 a weight counts as none.
constexpr double kLeast = -1000.0;
constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;

// One thread's share of a row's tile: NV vectors of kVec columns, `step` columns apart, as y (see ruled).  Y is double under rules; float
// where y is the logit itself.  Absent columns are -inf.  `bad` is set by a NaN.
template <typename E, bool RULES, int NV>
struct Tile {
    using Y = typename std::conditional<RULES, double, float>::type;
    Y y[NV][E::kVec];

    __device__ void load(const Row& w, const typename E::T* x, int64_t v0, int64_t step, int64_t width, const uint32_t* counts, bool* bad) {
        float f[NV][E::kVec];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (NV == 1 || v0 + k * step < width) load_cols<E>(x, v0 + k * step, width, f[k], -INFINITY);
            else
#pragma unroll
                for (int j = 0; j < E::kVec; j++) f[k][j] = -INFINITY;
        }
        bool nan = false;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t at = v0 + k * step;
            const uint32_t bits = !RULES || at >= width ? 0xFFu : allowed_bits(w, at);
#pragma unroll
            for (int j = 0; j < E::kVec; j++) {
                if (RULES) {
                    const bool here = at + j < width;
                    y[k][j] = ruled(w, f[k][j], here && counts ? counts[k * step + j] : 0u, bits >> j & 1, here ? at + j : 0);
                    if (!here) y[k][j] = -INFINITY;
                } else {
                    y[k][j] = f[k][j];
                }
                nan = nan || y[k][j] != y[k][j];
            }
        }
        *bad = nan;
    }
    __device__ Y max() const {
        Y m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int j = 0; j < E::kVec; j++) m = y[k][j] > m ? y[k][j] : m;
        return m;
    }
};

// ---- host side -------------------------------------------------------------------------------------------------------------------------
int check_matrix(const char* what, const void* data, int type, int64_t rows, int64_t width, int64_t stride);
int check_output(const char* what, const void* out, int type, int64_t rows, int64_t width, int64_t stride, const void* in, int64_t in_stride);
int check_rules(const gymhip_logit_rules* r, int64_t rows, int64_t width, Rules* out);
int check_keys(const gymhip_random_keys* k, Keys* out);
int check_actions(const void* actions, int dtype, int64_t rows);
int check_workspace(const void* workspace, size_t bytes, size_t needed);
int launched();

// Workgroups for n units of work: as many as there are, up to what keeps every CU busy several times over; kernels stride over the rest.
inline unsigned grid_for(int64_t n, int64_t most = 1 << 16) { return (unsigned)(n < most ? n : most); }

// f(E{}) for the element type of `type`.
template <typename F>
int with_type(int type, F f) {
    if (type == GYMHIP_TYPE_F32) f(F32{});
    else if (type == GYMHIP_TYPE_F16) f(F16{});
    else f(BF16{});
    return launched();
}
template <typename F>
void with_bool(bool v, F f) {
    if (v) f(std::true_type{});
    else f(std::false_type{});
}

}  // namespace policy
}  // namespace gymhip
