// policy_common.h — what the policy kernels (policy_*.hip) share: element types, the counter-based generator, the rules on logits, reductions
// over groups of lanes, and the host-side checks of the entry points.  Formulas: include/gymhip.h.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/gymhip.h"
#include "gymhip_internal.h"

namespace gymhip {
namespace policy {

constexpr int kBlock = 256;
constexpr int kWave = 64;

// ---- element types: kVec elements are 16 bytes; loads widen to float, stores round a float to nearest even -----------------------------
struct F32 {
    using T = float;
    static constexpr int kVec = 4;
    static constexpr uint32_t kNone = 0xFF800000u;   // -inf
    __device__ static float widen(const uint32_t* w, int j) { return __uint_as_float(w[j]); }
    __device__ static uint32_t narrow(const float* v) { return __float_as_uint(v[0]); }
};
struct F16 {
    using T = _Float16;
    static constexpr int kVec = 8;
    static constexpr uint32_t kNone = 0xFC00FC00u;
    __device__ static float widen(const uint32_t* w, int j) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(j & 1 ? w[j / 2] >> 16 : w[j / 2])); }
    __device__ static uint32_t narrow(const float* v) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[0]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16;
    }
};
struct BF16 {
    using T = __bf16;
    static constexpr int kVec = 8;
    static constexpr uint32_t kNone = 0xFF80FF80u;
    __device__ static float widen(const uint32_t* w, int j) { return __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16); }
    __device__ static uint32_t narrow(const float* v) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[0]) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[1]) << 16;
    }
};

// C adjacent elements of a row, as they lie in memory: C * sizeof(T) is 4, 8 or 16 bytes.  The address has the element's alignment only (odd
// strides, odd starts); the hardware takes 16-byte accesses at any such address, so a row needs no aligned middle of its own.
template <typename E, int C>
struct Raw {
    using T = typename E::T;
    static constexpr int kWords = C * (int)sizeof(T) / 4;
    uint32_t w[kWords];
    struct __attribute__((packed, aligned(sizeof(T)))) Packed { uint32_t w[kWords]; };

    // Columns from v0 on; those behind the row's end are -inf, and not read.
    __device__ void load(const T* row, int64_t v0, int64_t width) {
        if (v0 + C <= width) {
            const Packed p = *(const Packed*)(row + v0);
#pragma unroll
            for (int i = 0; i < kWords; i++) w[i] = p.w[i];
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i++) w[i] = E::kNone;
#pragma unroll
            for (int j = 0; j < C; j++)
                if (v0 + j < width) {
                    if (sizeof(T) == 4) w[j] = ((const uint32_t*)row)[v0 + j];
                    else {
                        const uint32_t e = ((const uint16_t*)row)[v0 + j];
                        w[j / 2] = j & 1 ? (w[j / 2] & 0xFFFFu) | e << 16 : (w[j / 2] & 0xFFFF0000u) | e;
                    }
                }
        }
    }
    __device__ float get(int j) const { return E::widen(w, j); }
    // get(j), and j set to v, for a j that is not known at compile time: by shifts, as a register has no index.
    __device__ float pick(int j) const {
        static_assert(kWords == 4, "");
        const uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
        constexpr int half = C / 2;
        const uint32_t e[1] = {(uint32_t)((j & half ? hi : lo) >> ((j & (half - 1)) * (int)sizeof(T) * 8))};
        return E::widen(e, 0);
    }
    __device__ void put(int j, float v) {
        static_assert(kWords == 4, "");
        constexpr int half = C / 2;
        const float pair[2] = {v, 0.f};
        const int shift = (j & (half - 1)) * (int)sizeof(T) * 8;
        const uint64_t m = (sizeof(T) == 4 ? 0xFFFFFFFFull : 0xFFFFull) << shift, bits = (uint64_t)E::narrow(pair) << shift;
        const uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
        const uint64_t l = j & half ? lo : (lo & ~m) | (bits & m), h = j & half ? (hi & ~m) | (bits & m) : hi;
        w[0] = (uint32_t)l;
        w[1] = (uint32_t)(l >> 32);
        w[2] = (uint32_t)h;
        w[3] = (uint32_t)(h >> 32);
    }
    // All ones in the places of those elements of word i whose bit is set.
    __device__ static uint32_t places(uint32_t bits, int i) {
        if (sizeof(T) == 4) return (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_sbfe((int)bits, 2 * i, 1), hi = (uint32_t)__builtin_amdgcn_sbfe((int)bits, 2 * i + 1, 1);
        return __builtin_amdgcn_perm(hi, lo, 0x05040100u);   // two bytes of each
    }
    // Elements whose bit is 0 become -inf, or 0.
    __device__ void keep(uint32_t bits) {
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            const uint32_t m = places(bits, i);
            w[i] = (w[i] & m) | (E::kNone & ~m);
        }
    }
    __device__ void clear(uint32_t bits) {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] &= places(bits, i);
    }
    __device__ void set(const float* v) {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = E::narrow(v + i * C / kWords);
    }
    __device__ void store(T* row, int64_t v0, int64_t width) const {
        if (v0 + C <= width) {
            Packed p;
#pragma unroll
            for (int i = 0; i < kWords; i++) p.w[i] = w[i];
            *(Packed*)(row + v0) = p;
        } else {
#pragma unroll
            for (int j = 0; j < C; j++)
                if (v0 + j < width) {
                    if (sizeof(T) == 4) ((uint32_t*)row)[v0 + j] = w[j];
                    else ((uint16_t*)row)[v0 + j] = (uint16_t)(j & 1 ? w[j / 2] >> 16 : w[j / 2]);
                }
        }
    }
};

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
    const double one_to_two = __hiloint2double((int)(0x3FF00000u | w.x >> 12), (int)(w.x << 20 | w.y >> 12));
    return one_to_two - 1.0 + 0x1p-53;
}

// ---- rules ---------------------------------------------------------------------------------------------------------------------------
// What a temperature makes of exponentials: exp(y / temp) is 2^(y k2).  From `least` on down that is below 2^-1000, up to `most` at most 2^900.
struct Heat {
    double temp, k2, least, most;
    bool greedy;
    static __host__ __device__ Heat of(float t) {
        Heat h;
        h.greedy = !(t > 0.f);
        h.temp = h.greedy ? 1.0 : t < INFINITY ? (double)t : 3.4028234663852886e38;   // an infinite one (values of tensors are not checked): as the greatest float
        h.k2 = 1.4426950408889634074 / h.temp;
        const double unit = h.temp * 0.69314718055994530942, most = 900.0 * unit;
        h.least = -1000.0 * unit;
        h.most = most < 3e38 ? most : 3e38;   // an infinite logit is above it
        return h;
    }
};

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
    float rep, pres, freq;
    Heat heat;   // of the one temperature where temp_rows is null, made on the host
    // y is the logit itself, or -inf where the mask does not allow it
    __host__ __device__ bool plain() const { return !bias && !hist; }
};

// One row's share of them.
struct Row : Heat {
    const uint32_t* mask;   // its line, or null where everything is allowed
    const float* bias;
    double rep, inv_rep, pres, freq;
    bool masked, biased;    // there is a mask, a bias at all: the same for all rows
    bool nothing;           // its line lies behind the mask's last one
};

// RULES: there is a bias or a history.
template <bool RULES>
__device__ inline Row row_of(const Rules& r, int64_t b) {
    Row w;
    // (all of it in the branch: a temperature of its own costs a division)
    if (r.temp_rows) (Heat&)w = Heat::of(r.temp_rows[b]);
    else (Heat&)w = r.heat;
    w.masked = r.mask != nullptr;
    w.biased = RULES && r.bias;
    w.mask = nullptr;
    w.bias = nullptr;
    w.nothing = false;
    w.rep = w.inv_rep = 1.0;
    w.pres = w.freq = 0.0;
    if (r.mask) {
        const int64_t line = r.mask_rows ? r.mask_rows[b] : (r.mask_lines == 1 ? 0 : b);
        w.nothing = line >= r.mask_lines;
        if (line >= 0 && !w.nothing) w.mask = r.mask + line * r.mask_stride;
    }
    if (RULES) {
        if (r.bias) w.bias = r.bias + b * r.bias_stride;
        if (r.hist) {
            w.rep = r.rep_rows ? r.rep_rows[b] : r.rep;
            w.inv_rep = 1.0 / w.rep;
            w.pres = r.pres_rows ? r.pres_rows[b] : r.pres;
            w.freq = r.freq_rows ? r.freq_rows[b] : r.freq;
        }
    }
    return w;
}

// x / d as IEEE rounds it, with inv = 1 / d rounded: the quotient's remainder is exact in one fma and corrects it (Markstein's theorem; x and d
// are far from a double's range, being floats or sums of a few).  Infinities and NaN, whose remainder is NaN, keep the first quotient.
__device__ inline double divided(double x, double d, double inv) {
    const double q = x * inv;
    const double c = __builtin_fma(__builtin_fma(-q, d, x), inv, q);
    return fabs(q) < INFINITY ? c : q;
}

// The mask's bits of C (at most 8) columns from v0 on, v0 a multiple of C; of none behind the row's end.
__device__ inline uint32_t allowed_bits(const Row& w, int64_t v0, int64_t width) {
    if (!w.masked) return 0xFFu;
    if (w.nothing) return 0u;
    return w.mask && v0 < width ? w.mask[v0 >> 5] >> (v0 & 31) : 0xFFu;
}

__device__ inline bool allowed(const Row& w, int64_t v) { return !w.nothing && (!w.mask || (w.mask[v >> 5] >> (v & 31) & 1u)); }

// x under the penalties of a count > 0.
__device__ inline double penalised(const Row& w, double x, uint32_t count) {
    const double y = x > 0 ? divided(x, w.rep, w.inv_rep) : x * w.rep;
    return y - w.freq * (double)count - w.pres;
}
// y of one column.
__device__ inline double ruled(const Row& w, float xf, uint32_t count, bool ok, int64_t v) {
    double y = xf;
    if (count) y = penalised(w, y, count);
    if (w.biased) y += (double)w.bias[v];
    return ok ? y : -INFINITY;
}

// The biases of C columns from v0 on.
template <int C>
__device__ inline void bias_cols(const Row& w, int64_t v0, int64_t width, float* f) {
    if (v0 + C <= width) {
        struct __attribute__((packed, aligned(4))) Packed { float f[C]; };
        const Packed p = *(const Packed*)(w.bias + v0);
#pragma unroll
        for (int j = 0; j < C; j++) f[j] = p.f[j];
    } else {
#pragma unroll
        for (int j = 0; j < C; j++) f[j] = v0 + j < width ? w.bias[v0 + j] : 0.f;
    }
}

// Workgroup i of rows * cuts, cuts to a row.  Adjacent workgroups go to the 8 XCDs in turn, each with an L2 of its own: eight rows are taken side by side, so that
// a row's cuts, which all read its history, share one; in another order each time, so that dearer rows at a regular distance are spread over the XCDs.
// (512 x 131,072 bf16 after 4,096 ids, us: process_logits 96 -> 85, sample_actions under all rules 196 -> 177.)
struct Cut {
    int64_t row;
    uint32_t cut;
    __device__ Cut(int64_t i, uint32_t cuts, int64_t rows) {
        if (cuts == 1) {
            row = i;
            cut = 0;
            return;
        }
        const int64_t eight = i / (8 * cuts);
        const uint32_t rest = (uint32_t)(i - eight * (8 * cuts)), side = rows - eight * 8 < 8 ? (uint32_t)(rows - eight * 8) : 8u;
        cut = rest / side;
        row = eight * 8 + (rest - cut * side + (uint32_t)(eight & 7)) % side;
    }
};

// How often ids occur in a tile of columns of n rows, in LDS: 32 bits each, or 16 where no history is longer than 65,535; and with `bits` a bit for
// each id that occurs at all, behind the counts (cap is a multiple of 32 then).
struct Counts {
    uint32_t* words;   // null: there is no history
    int cap, all;      // columns of a row's tile; of all n rows'
    bool half, bits;

    __device__ uint32_t* touched() const { return words + (half ? all / 2 : all); }
    __device__ int size() const { return (half ? all / 2 : all) + (bits ? all / 32 : 0); }
    __device__ uint32_t at(int i) const { return half ? words[i >> 1] >> (16 * (i & 1)) & 0xFFFFu : words[i]; }
    // C counts from i on, i a multiple of C.
    template <int C>
    __device__ void get(int i, uint32_t* c) const {
        if (half) {
#pragma unroll
            for (int j = 0; j < C / 2; j++) {
                const uint32_t v = words[i / 2 + j];
                c[2 * j] = v & 0xFFFFu;
                c[2 * j + 1] = v >> 16;
            }
        } else {
#pragma unroll
            for (int j = 0; j < C; j++) c[j] = words[i + j];
        }
    }
    // Which of the C columns from i on have a count.
    template <int C>
    __device__ uint32_t which(int i) const {
        if (bits) return touched()[i >> 5] >> (i & 31) & ((1u << C) - 1);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < C; j++) m |= at(i + j) ? 1u << j : 0u;
        return m;
    }
    // Whether any lane of the wave has a count among the columns of its vector at i (or it is not known without going through them).
    template <int C>
    __device__ bool any(int i) const { return words && (!bits || __any(which<C>(i))); }
};

// A vector as it is loaded: its columns, and the mask's bits for them.
template <typename E, int C>
struct Vector {
    Raw<E, C> raw;
    uint32_t bits;
    __device__ void load(const Row& w, const typename E::T* row, int64_t at, int64_t width) {
        raw.load(row, at, at < width ? width : 0);
        bits = allowed_bits(w, at, width);
    }
};

// y of C columns from v0 on: the logits after penalties and bias, before the temperature; -inf where the mask does not allow.  In double (which
// runs at the rate of float here): what is compared and summed must be the formula's value even where a bias or a penalty cancels most of
// the logit.  Straight-line code: a wave passes over the penalties only where none of its lanes has a count (`counted` false, or found here).  bits: allowed_bits of the columns.
template <typename E, int C>
__device__ inline void ruled_cols(const Row& w, const Raw<E, C>& raw, uint32_t bits, int64_t v0, int64_t width, const Counts& counts, int place, bool counted,
                                  double* y) {
#pragma unroll
    for (int j = 0; j < C; j++) y[j] = (double)raw.get(j);
    if (counted) {
        uint32_t c[C], any = 0;
        counts.get<C>(place, c);
#pragma unroll
        for (int j = 0; j < C; j++) any |= c[j];
        if (__any(any)) {
#pragma unroll
            for (int j = 0; j < C; j++) {
                const double p = penalised(w, y[j], c[j]);
                y[j] = c[j] ? p : y[j];
            }
        }
    }
    if (w.biased) {
        float f[C];
        bias_cols<C>(w, v0, width, f);
#pragma unroll
        for (int j = 0; j < C; j++) y[j] += (double)f[j];
    }
#pragma unroll
    for (int j = 0; j < C; j++) y[j] = bits >> j & 1 ? y[j] : -INFINITY;
}

// Counts the ids of columns [lo, lo + span) of a row's history, `step` lanes together of which this one is `first`, from place `base` on.
template <typename Id>
__device__ inline void count_row(const Id* ids, int64_t len, int64_t lo, uint32_t span, int first, int step, const Counts& c, int base, bool bits) {
    struct __attribute__((packed, aligned(sizeof(Id)))) Four { Id v[4]; };
    uint32_t* touched = c.touched();
    auto count = [&](Id id) {
        const uint64_t off = (uint64_t)((int64_t)id - lo);
        if (off < span) {
            const int at = base + (int)off;
            if (c.half) atomicAdd(&c.words[at >> 1], 1u << (16 * (at & 1)));
            else atomicAdd(&c.words[at], 1u);
            if (bits) atomicOr(&touched[at >> 5], 1u << (at & 31));
        }
    };
    for (int64_t i = (int64_t)first * 4; i < len; i += (int64_t)step * 4) {   // (2 or 4 loads under way: the same or, for their registers, slower)
        if (i + 4 <= len) {
            const Four f = *(const Four*)(ids + i);
#pragma unroll
            for (int j = 0; j < 4; j++) count(f.v[j]);
        } else {
            for (int64_t j = i; j < len; j++) count(ids[j]);
        }
    }
}
// Counts the ids of columns [lo, lo + cap) in the histories of rows [b0, b0 + n), n a power of two.  By the
// whole workgroup: every thread comes here, and counts may be read after it returns.  Integer LDS atomics, so their order is free.  Lanes that add to one
// word wait for each other, and ids repeat: where the row's columns leave most of its tile empty, adjacent lanes count in
// copies, added up afterwards (1,339 rows of 3 columns after 12,191 ids: 178 -> 71 us).  COPIES false: rows wider than a tile, which leave nothing.
template <bool COPIES = true>
__device__ inline void count_ids(const Rules& r, int64_t b0, int n, int64_t rows, int64_t width, int64_t lo, const Counts& c) {
    __syncthreads();
    for (int i = threadIdx.x; i < c.size() / 4; i += kBlock) ((uint4*)c.words)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const uint32_t span = (uint32_t)(lo + c.cap < width ? c.cap : width - lo);
    const int each = kBlock / n, mine = (int)threadIdx.x / each;   // `each` adjacent threads take a row
    const int first = (int)threadIdx.x & (each - 1);
    int pitch = c.cap, copies = 1;
    while (COPIES && copies < each && copies < 16 && pitch % 4 == 0 && span * 2 <= (uint32_t)pitch) {
        pitch /= 2;
        copies *= 2;
    }
    const int64_t b = b0 + mine;
    if (b < rows) {
        int64_t len = r.hist_cols;
        if (r.hist_len) {
            const int64_t have = r.len64 ? ((const int64_t*)r.hist_len)[b] : (int64_t)((const int32_t*)r.hist_len)[b];
            len = have < len ? have : len;
        }
        const int base = mine * c.cap + (first & (copies - 1)) * pitch;
        const bool bits = c.bits && copies == 1;
        if (r.hist64) count_row((const int64_t*)r.hist + b * r.hist_stride, len, lo, span, first, each, c, base, bits);
        else count_row((const int32_t*)r.hist + b * r.hist_stride, len, lo, span, first, each, c, base, bits);
    }
    __syncthreads();
    if (copies > 1) {
        // a word at a time (of 16-bit counts two, which no sum overflows): the copies' columns are cleared, nobody has them
        const int shift = c.half ? 1 : 0, words = (int)(span + shift) >> shift;
        for (int i = first; i < words; i += each) {
            uint32_t* w = c.words + (mine * c.cap >> shift) + i;
            uint32_t sum = w[0];
            for (int k = 1; k < copies; k++) {
                uint32_t* more = w + k * (pitch >> shift);
                sum += *more;
                *more = 0;
            }
            w[0] = sum;
            if (c.bits) {
                const int at = mine * c.cap + (i << shift);
                const uint32_t low = c.half ? sum & 0xFFFFu : sum, high = c.half ? sum >> 16 : 0u;
                const uint32_t set = (low ? 1u : 0u) | (high ? 2u : 0u);
                if (set) atomicOr(&c.touched()[at >> 5], set << (at & 31));
            }
        }
        __syncthreads();
    }
}

// A workgroup's tile of columns is kTile 16-byte vectors a lane at most; half as many where the counts take 32 bits, so that both fit the same LDS.
constexpr int kTile = 4;
template <typename E>
constexpr int counts_words() { return kBlock * E::kVec * kTile / 2 + kBlock * E::kVec * kTile / 32; }
inline bool half_counts(const Rules& r) { return r.hist_cols <= 65535; }
// Where a lane goes through its row vector by vector (sample_actions, action_log_prob) a workgroup's tile under a history is 8,192 columns whatever their type, or 4,096
// counted in 32 bits: 17 KB.  Of a wave's row it is half as much, for four rows 34 KB: four workgroups a CU, as many as there are registers for.
template <int G>
constexpr int strip_words() { return (G == kWave ? 2 : 1) * (8192 / 2 + 8192 / 32); }
template <typename E>
int strip_vectors(const Rules& r, int lanes) { return (lanes == kWave ? 2 : 1) * (half_counts(r) ? 8192 : 4096) / (kBlock * E::kVec); }

// Lanes that share a row which `least` lanes hold: more of them where a history is to be counted and the rows alone do not make the 2,048 workgroups that
// fill the chip (1,339 rows of 3 columns after 12,191 ids each, 256 lanes instead of one: 3,430 -> 178 us).
inline int lanes_for(const Rules& r, int64_t rows, int least) {
    int g = least;
    while (g < kBlock && r.hist && r.hist_cols > 4 * g && rows * g < 2048 * kBlock) g *= 2;
    return g;
}

// ---- reductions over G lanes: G <= 64 adjacent lanes of a wave by lane permutations in the vector unit, G = kBlock through LDS as well --------
template <int CTRL, int ROWS = 0xF>
__device__ inline uint32_t permuted(uint32_t v, uint32_t else_) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)else_, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS = 0xF, typename V>
__device__ inline V permuted_value(V v, V else_) {
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "");
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, permuted<CTRL, ROWS>(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, else_)));
    } else {
        const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, else_);
        const uint64_t lo = permuted<CTRL, ROWS>((uint32_t)a, (uint32_t)b), hi = permuted<CTRL, ROWS>((uint32_t)(a >> 32), (uint32_t)(b >> 32));
        return __builtin_bit_cast(V, hi << 32 | lo);
    }
}

template <int G, typename V, typename Op>
__device__ inline V group_reduce(V v, Op op, V* lds) {
    if (G >= 2) v = op(v, permuted_value<0xB1>(v, v));    // lane ^ 1
    if (G >= 4) v = op(v, permuted_value<0x4E>(v, v));    // lane ^ 2
    if (G >= 8) v = op(v, permuted_value<0x141>(v, v));   // 7 - lane: the other four, which by now hold one value
    if (G >= 16) v = op(v, permuted_value<0x140>(v, v));  // 15 - lane
    if (G >= 32) v = op(v, __shfl_xor(v, 16));
    if (G >= 64) v = op(v, __shfl_xor(v, 32));
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

// Sums over lanes 0 .. lane of each group of W <= 64 lanes.
template <int W>
__device__ inline double running_sum(double v, int lane) {
    if (W >= 2) { const double o = permuted_value<0x111>(v, 0.0); v += lane >= 1 ? o : 0.0; }
    if (W >= 4) { const double o = permuted_value<0x112>(v, 0.0); v += lane >= 2 ? o : 0.0; }
    if (W >= 8) { const double o = permuted_value<0x114>(v, 0.0); v += lane >= 4 ? o : 0.0; }
    if (W >= 16) { const double o = permuted_value<0x118>(v, 0.0); v += lane >= 8 ? o : 0.0; }
    if (W >= 32) v += permuted_value<0x142, 0xA>(v, 0.0);   // the last lane of a row of 16 to the next row
    if (W >= 64) v += permuted_value<0x143, 0xC>(v, 0.0);   // lane 31 to the upper half
    return v;
}

// Orders what the lanes of a group have written to LDS before what they read.
template <int G>
__device__ inline void group_sync() {
    if (G > kWave) {
        __syncthreads();
    } else {   // one wave's LDS accesses are in order: the compiler has to keep them so
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename V> struct Max { __device__ V operator()(V a, V b) const { return a > b ? a : b; } };   // of values without NaN
template <typename V> struct Min { __device__ V operator()(V a, V b) const { return a < b ? a : b; } };
template <typename V> struct Sum { __device__ V operator()(V a, V b) const { return a + b; } };

// 2^(d k) in double to 4e-14 of its value (and 1 for 0), for -1000 <= d k <= 1000: d k = n + f, |f| <= 1/2, and for (2^f - 1) / f the polynomial of
// degree 8 through the Chebyshev nodes.  14 instructions, all at the double (= float) rate.
__device__ inline double exp2_double(double d, double k) {
    const double shifted = __builtin_fma(d, k, 0x1.8p52);                    // n in the low word
    const double f = __builtin_fma(d, k, -(shifted - 0x1.8p52));
    double p = 0x1.b63880f05fbb6p-24;
    p = __builtin_fma(p, f, 0x1.63d136346743dp-20);
    p = __builtin_fma(p, f, 0x1.ffcb95155e91bp-17);
    p = __builtin_fma(p, f, 0x1.4308ac85ac496p-13);
    p = __builtin_fma(p, f, 0x1.5d87fe86fe9e5p-10);
    p = __builtin_fma(p, f, 0x1.3b2ab7181b749p-7);
    p = __builtin_fma(p, f, 0x1.c6b08d7047e52p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff823cedp-3);
    p = __builtin_fma(p, f, 0x1.62e42fefa39efp-1);
    p = __builtin_fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(shifted) << 20), __double2loint(p));
}
// log2 s for a normal s: its exponent, and of its mantissa a the float logarithm l with a 2^-l = 1 + e, |e| < 1e-6, whose logarithm is three terms
// of its series.
__device__ inline double log2_double(double s) {
    const int n = (int)(__double2hiint(s) >> 20) - 1023;
    const double a = __hiloint2double((__double2hiint(s) & 0xFFFFF) | 0x3FF00000, __double2loint(s));
    const double l = (double)__builtin_amdgcn_logf((float)a);
    const double e = __builtin_fma(a, exp2_double(-l, 1.0), -1.0);
    return __builtin_fma(__builtin_fma(__builtin_fma(e, 1.0 / 3.0, -0.5), e, 1.0) * e, 1.4426950408889634074, l) + (double)n;
}
// As a float that is not infinite: a temperature may be so low that its reciprocal overflows, and what is 0 beside it is to stay 0.
__device__ inline float finite(double v) { return (float)__builtin_fmin(v, 3e38); }
constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;

// ---- host side -------------------------------------------------------------------------------------------------------------------------
int check_matrix(const char* what, const void* data, int type, int64_t rows, int64_t width, int64_t stride);
int check_output(const char* what, const void* out, int type, int64_t rows, int64_t width, int64_t stride, const void* in, int64_t in_stride);
int check_rules(const gymhip_logit_rules* r, int64_t rows, int64_t width, Rules* out);
int check_keys(const gymhip_random_keys* k, Keys* out);
int check_actions(const void* actions, int dtype, int64_t rows);
int check_workspace(const void* workspace, size_t bytes, size_t needed);
struct Range {
    const char* what;
    const void* at;
    int64_t bytes;
};
int check_results(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, std::initializer_list<Range> results);
int launched();

// Workgroups for n units of work: as many as there are, up to `most`; kernels stride over the rest.
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
