// policy.hip — the policy's end of the VecEnv loop: rules on logits (penalties for repeated choices, biases, masks, temperature), the draw of
// an action, its log-probability and entropy with their gradients, and dropout.  Entry points and formulas: include/gymhip.h.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/gymhip.h"
#include "gymhip_internal.h"

namespace gymhip {
namespace {

constexpr int kBlock = 256;
constexpr int kChunk = 4096;   // columns whose history counts are held in LDS at a time

// ---- element types: 16-bit loads widen to float, stores round to nearest even --------------------------------------------------------
struct F32 {
    using T = float;
    __device__ static float load(const T* p) { return *p; }
    __device__ static void store(T* p, float v) { *p = v; }
};
struct F16 {
    using T = _Float16;
    __device__ static float load(const T* p) { return (float)*p; }
    __device__ static void store(T* p, float v) { *p = (_Float16)v; }
};
struct BF16 {
    using T = __bf16;
    __device__ static float load(const T* p) { return (float)*p; }
    __device__ static void store(T* p, float v) { *p = (__bf16)v; }
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
    int64_t hist_stride, hist_cols;
    const void* hist_len;
    int hist64, len64;
    const float *rep_rows, *pres_rows, *freq_rows, *temp_rows;
    float rep, pres, freq, temp;
};

// One row's share of them.
struct Row {
    double rep, pres, freq, temp;
    bool greedy;
    const uint32_t* mask;   // its line, or null where everything is allowed
    bool nothing;           // its line lies behind the mask's last one
    const float* bias;
    const int32_t* h32;
    const int64_t* h64;
    int64_t len;
};

__device__ inline Row row_of(const Rules& r, int64_t b) {
    Row w;
    w.rep = r.rep_rows ? r.rep_rows[b] : r.rep;
    w.pres = r.pres_rows ? r.pres_rows[b] : r.pres;
    w.freq = r.freq_rows ? r.freq_rows[b] : r.freq;
    const float t = r.temp_rows ? r.temp_rows[b] : r.temp;
    w.greedy = !(t > 0.f);
    w.temp = w.greedy ? 1.0 : (double)t;
    w.mask = nullptr;
    w.nothing = false;
    if (r.mask) {
        const int64_t line = r.mask_rows ? r.mask_rows[b] : (r.mask_lines == 1 ? 0 : b);
        w.nothing = line >= r.mask_lines;
        if (line >= 0 && !w.nothing) w.mask = r.mask + line * r.mask_stride;
    }
    w.bias = r.bias ? r.bias + b * r.bias_stride : nullptr;
    w.h32 = nullptr;
    w.h64 = nullptr;
    w.len = 0;
    if (r.hist) {
        if (r.hist64) w.h64 = (const int64_t*)r.hist + b * r.hist_stride;
        else w.h32 = (const int32_t*)r.hist + b * r.hist_stride;
        w.len = r.hist_cols;
        if (r.hist_len) {
            const int64_t n = r.len64 ? ((const int64_t*)r.hist_len)[b] : ((const int32_t*)r.hist_len)[b];
            w.len = n < 0 ? 0 : (n < w.len ? n : w.len);
        }
    }
    return w;
}

__device__ inline bool allowed(const Row& w, int64_t v) {
    return !w.nothing && (!w.mask || ((w.mask[v >> 5] >> (v & 31)) & 1u));
}

// z in double precision: double arithmetic runs at the rate of single here, and every use of z (rounded out, compared, summed) then sees
// the formula's value to 2^-52.
__device__ inline double ruled(const Row& w, float xf, uint32_t count, int64_t v) {
    if (!allowed(w, v)) return -INFINITY;
    double x = xf;
    if (count) {
        x = x > 0 ? x / w.rep : x * w.rep;
        x = x - w.freq * (double)count - w.pres;
    }
    if (w.bias) x = x + (double)w.bias[v];
    return x / w.temp;
}
__device__ inline double slope(const Row& w, float xf, uint32_t count, int64_t v) {
    if (!allowed(w, v)) return 0.0;
    double g = 1.0;
    if (count) g = xf > 0.f ? 1.0 / w.rep : w.rep;
    return g / w.temp;
}

// How often each id of columns [lo, lo + kChunk) occurs in the row's history, by the whole workgroup; integer atomics, so the order is free.
__device__ inline void count_chunk(const Row& w, int64_t lo, uint32_t* counts) {
    __syncthreads();
    for (int i = threadIdx.x; i < kChunk; i += kBlock) counts[i] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < w.len; i += kBlock) {
        const int64_t id = w.h64 ? w.h64[i] : (int64_t)w.h32[i];
        if (id >= lo && id < lo + kChunk) atomicAdd(&counts[id - lo], 1u);
    }
    __syncthreads();
}

template <typename V, typename Op>
__device__ inline V block_reduce(V v, Op op, V* scratch) {
    __syncthreads();
    scratch[threadIdx.x] = v;
    __syncthreads();
    for (int s = kBlock / 2; s > 0; s >>= 1) {
        if ((int)threadIdx.x < s) scratch[threadIdx.x] = op(scratch[threadIdx.x], scratch[threadIdx.x + s]);
        __syncthreads();
    }
    return scratch[0];
}

// Walks a row chunk by chunk: f(v, x, count) for every column, each by one thread.
template <typename E, typename F>
__device__ inline void each_column(const Row& w, const typename E::T* x, int64_t width, uint32_t* counts, F f) {
    for (int64_t lo = 0; lo < width; lo += kChunk) {
        if (w.len) count_chunk(w, lo, counts);
        const int64_t hi = lo + kChunk < width ? lo + kChunk : width;
        for (int64_t v = lo + threadIdx.x; v < hi; v += kBlock) f(v, E::load(x + v), w.len ? counts[v - lo] : 0u);
    }
}

// ---- kernels: one workgroup per row ----------------------------------------------------------------------------------------------------
template <typename E>
__global__ void __launch_bounds__(kBlock) process_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, Rules r,
                                                         typename E::T* out, int64_t out_stride) {
    __shared__ uint32_t counts[kChunk];
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Row w = row_of(r, b);
        each_column<E>(w, x + b * stride, width, counts,
                       [&](int64_t v, float xf, uint32_t c) { E::store(out + b * out_stride + v, (float)ruled(w, xf, c, v)); });
    }
}

template <typename E>
__global__ void __launch_bounds__(kBlock) process_backward_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, Rules r,
                                                                  const typename E::T* g, int64_t g_stride, typename E::T* out, int64_t out_stride) {
    __shared__ uint32_t counts[kChunk];
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Row w = row_of(r, b);
        each_column<E>(w, x + b * stride, width, counts, [&](int64_t v, float xf, uint32_t c) {
            const double s = slope(w, xf, c, v);
            E::store(out + b * out_stride + v, s == 0.0 ? 0.f : (float)((double)E::load(g + b * g_stride + v) * s));
        });
    }
}

template <typename E>
__global__ void __launch_bounds__(kBlock) sample_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r, Keys keys,
                                                        int32_t* actions, float* log_prob) {
    __shared__ uint32_t counts[kChunk];
    __shared__ double scratch[kBlock];
    __shared__ long long scratch_at[kBlock];
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Row w = row_of(r, b);
        const typename E::T* x = x0 + b * stride;
        double m = -INFINITY;
        long long at = width;
        each_column<E>(w, x, width, counts, [&](int64_t v, float xf, uint32_t c) {
            const double z = ruled(w, xf, c, v);
            if (z > m) { m = z; at = v; }
        });
        const double mine = m;
        m = block_reduce(m, [](double p, double q) { return p > q ? p : q; }, scratch);
        at = block_reduce(mine == m ? at : (long long)width, [](long long p, long long q) { return p < q ? p : q; }, scratch_at);
        const double base = m == -INFINITY ? 0.0 : m;
        double sum = 0;
        each_column<E>(w, x, width, counts, [&](int64_t v, float xf, uint32_t c) { sum += exp(ruled(w, xf, c, v) - base); });
        sum = block_reduce(sum, [](double p, double q) { return p + q; }, scratch);
        int32_t action = -1;
        float lp = sum == 0.0 ? -INFINITY : NAN;
        if (sum > 0.0 && sum < INFINITY) {
            if (!w.greedy) {
                // the running sum, 256 columns at a time; the least column that passes the level, or the last one with any weight
                const double level = row_uniform(keys, b) * sum;
                double before = 0;
                long long last = -1;
                at = -1;
                for (int64_t lo = 0; lo < width && at < 0; lo += kChunk) {
                    if (w.len) count_chunk(w, lo, counts);
                    for (int64_t base_v = lo; base_v < lo + kChunk && base_v < width && at < 0; base_v += kBlock) {
                        const int64_t v = base_v + threadIdx.x;
                        const double e = v < width ? exp(ruled(w, E::load(x + v), w.len ? counts[v - lo] : 0u, v) - base) : 0.0;
                        __syncthreads();
                        scratch[threadIdx.x] = e;
                        __syncthreads();
                        for (int s = 1; s < kBlock; s <<= 1) {
                            const double o = (int)threadIdx.x >= s ? scratch[threadIdx.x - s] : 0.0;
                            __syncthreads();
                            scratch[threadIdx.x] += o;
                            __syncthreads();
                        }
                        const double upto = before + scratch[threadIdx.x], all = before + scratch[kBlock - 1];
                        const long long hit = e > 0.0 && upto > level ? (long long)v : (long long)width;
                        const long long any = e > 0.0 ? (long long)v : -1;
                        const long long first = block_reduce(hit, [](long long p, long long q) { return p < q ? p : q; }, scratch_at);
                        const long long most = block_reduce(any, [](long long p, long long q) { return p > q ? p : q; }, scratch_at);
                        if (first < width) at = first;
                        last = most > last ? most : last;
                        before = all;
                    }
                }
                if (at < 0) at = last;
            }
            if (w.len) count_chunk(w, at, counts);   // the chosen column's own count, at counts[0]
            action = (int32_t)at;
            lp = (float)(ruled(w, E::load(x + at), w.len ? counts[0] : 0u, at) - base - log(sum));
        }
        if (threadIdx.x == 0) {
            actions[b] = action;
            log_prob[b] = lp;
        }
        __syncthreads();
    }
}

template <typename E>
__global__ void __launch_bounds__(kBlock) score_kernel(const typename E::T* x0, int64_t rows, int64_t width, int64_t stride, Rules r,
                                                       const void* actions, int act64, float* log_prob, float* entropy, double* log_sum) {
    __shared__ uint32_t counts[kChunk];
    __shared__ double scratch[kBlock];
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Row w = row_of(r, b);
        const typename E::T* x = x0 + b * stride;
        const int64_t act = act64 ? ((const int64_t*)actions)[b] : ((const int32_t*)actions)[b];
        double m = -INFINITY, za = -INFINITY;
        each_column<E>(w, x, width, counts, [&](int64_t v, float xf, uint32_t c) {
            const double z = ruled(w, xf, c, v);
            m = z > m ? z : m;
            if (v == act) za = z;
        });
        m = block_reduce(m, [](double p, double q) { return p > q ? p : q; }, scratch);
        // one thread holds the action's z; NaN must come through, so it is picked, not maximised
        __syncthreads();
        if (threadIdx.x == 0) scratch[0] = -INFINITY;
        __syncthreads();
        if (act >= 0 && act < width && (int)threadIdx.x == (int)((act % kChunk) % kBlock)) scratch[0] = za;
        __syncthreads();
        za = scratch[0];
        const double base = m == -INFINITY ? 0.0 : m;
        double sum = 0, dot = 0;
        each_column<E>(w, x, width, counts, [&](int64_t v, float xf, uint32_t c) {
            const double d = ruled(w, xf, c, v) - base;
            const double e = exp(d);
            sum += e;
            dot += d == -INFINITY ? 0.0 : e * d;
        });
        sum = block_reduce(sum, [](double p, double q) { return p + q; }, scratch);
        dot = block_reduce(dot, [](double p, double q) { return p + q; }, scratch);
        if (threadIdx.x == 0) {
            const double ls = log(sum);
            log_prob[b] = sum == 0.0 ? -INFINITY : (float)(za - base - ls);
            entropy[b] = sum == 0.0 ? 0.f : (float)(ls - dot / sum);
            log_sum[2 * b] = base;   // apart: beside a mask of the type's lowest value the sum of the two would lose log S
            log_sum[2 * b + 1] = sum == 0.0 ? -INFINITY : ls;
        }
        __syncthreads();
    }
}

template <typename E>
__global__ void __launch_bounds__(kBlock) score_backward_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, Rules r,
                                                                const void* actions, int act64, const float* log_prob, const float* entropy,
                                                                const double* log_sum, const float* g_lp, const float* g_ent,
                                                                typename E::T* out, int64_t out_stride) {
    __shared__ uint32_t counts[kChunk];
    for (int64_t b = blockIdx.x; b < rows; b += gridDim.x) {
        const Row w = row_of(r, b);
        const int64_t act = act64 ? ((const int64_t*)actions)[b] : ((const int32_t*)actions)[b];
        const double base = log_sum[2 * b], ls = log_sum[2 * b + 1], ent = entropy[b];
        const double gl = !g_lp || log_prob[b] == -INFINITY ? 0.0 : (double)g_lp[b];
        const double ge = g_ent ? (double)g_ent[b] : 0.0;
        each_column<E>(w, x + b * stride, width, counts, [&](int64_t v, float xf, uint32_t c) {
            const double lp = ruled(w, xf, c, v) - base - ls;
            const double s = slope(w, xf, c, v);
            double g = 0.0;
            if (ls != -INFINITY && s != 0.0 && lp != -INFINITY) {
                const double p = exp(lp);
                g = ((v == act ? gl : 0.0) - gl * p - ge * p * (lp + ent)) * s;
            }
            E::store(out + b * out_stride + v, (float)g);
        });
    }
}

template <typename E>
__global__ void __launch_bounds__(kBlock) dropout_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, uint32_t limit,
                                                         float scale, Keys keys, typename E::T* out, int64_t out_stride) {
    const int64_t blocks = (width + 7) / 8, n = rows * blocks;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
        const int64_t b = i / blocks, q = i % blocks;
        const uint4 w4 = row_words(keys, b, (uint32_t)q);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        for (int j = 0; j < 8 && q * 8 + j < width; j++) {
            const uint32_t h = (w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
            const float v = E::load(x + b * stride + q * 8 + j) * scale;
            E::store(out + b * out_stride + q * 8 + j, h >= limit ? v : 0.f);
        }
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------
int64_t element_size(int type) { return type == GYMHIP_TYPE_F32 ? 4 : 2; }

int check_matrix(const char* what, const void* data, int type, int64_t rows, int64_t width, int64_t stride) {
    if (type != GYMHIP_TYPE_F32 && type != GYMHIP_TYPE_F16 && type != GYMHIP_TYPE_BF16) return fail(GYMHIP_EINVAL, "type must be GYMHIP_TYPE_F32, _F16 or _BF16");
    if (rows < 0 || width < 0 || width > GYMHIP_POLICY_MAX_WIDTH) return fail(GYMHIP_EINVAL, "rows or width out of range (width <= 2^24)");
    if (rows && width && !data) return fail(GYMHIP_EINVAL, "%s is null", what);
    if (stride < 0 || (rows > 1 && stride > (int64_t)0x7fffffffffffffffll / 8 / rows)) return fail(GYMHIP_EINVAL, "%s: stride out of range", what);
    if ((uintptr_t)data % (uintptr_t)element_size(type)) return fail(GYMHIP_EINVAL, "%s is not aligned to its type", what);
    return GYMHIP_OK;
}

// An output's rows must not share elements, and it may coincide with an input only element for element.
int check_output(const char* what, const void* out, int type, int64_t rows, int64_t width, int64_t stride, const void* in, int64_t in_stride) {
    if (int rc = check_matrix(what, out, type, rows, width, stride)) return rc;
    if (rows > 1 && stride < width) return fail(GYMHIP_EINVAL, "%s: rows overlap (stride < width)", what);
    if (!in || !rows || !width || (in == out && (in_stride == stride || rows == 1))) return GYMHIP_OK;
    const uintptr_t e = (uintptr_t)element_size(type);
    const uintptr_t a = (uintptr_t)out, a1 = a + ((uintptr_t)(rows - 1) * (uintptr_t)stride + (uintptr_t)width) * e;
    const uintptr_t c = (uintptr_t)in, c1 = c + ((uintptr_t)(rows - 1) * (uintptr_t)in_stride + (uintptr_t)width) * e;
    if (a < c1 && c < a1) return fail(GYMHIP_EINVAL, "%s overlaps an input", what);
    return GYMHIP_OK;
}

int check_rules(const gymhip_logit_rules* r, int64_t rows, int64_t width, Rules* out) {
    *out = Rules{};
    out->rep = out->temp = 1.f;
    if (!r) return GYMHIP_OK;
    if (r->struct_size != (int32_t)sizeof(gymhip_logit_rules)) return fail(GYMHIP_EINVAL, "bad gymhip_logit_rules.struct_size");
    if (r->mask) {
        if (r->mask_lines < 1) return fail(GYMHIP_EINVAL, "mask_lines must be positive");
        if (!r->mask_rows && r->mask_lines != 1 && r->mask_lines != rows) return fail(GYMHIP_EINVAL, "without mask_rows, mask_lines must be 1 or rows");
        if (r->mask_stride < 0 || (r->mask_lines > 1 && r->mask_stride < (width + 31) / 32)) return fail(GYMHIP_EINVAL, "mask lines are shorter than ceil(width / 32) words");
    } else if (r->mask_rows) {
        return fail(GYMHIP_EINVAL, "mask_rows without a mask");
    }
    if (r->bias && r->bias_stride < 0) return fail(GYMHIP_EINVAL, "bias_stride must not be negative");
    if (r->history) {
        if (r->history_dtype != GYMHIP_ACT_I32 && r->history_dtype != GYMHIP_ACT_I64) return fail(GYMHIP_EINVAL, "history_dtype must be GYMHIP_ACT_I32 or _I64");
        if (r->history_len && r->history_len_dtype != GYMHIP_ACT_I32 && r->history_len_dtype != GYMHIP_ACT_I64)
            return fail(GYMHIP_EINVAL, "history_len_dtype must be GYMHIP_ACT_I32 or _I64");
        if (r->history_cols < 0 || r->history_cols > 0x7fffffff || r->history_stride < 0) return fail(GYMHIP_EINVAL, "history size out of range");
    } else if (r->history_len) {
        return fail(GYMHIP_EINVAL, "history_len without a history");
    }
    if (!r->repetition_rows && !(r->repetition > 0.f && std::isfinite(r->repetition))) return fail(GYMHIP_EINVAL, "repetition must be positive and finite");
    if (!r->temperature_rows && !(r->temperature >= 0.f && std::isfinite(r->temperature))) return fail(GYMHIP_EINVAL, "temperature must be finite and not negative");
    if ((!r->presence_rows && !std::isfinite(r->presence)) || (!r->frequency_rows && !std::isfinite(r->frequency)))
        return fail(GYMHIP_EINVAL, "presence and frequency must be finite");
    out->mask = r->mask; out->mask_stride = r->mask_stride; out->mask_lines = r->mask_lines; out->mask_rows = r->mask_rows;
    out->bias = r->bias; out->bias_stride = r->bias_stride;
    if (r->history && r->history_cols > 0) {
        out->hist = r->history; out->hist_stride = r->history_stride; out->hist_cols = r->history_cols; out->hist_len = r->history_len;
        out->hist64 = r->history_dtype == GYMHIP_ACT_I64; out->len64 = r->history_len_dtype == GYMHIP_ACT_I64;
    }
    out->rep_rows = r->repetition_rows; out->pres_rows = r->presence_rows; out->freq_rows = r->frequency_rows; out->temp_rows = r->temperature_rows;
    out->rep = r->repetition; out->pres = r->presence; out->freq = r->frequency; out->temp = r->temperature;
    return GYMHIP_OK;
}

int check_keys(const gymhip_random_keys* k, Keys* out) {
    if (!k || k->struct_size != (int32_t)sizeof(gymhip_random_keys)) return fail(GYMHIP_EINVAL, "keys: null, or bad gymhip_random_keys.struct_size");
    out->seed = k->seed; out->row = k->row; out->step = k->step; out->rows = k->rows; out->steps = k->steps; out->steps_per_row = k->steps_per_row != 0;
    return GYMHIP_OK;
}

int check_actions(const void* actions, int dtype, int64_t rows) {
    if (rows && !actions) return fail(GYMHIP_EINVAL, "actions is null");
    if (dtype != GYMHIP_ACT_I32 && dtype != GYMHIP_ACT_I64) return fail(GYMHIP_EINVAL, "action_dtype must be GYMHIP_ACT_I32 or GYMHIP_ACT_I64");
    return GYMHIP_OK;
}

unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 16) ? rows : (1 << 16)); }

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GYMHIP_OK : fail(GYMHIP_EHIP, "launch failed: %s", hipGetErrorString(e));
}

// f(E{}) for the element type of `type`.
template <typename F>
int with_type(int type, F f) {
    if (type == GYMHIP_TYPE_F32) f(F32{});
    else if (type == GYMHIP_TYPE_F16) f(F16{});
    else f(BF16{});
    return launched();
}

}  // namespace
}  // namespace gymhip

using namespace gymhip;

extern "C" {

int gymhip_process_logits(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules, void* out,
                          int64_t out_stride, void* stream) {
    Rules r;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_output("out", out, type, rows, width, out_stride, logits, stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (!rows || !width) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        using T = typename E::T;
        hipLaunchKernelGGL(process_kernel<E>, dim3(row_grid(rows)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)logits, rows, width, stride, r, (T*)out, out_stride);
    });
}

int gymhip_process_logits_backward(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules,
                                   const void* grad_out, int64_t grad_out_stride, void* grad_in, int64_t grad_in_stride, void* stream) {
    Rules r;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_matrix("grad_out", grad_out, type, rows, width, grad_out_stride)) return rc;
    if (int rc = check_output("grad_in", grad_in, type, rows, width, grad_in_stride, logits, stride)) return rc;
    if (int rc = check_output("grad_in", grad_in, type, rows, width, grad_in_stride, grad_out, grad_out_stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (!rows || !width) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        using T = typename E::T;
        hipLaunchKernelGGL(process_backward_kernel<E>, dim3(row_grid(rows)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)logits, rows, width, stride, r,
                           (const T*)grad_out, grad_out_stride, (T*)grad_in, grad_in_stride);
    });
}

size_t gymhip_sample_workspace_bytes(int64_t rows, int64_t width) { (void)rows; (void)width; return 0; }

int gymhip_sample_actions(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules,
                          const gymhip_random_keys* keys, int32_t* actions, float* log_prob, void* workspace, size_t workspace_bytes, void* stream) {
    Rules r;
    Keys k;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (int rc = check_keys(keys, &k)) return rc;
    if (rows && (!actions || !log_prob)) return fail(GYMHIP_EINVAL, "actions or log_prob is null");
    if (workspace_bytes < gymhip_sample_workspace_bytes(rows, width)) return fail(GYMHIP_EINVAL, "workspace too small");
    (void)workspace;
    if (!rows) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        using T = typename E::T;
        hipLaunchKernelGGL(sample_kernel<E>, dim3(row_grid(rows)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)logits, rows, width, stride, r, k, actions, log_prob);
    });
}

size_t gymhip_action_log_prob_workspace_bytes(int64_t rows, int64_t width) { (void)rows; (void)width; return 0; }

int gymhip_action_log_prob(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules,
                           const void* actions, int action_dtype, float* log_prob, float* entropy, double* log_sum, void* workspace,
                           size_t workspace_bytes, void* stream) {
    Rules r;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (int rc = check_actions(actions, action_dtype, rows)) return rc;
    if (rows && (!log_prob || !entropy || !log_sum)) return fail(GYMHIP_EINVAL, "log_prob, entropy or log_sum is null");
    if (workspace_bytes < gymhip_action_log_prob_workspace_bytes(rows, width)) return fail(GYMHIP_EINVAL, "workspace too small");
    (void)workspace;
    if (!rows) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        using T = typename E::T;
        hipLaunchKernelGGL(score_kernel<E>, dim3(row_grid(rows)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)logits, rows, width, stride, r, actions,
                           (int)(action_dtype == GYMHIP_ACT_I64), log_prob, entropy, log_sum);
    });
}

int gymhip_action_log_prob_backward(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, const gymhip_logit_rules* rules,
                                    const void* actions, int action_dtype, const float* log_prob, const float* entropy, const double* log_sum,
                                    const float* grad_log_prob, const float* grad_entropy, void* grad_in, int64_t grad_in_stride, void* stream) {
    Rules r;
    if (int rc = check_matrix("logits", logits, type, rows, width, stride)) return rc;
    if (int rc = check_output("grad_in", grad_in, type, rows, width, grad_in_stride, logits, stride)) return rc;
    if (int rc = check_rules(rules, rows, width, &r)) return rc;
    if (int rc = check_actions(actions, action_dtype, rows)) return rc;
    if (rows && (!log_prob || !entropy || !log_sum)) return fail(GYMHIP_EINVAL, "log_prob, entropy or log_sum is null");
    if (!rows || !width) return GYMHIP_OK;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        using T = typename E::T;
        hipLaunchKernelGGL(score_backward_kernel<E>, dim3(row_grid(rows)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)logits, rows, width, stride, r, actions,
                           (int)(action_dtype == GYMHIP_ACT_I64), log_prob, entropy, log_sum, grad_log_prob, grad_entropy, (T*)grad_in, grad_in_stride);
    });
}

int gymhip_dropout(const void* x, int type, int64_t rows, int64_t width, int64_t stride, double p, const gymhip_random_keys* keys, void* out,
                   int64_t out_stride, void* stream) {
    Keys k;
    if (int rc = check_matrix("x", x, type, rows, width, stride)) return rc;
    if (int rc = check_output("out", out, type, rows, width, out_stride, x, stride)) return rc;
    if (int rc = check_keys(keys, &k)) return rc;
    if (!(p >= 0.0 && p < 1.0) || std::nearbyint(p * 65536.0) > 65535.0) return fail(GYMHIP_EINVAL, "p must lie in [0, 1) and round to less than 65536 / 65536");
    if (!rows || !width) return GYMHIP_OK;
    const uint32_t limit = (uint32_t)std::nearbyint(p * 65536.0);
    const float scale = (float)(65536.0 / (65536.0 - limit));
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        using T = typename E::T;
        const int64_t blocks = rows * ((width + 7) / 8), grid = (blocks + kBlock - 1) / kBlock;
        hipLaunchKernelGGL(dropout_kernel<E>, dim3((unsigned)(grid < 65536 ? grid : 65536)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)x, rows, width,
                           stride, limit, scale, k, (T*)out, out_stride);
    });
}

}  // extern "C"
