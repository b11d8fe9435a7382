// policy_rules.hip — element by element: the rules on logits with their gradient, and the gradient of an action's score.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

// A workgroup takes a tile of R rows by C columns, C = lanes * kVec * nv with `lanes` a power of two: a row of at most kBlock * kVec * kTile
// columns is one tile's row (and several of them share a workgroup), a wider one is cut into tiles along its columns.
struct Tiling {
    int lanes_log2;      // lanes that share a row
    int nv;              // vectors a lane, <= kTile
    int64_t cuts;        // tiles along a row
    int64_t bands, tiles;   // tiles across, and in all
    bool half;           // counts of 16 bits
};

template <typename E>
Tiling tiling(int64_t rows, int64_t width, const Rules& r) {
    Tiling t;
    t.half = half_counts(r);
    const int64_t most = r.hist && !t.half ? kTile / 2 : kTile;
    // As few lanes as hold a row in `most` vectors each, for what a row costs beside its columns is paid by each of its waves; more where rows are too few for 2,048
    // workgroups, or a lane would have more than 80 ids to count.  us against a vector a lane: 18,315 x 1,086 f16 after 10 ids 82 -> 37, 1,000,000 x 18 f32 with a
    // bias 76 -> 40, none 41 -> 36; after 300 ids 410 -> 360 (462 without the rule for ids, 430 and 1,130 for 9 bf16 columns).
    t.lanes_log2 = 0;
    while (t.lanes_log2 < 8 && ((int64_t)E::kVec << t.lanes_log2) * (width <= E::kVec ? 1 : most) < width) t.lanes_log2++;
    while (t.lanes_log2 < 8 && ((int64_t)E::kVec << t.lanes_log2) < width && (rows << t.lanes_log2 < 2048 * kBlock || (r.hist && r.hist_cols > 80u << t.lanes_log2)))
        t.lanes_log2++;
    for (const int lanes = lanes_for(r, rows, 1 << t.lanes_log2); 1 << t.lanes_log2 < lanes;) t.lanes_log2++;
    const int64_t step = (int64_t)E::kVec << t.lanes_log2;
    const int64_t need = (width + step - 1) / step;
    t.nv = (int)(need < most ? need : most);
    t.cuts = (width + step * t.nv - 1) / (step * t.nv);
    const int64_t per = kBlock >> t.lanes_log2;
    t.bands = (rows + per - 1) / per;
    t.tiles = t.bands * t.cuts;
    return t;
}

// Goes through a workgroup's tiles.  begin(b) makes a row's state; f(state, raw, b, first column, its mask bits, its place in the counts, apart) is called for
// each of the lane's vectors of `src`, and changes raw into what is stored at `out`.  apart: which of its columns have a count, for f to go
// through one by one after its straight pass over all.
// Without rules all vectors are loaded first; under them it goes one at a time, with the next one's load under way, in fewer registers.
template <typename E, bool RULES, typename Begin, typename F>
__device__ inline void each_vector(const Rules& r, const Tiling& t, const typename E::T* src, int64_t src_stride, int64_t rows, int64_t width,
                                   typename E::T* out, int64_t out_stride, const Counts& counts, Begin begin, F f) {
    constexpr int C = E::kVec;
    const int lanes = 1 << t.lanes_log2, per = kBlock >> t.lanes_log2, step = C << t.lanes_log2, cap = counts.cap;
    const int mine = (int)threadIdx.x >> t.lanes_log2, lane = (int)threadIdx.x & (lanes - 1);
    for (int64_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
        const Cut at_tile(tile, (uint32_t)t.cuts, t.bands);
        const int64_t band = at_tile.row, lo = (int64_t)at_tile.cut * cap;
        const int64_t b = band * per + mine, v0 = lo + lane * C, end = b < rows ? width : 0;
        const int place = mine * cap + lane * C;
        const typename E::T* from = src + b * src_stride;
        typename E::T* to = out + b * out_stride;
        if constexpr (RULES) {
            Raw<E, C> next;
            if (v0 < end) next.load(from, v0, width);
            if (counts.words) count_ids(r, band * per, per, rows, width, lo, counts);
            if (b >= rows) continue;
            const auto state = begin(b);
            uint32_t next_bits = allowed_bits(state, v0, width);
#pragma unroll 1
            for (int k = 0; k < t.nv; k++) {
                const int64_t at = v0 + k * step;
                if (at >= width) break;
                const uint32_t apart = counts.words ? counts.which<C>(place + k * step) : 0u;
                Raw<E, C> raw = next;
                const uint32_t bits = next_bits;
                if (k + 1 < t.nv && at + step < width) {
                    next.load(from, at + step, width);
                    next_bits = allowed_bits(state, at + step, width);
                }
                f(state, raw, b, at, bits, place + k * step, apart);
                raw.store(to, at, width);
            }
        } else {
            if (b >= rows) continue;
            Raw<E, C> raw[kTile];
#pragma unroll
            for (int k = 0; k < kTile; k++)
                if (k < t.nv && v0 + k * step < width) raw[k].load(from, v0 + k * step, width);
            const auto state = begin(b);
#pragma unroll
            for (int k = 0; k < kTile; k++) {
                const int64_t at = v0 + k * step;
                if (k >= t.nv || at >= width) continue;
                f(state, raw[k], b, at, 0u, 0, 0u);
                raw[k].store(to, at, width);
            }
        }
    }
}

// The kernels' launch bounds under rules: the waves a SIMD that the compiler has to leave registers for.  Measured, us, of process_logits 512 x 131,072 bf16 with a bias,
// 4 and 5 waves: 61, 82; of f32 2,483 x 20,236 with a history 101, 89; of the gradients there 123, 109.

// The LDS of the counts, and what is in it.
#define GYMHIP_POLICY_COUNTS(E, RULES)                                                      \
    __shared__ __align__(16) uint32_t words[RULES ? counts_words<E>() : 4];                  \
    const Counts counts { RULES && r.hist ? words : nullptr, (E::kVec << t.lanes_log2) * t.nv, kBlock * E::kVec * t.nv, t.half, t.lanes_log2 >= 3 }

// z = x / d of floats as IEEE rounds it (z may be x).  inv = 1 / d, or 0 where d is not between 2^-20 and 2^20: then, and where the quotient is not
// between 2^-60 and 2^100, the remainder may not be exact (see `divided`) and the division itself is made.  Straight-line code but for lanes that
// hold such a quotient: a zero, an infinity, or what hardly occurs.
template <int C>
__device__ inline void divide_cols(const float* x, float d, float inv, float* z) {
    bool odd = false;
    float c[C];
#pragma unroll
    for (int j = 0; j < C; j++) {
        const float q = x[j] * inv, a = fabsf(q);
        c[j] = __builtin_fmaf(__builtin_fmaf(-q, d, x[j]), inv, q);
        odd = odd || !(a > 0x1p-60f && a < 0x1p100f);
    }
    if (odd) {
#pragma unroll
        for (int j = 0; j < C; j++) {
            const float a = fabsf(x[j] * inv);
            if (!(a > 0x1p-60f && a < 0x1p100f)) c[j] = x[j] == 0.f || fabsf(x[j]) == INFINITY ? x[j] : x[j] / d;
        }
    }
#pragma unroll
    for (int j = 0; j < C; j++) z[j] = c[j];
}

struct ProcessRow : Row {
    double inv_temp;
    float tempf, inv_tempf;
    bool undivided;   // every row's temperature is 1 (or 0)

    // y / T on its way to a float: divided, or for 2-byte results, whose rounding hides 1e-16, multiplied by the reciprocal (2,048 x 49,999 bf16 under all rules: 208 -> 180 us).
    template <typename E>
    __device__ double over(double y) const { return sizeof(typename E::T) == 2 ? y * inv_temp : divided(y, temp, inv_temp); }
    // (RULES: where vector instructions cost time; without them the float division is as fast, 79 and 86 us of 2,048 x 49,999 bf16.)
    template <typename E, bool RULES, int C>
    __device__ void over_cols(float* v) const {
        if (undivided) return;
        if (RULES && sizeof(typename E::T) == 2) {
#pragma unroll
            for (int j = 0; j < C; j++) v[j] = (float)((double)v[j] * inv_temp);
        } else {
            divide_cols<C>(v, tempf, inv_tempf, v);
        }
    }
};
template <bool RULES>
__device__ inline ProcessRow process_row(const Rules& r, int64_t b) {
    ProcessRow p;
    (Row&)p = row_of<RULES>(r, b);
    p.inv_temp = 1.0 / p.temp;
    p.tempf = (float)p.temp;
    p.undivided = !r.temp_rows && r.heat.temp == 1.0;
    p.inv_tempf = p.tempf >= 0x1p-20f && p.tempf <= 0x1p20f ? 1.f / p.tempf : 0.f;
    return p;
}

// z = y / T: a correctly rounded float division where y is the logit itself; under a penalty or a bias y is a double, divided and rounded to float32.  2-byte results are
// rounded twice, to float32 and then to their type: 2^-24 of z more than one rounding, which would take the quotient's remainder along for it.
template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock, RULES ? (sizeof(typename E::T) == 4 ? 5 : 4) : 1) process_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, Rules r, Tiling t,
                                                         typename E::T* out, int64_t out_stride) {
    GYMHIP_POLICY_COUNTS(E, RULES);
    constexpr int C = E::kVec;
    each_vector<E, RULES>(r, t, x, stride, rows, width, out, out_stride, counts, [&](int64_t b) { return process_row<RULES>(r, b); },
                          [&](const ProcessRow& p, Raw<E, C>& raw, int64_t, int64_t at, uint32_t bits, int place, uint32_t apart) {
        float z[C];
        const Raw<E, C> whole = raw;
        if (RULES && p.biased) {
            float f[C];
            bias_cols<C>(p, at, width, f);
#pragma unroll
            for (int j = 0; j < C; j++) {
                const double y = (double)raw.get(j) + (double)f[j];
                z[j] = (float)(p.undivided ? y : p.template over<E>(y));
            }
        } else {
#pragma unroll
            for (int j = 0; j < C; j++) z[j] = raw.get(j);
            p.template over_cols<E, RULES, C>(z);
        }
        raw.set(z);
        if (RULES) {
            while (apart) {
                const int j = __ffs((int)apart) - 1;
                apart &= apart - 1;
                raw.put(j, (float)p.template over<E>(ruled(p, whole.pick(j), counts.at(place + j), true, at + j)));
            }
        }
        if (p.masked) raw.keep(RULES ? bits : allowed_bits(p, at, width));
    });
}

// g dz/dx.  Of the logit only its sign matters, and only under a penalty: it is read for the columns with a count alone.
template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock, RULES ? 5 : 1) process_backward_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, Rules r, Tiling t,
                                                                  const typename E::T* g, int64_t g_stride, typename E::T* out, int64_t out_stride) {
    GYMHIP_POLICY_COUNTS(E, RULES);
    constexpr int C = E::kVec;
    each_vector<E, RULES>(r, t, g, g_stride, rows, width, out, out_stride, counts, [&](int64_t b) { return process_row<RULES>(r, b); },
                          [&](const ProcessRow& p, Raw<E, C>& raw, int64_t b, int64_t at, uint32_t bits, int, uint32_t apart) {
        float u[C];
        const Raw<E, C> whole = raw;
#pragma unroll
        for (int j = 0; j < C; j++) u[j] = raw.get(j);
        p.template over_cols<E, RULES, C>(u);
        raw.set(u);
        if (RULES) {
            while (apart) {
                const int j = __ffs((int)apart) - 1;
                apart &= apart - 1;
                const float xf = (float)x[b * stride + at + j];
                raw.put(j, (float)((double)whole.pick(j) * (xf > 0.f ? p.inv_rep : p.rep) * p.inv_temp));
            }
        }
        if (p.masked) raw.clear(RULES ? bits : allowed_bits(p, at, width));
    });
}

struct ScoreRow : Row {
    int64_t act;
    double base;            // max y
    float k, ls2, gl, ge, ent, inv_temp, repf, inv_repf;
    bool empty;

    // (delta gl - p (gl + ge (log p + H))) / T with p = 2^((y - max y) log2 e / T - log2 S), d = y - max y
    __device__ float slope(float d, bool hot) const {
        const float lp2 = __builtin_fmaf(d, k, -ls2);
        const float p = __builtin_amdgcn_exp2f(lp2);
        const float lp = (lp2 < -200.f ? -200.f : lp2) * (float)kLn2;   // p is 0 there; keeps 0 * inf out
        return ((hot ? gl : 0.f) - p * __builtin_fmaf(ge, lp + ent, gl)) * inv_temp;
    }
};

// dx = that times dy/dx, in float32; y - max y is taken before anything is rounded, so p is as exact far from 0 as near it.
template <typename E, bool RULES>
__global__ void __launch_bounds__(kBlock, RULES ? 5 : 1) score_backward_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, Rules r, Tiling t,
                                                                const void* actions, int act64, const float* log_prob, const float* entropy,
                                                                const double* log_sum, const float* g_lp, const float* g_ent,
                                                                typename E::T* out, int64_t out_stride) {
    GYMHIP_POLICY_COUNTS(E, RULES);
    constexpr int C = E::kVec;
    each_vector<E, RULES>(r, t, x, stride, rows, width, out, out_stride, counts, [&](int64_t b) {
        ScoreRow s;
        (Row&)s = row_of<RULES>(r, b);
        s.act = act64 ? ((const int64_t*)actions)[b] : (int64_t)((const int32_t*)actions)[b];
        s.base = log_sum[2 * b];
        const double ls = log_sum[2 * b + 1];
        s.empty = ls == -INFINITY;
        s.ls2 = (float)(ls * kLog2e);
        s.inv_temp = finite(1.0 / s.temp);
        s.k = finite(s.k2);
        s.gl = !g_lp || log_prob[b] == -INFINITY ? 0.f : g_lp[b];
        s.ge = g_ent ? g_ent[b] : 0.f;
        s.ent = entropy[b];
        s.repf = (float)s.rep;
        s.inv_repf = (float)s.inv_rep;
        return s;
    }, [&](const ScoreRow& s, Raw<E, C>& raw, int64_t, int64_t at, uint32_t bits, int place, uint32_t apart) {
        const int64_t hot = s.act - at;
        float g[C];
        const Raw<E, C> whole = raw;
        if (RULES && s.biased) {
            float f[C];
            bias_cols<C>(s, at, width, f);
#pragma unroll
            for (int j = 0; j < C; j++) g[j] = (float)((double)raw.get(j) + (double)f[j] - s.base);
        } else if (RULES) {
#pragma unroll
            for (int j = 0; j < C; j++) g[j] = (float)((double)raw.get(j) - s.base);
        } else {
#pragma unroll
            for (int j = 0; j < C; j++) g[j] = raw.get(j) - (float)s.base;   // the greatest logit: exact in float
        }
#pragma unroll
        for (int j = 0; j < C; j++) g[j] = s.slope(g[j], hot == j);
        raw.set(g);
        if (RULES) {
            while (apart) {
                const int j = __ffs((int)apart) - 1;
                apart &= apart - 1;
                const float xf = whole.pick(j);
                const double y = ruled(s, xf, counts.at(place + j), true, at + j);
                raw.put(j, s.slope((float)(y - s.base), hot == j) * (xf > 0.f ? s.inv_repf : s.repf));
            }
        }
        if (s.empty) raw.clear(0u);
        else if (s.masked) raw.clear(RULES ? bits : allowed_bits(s, at, width));
    });
}

int64_t element_size(int type) { return type == GYMHIP_TYPE_F32 ? 4 : 2; }

}  // namespace

// ---- host side: the checks every policy entry point makes ----------------------------------------------------------------------------------
int check_matrix(const char* what, const void* data, int type, int64_t rows, int64_t width, int64_t stride) {
    if (type != GYMHIP_TYPE_F32 && type != GYMHIP_TYPE_F16 && type != GYMHIP_TYPE_BF16) return fail(GYMHIP_EINVAL, "type must be GYMHIP_TYPE_F32, _F16 or _BF16");
    if (rows < 0 || rows > (1ll << 40) || width < 0 || width > GYMHIP_POLICY_MAX_WIDTH) return fail(GYMHIP_EINVAL, "rows or width out of range (width <= 2^24)");
    if (rows && width && !data) return fail(GYMHIP_EINVAL, "%s is null", what);
    if (stride < 0 || (rows > 1 && stride > 0x7fffffffffffffffll / 8 / rows)) return fail(GYMHIP_EINVAL, "%s: stride out of range", what);
    if ((uintptr_t)data % (uintptr_t)element_size(type)) return fail(GYMHIP_EINVAL, "%s is not aligned to its type", what);
    return GYMHIP_OK;
}

// An output's rows must not share elements, and it may coincide with an input only element for element.  Rows equally far apart may lie between each other (the halves
// of a buffer's rows); of other layouts the whole ranges must be apart.
int check_output(const char* what, const void* out, int type, int64_t rows, int64_t width, int64_t stride, const void* in, int64_t in_stride) {
    if (int rc = check_matrix(what, out, type, rows, width, stride)) return rc;
    if (rows > 1 && stride < width) return fail(GYMHIP_EINVAL, "%s: rows overlap (stride < width)", what);
    if (!in || !rows || !width || (in == out && (in_stride == stride || rows == 1))) return GYMHIP_OK;
    const uintptr_t e = (uintptr_t)element_size(type);
    const uintptr_t a = (uintptr_t)out, a1 = a + ((uintptr_t)(rows - 1) * (uintptr_t)stride + (uintptr_t)width) * e;
    const uintptr_t c = (uintptr_t)in, c1 = c + ((uintptr_t)(rows - 1) * (uintptr_t)in_stride + (uintptr_t)width) * e;
    if (a >= c1 || c >= a1) return GYMHIP_OK;
    if (rows > 1 && in_stride == stride) {   // from a row of the input to the output's next one, and on to the input's next
        const uintptr_t s = (uintptr_t)stride * e, w = (uintptr_t)width * e, d = a >= c ? (a - c) % s : (s - (c - a) % s) % s;
        if (d >= w && s - d >= w) return GYMHIP_OK;
    }
    return fail(GYMHIP_EINVAL, "%s overlaps an input", what);
}

int check_rules(const gymhip_logit_rules* r, int64_t rows, int64_t width, Rules* out) {
    *out = Rules{};
    out->rep = 1.f;
    out->heat = Heat::of(1.f);
    if (!r) return GYMHIP_OK;
    if (r->struct_size != (int32_t)sizeof(gymhip_logit_rules)) return fail(GYMHIP_EINVAL, "bad gymhip_logit_rules.struct_size");
    if (!rows || !width) return GYMHIP_OK;   // there is nothing to rule, and the pointers to a row's things may be null without meaning that there are none
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
        out->hist = r->history; out->hist_stride = r->history_stride; out->hist_cols = (uint32_t)r->history_cols; out->hist_len = r->history_len;
        out->hist64 = r->history_dtype == GYMHIP_ACT_I64; out->len64 = r->history_len_dtype == GYMHIP_ACT_I64;
    }
    out->rep_rows = r->repetition_rows; out->pres_rows = r->presence_rows; out->freq_rows = r->frequency_rows; out->temp_rows = r->temperature_rows;
    out->rep = r->repetition; out->pres = r->presence; out->freq = r->frequency; 
    if (!r->temperature_rows) out->heat = Heat::of(r->temperature);
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

int check_workspace(const void* workspace, size_t bytes, size_t needed) {
    if (!needed) return GYMHIP_OK;
    if (!workspace || bytes < needed) return fail(GYMHIP_EINVAL, "workspace: %zu bytes needed, %zu given", needed, workspace ? bytes : (size_t)0);
    if ((uintptr_t)workspace % 16) return fail(GYMHIP_EINVAL, "workspace is not 16-byte aligned");
    return GYMHIP_OK;
}

// What is written per row must lie in none of the logits, of which other rows are still read then, nor in another result.
int check_results(const void* logits, int type, int64_t rows, int64_t width, int64_t stride, std::initializer_list<Range> results) {
    if (!rows) return GYMHIP_OK;
    const Range x{"logits", logits, width ? ((rows - 1) * stride + width) * element_size(type) : 0};
    const auto cross = [](const Range& a, const Range& b) { return (uintptr_t)a.at < (uintptr_t)b.at + (uintptr_t)b.bytes && (uintptr_t)b.at < (uintptr_t)a.at + (uintptr_t)a.bytes; };
    for (const Range* r = results.begin(); r != results.end(); r++) {
        if (cross(*r, x)) return fail(GYMHIP_EINVAL, "%s overlaps the logits", r->what);
        for (const Range* q = results.begin(); q != r; q++)
            if (cross(*r, *q)) return fail(GYMHIP_EINVAL, "%s overlaps %s", r->what, q->what);
    }
    return GYMHIP_OK;
}

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GYMHIP_OK : fail(GYMHIP_EHIP, "launch failed: %s", hipGetErrorString(e));
}

}  // namespace policy
}  // namespace gymhip

using namespace gymhip;
using namespace gymhip::policy;

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
        with_bool(!r.plain(), [&](auto ruled_) {
            const Tiling t = tiling<E>(rows, width, r);
            hipLaunchKernelGGL((process_kernel<E, decltype(ruled_)::value>), dim3(grid_for(t.tiles)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)logits, rows,
                               width, stride, r, t, (T*)out, out_stride);
        });
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
        with_bool(!r.plain(), [&](auto ruled_) {
            const Tiling t = tiling<E>(rows, width, r);
            hipLaunchKernelGGL((process_backward_kernel<E, decltype(ruled_)::value>), dim3(grid_for(t.tiles)), dim3(kBlock), 0, (hipStream_t)stream,
                               (const T*)logits, rows, width, stride, r, t, (const T*)grad_out, grad_out_stride, (T*)grad_in, grad_in_stride);
        });
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
        with_bool(!r.plain(), [&](auto ruled_) {
            const Tiling t = tiling<E>(rows, width, r);
            hipLaunchKernelGGL((score_backward_kernel<E, decltype(ruled_)::value>), dim3(grid_for(t.tiles)), dim3(kBlock), 0, (hipStream_t)stream,
                               (const T*)logits, rows, width, stride, r, t, actions, (int)(action_dtype == GYMHIP_ACT_I64), log_prob, entropy, log_sum,
                               grad_log_prob, grad_entropy, (T*)grad_in, grad_in_stride);
        });
    });
}

}  // extern "C"
