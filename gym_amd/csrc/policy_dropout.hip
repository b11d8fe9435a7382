// policy_dropout.hip — dropout whose mask is a function of (seed, row key, step, column): forward and backward are the same call.
//
// Eight columns take their 16 bits each from one block of the generator (14 wide multiplies), so the arithmetic stays below the traffic of
// one read and one write per element.
#include "policy_common.h"

namespace gymhip {
namespace policy {
namespace {

template <typename E>
__global__ void __launch_bounds__(kBlock) dropout_kernel(const typename E::T* x, int64_t rows, int64_t width, int64_t stride, uint32_t limit, float scale,
                                                         Keys keys, typename E::T* out, int64_t out_stride) {
    const int64_t blocks = (width + 7) / 8, n = rows * blocks;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
        const int64_t b = n >> 32 ? i / blocks : (int64_t)((uint32_t)i / (uint32_t)blocks), q = i - b * blocks;
        const uint4 w4 = row_words(keys, b, (uint32_t)q);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        constexpr int N = 8 / E::kVec;
        Raw<E, E::kVec> raw[N];
#pragma unroll
        for (int h = 0; h < N; h++)
            if (q * 8 + h * E::kVec < width) raw[h].load(x + b * stride, q * 8 + h * E::kVec, width);
#pragma unroll
        for (int h = 0; h < N; h++) {
            const int64_t at = q * 8 + h * E::kVec;
            if (at >= width) continue;
            float v[E::kVec];
#pragma unroll
            for (int j = 0; j < E::kVec; j++) {
                const int lane = h * E::kVec + j;
                const uint32_t bits = lane & 1 ? w[lane >> 1] >> 16 : w[lane >> 1] & 0xFFFFu;
                v[j] = bits >= limit ? raw[h].get(j) * scale : 0.f;
            }
            raw[h].set(v);
            raw[h].store(out + b * out_stride, at, width);
        }
    }
}

}  // namespace
}  // namespace policy
}  // namespace gymhip

using namespace gymhip;
using namespace gymhip::policy;

extern "C" int gymhip_dropout(const void* x, int type, int64_t rows, int64_t width, int64_t stride, double p, const gymhip_random_keys* keys, void* out,
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
        const int64_t blocks = rows * ((width + 7) / 8);
        hipLaunchKernelGGL(dropout_kernel<E>, dim3(grid_for((blocks + kBlock - 1) / kBlock)), dim3(kBlock), 0, (hipStream_t)stream, (const T*)x, rows, width,
                           stride, limit, scale, k, (T*)out, out_stride);
    });
}
