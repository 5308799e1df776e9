// tanh of capped attention scores, for the prompt kernels (flash_attn_scored.cuh) and the one-token kernel (paged_step.cu).
#pragma once
#include "attn_math.cuh"
#include "flash_tc_utils.cuh"

namespace lmoe {
namespace fatc {

// v -> tanh(a v).  The special-function pipe (16 a clock) would be the bound: two operations here and one in the softmax.  So small |a v| take an odd polynomial on the FMA pipe, two numbers
// at a time: minimax fits of tanh(y) / y in y^2, of degree 4 up to 0.75 (relative error 6e-7, 7e-7 as evaluated) and of degree 7 up to 1.5 (7e-7, 9e-7).  Only where a warp holds a larger one
// 1 - 2 / (e^2y + 1) is taken (2e-7 of one: of a small tanh under a large cap that would leave nothing, 0.1 of a score under a cap of 10^6).  The shorter one, scores of 6 under a cap of 50: both passes of packed documents 355 -> 338 us.
template <int N, int K> __device__ __forceinline__ void tanh_poly(uint32_t (&v)[N], float a, const float (&C)[K]) {
    const float2 a2 = make_float2(a, a);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 y = __fmul2_rn(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), a2), z = __fmul2_rn(y, y);
        float2 p = make_float2(C[K - 1], C[K - 1]);
#pragma unroll
        for (int k = K - 2; k >= 0; --k) p = __ffma2_rn(p, z, make_float2(C[k], C[k]));
        p = __fmul2_rn(p, y);
        v[i] = __float_as_uint(p.x), v[i + 1] = __float_as_uint(p.y);
    }
}
template <int N> __device__ __forceinline__ void tanh_short(uint32_t (&v)[N], float a) {
    constexpr float C[5] = {0.9999994349175398f, -0.3332825150562937f, 0.13258982968967536f, -0.050056294660209305f, 0.012929624292536307f};
    tanh_poly(v, a, C);
}
template <int N> __device__ __forceinline__ void tanh_long(uint32_t (&v)[N], float a) {
    constexpr float C[8] = {0.9999993443489075f, -0.33329397439956665f, 0.1329476684331894f, -0.0524832084774971f, 0.01892727054655552f, -0.0054357172921299934f,
                            0.0010218708775937557f, -8.942410931922495e-05f};
    tanh_poly(v, a, C);
}
template <int N> __device__ __forceinline__ void tanh_of(uint32_t (&v)[N], float a) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) top = max3(top, fabsf(__uint_as_float(v[i])), fabsf(__uint_as_float(v[i + 1])));
    if (!__any_sync(0xffffffffu, top * a > 0.75f)) tanh_short(v, a);
    else if (!__any_sync(0xffffffffu, top * a > 1.5f)) tanh_long(v, a);
    else {
        const float a2 = a * 2.f * LOG2E;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __float_as_uint(1.f - 2.f * rcp(ex2(__uint_as_float(v[i]) * a2) + 1.f));
    }
}
// The same number by number, without a vote, for the one-token kernel, which waits for memory and whose chains count: the exponentials and the shorter polynomial side by side.  (Replayed: 64
// requests of up to 8192 keys 187.6 us with exponentials alone, 188.6 with this; eight of up to 2048 8.6 / 8.8 us.)
template <int N> __device__ __forceinline__ void tanh_each(uint32_t (&v)[N], float a) {
    uint32_t p[N];
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v[i];
    tanh_short(p, a);
    const float a2 = a * 2.f * LOG2E;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = __uint_as_float(v[i]), e = 1.f - 2.f * rcp(ex2(x * a2) + 1.f);
        v[i] = fabsf(x * a) <= 0.75f ? p[i] : __float_as_uint(e);
    }
}

}  // namespace fatc
}  // namespace lmoe
