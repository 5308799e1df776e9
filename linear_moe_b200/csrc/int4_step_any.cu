// Attention of one new token per request over a paged cache of 4 bits a number (int4_cache.cuh), for any query type and heads of up to 256 numbers:
//   x_j = cap tanh(scale q k_j / cap) - slope_h (n - 1 - j),   o = sum_j softmax_j(x_j) v_j   over the keys  max(0, n - window) <= j < n
// A block per (request, query head), a warp per key, a lane for a number of every group; 32 bits throughout, compiled without approximate functions.
#include "int4_step.cuh"

namespace lmoe {
namespace int4 {

constexpr int ANY_WARPS = 8;

template <typename T, int N>                             // N: groups of a head
__global__ void __launch_bounds__(ANY_WARPS * 32) int4_step_any_kernel(const StepArgs a) {
    __shared__ float O[ANY_WARPS][32 * N], M[ANY_WARPS], L[ANY_WARPS];
    const int h = blockIdx.x, b = blockIdx.y, hk = h / (a.H / a.G), w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* q = (const T*)a.q + b * a.q_b + h * a.q_h;
    const Share sh = share_of(a, b);
    if (threadIdx.x == 0 && h == 0 && a.lengths[b] != sh.len) atomicCAS(a.err, 0, 0x42000);
    const long long bytes = page_bytes(a.page, 32 * N);
    float x[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = val(q[lane + 32 * i]) * a.scale, o[i] = 0.f;
    const float slope = a.slopes != nullptr ? a.slopes[h] : 0.f;
    auto number = [&](const unsigned char* at, int row, int i) -> float {
        const int code = at[row * 16 * N + place(N, row, i) * 16 + lane / 2] >> (4 * (lane & 1)) & 15;
        const uint16_t* s = reinterpret_cast<const uint16_t*>(at + a.page * 16 * N + row * 4 * N);
        return __uint_as_float((uint32_t)s[i] << 16) + __uint_as_float((uint32_t)s[N + i] << 16) * (float)code;
    };
    for (int key = sh.lo + w; key < sh.len; key += ANY_WARPS) {
        const int page = a.table[b * a.table_ld + key / a.page], row = key % a.page;
        if (page < 0 || page >= a.pages) {
            if (lane == 0) atomicCAS(a.err, 0, 0x43000);
            continue;
        }
        const unsigned char *kp = a.k + ((long long)page * a.G + hk) * bytes, *vp = a.v + ((long long)page * a.G + hk) * bytes;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += x[i] * number(kp, row, i);
        s = warp_sum(s);
        if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
        s -= slope * (float)(sh.len - 1 - key);
        // (a NaN score raises no maximum and has a weight of NaN, which stays in the sum and the output)
        const float top = fmaxf(m, s), f = m == top ? 1.f : expf(m - top), p = expf(s - (top == -INFINITY ? 0.f : top));
        m = top;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * f + p * number(vp, row, i);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) O[w][lane + 32 * i] = o[i];
    if (lane == 0) M[w] = m, L[w] = l;
    __syncthreads();
    float top = M[0], sum = 0.f, f[ANY_WARPS];
#pragma unroll
    for (int i = 1; i < ANY_WARPS; ++i) top = fmaxf(top, M[i]);
#pragma unroll
    for (int i = 0; i < ANY_WARPS; ++i) {
        f[i] = M[i] == -INFINITY ? 0.f : expf(M[i] - top);      // times NaN: NaN
        sum += f[i] * L[i];
    }
    for (int d = threadIdx.x; d < 32 * N; d += ANY_WARPS * 32) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < ANY_WARPS; ++i) y += f[i] * O[i][d];
        ((T*)a.out)[((long long)b * a.H + h) * 32 * N + d] = num<T>(sum == 0.f ? 0.f : y / sum);             // zero: nothing seen
    }
}

template <typename T>
static int launch_any(const StepArgs& a, cudaStream_t st) {
    const dim3 grid(a.H, a.B);
    switch (a.D / UNIT) {
        case 1: int4_step_any_kernel<T, 1><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        case 2: int4_step_any_kernel<T, 2><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        case 3: int4_step_any_kernel<T, 3><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        case 4: int4_step_any_kernel<T, 4><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        case 5: int4_step_any_kernel<T, 5><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        case 6: int4_step_any_kernel<T, 6><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        case 7: int4_step_any_kernel<T, 7><<<grid, ANY_WARPS * 32, 0, st>>>(a); break;
        default: int4_step_any_kernel<T, 8><<<grid, ANY_WARPS * 32, 0, st>>>(a);
    }
    return (int)cudaGetLastError();
}

}  // namespace int4
}  // namespace lmoe

// type: 0 fp32, 1 bf16, 2 fp16.
LMOE_API int lmoe_int4_step_any(const lmoe::int4::StepArgs* ap, int type, cudaStream_t st) {
    using namespace lmoe::int4;
    const StepArgs& a = *ap;
    if (!fits(a) || a.splits != 1) return -1;
    return type == 0 ? launch_any<float>(a, st) : type == 1 ? launch_any<lmoe::bf16>(a, st) : launch_any<__half>(a, st);
}
