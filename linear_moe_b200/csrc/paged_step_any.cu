// The function of paged_step.cu for what its tensor-core kernel does not take: fp32, heads of more than 128 numbers or no multiple of 8, rows off 16-byte boundaries, pages of any
// size.  A block per (request, query head); a warp per key, lanes along the head; fp32 throughout, compiled without approximate functions.  Every query head reads its key head's rows by
// itself (they meet in L1 and L2), and a request's keys are not shared out.  Bound by the chain of a key: score, sum over the warp, exponential, the output's scaling.
// Measured, replayed, keys of one length, 32 over 8 heads of 128 in bf16 on the tensor cores / here in pages of 24 rows / here in fp32 / here with heads of 256 (bf16): 8 requests of 2048 keys 15 / 240 / 225 / 362 us,
// 64 of 4096 172 / 1691 / 1585 / 2925; 2 of 65536 (16 over 2 heads) 31 / 7153 / 7008 / 10907; 1 of 300 (16 over 4) 5.2 / 25 / 23 / 32.  So it is what runs where nothing else does, and no more.
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged_step.cuh"

namespace lmoe {
namespace paged {

__device__ __forceinline__ float val(float x) { return x; }
__device__ __forceinline__ float val(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float val(__half x) { return __half2float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(bf16* p, float x) { *p = __float2bfloat16(x); }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half(x); }

constexpr int ANY_WARPS = 8;

template <typename T, int PER>                           // PER: numbers of a head per lane
__global__ void __launch_bounds__(ANY_WARPS * 32) paged_step_any_kernel(const Args a) {
    __shared__ float O[ANY_WARPS][32 * PER], M[ANY_WARPS], L[ANY_WARPS];
    const int h = blockIdx.x, b = blockIdx.y, hk = h / (a.H / a.G), w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T *q = (const T*)a.q + b * a.q_b + h * a.q_h, *kn = (const T*)a.k_new + b * a.n_b + hk * a.n_h, *vn = (const T*)a.v_new + b * a.m_b + hk * a.m_h;
    T *kc = (T*)a.k + hk * a.k_head, *vc = (T*)a.v + hk * a.v_head;
    const Share sh = share_of(a, b);
    if (threadIdx.x == 0 && h == 0 && a.lengths[b] != sh.len) atomicCAS(a.err, 0, 0x11000);
    const bool fresh = a.k_new != nullptr;
    if (fresh && h % (a.H / a.G) == 0 && sh.len > 0) {
        const int key = sh.len - 1, page = a.table[b * a.table_ld + key / a.page];
        if (page >= 0 && page < a.pages)
            for (int d = threadIdx.x; d < a.D; d += ANY_WARPS * 32) {
                kc[page * a.k_page + key % a.page * a.k_row + d] = kn[d];
                vc[page * a.v_page + key % a.page * a.v_row + d] = vn[d];
            }
    }
    float x[PER], o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int d = lane + 32 * i;
        x[i] = d < a.D ? val(q[d]) * a.scale : 0.f;
        o[i] = 0.f;
    }
    const float slope = a.slopes != nullptr ? a.slopes[h] : 0.f;
    for (int key = sh.lo + w; key < sh.len; key += ANY_WARPS) {
        const int page = a.table[b * a.table_ld + key / a.page];
        if (page < 0 || page >= a.pages) {
            if (lane == 0) atomicCAS(a.err, 0, 0x12000);
            continue;
        }
        const bool mine = fresh && key == sh.len - 1;
        const T* kr = mine ? kn : kc + page * a.k_page + key % a.page * a.k_row;
        const T* vr = mine ? vn : vc + page * a.v_page + key % a.page * a.v_row;
        float s = 0.f, v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int d = lane + 32 * i;
            v[i] = d < a.D ? val(vr[d]) : 0.f;
            s += d < a.D ? x[i] * val(kr[d]) : 0.f;
        }
        s = warp_sum(s);
        if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
        s -= slope * (float)(sh.len - 1 - key);
        // (a NaN score raises no maximum and has a weight of NaN, which stays in the sum and the output)
        const float top = fmaxf(m, s), f = m == top ? 1.f : expf(m - top), p = expf(s - (top == -INFINITY ? 0.f : top));
        m = top;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = o[i] * f + p * v[i];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) O[w][lane + 32 * i] = o[i];
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
    for (int d = threadIdx.x; d < a.D; d += ANY_WARPS * 32) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < ANY_WARPS; ++i) y += f[i] * O[i][d];
        put((T*)a.out + ((long long)b * a.H + h) * a.D + d, sum == 0.f ? 0.f : y / sum);             // zero: nothing seen
    }
}

template <typename T>
static int launch_any(const Args& a, cudaStream_t st) {
    const dim3 grid(a.H, a.B);
    if (a.D <= 64) paged_step_any_kernel<T, 2><<<grid, ANY_WARPS * 32, 0, st>>>(a);
    else if (a.D <= 128) paged_step_any_kernel<T, 4><<<grid, ANY_WARPS * 32, 0, st>>>(a);
    else if (a.D <= 256) paged_step_any_kernel<T, 8><<<grid, ANY_WARPS * 32, 0, st>>>(a);
    else paged_step_any_kernel<T, 16><<<grid, ANY_WARPS * 32, 0, st>>>(a);
    return (int)cudaGetLastError();
}

}  // namespace paged
}  // namespace lmoe

// type: 0 fp32, 1 bf16, 2 fp16.  Heads of up to 512.
LMOE_API int lmoe_paged_step_any(const lmoe::paged::Args* ap, int type, cudaStream_t st) {
    using namespace lmoe::paged;
    const Args& a = *ap;
    if (a.B <= 0 || a.B > 65535 || a.G <= 0 || a.H % a.G != 0 || a.D <= 0 || a.D > 512 || a.page <= 0 || a.table_n < 0 || a.splits != 1 ||
        (long long)a.table_n * a.page > 0x7fffffff - GROUP) return -1;
    return type == 0 ? launch_any<float>(a, st) : type == 1 ? launch_any<lmoe::bf16>(a, st) : launch_any<__half>(a, st);
}
