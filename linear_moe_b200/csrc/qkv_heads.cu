// Heads out of a fused projection: rows [G, r + 2, D] of a token (r query heads, the key and the value of every group) become queries [G r, D], keys [G, D] and values [G, D]; query and key heads are
// normed by their root mean square and turned by their position:
//   y = w x / sqrt(mean x^2 + eps),  (z_a, z_b) = (y_a cos - y_b sin, y_a sin + y_b cos)    over the pairs (a, b) = (i, i + R/2), or (2i, 2i + 1), of the first R numbers
// and back again:  (dy_a, dy_b) = (dz_a cos + dz_b sin, dz_b cos - dz_a sin),  dw = sum dy x / rms,  dx = (dy w - x' mean(dy w x')) / rms  with x' = x / rms.
//
// Bound by reading the projection once and writing the heads once (backward: the heads' gradients and the normed part of the projection once, its gradient once); the norm's factor is computed again
// instead of being kept.  32-bit arithmetic, one rounding per number; compiled without approximate functions.
#include <cuda_fp16.h>

#include "common.cuh"

namespace lmoe {
namespace heads {

struct Args {
    const void *x, *wq, *wk;                          // [rows, G, r + 2, D] (rows b T + t, at b x_b + t x_t); [D] or null
    void *q, *k, *v;                                  // [rows, G r, D], [rows, G, D] twice
    const float *cos, *sin;                           // [tokens, R / 2]; R 0: no rotation
    const void* at;                                   // [rows], the tables' row of every token; null: token t of a sequence has row t
    const void *dq, *dk, *dv;                         // backward; null: zeros
    void *dx, *dwq, *dwk;
    float* part;                                      // [parts, 2, D]
    long long x_b, x_t, rows;
    int T, G, r, D, R, tokens, interleaved, at_wide, w_type, parts;
    float eps;
    int* err;
};

__device__ __forceinline__ float val(float x) { return x; }
__device__ __forceinline__ float val(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float val(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T num(float x);
template <> __device__ __forceinline__ float num<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 num<bf16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half num<__half>(float x) { return __float2half(x); }
// types of the weights: 0 fp32, 1 bf16, 2 fp16
__device__ __forceinline__ float weight(const void* w, int type, int i) {
    return type == 0 ? ((const float*)w)[i] : type == 1 ? val(((const bf16*)w)[i]) : val(((const __half*)w)[i]);
}

// The tables' row of a token; one that lies outside is reported and taken as the nearest that there is.
__device__ __forceinline__ long long row_of(const Args& a, long long row) {
    if (a.at == nullptr) return row % a.T;
    const long long p = a.at_wide ? ((const long long*)a.at)[row] : ((const int*)a.at)[row];
    if (p >= 0 && p < a.tokens) return p;
    atomicCAS(a.err, 0, 0x41000);
    return p < 0 ? 0 : a.tokens - 1;
}

// Any head of up to 1024 numbers: a warp per head, a lane for every 32nd number; the other one of a pair is read where it lies.
constexpr int WARPS = 8;
template <typename T, int PER>
__global__ void __launch_bounds__(WARPS * 32) heads_any_kernel(const Args a) {
    const int lane = threadIdx.x & 31, S = a.r + 2, half = a.R / 2;
    const long long items = a.rows * a.G * S;
    for (long long it = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); it < items; it += (long long)gridDim.x * WARPS) {
        const long long row = it / (a.G * S);
        const int slot = it % (a.G * S), g = slot / S, i = slot % S;
        const T* x = (const T*)a.x + row / a.T * a.x_b + row % a.T * a.x_t + (long long)slot * a.D;
        T* y = i < a.r ? (T*)a.q + ((row * a.G + g) * a.r + i) * a.D : (i == a.r ? (T*)a.k : (T*)a.v) + (row * a.G + g) * a.D;
        if (i > a.r) {
            for (int d = lane; d < a.D; d += 32) y[d] = x[d];
            continue;
        }
        const void* w = i < a.r ? a.wq : a.wk;
        float v[PER], sum = 0.f;
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            v[c] = lane + 32 * c < a.D ? val(x[lane + 32 * c]) : 0.f;
            sum += v[c] * v[c];
        }
        const float inv = w != nullptr ? 1.f / sqrtf(warp_sum(sum) / a.D + a.eps) : 1.f;
        const long long pos = a.R ? row_of(a, row) : 0;
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            const int d = lane + 32 * c;
            if (d >= a.D) break;
            float z = v[c] * inv * (w != nullptr ? weight(w, a.w_type, d) : 1.f);
            if (d < a.R) {
                const int f = a.interleaved ? d / 2 : d % half, o = a.interleaved ? d ^ 1 : d < half ? d + half : d - half;
                const float u = val(x[o]) * inv * (w != nullptr ? weight(w, a.w_type, o) : 1.f), cs = a.cos[pos * half + f], sn = a.sin[pos * half + f];
                z = o > d ? z * cs - u * sn : z * cs + u * sn;
            }
            y[d] = num<T>(z);
        }
    }
}

template <typename T, int PER>
__global__ void __launch_bounds__(WARPS * 32) heads_any_bwd_kernel(const Args a) {
    __shared__ float red[WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, S = a.r + 2, half = a.R / 2;
    const long long items = a.rows * a.G * S;
    float dw[2][PER];
#pragma unroll
    for (int c = 0; c < PER; ++c) dw[0][c] = dw[1][c] = 0.f;
    for (long long it = (long long)blockIdx.x * WARPS + warp; it < items; it += (long long)gridDim.x * WARPS) {
        const long long row = it / (a.G * S);
        const int slot = it % (a.G * S), g = slot / S, i = slot % S;
        T* dx = (T*)a.dx + it * a.D;
        const void* from = i < a.r ? a.dq : i == a.r ? a.dk : a.dv;
        const T* dz = (const T*)from + (i < a.r ? (row * a.G + g) * a.r + i : row * a.G + g) * a.D;
        if (from == nullptr || i > a.r) {
            for (int d = lane; d < a.D; d += 32) dx[d] = from == nullptr ? num<T>(0.f) : dz[d];
            continue;
        }
        const void* w = i < a.r ? a.wq : a.wk;
        const T* x = (const T*)a.x + row / a.T * a.x_b + row % a.T * a.x_t + (long long)slot * a.D;
        const long long pos = a.R ? row_of(a, row) : 0;
        float v[PER], dy[PER], sum = 0.f, dot = 0.f;
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            const int d = lane + 32 * c;
            const bool in = d < a.D;
            v[c] = in && w != nullptr ? val(x[d]) : 0.f;
            sum += v[c] * v[c];
            dy[c] = in ? val(dz[d]) : 0.f;
            if (d < a.R) {
                const int f = a.interleaved ? d / 2 : d % half, o = a.interleaved ? d ^ 1 : d < half ? d + half : d - half;
                const float u = val(dz[o]), cs = a.cos[pos * half + f], sn = a.sin[pos * half + f];
                dy[c] = o > d ? dy[c] * cs + u * sn : dy[c] * cs - u * sn;
            }
        }
        const float inv = w != nullptr ? 1.f / sqrtf(warp_sum(sum) / a.D + a.eps) : 1.f;
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            v[c] *= inv;
            if (w == nullptr) continue;
            if (i < a.r) dw[0][c] += dy[c] * v[c];
            else dw[1][c] += dy[c] * v[c];
            dy[c] *= lane + 32 * c < a.D ? weight(w, a.w_type, lane + 32 * c) : 0.f;
            dot += dy[c] * v[c];
        }
        dot = w != nullptr ? warp_sum(dot) / a.D : 0.f;
#pragma unroll
        for (int c = 0; c < PER; ++c)
            if (lane + 32 * c < a.D) dx[lane + 32 * c] = num<T>((dy[c] - v[c] * dot) * inv);
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            __syncthreads();
            red[warp][lane] = dw[n][c];
            __syncthreads();
            if (warp == 0 && lane + 32 * c < a.D) {
                float s = 0.f;
#pragma unroll
                for (int y = 0; y < WARPS; ++y) s += red[y][lane];
                a.part[((long long)blockIdx.x * 2 + n) * a.D + lane + 32 * c] = s;
            }
        }
}

// Weights' gradients out of the blocks' parts, in the order of the blocks: a block for 32 numbers of one weight, its warps take the parts in turn.
constexpr int SUM_WARPS = 16;
__global__ void __launch_bounds__(SUM_WARPS * 32) heads_sum_kernel(const Args a) {
    __shared__ float red[SUM_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane, n = blockIdx.y;
    pdl_wait();
    float s = 0.f;
    if (d < a.D)
        for (int p = warp; p < a.parts; p += SUM_WARPS) s += a.part[((long long)p * 2 + n) * a.D + d];
    red[warp][lane] = s;
    __syncthreads();
    if (warp > 0 || d >= a.D) return;
    s = 0.f;
#pragma unroll
    for (int y = 0; y < SUM_WARPS; ++y) s += red[y][lane];
    void* out = n == 0 ? a.dwq : a.dwk;
    if (out == nullptr) return;
    if (a.w_type == 0) ((float*)out)[d] = s;
    else if (a.w_type == 1) ((bf16*)out)[d] = num<bf16>(s);
    else ((__half*)out)[d] = num<__half>(s);
}

template <typename T, int PER>
static int run_any(const Args& a, bool back, cudaStream_t st) {
    const long long blocks = (a.rows * a.G * (a.r + 2) + WARPS - 1) / WARPS;
    if (!back) {
        heads_any_kernel<T, PER><<<(unsigned)(blocks < 65536 ? blocks : 65536), WARPS * 32, 0, st>>>(a);
        return (int)cudaGetLastError();
    }
    heads_any_bwd_kernel<T, PER><<<a.parts, WARPS * 32, 0, st>>>(a);
    const int rc = (int)cudaGetLastError();
    if (rc || a.part == nullptr) return rc;
    heads_sum_kernel<<<dim3((a.D + 31) / 32, 2), SUM_WARPS * 32, 0, st>>>(a);
    return (int)cudaGetLastError();
}
template <typename T>
static int by_width(const Args& a, bool back, cudaStream_t st) {
    if (a.D <= 128) return run_any<T, 4>(a, back, st);
    if (a.D <= 256) return run_any<T, 8>(a, back, st);
    return run_any<T, 32>(a, back, st);
}

}  // namespace heads
}  // namespace lmoe

// type: 0 fp32, 1 bf16, 2 fp16.  back: the gradients (a.parts blocks, whose parts of the weights' gradients a second launch adds up).
LMOE_API int lmoe_qkv_heads(const lmoe::heads::Args* ap, int type, int back, cudaStream_t st) {
    using namespace lmoe::heads;
    const Args& a = *ap;
    if (a.rows <= 0 || a.T <= 0 || a.G <= 0 || a.r <= 0 || a.D <= 0 || a.D > 1024 || a.R < 0 || a.R > a.D || a.R % 2 != 0 || (a.R > 0 && a.tokens <= 0) || (back && a.parts <= 0)) return -1;
    return type == 0 ? by_width<float>(a, back, st) : type == 1 ? by_width<lmoe::bf16>(a, back, st) : by_width<__half>(a, back, st);
}
