// Heads out of a fused projection: rows [G, r + 2, D] of a token (r query heads, the key and the value of every group) become queries [G r, D], keys [G, D] and values [G, D]; query and key heads are
// normed by their root mean square and turned by their position:
//   y = w x / sqrt(mean x^2 + eps),  (z_a, z_b) = (y_a cos - y_b sin, y_a sin + y_b cos)    over the pairs (a, b) = (i, i + R/2), or (2i, 2i + 1), of the first R numbers
// and back again:  (dy_a, dy_b) = (dz_a cos + dz_b sin, dz_b cos - dz_a sin),  dw = sum dy x / rms,  dx = (dy w - x' mean(dy w x')) / rms  with x' = x / rms.
//
// Bound by reading the projection once and writing the heads once (backward: the heads' gradients and the normed part of the projection once, its gradient once); the norm's factor is computed again
// instead of being kept.  32-bit arithmetic, one rounding per number; compiled without approximate functions.
// 16384 tokens, 32 over 8 heads of 128, bf16: forward 402 MB in 74 us (5.4 TB/s), backward 571 MB in 130 us (4.4 TB/s) and 7 us for the sums of the weights' gradients.  A warp per head with a number every 32nd lane
// took 1279 us for both; 16 bytes a thread, blocks of queries, keys and values 365; the next head's numbers loaded ahead, index divisions as products, arithmetic two numbers at a time 209.
// Two heads ahead, with the norms' weights in shared memory to make room for them, took 276: the forward pass spills at its 64 registers, the backward pass goes from 130 to 144.
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
    float* part;                                      // of the weights' gradients: [parts, 2, D]; heads of vectors [parts, D], those of queries and then those of keys
    long long x_b, x_t, rows;
    int T, G, r, D, R, tokens, interleaved, at_wide, w_type, parts;
    unsigned div[4][2];                               // heads of vectors: divisors G r, G, r and T (`over`)
    int vectors, parts_q, parts_k;                    // heads of vectors: blocks of queries and of keys (the rest are values'); backward: one part each
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

// Heads of vectors: 16 bytes of a thread, twice.  A head is up to 32 threads', and what turns together one thread's: numbers from E j and from R / 2 + E j on (behind R: E neighbours twice), or, where
// neighbours turn, from E j and from D / 2 + E j on.  A block works on queries, keys or values alone, so that a thread keeps its numbers' weights, and their gradients, in registers.
constexpr int VT = 256;
template <typename T> struct Chunk { static constexpr int E = 16 / sizeof(T); };      // numbers of a vector
template <typename T> __device__ __forceinline__ float2 pair_of(const uint4& raw, int i);      // numbers 2 i, 2 i + 1
template <> __device__ __forceinline__ float2 pair_of<float>(const uint4& raw, int i) { return reinterpret_cast<const float2*>(&raw)[i]; }
template <> __device__ __forceinline__ float2 pair_of<bf16>(const uint4& raw, int i) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&raw)[i];
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 pair_of<__half>(const uint4& raw, int i) { return __half22float2(reinterpret_cast<const __half2*>(&raw)[i]); }
template <typename T> __device__ __forceinline__ void unpack(const uint4& raw, float2* x) {
#pragma unroll
    for (int i = 0; i < Chunk<T>::E / 2; ++i) x[i] = pair_of<T>(raw, i);
}
template <typename T> __device__ __forceinline__ void store_chunk(T* p, const float2* x) {
    __align__(16) T y[Chunk<T>::E];
#pragma unroll
    for (int i = 0; i < Chunk<T>::E / 2; ++i) y[2 * i] = num<T>(x[i].x), y[2 * i + 1] = num<T>(x[i].y);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(y);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// n / d for n < 2^31 by a product (Granlund and Montgomery, "Division by invariant integers using multiplication"): d's multiplier and shift come from the host
__device__ __forceinline__ unsigned over(unsigned n, const unsigned (&d)[2]) { return (__umulhi(n, d[0]) + n) >> d[1]; }
template <int TPH> __device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int o = TPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
struct Place { int kind, block, blocks, at[2]; bool in, turns[2]; };      // kind: 0 queries, 1 keys, 2 values; first numbers of a thread's vectors
template <typename T, int TPH> __device__ __forceinline__ Place place_of(const Args& a) {
    constexpr int E = Chunk<T>::E;
    Place p;
    const int b = blockIdx.x, j = threadIdx.x % TPH;
    p.kind = b < a.parts_q ? 0 : b < a.parts_q + a.parts_k ? 1 : 2;
    p.block = p.kind == 0 ? b : p.kind == 1 ? b - a.parts_q : b - a.parts_q - a.parts_k;
    p.blocks = p.kind == 0 ? a.parts_q : p.kind == 1 ? a.parts_k : gridDim.x - a.parts_q - a.parts_k;
    p.in = j < a.D / (2 * E);
    if (a.interleaved) p.at[0] = E * j, p.at[1] = a.D / 2 + E * j;
    else if (E * j < a.R / 2) p.at[0] = E * j, p.at[1] = a.R / 2 + E * j;
    else p.at[0] = 2 * E * j, p.at[1] = p.at[0] + E;
    p.turns[0] = p.at[0] < a.R, p.turns[1] = p.at[1] < a.R;
    return p;
}
// Cosines or sines, N in a row
template <int N> __device__ __forceinline__ void load_table(const float* p, float2* x) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
        if constexpr (N % 4 == 0) {
            const float4 y = __ldg(reinterpret_cast<const float4*>(p + i));
            x[i / 2] = make_float2(y.x, y.y), x[i / 2 + 1] = make_float2(y.z, y.w);
        } else x[i / 2] = __ldg(reinterpret_cast<const float2*>(p + i));
}
// (a, b) -> (a cos - b sin, a sin + b cos), with the sine's sign
template <typename T, bool INTER> __device__ __forceinline__ void turn(const Args& a, const Place& p, long long pos, float sign, float2* x) {
    constexpr int E = Chunk<T>::E;
    const int half = a.R / 2;
    const float *cos = a.cos + pos * half, *sin = a.sin + pos * half;
    if constexpr (!INTER) {
        if (!p.turns[0]) return;
        float2 c[E / 2], s[E / 2];
        load_table<E>(cos + p.at[0], c);
        load_table<E>(sin + p.at[0], s);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const float2 u = x[i], v = x[E / 2 + i], sn = __fmul2_rn(s[i], both(sign));
            x[i] = __ffma2_rn(v, make_float2(-sn.x, -sn.y), __fmul2_rn(u, c[i]));
            x[E / 2 + i] = __ffma2_rn(u, sn, __fmul2_rn(v, c[i]));
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!p.turns[h]) continue;
            float2 c[E / 4], s[E / 4];
            load_table<E / 2>(cos + p.at[h] / 2, c);
            load_table<E / 2>(sin + p.at[h] / 2, s);
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                float2& y = x[h * (E / 2) + i];
                const float cs = i & 1 ? c[i / 2].y : c[i / 2].x, sn = sign * (i & 1 ? s[i / 2].y : s[i / 2].x);
                y = make_float2(y.x * cs - y.y * sn, y.x * sn + y.y * cs);
            }
        }
    }
}
// Head `it` of a kind: its token, its row in the tables if it is its place, and where it lies in the projection
struct Head { unsigned row, t; long long from; };
__device__ __forceinline__ Head head_of(const Args& a, int kind, unsigned it, long long ld_b, long long ld_t) {
    Head y;
    y.row = over(it, a.div[kind == 0 ? 0 : 1]);
    const unsigned h = it - y.row * (kind == 0 ? a.G * a.r : a.G), b = over(y.row, a.div[3]);
    y.t = y.row - b * a.T;
    y.from = b * ld_b + y.t * ld_t + (long long)(kind == 0 ? h + 2 * over(h, a.div[2]) : h * (a.r + 2) + a.r + kind - 1) * a.D;
    return y;
}
__device__ __forceinline__ uint4 load16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

template <typename T, int TPH, bool INTER>
__global__ void __launch_bounds__(VT, 4) heads_vec_kernel(const Args a) {
    constexpr int E = Chunk<T>::E, HEADS = VT / TPH;
    const Place p = place_of<T, TPH>(a);
    const void* wp = p.kind == 0 ? a.wq : p.kind == 1 ? a.wk : nullptr;
    float2 w[E];
    if (wp != nullptr && p.in)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int d = p.at[2 * i / E] + 2 * i % E;
            w[i] = make_float2(weight(wp, a.w_type, d), weight(wp, a.w_type, d + 1));
        }
    T* out = (T*)(p.kind == 0 ? a.q : p.kind == 1 ? a.k : a.v);
    const unsigned items = (unsigned)(a.rows * a.G) * (p.kind == 0 ? a.r : 1), step = p.blocks * HEADS;
    unsigned it = p.block * HEADS + threadIdx.x / TPH;
    // the next head's numbers are on their way while this one's are worked on
    Head next;
    uint4 raw[2] = {};
    auto fetch = [&](unsigned i) {
        if (!p.in || i >= items) return;
        next = head_of(a, p.kind, i, a.x_b, a.x_t);
        const T* x = (const T*)a.x + next.from;
        raw[0] = load16(x + p.at[0]), raw[1] = load16(x + p.at[1]);
    };
    fetch(it);
    for (unsigned it0 = p.block * HEADS; it0 < items; it0 += step, it += step) {
        const bool there = p.in && it < items;
        const Head h = next;
        float2 x[E];
        unpack<T>(raw[0], x), unpack<T>(raw[1], x + E / 2);
        fetch(it + step);
        if (wp != nullptr) {
            float2 sum = both(0.f);
#pragma unroll
            for (int i = 0; i < E; ++i) sum = __ffma2_rn(x[i], x[i], sum);
            const float inv = 1.f / sqrtf(head_sum<TPH>(p.in ? sum.x + sum.y : 0.f) / a.D + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = __fmul2_rn(__fmul2_rn(x[i], both(inv)), w[i]);
        }
        if (!there) continue;
        if (a.R > 0 && p.kind < 2) turn<T, INTER>(a, p, a.at == nullptr ? h.t : row_of(a, h.row), 1.f, x);
        store_chunk(out + (long long)it * a.D + p.at[0], x);
        store_chunk(out + (long long)it * a.D + p.at[1], x + E / 2);
    }
}

template <typename T, int TPH, bool INTER>
__global__ void __launch_bounds__(VT, 2) heads_vec_bwd_kernel(const Args a) {
    constexpr int E = Chunk<T>::E, HEADS = VT / TPH;
    __shared__ float red[HEADS][TPH * 2 * E];
    const Place p = place_of<T, TPH>(a);
    pdl_trigger();
    const T* from = (const T*)(p.kind == 0 ? a.dq : p.kind == 1 ? a.dk : a.dv);
    const void *weights = p.kind == 0 ? a.wq : p.kind == 1 ? a.wk : nullptr, *wp = from != nullptr ? weights : nullptr;      // (what nothing asks of is not looked at: zero whatever lies there)
    float2 w[E], dw[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int d = p.at[2 * i / E] + 2 * i % E;
        dw[i] = both(0.f);
        w[i] = wp != nullptr && p.in ? make_float2(weight(wp, a.w_type, d), weight(wp, a.w_type, d + 1)) : both(0.f);
    }
    const unsigned items = (unsigned)(a.rows * a.G) * (p.kind == 0 ? a.r : 1), step = p.blocks * HEADS;
    const long long ld = (long long)a.G * (a.r + 2) * a.D;
    const bool same = a.x_t == ld && a.x_b == ld * a.T;                // the projection and its gradient lie alike
    unsigned it = p.block * HEADS + threadIdx.x / TPH;
    Head next;
    uint4 raw_x[2] = {}, raw_d[2] = {};
    auto fetch = [&](unsigned i) {
        if (!p.in || i >= items) return;
        next = head_of(a, p.kind, i, ld * a.T, ld);
        if (from != nullptr) raw_d[0] = load16(from + (long long)i * a.D + p.at[0]), raw_d[1] = load16(from + (long long)i * a.D + p.at[1]);
        if (wp != nullptr) {
            const T* x = (const T*)a.x + (same ? next.from : head_of(a, p.kind, i, a.x_b, a.x_t).from);
            raw_x[0] = load16(x + p.at[0]), raw_x[1] = load16(x + p.at[1]);
        }
    };
    fetch(it);
    for (unsigned it0 = p.block * HEADS; it0 < items; it0 += step, it += step) {
        const bool there = p.in && it < items;
        const Head h = next;
        float2 x[E], dy[E];
        unpack<T>(raw_x[0], x), unpack<T>(raw_x[1], x + E / 2);
        unpack<T>(raw_d[0], dy), unpack<T>(raw_d[1], dy + E / 2);
        fetch(it + step);
        if (there && a.R > 0 && p.kind < 2 && from != nullptr) turn<T, INTER>(a, p, a.at == nullptr ? h.t : row_of(a, h.row), -1.f, dy);
        if (wp != nullptr) {
            float2 sum = both(0.f), dot = both(0.f);
#pragma unroll
            for (int i = 0; i < E; ++i) sum = __ffma2_rn(x[i], x[i], sum);
            const float rms = sqrtf(head_sum<TPH>(p.in ? sum.x + sum.y : 0.f) / a.D + a.eps), inv = there ? 1.f / rms : 0.f;      // (threads without a head add nothing)
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x[i] = __fmul2_rn(x[i], both(inv));
                dw[i] = __ffma2_rn(dy[i], x[i], dw[i]);
                dy[i] = __fmul2_rn(dy[i], w[i]);
                dot = __ffma2_rn(dy[i], x[i], dot);
            }
            const float mean = head_sum<TPH>(there ? dot.x + dot.y : 0.f) / a.D;
#pragma unroll
            for (int i = 0; i < E; ++i) dy[i] = __fmul2_rn(__ffma2_rn(x[i], both(-mean), dy[i]), both(inv));
        }
        if (!there) continue;
        store_chunk((T*)a.dx + h.from + p.at[0], dy);
        store_chunk((T*)a.dx + h.from + p.at[1], dy + E / 2);
    }
    if (a.part == nullptr || weights == nullptr) return;
    if (p.in)
#pragma unroll
        for (int i = 0; i < E; ++i) *reinterpret_cast<float2*>(&red[threadIdx.x / TPH][p.at[2 * i / E] + 2 * i % E]) = dw[i];
    __syncthreads();
    float* out = a.part + (long long)(p.kind == 0 ? p.block : a.parts_q + p.block) * a.D;
    for (int d = threadIdx.x; d < a.D; d += VT) {
        float s = 0.f;
#pragma unroll 8
        for (int y = 0; y < HEADS; ++y) s += red[y][d];
        out[d] = s;
    }
}

// Weights' gradients out of the blocks' parts, in the order of the blocks: a block for 32 numbers of one weight, its warps take the parts in turn.
constexpr int SUM_WARPS = 16;
__global__ void __launch_bounds__(SUM_WARPS * 32) heads_sum_kernel(Args a) {
    __shared__ float red[SUM_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane, n = blockIdx.y;
    pdl_wait();
    const int count = a.vectors ? (n == 0 ? a.parts_q : a.parts_k) : a.parts;
    const float* part = a.part + (long long)(a.vectors ? n * a.parts_q : n) * a.D + d;
    const long long ld = a.vectors ? a.D : 2 * a.D;
    float s = 0.f;
    if (d < a.D && (n == 0 ? a.dwq : a.dwk) != nullptr)
#pragma unroll 8
        for (int p = warp; p < count; p += SUM_WARPS) s += part[p * ld];
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

static int sum_up(const Args& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.D + 31) / 32, 2);
    cfg.blockDim = dim3(SUM_WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, heads_sum_kernel, a);
    return (int)cudaGetLastError();
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
    return sum_up(a, st);
}
template <typename T, int TPH, bool INTER>
static int run_vec(const Args& a, bool back, cudaStream_t st) {
    if (back) heads_vec_bwd_kernel<T, TPH, INTER><<<a.parts, VT, 0, st>>>(a);
    else heads_vec_kernel<T, TPH, INTER><<<a.parts, VT, 0, st>>>(a);
    const int rc = (int)cudaGetLastError();
    return rc || !back || a.part == nullptr ? rc : sum_up(a, st);
}
template <typename T, int TPH>
static int run_vec(const Args& a, bool back, cudaStream_t st) { return a.interleaved ? run_vec<T, TPH, true>(a, back, st) : run_vec<T, TPH, false>(a, back, st); }
template <typename T>
static int by_width(const Args& a, bool back, cudaStream_t st) {
    if (a.vectors) {
        const int threads = a.D / (2 * Chunk<T>::E);
        if (threads > 32 || a.D % (2 * Chunk<T>::E) || a.R % (2 * Chunk<T>::E) || a.rows * a.G * a.r > 0x7fffffffll || a.parts_q < 1 || a.parts_k < 1 || a.parts <= a.parts_q + a.parts_k) return -1;
        if (threads <= 4) return run_vec<T, 4>(a, back, st);
        if (threads <= 8) return run_vec<T, 8>(a, back, st);
        if (threads <= 16) return run_vec<T, 16>(a, back, st);
        return run_vec<T, 32>(a, back, st);
    }
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
