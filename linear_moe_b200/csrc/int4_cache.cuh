// A paged cache of 4 bits a number.  A head's row goes in groups of 32 numbers, x = low + size * code with codes of 0 to 15 and low and size in bf16.  A page [G, page (D / 2 + D / 8) bytes] holds, head
// by head, the codes of its rows (D / 2 bytes each, 16 a group, the lower half of a byte first) and then every row's n = D / 32 lows and n sizes.
//
// Eight neighbouring rows, or every second one of eight, are read 16 bytes a row at once (csrc/int4_step.cu), which has to come from all banks of shared memory.  So groups change places from row to row where rows
// are 32 or 64 bytes long: group c of row j lies at place c ^ (j / 4 % 2) with two groups, c ^ (j / 2 % 4) with four.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace lmoe {
namespace int4 {

constexpr int UNIT = 32;

__host__ __device__ __forceinline__ int place(int n, int row, int c) { return n == 4 ? c ^ (row >> 1 & 3) : n == 2 ? c ^ (row >> 2 & 1) : c; }
__host__ __device__ __forceinline__ long long page_bytes(int page, int D) { return (long long)page * (D / 2 + D / 8); }

__device__ __forceinline__ float val(float x) { return x; }
__device__ __forceinline__ float val(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float val(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T num(float x);
template <> __device__ __forceinline__ float num<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 num<bf16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half num<__half>(float x) { return __float2half(x); }

// K consecutive numbers (a multiple of eight), 16-byte aligned
template <int K, typename T> __device__ __forceinline__ void load_row(const T* p, float (&x)[K]) {
#pragma unroll
    for (int i = 0; i < K * (int)sizeof(T) / 16; ++i) {
        const uint4 raw = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); ++j) x[i * (16 / (int)sizeof(T)) + j] = val(reinterpret_cast<const T*>(&raw)[j]);
    }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) { load_row<8>(p, x); }
template <int K, typename T> __device__ __forceinline__ void store_row(T* p, const float (&x)[K]) {
#pragma unroll
    for (int i = 0; i < K * (int)sizeof(T) / 16; ++i) {
        __align__(16) T y[16 / sizeof(T)];
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); ++j) y[j] = num<T>(x[i * (16 / (int)sizeof(T)) + j]);
        reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(y);
    }
}

}  // namespace int4
}  // namespace lmoe
