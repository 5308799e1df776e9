// Rows into a paged cache of 4 bits a number, and rows out of it (the layout: int4_cache.cuh).
//   low = the least number of a group, down to bf16;  size = (greatest - low) / 15, up to bf16;  code = (x - low) / size, to the nearest
// so that every number of the group lies between low and low + 15 size and comes back within size / 2.  Each step is one IEEE operation in 32 bits (compiled without approximate functions), so the codes
// are the same wherever they are computed.  A group with a number that is not finite, or whose range 32 bits do not hold, comes back as NaN.
//
// Bound by memory: a thread takes eight numbers, four threads a group, neighbouring threads neighbouring rows of one head, so that codes and scales are written and read in whole sectors.
#include "int4_cache.cuh"

namespace lmoe {
namespace int4 {

struct RowArgs {
    void* x[2];                          // keys and values [B, T, G, D]: read by store, written (dense) by read
    unsigned char* pool[2];              // [pages, G, page bytes]
    const int *table, *lengths;          // [B, table_n], [B]
    long long x_b[2], x_t[2], x_g[2], table_ld;
    int B, T, G, D, page, pages, table_n;
    int* err;
};

struct Item { int b, g, t, u; };         // eight numbers: u-th of row t of head g
__device__ __forceinline__ bool item_of(const RowArgs& a, Item& it) {
    const int units = a.D / 8;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)a.B * a.G * a.T * units) return false;
    const long long row = i / units;
    it.u = i - row * units;
    it.t = row % a.T;
    it.g = row / a.T % a.G;
    it.b = row / a.T / a.G;
    return true;
}
// The page of a request's key; -1: none (reported)
__device__ __forceinline__ int page_of(const RowArgs& a, int b, int key) {
    const int p = a.table[b * a.table_ld + key / a.page];
    if (p >= 0 && p < a.pages) return p;
    atomicCAS(a.err, 0, 0x43000);
    return -1;
}

template <typename T>
__global__ void __launch_bounds__(256) int4_store_kernel(const RowArgs a) {
    Item it;
    const bool in = item_of(a, it);                  // a group's four threads are in or out together
    if (!in) return;
    const unsigned group = 0xfu << (threadIdx.x & 28);
    const int n = a.lengths[it.b], key = n - a.T + it.t;
    if (n < 0 || n > a.table_n * a.page) {
        if (it.u == 0) atomicCAS(a.err, 0, 0x42000);
        return;
    }
    if (key < 0) return;                             // in front of the request's first row
    const int page = page_of(a, it.b, key), row = key % a.page, z = blockIdx.y;
    if (page < 0) return;
    float x[8];
    load8((const T*)a.x[z] + it.b * a.x_b[z] + it.t * a.x_t[z] + it.g * a.x_g[z] + it.u * 8, x);
    float least = x[0], most = x[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        least = fminf(least, x[i]);
        most = fmaxf(most, x[i]);
        finite = finite && fabsf(x[i]) <= 3.402823466e38f;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        least = fminf(least, __shfl_xor_sync(group, least, o));
        most = fmaxf(most, __shfl_xor_sync(group, most, o));
    }
    const uint32_t lb = least == 0.f ? 0u : __float_as_uint(least);      // of zeros the positive one
    float low = __uint_as_float((lb >> 31 ? lb + 0xffffu : lb) & 0xffff0000u);
    float size = __uint_as_float((__float_as_uint(__fmul_rn(__fsub_rn(most, low), 1.f / 15.f)) + 0xffffu) & 0xffff0000u);
    finite = __all_sync(group, finite) && fabsf(low) <= 3.402823466e38f && size <= 3.402823466e38f;
    if (!finite) low = __uint_as_float(0x7fc00000u), size = 0.f;
    uint32_t code = 0;
    if (size > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) code |= (uint32_t)fminf(rintf(__fdiv_rn(__fsub_rn(x[i], low), size)), 15.f) << (4 * i);
    }
    const int units = a.D / UNIT, c = it.u / 4;
    unsigned char* at = a.pool[z] + ((long long)page * a.G + it.g) * page_bytes(a.page, a.D);
    reinterpret_cast<uint32_t*>(at + row * (a.D / 2) + place(units, row, c) * 16)[it.u % 4] = code;
    if (it.u % 4 == 0) {
        uint16_t* s = reinterpret_cast<uint16_t*>(at + a.page * (a.D / 2) + row * (a.D / 8));
        s[c] = __float_as_uint(low) >> 16;
        s[units + c] = __float_as_uint(size) >> 16;
    }
}

// Rows behind a request's last one are zeros.
template <typename T>
__global__ void __launch_bounds__(256) int4_read_kernel(const RowArgs a) {
    Item it;
    if (!item_of(a, it)) return;
    const int z = blockIdx.y, n = a.lengths[it.b];
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (n < 0 || n > a.table_n * a.page) {
        if (it.u == 0) atomicCAS(a.err, 0, 0x42000);
    }
    if (it.t < min(n, a.table_n * a.page)) {
        const int page = page_of(a, it.b, it.t), row = it.t % a.page;
        if (page >= 0) {
            const int units = a.D / UNIT, c = it.u / 4;
            const unsigned char* at = a.pool[z] + ((long long)page * a.G + it.g) * page_bytes(a.page, a.D);
            const uint32_t code = reinterpret_cast<const uint32_t*>(at + row * (a.D / 2) + place(units, row, c) * 16)[it.u % 4];
            const uint16_t* s = reinterpret_cast<const uint16_t*>(at + a.page * (a.D / 2) + row * (a.D / 8));
            const float low = __uint_as_float((uint32_t)s[c] << 16), size = __uint_as_float((uint32_t)s[units + c] << 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = low + size * (float)(code >> (4 * i) & 15);
        }
    }
    store8((T*)a.x[z] + (((long long)it.b * a.T + it.t) * a.G + it.g) * a.D + it.u * 8, x);
}

template <typename T>
static int run(const RowArgs& a, bool read, cudaStream_t st) {
    const dim3 grid((unsigned)(((long long)a.B * a.G * a.T * (a.D / 8) + 255) / 256), 2);
    if (read) int4_read_kernel<T><<<grid, 256, 0, st>>>(a);
    else int4_store_kernel<T><<<grid, 256, 0, st>>>(a);
    return (int)cudaGetLastError();
}

}  // namespace int4
}  // namespace lmoe

// type: 0 fp32, 1 bf16, 2 fp16.  Rows of 16-byte boundaries; D a multiple of 32, pages of a multiple of 16 rows, pools from 16-byte boundaries.
LMOE_API int lmoe_int4_rows(const lmoe::int4::RowArgs* ap, int type, int read, cudaStream_t st) {
    using namespace lmoe::int4;
    const RowArgs& a = *ap;
    if (a.B <= 0 || a.T <= 0 || a.G <= 0 || a.D <= 0 || a.D > 256 || a.D % UNIT != 0 || a.page <= 0 || a.page % 16 != 0 || a.pages < 0 || a.table_n < 0 || (long long)a.table_n * a.page > 0x7fffffff - 16 ||
        ((long long)a.B * a.G * a.T * (a.D / 8) + 255) / 256 > 0x7fffffff) return -1;
    return type == 0 ? run<float>(a, read, st) : type == 1 ? run<lmoe::bf16>(a, read, st) : run<__half>(a, read, st);
}
