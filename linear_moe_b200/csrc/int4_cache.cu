// Rows into a paged cache of 4 bits a number, and rows out of it (the layout: int4_cache.cuh).
//   low = the least number of a group, down to bf16;  size = (greatest - low) / 15, up to bf16;  code = (x - low) / size, to the nearest
// so that every number of the group lies between low and low + 15 size and comes back within size / 2.  Each step is one IEEE operation in 32 bits (compiled without approximate functions), so the codes
// are the same wherever they are computed.  A group with a number that is not finite, or whose range 32 bits do not hold, comes back as NaN.
//
// Bound by memory, if few instructions are spent on a number: a thread takes half a group of each of four rows, a block the rows of one head of a request, so that codes and scales are written and read in whole
// sectors and four loads are on their way at once.
#include "int4_cache.cuh"

namespace lmoe {
namespace int4 {

struct RowArgs {
    void* x[2];                          // keys and values [B, T, G, D]: read by store, written (dense) by read
    unsigned char* pool[2];              // [pages, G, page bytes]
    const int *table, *lengths;          // [B, table_n], [B]
    long long x_b[2], x_t[2], x_g[2], table_ld;
    int B, T, G, D, page, pages, table_n, page_bits;      // page_bits: pages of 2^page_bits rows, or -1
    int* err;
};
__device__ __forceinline__ int over_page(const RowArgs& a, int key) { return a.page_bits >= 0 ? key >> a.page_bits : key / a.page; }

constexpr int ROWS = 4;                  // of a thread
// The page of a request's key; -1: none (reported)
__device__ __forceinline__ int page_of(const RowArgs& a, int b, int key) {
    const int p = a.table[b * a.table_ld + over_page(a, key)];
    if (p >= 0 && p < a.pages) return p;
    atomicCAS(a.err, 0, 0x43000);
    return -1;
}

// N: groups of a head.  Block (x, y, z): rows of head y / 2, keys or values, of request z.
template <typename T, int N>
__global__ void __launch_bounds__(256) int4_store_kernel(const RowArgs a) {
    constexpr int UNITS = 2 * N, D = 32 * N;
    const int z = blockIdx.y & 1, g = blockIdx.y >> 1, b = blockIdx.z, step = blockDim.x / UNITS, u = threadIdx.x % UNITS, first = blockIdx.x * step * ROWS + threadIdx.x / UNITS;
    if (threadIdx.x >= step * UNITS) return;         // (a group's two threads stay or go together)
    const unsigned group = 3u << (threadIdx.x & 30);
    const int n = a.lengths[b];
    if (n < 0 || n > a.table_n * a.page) {
        if (u == 0) atomicCAS(a.err, 0, 0x42000);
        return;
    }
    const int c = u / 2;
    const T* from = (const T*)a.x[z] + b * a.x_b[z] + g * a.x_g[z] + u * 16;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int t = first + i * step, key = n - a.T + t;
        if (t >= a.T || key < 0) continue;           // (in front of the request's first row)
        float x[16];
        load_row<16>(from + t * a.x_t[z], x);
        const int page = page_of(a, b, key), row = key - over_page(a, key) * a.page;
        if (page < 0) continue;
        float least = x[0], most = x[0], sum = x[0] * 0.f;
#pragma unroll
        for (int j = 1; j < 16; ++j) {
            least = fminf(least, x[j]);
            most = fmaxf(most, x[j]);
            sum = fmaf(x[j], 0.f, sum);              // NaN of infinities and NaN, which least and most pass over
        }
        least = fminf(least, __shfl_xor_sync(group, least, 1));
        most = fmaxf(most, __shfl_xor_sync(group, most, 1));
        sum += __shfl_xor_sync(group, sum, 1);
        const uint32_t lb = least == 0.f ? 0u : __float_as_uint(least);      // of zeros the positive one
        float low = __uint_as_float((lb >> 31 ? lb + 0xffffu : lb) & 0xffff0000u);
        float size = __uint_as_float((__float_as_uint(fabsf(__fmul_rn(__fsub_rn(most, low), 1.f / 15.f))) + 0xffffu) & 0xffff0000u);      // (not -0: sizes are compared by their bits)
        if (!(sum == 0.f && fabsf(low) <= 3.402823466e38f && size <= 3.402823466e38f)) low = __uint_as_float(0x7fc00000u), size = 0.f;
        // The quotient by a product with the reciprocal is off by less than 4 2^-20 (of 16 at most): where it is that near to a border between two codes, and for sizes whose reciprocal may overflow,
        // it is divided out.
        uint32_t code[2] = {0, 0};
        if (size > 0.f) {
            const float inverse = __fdiv_rn(1.f, size), magic = 12582912.f;      // 1.5 2^23: what is added to it is rounded to a whole number, which its lowest bits are
            float far = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float q = fminf(__fmul_rn(__fsub_rn(x[j], low), inverse), 15.25f), r = __fadd_rn(q, magic);
                far = fmaxf(far, fabsf(__fsub_rn(q, __fsub_rn(r, magic))));
                code[j / 8] |= (__float_as_uint(r) & 15u) << (4 * (j % 8));
            }
            if (!(far < 0.49998f && size > 1e-30f)) {
                code[0] = code[1] = 0;
#pragma unroll
                for (int j = 0; j < 16; ++j) code[j / 8] |= (uint32_t)fminf(rintf(__fdiv_rn(__fsub_rn(x[j], low), size)), 15.f) << (4 * (j % 8));
            }
        }
        unsigned char* at = a.pool[z] + ((long long)page * a.G + g) * page_bytes(a.page, D);
        *reinterpret_cast<uint2*>(at + row * (D / 2) + place(N, row, c) * 16 + (u & 1) * 8) = make_uint2(code[0], code[1]);
        reinterpret_cast<uint16_t*>(at + a.page * (D / 2) + row * (D / 8))[u & 1 ? N + c : c] = __float_as_uint(u & 1 ? size : low) >> 16;
    }
}

// Rows behind a request's last one are zeros.
template <typename T, int N>
__global__ void __launch_bounds__(256) int4_read_kernel(const RowArgs a) {
    constexpr int UNITS = 2 * N, D = 32 * N;
    const int z = blockIdx.y & 1, g = blockIdx.y >> 1, b = blockIdx.z, step = blockDim.x / UNITS, u = threadIdx.x % UNITS, first = blockIdx.x * step * ROWS + threadIdx.x / UNITS;
    if (threadIdx.x >= step * UNITS) return;
    const int n = a.lengths[b], c = u / 2;
    int pages[ROWS];                                 // (asked for ahead of the length)
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int at = over_page(a, first + i * step);
        pages[i] = at < a.table_n ? a.table[b * a.table_ld + at] : -1;
    }
    const int last = min(n, a.table_n * a.page);
    if (n != max(last, 0) && u == 0) atomicCAS(a.err, 0, 0x42000);
    uint2 code[ROWS];
    float low[ROWS], size[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int t = first + i * step;
        code[i] = make_uint2(0, 0), low[i] = size[i] = 0.f;
        if (t >= last || t >= a.T) continue;
        const int page = pages[i], row = t - over_page(a, t) * a.page;
        if (page < 0 || page >= a.pages) {
            atomicCAS(a.err, 0, 0x43000);
            continue;
        }
        const unsigned char* at = a.pool[z] + ((long long)page * a.G + g) * page_bytes(a.page, D);
        code[i] = *reinterpret_cast<const uint2*>(at + row * (D / 2) + place(N, row, c) * 16 + (u & 1) * 8);
        const uint16_t* s = reinterpret_cast<const uint16_t*>(at + a.page * (D / 2) + row * (D / 8));
        low[i] = __uint_as_float((uint32_t)s[c] << 16), size[i] = __uint_as_float((uint32_t)s[N + c] << 16);
    }
    T* to = (T*)a.x[z] + ((long long)b * a.T * a.G + g) * D + u * 16;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int t = first + i * step;
        if (t >= a.T) continue;
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {               // (2^23 + code: no conversion)
            const uint32_t w = j < 8 ? code[i].x : code[i].y;
            x[j] = low[i] + size[i] * (__uint_as_float((w >> (4 * (j % 8)) & 15u) | 0x4b000000u) - 8388608.f);
        }
        store_row<16>(to + (long long)t * a.G * D, x);
    }
}

template <typename T, int N>
static int run(const RowArgs& a, bool read, cudaStream_t st) {
    // blocks of few threads where there are few rows
    const int units = 2 * N, want = (a.T < 64 ? (a.T * units + 31) / 32 * 32 : 256), threads = want < 32 ? 32 : want < 256 ? want : 256, rows = threads / units * ROWS;
    const dim3 grid((unsigned)((a.T + rows - 1) / rows), 2 * a.G, a.B);
    if (read) int4_read_kernel<T, N><<<grid, threads, 0, st>>>(a);
    else int4_store_kernel<T, N><<<grid, threads, 0, st>>>(a);
    return (int)cudaGetLastError();
}
template <typename T>
static int by_width(const RowArgs& a, bool read, cudaStream_t st) {
    switch (a.D / UNIT) {
        case 1: return run<T, 1>(a, read, st);
        case 2: return run<T, 2>(a, read, st);
        case 3: return run<T, 3>(a, read, st);
        case 4: return run<T, 4>(a, read, st);
        case 5: return run<T, 5>(a, read, st);
        case 6: return run<T, 6>(a, read, st);
        case 7: return run<T, 7>(a, read, st);
        default: return run<T, 8>(a, read, st);
    }
}

}  // namespace int4
}  // namespace lmoe

// type: 0 fp32, 1 bf16, 2 fp16.  Rows of 16-byte boundaries; D a multiple of 32, pages of a multiple of 16 rows, pools from 16-byte boundaries.
LMOE_API int lmoe_int4_rows(const lmoe::int4::RowArgs* ap, int type, int read, cudaStream_t st) {
    using namespace lmoe::int4;
    const RowArgs& a = *ap;
    if (a.B <= 0 || a.B > 65535 || a.T <= 0 || a.G <= 0 || a.G > 32767 || a.D <= 0 || a.D > 256 || a.D % UNIT != 0 || a.page <= 0 || a.page > 65536 || a.page % 16 != 0 || a.pages < 0 || a.table_n < 0 ||
        (long long)a.table_n * a.page > 0x7fffffff - 4096) return -1;
    return type == 0 ? by_width<float>(a, read, st) : type == 1 ? by_width<lmoe::bf16>(a, read, st) : by_width<__half>(a, read, st);
}
