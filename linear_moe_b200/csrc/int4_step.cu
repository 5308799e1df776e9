// Attention of one new token per request over a paged cache of 4 bits a number (int4_cache.cuh), bf16 and fp16 queries, heads of 32, 64, 96 and 128:
//   x_j = cap tanh(scale q k_j / cap) - slope_h (n - 1 - j),   o = sum_j softmax_j(x_j) v_j   over the keys  max(0, n - window) <= j < n
//
// Bound by reading the visible rows once, 5/8 byte a number.  That is less than a third of what bf16 rows take, so a key has to be worked through in a third of the time, and what is spent on it is the
// conversion of codes; they go to the tensor cores as they are, two at a time by one mask: a code in the lowest bits of an fp16 number is code 2^-24, the next one above it 16 code 2^-24 (both exact: numbers below
// 2^-13 are 2^-24 apart).  So
//   q k_j = sum_c size_jc (q code_j)_c + sum_c low_jc Q_c        c: groups of 32, Q_c the query's sum over the group
//   o = sum_j (p_j size_jc) code_j + sum_j p_j low_jc
// The first sums are products of fp16 numbers with one result per group of a row (keys: 16 rows at a time, the heads are the 8 columns of an m16n8k16 product; values: 16 numbers of a group at a time).  The
// second ones are one small product each of bf16 numbers, whose other operand is the row's lows as they lie in the cache; Q in three parts, p in two.
// Queries go in scaled by a power of two per head, which fp16 holds exactly but for what is below 2^-35 of the head's largest number.  p size goes in as two fp16 numbers, what it is rounded to and the rest of it, together
// 22 bits: where a key head has up to four query heads the columns 4 to 7 of the products, which would be empty, take the heads 0 to 3 once more with the rests, otherwise there are second products.  (The
// rounded one alone, 11 bits, put one bf16 output in seven on the wrong neighbour of the 64-bit value.  64 requests of up to 8192 keys, four heads a key head: 106 us without the rests, 111 with them; eight: 106 and 117.  In three bf16 parts instead of two, p beside
// the lows changed nothing that could be measured: scores are off by more, 2^-23 of their products' largest part a step of 16.)  A power of two per warp keeps p size at 2^15 at most, where p is 1 and size the largest
// one seen at 2^7 (fp16 tells 2^-24 apart there).
//
// A CTA of four warps takes one key head, up to 8 of its query heads and a range of keys, 128 at a time: a stage of a ring of two, of which a warp reads 32 keys.  The warps take turns in filling the stages by bulk
// copies, a lane per copy (64 rows of a page lie together: eight copies a stage; pages of other sizes: 32).  Maxima lag by up to 2^8: unless a score runs ahead of that, nothing is exchanged between lanes and nothing rescaled.
//
// 64 requests of up to 8192 keys, 32 over 8 heads of 128, capped (390 MB, 59 us at the copy rate): 111 us.  Issue slots are what it runs out of (60 % at 16 warps per SM): 453 instructions of a warp for 16 keys, the CTAs' starts and ends among
// them, half of them on the ALU pipe.  What took it there (with 11 bits of p size, 106 in the end): heads as the rows of the score products, codes as 128 + code in bf16 and their sums taken out again 185; keys as the rows, addresses of 32 bits 152; two groups of 16 keys at a time 137; codes
// as small fp16 numbers 129; rings of the CTA instead of the warps' own (fewer, larger copies) 121; four CTAs per SM with two stages instead of three with three 113.  Two of up to 100001 keys, 16 over 2 heads of 64: 21 us.
// (Keys and values in five places of their own, more of them on their way: 123, for a second wait in every stage.)
// Rows of a group that are hidden (behind the last key, in front of the window, on a page that is none) are masked, and their values' scales set to zero in the ring, so that nothing stale meets a weight of zero.
// A NaN score raises no maximum, so what has seen nothing is told by its sum of zero, not by its maximum: a head that sees NaN gives NaN.
//
// The keys of a request are shared by up to 8 CTAs of a cluster, which join their maxima, sums and outputs in distributed shared memory; long contexts with few heads take more CTAs, which leave their parts
// in fp32 for a second launch.
#include <cooperative_groups.h>
#include <type_traits>

#include "attn_math.cuh"
#include "flash_tc_utils.cuh"
#include "int4_step.cuh"
#include "tanh_cap.cuh"

namespace lmoe {
namespace int4 {
namespace cg = cooperative_groups;

constexpr int CTAS = 4, WARPS = 4, STAGES = 2, MAX_CLUSTER = 8, HEADS = 8, ROWS = 64;
constexpr float LOG2E = 1.4426950408889634f, LAG = 8.f;

__device__ __forceinline__ uint32_t pack2(float x, float y) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ float lower(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float upper(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float2 x) { return pack2(x.x, x.y); }
// What rounding two numbers to bf16 took away, rounded itself
__device__ __forceinline__ uint32_t rest(float2 x, uint32_t rounded) { return pack2(__ffma2_rn(make_float2(lower(rounded), upper(rounded)), make_float2(-1.f, -1.f), x)); }
// Shared memory by its 32-bit addresses, with the constant part in the instruction
template <int AT> __device__ __forceinline__ uint32_t lds32(uint32_t a) { uint32_t x; asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(x) : "r"(a), "n"(AT)); return x; }
template <int AT> __device__ __forceinline__ uint32_t lds16(uint32_t a) { uint32_t x; asm volatile("ld.shared.u16 %0, [%1+%2];" : "=r"(x) : "r"(a), "n"(AT)); return x; }
template <int AT> __device__ __forceinline__ uint2 lds64(uint32_t a) { uint2 x; asm volatile("ld.shared.v2.u32 {%0, %1}, [%2+%3];" : "=r"(x.x), "=r"(x.y) : "r"(a), "n"(AT)); return x; }
// An 8 x 8 matrix of 32-bit numbers, whose row g lies in the lanes 4 g + t, two numbers each: turned
__device__ __forceinline__ void turn(float2 x, uint32_t& a, uint32_t& b) {
    const uint32_t x0 = __float_as_uint(x.x), x1 = __float_as_uint(x.y);
    uint32_t lo = __byte_perm(x0, x1, 0x5410), hi = __byte_perm(x0, x1, 0x7632);
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(lo));
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(hi));
    a = __byte_perm(lo, hi, 0x5410);
    b = __byte_perm(lo, hi, 0x7632);
}
// A row's N sizes, behind its N lows: as they lie (two to a word, what is not a size set to zero), and one of them
template <int N> struct Sizes { uint32_t w[N == 4 || N == 3 ? 2 : 1]; };
template <int N, int AT> __device__ __forceinline__ Sizes<N> sizes(uint32_t row) {
    Sizes<N> s;
    if constexpr (N == 4) {
        const uint2 x = lds64<AT + 8>(row);
        s.w[0] = x.x, s.w[1] = x.y;
    } else if constexpr (N == 3) {
        s.w[0] = lds32<AT + 4>(row) & 0xffff0000u, s.w[1] = lds32<AT + 8>(row);
    } else if constexpr (N == 2) s.w[0] = lds32<AT + 4>(row);
    else s.w[0] = lds32<AT>(row) & 0xffff0000u;
    return s;
}
template <int N> __device__ __forceinline__ float size_of(const Sizes<N>& s, int c) {
    const int i = N % 2 + c;
    return i % 2 ? upper(s.w[i / 2]) : lower(s.w[i / 2]);
}
template <int N> __device__ __forceinline__ uint32_t larger(uint32_t most, const Sizes<N>& s) {      // of the even and of the odd ones, as bits
    if constexpr (N >= 3) return __vimax3_u16x2(most, s.w[0], s.w[1]);
    else return __vmaxu2(most, s.w[0]);
}
// Two bf16 numbers times a power of two.  (No .ftz: sizes below 2^-126 are numbers too.)
__device__ __forceinline__ uint32_t scaled(uint32_t w, float f) {
    float x, y;
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(x) : "f"(lower(w)), "f"(f));
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(y) : "f"(upper(w)), "f"(f));
    return __float_as_uint(x) >> 16 | (__float_as_uint(y) & 0xffff0000u);
}
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }      // zero: nothing seen
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Codes 0 and 4 of eight as fp16 numbers, in units of 2^-24; codes 1 and 5, in units of 2^-20 (2 and 6, 3 and 7: of w >> 8)
__device__ __forceinline__ uint32_t even(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t odd(uint32_t w) { return w & 0x00f000f0u; }
__device__ __forceinline__ uint32_t pack16(float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
// What rounding two numbers to fp16 took away, rounded itself (by -1), or the numbers rounded (by 0)
__device__ __forceinline__ uint32_t rest16(float2 x, uint32_t rounded, float by) {
    const float2 r = __ffma2_rn(__half22float2(*reinterpret_cast<const __half2*>(&rounded)), make_float2(by, by), x);
    return pack16(r.x, r.y);
}
__device__ __forceinline__ float two_to(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }      // -126 <= n <= 127
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" :: "r"(tc::s32(dst)), "l"(src), "r"(bytes), "r"(tc::s32(bar)) : "memory");
}
template <typename T> __device__ __forceinline__ uint32_t out2(float x, float y);
template <> __device__ __forceinline__ uint32_t out2<bf16>(float x, float y) { return pack2(x, y); }
template <> __device__ __forceinline__ uint32_t out2<__half>(float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }

// N: groups of a head.  TWICE: up to four query heads, columns 4 to 7 are those of 0 to 3 (the same scores, weights and sums; a product's column depends on nothing but its own operands).
// The pointers are read behind pdl_wait by plain loads: the kernel may start while the one before it runs.
template <typename T, int N, bool TWICE>
__global__ void __launch_bounds__(WARPS * 32, CTAS) int4_step_kernel(const StepArgs a) {
    constexpr int D = 32 * N, CODES = ROWS * D / 2, HALF = CODES + ROWS * D / 8, PART = 2 * HALF, STAGE = 2 * PART;      // bytes: keys' or values' codes of 64 rows, with their scales, both, twice
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];
    __shared__ uint32_t there_of[STAGES];                              // a bit per copy's lane: the groups that are there
    __shared__ float part_m[WARPS][HEADS], part_l[WARPS][HEADS], cta_m[HEADS], cta_l[HEADS];
    __shared__ int abort_flag, drain_flag, chosen, lens[WARPS * 32];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, gh = TWICE ? g & 3 : g;      // gh: the head of column g
    const int qpg = a.H / a.G, tiles = (qpg + HEADS - 1) / HEADS;
    int b = blockIdx.z;
    const int hk = blockIdx.y / tiles, tile = blockIdx.y % tiles, split = blockIdx.x;
    const int h0 = hk * qpg + tile * HEADS, nh = min(HEADS, hk * qpg + qpg - h0);
    if (threadIdx.x == 0) {
        abort_flag = drain_flag = 0;
        for (int s = 0; s < STAGES; ++s) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    if (a.sorted) {                                                    // this CTA's request: the one with blockIdx.z longer ones (up to 128 requests)
        const int mine = threadIdx.x < a.B ? a.lengths[threadIdx.x] : 0;
        lens[threadIdx.x] = mine;
        __syncthreads();
        int rank = 0;
        if (w * 32 < a.B)
            for (int i = 0; i < a.B; ++i) rank += lens[i] > mine || (lens[i] == mine && i < threadIdx.x);
        if (threadIdx.x < a.B && rank == blockIdx.z) chosen = threadIdx.x;
        __syncthreads();
        b = chosen;
    }
    const Share sh = share_of(a, b);
    const int beg = sh.first + split * sh.per, end = min(sh.last, beg + sh.per);
    if (threadIdx.x == 0 && split == 0 && blockIdx.y == 0 && a.lengths[b] != sh.len) atomicCAS(a.err, 0, 0x42000);
    if (beg >= end && a.splits > MAX_CLUSTER) return;                  // (a cluster's CTAs all stay, and one of them writes zeros where there is nothing to see)

    // Stages of eight groups, of which a warp reads two; the warps take turns in filling them.
    const int n_stages = beg < end ? (end - beg + 7) / 8 : 0;
    const bool blocks = a.page % ROWS == 0;                            // 64 rows lie together: a copy each for their codes and their scales, otherwise for a group's
    // a lane's copy: codes or scales, of keys or of values, of group lane / 4
    const unsigned char* from = (lane & 2 ? a.v : a.k) + (lane & 1 ? (long long)a.page * (D / 2) : 0);
    const int row_bytes = lane & 1 ? D / 8 : D / 2, copy_bytes = (blocks ? ROWS : GROUP) * row_bytes;
    unsigned char* to = smem + (lane >> 4) * PART + (lane >> 1 & 1) * HALF + (lane & 1) * CODES + (lane >> 2 & 3) * GROUP * row_bytes;
    int filled = w - WARPS;                                            // the last stage that this warp has filled
    long long page_at = -1;                                            // for the next one: where the page and head lie of this lane's group (-1: not there), and its row
    int row_at = 0;
    auto look_up = [&]() {
        const int gi = beg + 8 * (filled + WARPS) + (lane >> 2);
        page_at = -1;
        if (gi < end && (!blocks || (lane & 12) == 0)) {
            const int at = gi * GROUP / a.page, page = a.table[b * a.table_ld + at];
            row_at = gi * GROUP - at * a.page;
            if (page >= 0 && page < a.pages) page_at = ((long long)page * a.G + hk) * page_bytes(a.page, D);
            else atomicCAS(a.err, 0, 0x43000);
        }
    };
    auto fill = [&]() {
        filled += WARPS;
        const int st = filled % STAGES;
        const uint32_t lanes = __ballot_sync(0xffffffffu, page_at >= 0);
        if (lane == 0) {
            there_of[st] = blocks ? (lanes & 1u ? 0xffffu : 0u) | (lanes >> 16 & 1u ? 0xffff0000u : 0u) : lanes;
            if (lanes) tc::mbar_expect_tx(&full[st], __popc(lanes) / 4 * (blocks ? ROWS : GROUP) * (D + D / 4));
            else tc::mbar_arrive(&full[st]);
        }
        __syncwarp();
        if (page_at >= 0) bulk_load(to + st * STAGE, from + page_at + row_at * row_bytes, copy_bytes, &full[st]);
        look_up();
    };
    look_up();
    if (filled + WARPS < min(STAGES - 1, n_stages)) fill();

    // Queries: a lane's numbers 8 t .. 8 t + 7 of every group of head g, in the order of the codes, scaled by a power of two; beside the rows' lows their sums, in three parts
    uint32_t qa[N][4], sums[3] = {0, 0, 0};
    const bool there = gh < nh;
    const float slope = there && a.slopes != nullptr ? a.slopes[h0 + gh] * LOG2E : 0.f;
    float unit_q, more_q;                                              // of the scores: up to 2^137, for queries next to the largest number, in two factors
    {
        float q[N][8], most = 0.f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[c][i] = 0.f;
            const T* row = (const T*)a.q + b * a.q_b + (h0 + gh) * a.q_h + c * 32 + 8 * t;
            if (there && a.q_rows) load8(row, q[c]);
            else if (there)
#pragma unroll
                for (int i = 0; i < 8; ++i) q[c][i] = val(row[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(q[c][i]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int top = most > 0.f ? max((int)(__float_as_uint(fminf(most, 3.402823466e38f)) >> 23) - 127, -100) : 0;      // up to 2^15, the odd codes' numbers up to 2^11
        const float scale = two_to(14 - top);
        unit_q = two_to(10 + min(top, 100));
        more_q = two_to(max(top - 100, 0));
#pragma unroll
        for (int c = 0; c < N; ++c) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                qa[c][i] = pack16(q[c][i] * (i & 1 ? scale * 0.0625f : scale), q[c][i + 4] * (i & 1 ? scale * 0.0625f : scale));
                sum += q[c][i] * scale + q[c][i + 4] * scale;
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= two_to(-24);                                        // as the codes'
            if (c / 2 == t) {
#pragma unroll
                for (int y = 0; y < 3; ++y) {
                    const uint32_t part = pack2(sum, 0.f);
                    sums[y] |= part << (c & 1 ? 16 : 0);
                    sum -= lower(part);
                }
            }
        }
    }
    const float pre = (a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E) * unit_q, unit = a.cap > 0.f ? a.cap * LOG2E : pre;      // (scores of head g)
    // Weights are 2^(score - m + shift), with which p size is at most 2^(LAG + 7) where no size is above 2^(7 - shift).  Beyond 2^40 and below 2^-20 the sizes are scaled by 2^wide as well (before the
    // weights, which alone would leave fp32): the sums of weights and of weights times lows have to stay within it.
    float m = -INFINITY, l = 0.f, shift = 7.f;
    int wide = 0;
    uint32_t bound = 0;                                                // the power of two that no size so far is above, as the upper bits of a bf16 number, twice
    // o: numbers 4 g + 2 u, 4 g + 2 u + 1 (times 16) of group c, heads 2 t, 2 t + 1;  e: head g, numbers 2 t, 2 t + 1 of the scales
    float o[2 * N][4], e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    // What a lane reads of a stage: of keys, the words t and the sizes of rows g and g + 8; of values, the half-words g and the sizes of rows 2 t, 2 t + 1, 2 t + 8 and 2 t + 9
    const uint32_t part = (w >> 1) * PART, codes_at = part + (w & 1) * 2 * GROUP * (D / 2), scales_at = part + (w & 1) * 2 * GROUP * (D / 8);
    const uint32_t at_k = codes_at + g * (D / 2) + place(N, g, 0) * 16 + 4 * t, at_v = codes_at + 2 * t * (D / 2) + place(N, 2 * t, 0) * 16 + 2 * g, at_s = scales_at + g * (D / 8), at_ks = at_s + 4 * t, at_v2 = scales_at + 2 * t * (D / 8), at_vs = at_v2 + 2 * g;
    auto chunk = [](uint32_t a, int c) -> uint32_t { return N == 2 || N == 4 ? a ^ (16u * c) : a + 16u * c; };
    const bool far = __any_sync(0xffffffffu, more_q != 1.f);
    const float rests = TWICE && g < 4 ? 0.f : -1.f;
    bool alive = true;
    int j = 0;
    for (; j < n_stages; ++j) {
        const int st = j % STAGES, key0 = (beg + 8 * j + 2 * w) * GROUP;
        if (filled + WARPS == j + STAGES - 1 && j + STAGES - 1 < n_stages) {      // this warp's turn, into the stage that was read last
            if (j > 0) alive = fatc::mbar_wait_warp(&empty[(j - 1) % STAGES], (j - 1) / STAGES & 1, &abort_flag, a.err, 0x44020);
            if (!alive) break;
            fill();
        }
        alive = fatc::mbar_wait_warp(&full[st], j / STAGES & 1, &abort_flag, a.err, 0x44000 | st);
        if (!alive) break;
        const uint32_t here = there_of[st] >> (8 * w), groups = (here & 1u) | (here >> 3 & 2u);
        const bool edge = groups != 3u || key0 < sh.lo || key0 + 2 * GROUP > sh.len;
        auto seen = [&](int key) -> bool { return (groups >> ((key - key0) / GROUP) & 1u) && key >= sh.lo && key < sh.len; };
        if (edge) {                                                    // hidden rows get scales of zero
            uint32_t* scales = reinterpret_cast<uint32_t*>(smem + st * STAGE + (w >> 1) * PART + HALF + CODES + (w & 1) * 2 * GROUP * (D / 8));
            for (int i = lane; i < 2 * GROUP * N; i += 32)
                if (!seen(key0 + i / N)) scales[i] = 0;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // ahead of the next copy into this stage
            __syncwarp();
        }
        // (where a group of 32 numbers lies depends on the row modulo 8 alone, in rows of a power of two of bytes: an exclusive or of the address)
        const uint32_t base = tc::s32(smem) + st * STAGE;
        uint32_t v[8];                                                 // scores: head g, keys 8 (e >> 1) + 2 t + (e & 1)
        // Scores of rows g and g + 8 of a group, heads 2 t and 2 t + 1.  (The other way round, heads as the 16 rows: twice the products, and the rows that no head has have to be put beside every operand.)
        auto scores = [&](auto which) {
            constexpr int AT = decltype(which)::value * GROUP * (D / 2), S = CODES + decltype(which)::value * GROUP * (D / 8), E = decltype(which)::value * 4;
            float2 s0, s1;
            const uint32_t c0 = 2 * t < N ? lds32<S>(base + at_ks) : 0u, c1 = 2 * t < N ? lds32<S + D>(base + at_ks) : 0u;
            float x[4];
            mma_first(x, c0, c1, c0, c1, sums[0], sums[1]);
            mma(x, c0, c1, 0u, 0u, sums[2], 0u);
            s0 = make_float2(x[0], x[1]), s1 = make_float2(x[2], x[3]);
            const Sizes<N> k0 = sizes<N, S>(base + at_s), k1 = sizes<N, S + D>(base + at_s);
#pragma unroll
            for (int c = 0; c < N; ++c) {
                const uint32_t row = chunk(base + at_k, c), y = lds32<AT>(row), z = lds32<AT + 4 * D>(row);
                float d[4];
                mma16_first(d, even(y), even(z), odd(y), odd(z), qa[c][0], qa[c][1]);
                mma16(d, even(y >> 8), even(z >> 8), odd(y >> 8), odd(z >> 8), qa[c][2], qa[c][3]);
                const float f0 = size_of(k0, c), f1 = size_of(k1, c);
                s0 = __ffma2_rn(make_float2(f0, f0), make_float2(d[0], d[1]), s0);
                s1 = __ffma2_rn(make_float2(f1, f1), make_float2(d[2], d[3]), s1);
            }
            turn(s0, v[E], v[E + 1]);                                  // by halves of their bits
            turn(s1, v[E + 2], v[E + 3]);
        };
        scores(std::integral_constant<int, 0>());
        scores(std::integral_constant<int, 1>());
        if (far) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * more_q);
        }
        if (a.cap > 0.f) fatc::tanh_of(v, pre);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[i]) * unit;
        if (a.slopes != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] -= slope * (float)(sh.len - 1 - (key0 + 8 * (i >> 1) + 2 * t + (i & 1)));
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!seen(key0 + 8 * (i >> 1) + 2 * t + (i & 1))) x[i] = -INFINITY;
        }
        // sizes of the values of keys 8 (e >> 1) + 2 t + (e & 1)
        Sizes<N> vs[8] = {sizes<N, HALF + CODES>(base + at_v2), sizes<N, HALF + CODES + D / 8>(base + at_v2), sizes<N, HALF + CODES + D>(base + at_v2), sizes<N, HALF + CODES + 9 * (D / 8)>(base + at_v2),
                                sizes<N, HALF + CODES + 2 * D>(base + at_v2), sizes<N, HALF + CODES + 17 * (D / 8)>(base + at_v2), sizes<N, HALF + CODES + 3 * D>(base + at_v2),
                                sizes<N, HALF + CODES + 25 * (D / 8)>(base + at_v2)};
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = larger(largest, vs[i]);
        const float most = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__any_sync(0xffffffffu, most > m + LAG || __vmaxu2(largest, bound) != bound)) {      // the first visible keys too
            float mx = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mx = fmaxf(mx, m);
            const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(largest & 0xffffu, largest >> 16), bound >> 16));
            const int power = top == 0 ? 0 : (int)((top + 0x7fu) >> 7) - 127, kept = min(max(power, -20), 40);      // no size is above 2^power
            bound = min(top + 0x7fu, 0x7f80u) & 0xff80u;
            bound |= bound << 16;
            const float shift_now = 7.f - (float)kept;
            const float corr = m == -INFINITY ? 1.f : ex2(m - mx + (shift_now - shift));      // nothing has been summed up in front of the first one
            const float corr_o = corr * two_to(max(-126, kept - power - wide));
            m = mx, shift = shift_now, wide = kept - power;
            l *= corr;
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] *= corr;
            const float c0 = __shfl_sync(0xffffffffu, corr_o, 8 * t), c1 = __shfl_sync(0xffffffffu, corr_o, 8 * t + 4);      // of heads 2 t, 2 t + 1
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) o[i][0] *= c0, o[i][1] *= c1, o[i][2] *= c0, o[i][3] *= c1;
        }
        if (wide != 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (uint32_t& y : vs[i].w) y = scaled(y, two_to(wide));
        }
        const float low = (m == -INFINITY ? 0.f : m) - shift;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ex2(x[i] - low);
        l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        auto values = [&](auto which) {
            constexpr int AT = HALF + decltype(which)::value * GROUP * (D / 2), S = HALF + CODES + decltype(which)::value * GROUP * (D / 8), E = decltype(which)::value * 4;
            const float2 w0 = make_float2(x[E], x[E + 1]), w1 = make_float2(x[E + 2], x[E + 3]);
            {                                                          // the weights' sums of lows
                const uint32_t p0 = pack2(w0), p1 = pack2(w1);
                uint32_t b0 = 0, b1 = 0;
                if (g < N) {
                    b0 = lds16<S>(base + at_vs) | lds16<S + D / 8>(base + at_vs) << 16;
                    b1 = lds16<S + D>(base + at_vs) | lds16<S + 9 * (D / 8)>(base + at_vs) << 16;
                }
                mma(e, p0, rest(w0, p0), p1, rest(w1, p1), b0, b1);
            }
#pragma unroll
            for (int c = 0; c < N; ++c) {
                const float2 y0 = __fmul2_rn(w0, make_float2(size_of(vs[E], c), size_of(vs[E + 1], c))), y1 = __fmul2_rn(w1, make_float2(size_of(vs[E + 2], c), size_of(vs[E + 3], c)));
                uint32_t p0 = pack16(y0.x, y0.y), p1 = pack16(y1.x, y1.y);
                const uint32_t r0 = rest16(y0, p0, rests), r1 = rest16(y1, p1, rests);
                if constexpr (TWICE) p0 = r0, p1 = r1;
                // four codes of keys 2 t and 2 t + 1, and of 2 t + 8 and 2 t + 9
                const uint32_t row = chunk(base + at_v, c), z0 = lds16<AT>(row) | lds16<AT + D / 2>(row) << 16, z1 = lds16<AT + 4 * D>(row) | lds16<AT + 9 * (D / 2)>(row) << 16;
                mma16(o[2 * c], even(z0), odd(z0), even(z1), odd(z1), p0, p1);
                mma16(o[2 * c + 1], even(z0 >> 8), odd(z0 >> 8), even(z1 >> 8), odd(z1 >> 8), p0, p1);
                if constexpr (!TWICE) {
                    mma16(o[2 * c], even(z0), odd(z0), even(z1), odd(z1), r0, r1);
                    mma16(o[2 * c + 1], even(z0 >> 8), odd(z0 >> 8), even(z1 >> 8), odd(z1 >> 8), r0, r1);
                }
            }
        };
        values(std::integral_constant<int, 0>());
        values(std::integral_constant<int, 1>());
        __syncwarp();                                                  // the stage is read
        if (lane == 0) tc::mbar_arrive(&empty[st]);
    }
    if (!alive && filled >= j) fatc::mbar_wait_suspend(&full[filled % STAGES], filled / STAGES & 1, &drain_flag, a.err, 0x44010);      // after a wait that ran out: copies in flight, again within a limit

    // the warps' parts meet in shared memory
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) part_m[w][g] = m, part_l[w][g] = l * ex2(-shift);
    __syncthreads();
    constexpr int LD = D + 4;
    float *O = reinterpret_cast<float*>(smem), *E = O + WARPS * HEADS * LD;      // [WARPS][HEADS][LD], [WARPS][HEADS][8], over the rings
    // This warp's share of a head: what its weights are multiplied by for a sum of one over the CTA.  (Averages are what is joined, here and further on: sums of values leave fp32 earlier.)
    auto factor = [&](int head) -> float {
        float top = part_m[0][head], sum = 0.f;
#pragma unroll
        for (int y = 1; y < WARPS; ++y) top = fmaxf(top, part_m[y][head]);
#pragma unroll
        for (int y = 0; y < WARPS; ++y) sum += part_l[y][head] == 0.f ? 0.f : part_l[y][head] * ex2(part_m[y][head] - top);
        return inverse(sum) * (part_m[w][head] == -INFINITY ? 0.f : ex2(part_m[w][head] - top));
    };
    // (the weights' shift is in l, o and e alike and is taken out here; codes are in units of 2^-24, the odd ones of 2^-20.  24 - shift - wide is up to 145, for values next to the largest number: two factors)
    const int back = 24 - (int)shift - wide, some = min(back, 100);
    const float unshift = ex2(-shift), unscale = two_to(some), more = two_to(back - some), f0 = factor(2 * t), f1 = factor(2 * t + 1), fg = factor(g);
    auto number = [&](float f, float x) -> float { return f * x * unscale * more; };
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        const int d = i / 2 * 32 + 4 * g + 2 * (i & 1);
        *reinterpret_cast<float2*>(O + (w * HEADS + 2 * t) * LD + d) = make_float2(number(f0, o[i][0]), number(f0 * 0.0625f, o[i][2]));
        *reinterpret_cast<float2*>(O + (w * HEADS + 2 * t + 1) * LD + d) = make_float2(number(f1, o[i][1]), number(f1 * 0.0625f, o[i][3]));
    }
    *reinterpret_cast<float2*>(E + (w * HEADS + g) * 8 + 2 * t) = make_float2(fg * (e[0] + e[2]) * unshift, fg * (e[1] + e[3]) * unshift);
    if (threadIdx.x < HEADS) {
        float top = part_m[0][threadIdx.x], sum = 0.f;
#pragma unroll
        for (int y = 1; y < WARPS; ++y) top = fmaxf(top, part_m[y][threadIdx.x]);
#pragma unroll
        for (int y = 0; y < WARPS; ++y) sum += part_l[y][threadIdx.x] == 0.f ? 0.f : part_l[y][threadIdx.x] * ex2(part_m[y][threadIdx.x] - top);
        cta_m[threadIdx.x] = top;
        cta_l[threadIdx.x] = sum;
    }
    __syncthreads();
    const bool cluster = a.splits > 1 && a.splits <= MAX_CLUSTER;
    for (int i = threadIdx.x; i < nh * (D / 4); i += WARPS * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, c = d / 32;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        float rest_ = 0.f;
#pragma unroll
        for (int x = 0; x < WARPS; ++x) {
            const float4 z = load4(O + (x * HEADS + r) * LD + d);
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            if constexpr (TWICE) {
                const float4 u = load4(O + (x * HEADS + r + 4) * LD + d);
                y.x += u.x; y.y += u.y; y.z += u.z; y.w += u.w;
            }
            rest_ += E[(x * HEADS + r) * 8 + c];
        }
        y.x += rest_; y.y += rest_; y.z += rest_; y.w += rest_;
        const long long bh = (long long)b * a.H + h0 + r;
        if (cluster) store4(O + r * LD + d, y);                        // (only this thread reads what lies there)
        else if (a.splits == 1) *reinterpret_cast<uint2*>((T*)a.out + bh * D + d) = make_uint2(out2<T>(y.x, y.y), out2<T>(y.z, y.w));
        else {
            store4(a.part + (bh * a.splits + split) * D + d, y);
            if (d == 0) *reinterpret_cast<float2*>(a.ml + (bh * a.splits + split) * 2) = make_float2(cta_m[r], cta_l[r]);
        }
    }
    if (!cluster) return;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (int i = split * WARPS * 32 + threadIdx.x; i < nh * (D / 4); i += a.splits * WARPS * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float ms[MAX_CLUSTER], ls[MAX_CLUSTER], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
            ms[c] = c < a.splits ? *cl.map_shared_rank(&cta_m[r], c) : -INFINITY;
            ls[c] = c < a.splits ? *cl.map_shared_rank(&cta_l[r], c) : 0.f;
            top = fmaxf(top, ms[c]);
        }
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
            if (ls[c] != 0.f) ls[c] *= ex2(ms[c] - top);
            sum += ls[c];
        }
        const float inv = inverse(sum);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
            if (ls[c] == 0.f) continue;
            const float f = ls[c] * inv;
            const float4 z = load4(cl.map_shared_rank(O + r * LD + d, c));
            y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
        }
        *reinterpret_cast<uint2*>((T*)a.out + ((long long)b * a.H + h0 + r) * D + d) = make_uint2(out2<T>(y.x, y.y), out2<T>(y.z, y.w));
    }
    cl.sync();                                                         // the other CTAs have read this one's part
}

// The parts of a request's CTAs: a block per (request, query head), a lane per four numbers of a part, as many parts a warp as it has lanes for.  (A part a warp, eight warps: 148 parts of 64 numbers 24.8 us with
// the kernel ahead of it, now 22.8, replayed.)
constexpr int JOIN_WARPS = 16;
template <typename T, int N>
__global__ void __launch_bounds__(JOIN_WARPS * 32) int4_join_kernel(StepArgs a) {
    constexpr int D = 32 * N, LANES = N == 3 ? 32 : D / 4, SUB = 32 / LANES;
    __shared__ float4 O[JOIN_WARPS][LANES];
    pdl_wait();
    const int bh = blockIdx.x, b = bh / a.H, w = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane % LANES * 4;
    const Share sh = share_of(a, b);
    const int n = (sh.last - sh.first + sh.per - 1) / sh.per;
    const float* ml = a.ml + (long long)bh * a.splits * 2;
    const float* part = a.part + (long long)bh * a.splits * D + d;
    const bool mine = d < D;
    float seen = -INFINITY, sum = 0.f;                                 // of all parts, first: then no part waits for the one before it
    for (int s = lane; s < n; s += 32) {
        const float2 x = *reinterpret_cast<const float2*>(ml + 2 * s);
        const float high = fmaxf(seen, x.x);
        sum = (sum == 0.f ? 0.f : sum * ex2(seen - high)) + (x.y == 0.f ? 0.f : x.y * ex2(x.x - high));
        seen = high;
    }
    const float top = warp_max(seen), inv = inverse(warp_sum(sum == 0.f ? 0.f : sum * ex2(seen - top)));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = w * SUB + lane / LANES; s < n; s += JOIN_WARPS * SUB) {
        const float2 x = *reinterpret_cast<const float2*>(ml + 2 * s);
        const float4 y = mine ? load4(part + (long long)s * D) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float f = x.y == 0.f ? 0.f : x.y * ex2(x.x - top) * inv;
        o.x += y.x * f; o.y += y.y * f; o.z += y.z * f; o.w += y.w * f;
    }
#pragma unroll
    for (int x = LANES; x < 32; x <<= 1) {
        o.x += __shfl_xor_sync(0xffffffffu, o.x, x);
        o.y += __shfl_xor_sync(0xffffffffu, o.y, x);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, x);
        o.w += __shfl_xor_sync(0xffffffffu, o.w, x);
    }
    if (lane < LANES) O[w][lane] = o;
    __syncthreads();
    if (w > 0 || lane >= LANES) return;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < JOIN_WARPS; ++x) {
        const float4 y = O[x][lane];
        o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
    }
    if (mine) *reinterpret_cast<uint2*>((T*)a.out + (long long)bh * D + d) = make_uint2(out2<T>(o.x, o.y), out2<T>(o.z, o.w));
}

template <typename T, int N, bool TWICE>
static int launch(const StepArgs& a, cudaStream_t st) {
    constexpr int D = 32 * N, ring = STAGES * 4 * ROWS * (D / 2 + D / 8), ends = WARPS * HEADS * (D + 4 + 8) * 4, smem = ring > ends ? ring : ends;
    int rc = (int)cudaFuncSetAttribute(int4_step_kernel<T, N, TWICE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc) return rc;
    const int tiles = (a.H / a.G + HEADS - 1) / HEADS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.splits, a.G * tiles, a.B);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.splits > 1 && a.splits <= MAX_CLUSTER ? 2 : 1;
    cudaLaunchKernelEx(&cfg, int4_step_kernel<T, N, TWICE>, a);
    rc = (int)cudaGetLastError();
    if (rc || a.splits <= MAX_CLUSTER) return rc;
    return launch_early(int4_join_kernel<T, N>, (int64_t)a.B * a.H, JOIN_WARPS * 32, st, a);
}
template <typename T, int N>
static int launch(const StepArgs& a, cudaStream_t st) { return a.H / a.G <= 4 ? launch<T, N, true>(a, st) : launch<T, N, false>(a, st); }
template <typename T>
static int by_width(const StepArgs& a, cudaStream_t st) {
    switch (a.D / 32) {
        case 1: return launch<T, 1>(a, st);
        case 2: return launch<T, 2>(a, st);
        case 3: return launch<T, 3>(a, st);
        default: return launch<T, 4>(a, st);
    }
}

}  // namespace int4
}  // namespace lmoe

// half: fp16, else bf16.  Heads of up to 128.
LMOE_API int lmoe_int4_step(const lmoe::int4::StepArgs* ap, int half, cudaStream_t st) {
    using namespace lmoe::int4;
    const StepArgs& a = *ap;
    if (!fits(a) || a.D > 128 || (a.sorted && a.B > WARPS * 32) || (long long)a.G * ((a.H / a.G + HEADS - 1) / HEADS) > 65535 || (a.splits > MAX_CLUSTER && (a.part == nullptr || a.ml == nullptr))) return -1;
    return half ? by_width<__half>(a, st) : by_width<lmoe::bf16>(a, st);
}
