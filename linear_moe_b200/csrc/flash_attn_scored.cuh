// Attention with a range of visible keys per query, capped scores and a bias by distance, for bf16 and fp16 with heads of up to 128 (flash_attn_scored.cu, flash_attn_scored_fp16.cu):
//   x_ij = cap tanh(scale q_i k_j / cap) - slope_h |p_i - j|,  visible: first_i <= j < stop_i, causality with a query offset and a window if wanted;  o = softmax(x) v
//   ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do
// The products and their operands are laid out as in flash_attn_tc.cu: tcgen05 with accumulators in tensor memory, weights back into tensor memory as the A operand, sixteen softmax warps.
// What differs is the work.  A query's visible keys are one interval, whatever it comes from; a query tile's key tiles are the union of its rows' intervals, and only tiles that are not inside
// all of them are masked.  Packed documents leave a tile of queries few key tiles (five, for documents of 700 tokens), and then what a CTA does around its loop is half of its time: with a CTA
// per query tile 2200 cycles until its tensor memory and barriers are there, 2400 for Q, 2700 for its output in pieces of 16 bytes, 1600 until the next CTA is there; a key tile takes 2500.
// So the query-side kernels keep their CTAs: warp 3 asks the hardware for the tile of a CTA that has not started yet (clusterlaunchcontrol), one tile ahead, and works out its interval; loads,
// products and softmax go on from tile to tile, the rings and their phases counted through.  The dk / dv kernel, whose tiles of a long document have many times the work of others, shares the
// query heads of a key head between two CTAs, each of which finishes one of the two sums.
// Measured, kernel by kernel (one B200): (a) 2 x 4096 queries in packed documents of 700 on average, 16 over 4 heads of 128, capped at 50, (b) 8192 queries, 16 heads of 128, slopes, window
// of 2048.  Matrix rates in TFLOP/s, with the tensor pipe's active cycles:
//   forward  (a) 112 us, 270, 18 %  (b) 173 us, 596, 32 %     a tile's chain: scores 800 cycles, softmax 3400 (capped 5000), P V 950; two groups of warps take turns
//   delta    16 us for 84 MB, 5.2 TB/s
//   dq       (a) 105 us, 431, 30 %  (b) 159 us, 972, 55 %
//   dk / dv  (a) 130 us, 464, 33 %  (b) 260 us, 793, 45 %     of 3700 cycles a tile (uncapped) 2500 are products being issued: with 64 queries at a time K and V are read twice as often
// What is left: the forward chain, which ends only where P no longer lies over S (tensor memory is full with 128-wide heads); two query tiles in flight, one for each group of warps, with
// everything around the loop hidden, took as long (what one group does, the other one's issue slots pay for) and lost where few tiles of queries share the GPU.
// Every wait is bounded; the softmax warps, which meet in barriers, agree at every tile's end on whether to go on.
#pragma once
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "attn_math.cuh"
#include "flash_tc_utils.cuh"
#include "tanh_cap.cuh"

namespace lmoe {
namespace fatc {
namespace cg = cooperative_groups;

struct Ranges {
    const int *first, *stop;              // [B, Tq] with strides (first_b, 1), (stop_b, 1); null: 0 and Tk
    long long first_b, stop_b;
    const float* slopes;                  // [Hq]; null: no bias
    int8_t* low;                          // [B, Tq, Hq, d rounded up to 16]: the next eight bits of the output (residue); null: not wanted
    int4* tiles;                          // [B, query tiles]: union of the rows' intervals, then their intersection
    float cap;
    int causal, d;                        // d: head size, a multiple of 8 up to D (tensor maps fill the rest with zeros)
};
struct Args {
    bf16* out;                            // [B, Tq, Hq, d]
    float* lse;                           // [B, Hq, Tq]
    int B, Tq, Tk, Hq, Hkv;
    int q_offset, window;                 // window <= 0: none
    float scale;
    int* err;
    Ranges x;
};
struct BwdArgs {
    const float *lse, *delta;             // [B, Hq, Tq]: log-sum-exp of the forward pass, rowsum(dO * O)
    bf16 *dq, *dk, *dv;                   // [B, Tq, Hq, d], [B, Tk, Hkv, d] twice
    int B, Tq, Tk, Hq, Hkv;
    int q_offset, window;
    float scale;
    int* err;
    Ranges x;
};

// SCORE_CAP with the bias too, where there are slopes.
enum { SCORE_PLAIN, SCORE_BIAS, SCORE_CAP };
template <int S, bool H> struct Form { static constexpr bool HALF = H; static constexpr int SCORE = S; };
constexpr int BLK = BM * 128;             // one 64-column block of a 128-row tile
constexpr int MAX_TILES = 8192;           // query tiles that a dk / dv CTA can list: 2^20 queries

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                    "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
template <class F> __device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (F::HALF) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else return pack_bf16(a, b);
}
template <class F> __device__ __forceinline__ float2 unpack16(uint32_t x) {
    if constexpr (F::HALF) return __half22float2(*reinterpret_cast<const __half2*>(&x));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}
// What the output's rounding took away.  delta = do . o is subtracted from dp, nearly its equal where one weight is large: with the rounded o alone dq and dk were off by 0.0042 at scores
// of 6 in root mean square, with eight bits more 0.0025 (their own rounding: 0.0017).  Both numbers have the same sign, so their patterns differ by an integer: at most half a step, 2^15
// (fp16: 2^12; 2^15 after a shift), of which the upper eight bits are kept.  Four numbers and the two pairs that they were rounded to -> four bytes.
template <class F> __device__ __forceinline__ uint32_t residues(float a, float b, float c, float d, uint32_t ab, uint32_t cd) {
    const float2 x = unpack16<F>(ab), y = unpack16<F>(cd);
    int e[4] = {__float_as_int(a) - __float_as_int(x.x), __float_as_int(b) - __float_as_int(x.y), __float_as_int(c) - __float_as_int(y.x), __float_as_int(d) - __float_as_int(y.y)};
    if constexpr (F::HALF) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = min(max(e[i], -4096), 4096) * 8;                       // (in fp16's subnormals a step is more)
    }
    uint32_t p, q;
    asm("cvt.pack.sat.s16.s32 %0, %1, %2;" : "=r"(p) : "r"(e[1]), "r"(e[0]));
    asm("cvt.pack.sat.s16.s32 %0, %1, %2;" : "=r"(q) : "r"(e[3]), "r"(e[2]));
    return __byte_perm(p, q, 0x7531);
}
template <class F> __device__ __forceinline__ float with_residue(float kept, int r) { return __int_as_float(__float_as_int(kept) + r * (F::HALF ? 32 : 256)); }
// operand types of the instruction descriptor: bits 7 and 10 set for bf16, clear for fp16
template <class F, bool B_MN, int N> __host__ __device__ constexpr uint32_t idesc_of() {
    return F::HALF ? idesc_bf16<B_MN, N>() & ~((1u << 7) | (1u << 10)) : idesc_bf16<B_MN, N>();
}

// Visible keys [lo, hi) of query `row`, clipped to the keys that there are; a query that sees nothing has lo >= hi.  Neither is negative.
template <class A> __device__ __forceinline__ int2 visible_range(const A& a, int b, int row) {
    int lo = a.x.first != nullptr ? max(__ldg(a.x.first + b * a.x.first_b + row), 0) : 0;
    int hi = a.x.stop != nullptr ? min(__ldg(a.x.stop + b * a.x.stop_b + row), a.Tk) : a.Tk;
    const int at = a.q_offset + row;
    if (a.x.causal) hi = min(hi, at + 1);
    if (a.window > 0 && at >= 0) lo = max(lo, at - a.window + 1);
    return make_int2(lo, max(hi, 0));
}

// Scores as the kernels hold them, and what they are multiplied by to be exponents of 2 (`unit`):
//   SCORE_PLAIN   q k, unit scale / ln 2          SCORE_BIAS   scale q k / ln 2 - bias, unit 1
//   SCORE_CAP     tanh(scale q k / cap) - bias / cap, unit cap / ln 2
// `a`: factor of q k; `sl`: slope in the score's units.
struct ScoreOf { float a, sl, unit; };
template <class F> __device__ __forceinline__ ScoreOf score_of(float scale, const Ranges& x, int h) {
    ScoreOf s{1.f, 0.f, scale * LOG2E};
    if constexpr (F::SCORE == SCORE_BIAS) s = {scale * LOG2E, __ldg(x.slopes + h) * LOG2E, 1.f};
    if constexpr (F::SCORE == SCORE_CAP) s = {scale / x.cap, x.slopes != nullptr ? __ldg(x.slopes + h) / x.cap : 0.f, x.cap * LOG2E};
    return s;
}
// v -> a v - the bias of N neighbouring keys (queries), the first of them `dist` away.  Where no one is on the other side for any row of the warp (all but a causal sequence's diagonal tiles)
// the distance needs no absolute value: a product with the column's number and one for two scores, instead of a sum, a product and another one for each.  8192 queries x 16 heads, window of
// 2048: forward 218 / 212 us, dq 177 / 159 us, dk / dv 267 / 257 us.
template <int N> __device__ __forceinline__ void biased(uint32_t (&v)[N], float a, float slope, float dist) {
    const bool before = dist <= 1 - N;
    if (__all_sync(0xffffffffu, before) || __all_sync(0xffffffffu, dist >= 0.f)) {
        const float t = before ? slope : -slope, base = t * dist;
        const float2 a2 = make_float2(a, a);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), a2, make_float2(fmaf(t, i, base), fmaf(t, i + 1, base)));
            v[i] = __float_as_uint(x.x), v[i + 1] = __float_as_uint(x.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * a - slope * fabsf(dist + i));
    }
}
template <class F, int N> __device__ __forceinline__ void scored(uint32_t (&v)[N], const ScoreOf& s, const Ranges& x, float dist) {
    if constexpr (F::SCORE == SCORE_BIAS) biased(v, s.a, s.sl, dist);
    else if constexpr (F::SCORE == SCORE_CAP) {
        tanh_of(v, s.a);
        if (x.slopes != nullptr) biased(v, 1.f, s.sl, dist);
    }
}

// Bounded waits.  (Without the time hint of mbar_wait_suspend, and with several tries between two looks at the flag and the clock: these cost the other warps' turns.  Forward kernel of a batch
// with prefixes 92 -> 85 us.)
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(s32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    if (try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
            if (try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > WAIT_CYCLES) break;
    }
    *abort_flag = 1;
    atomicCAS(err, 0, code);
    return false;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    return __all_sync(0xffffffffu, wait_for(bar, parity, abort_flag, err, code));
}

// ---- work ----------------------------------------------------------------------------------------------------------------------------
// Which tile a CTA takes: the last (longest) tiles of a sequence first, over `group` (batch, head) pairs at a time, whose streamed rows share the L2.
struct TileOf { int rank, pair; };
__device__ __forceinline__ TileOf longest_first(int idx, int tiles, int pairs, int group) {
    const int sec = idx / (tiles * group), rem = idx - sec * tiles * group;
    const int n = min(group, pairs - sec * group);
    return {rem / n, sec * group + rem % n};
}
// Pairs whose streamed tensors (two of `rows` x D 16-bit numbers per `share` pairs) stay within half of the L2 together.
static int pairs_in_l2(int pairs, long long rows, int D, int share) {
    const long long n = (64LL << 20) / max(rows * D * 4, 1LL);
    return (int)min((long long)pairs, max(n, 1LL) * share);
}
// The hardware's next CTA that has not started: asked for by one thread, answered in 16 bytes of shared memory; its index, or -1 where there is none (after which nothing may be asked).
__device__ __forceinline__ void ask_work(void* answer, uint64_t* bar) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // the last answer has been read
    mbar_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" :: "r"(s32(answer)), "r"(s32(bar)) : "memory");
}
__device__ __forceinline__ int work_of(const void* answer) {
    uint32_t id;
    asm volatile("{\n.reg .pred p;\n.reg .b128 h;\n.reg .b32 y, z, w;\nmov.u32 %0, 0xffffffff;\nld.shared.b128 h, [%1];\n"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, h;\n}" : "=r"(id) : "r"(s32(answer)) : "memory");
    return (int)id;
}
// The tiles that a CTA works through, two slots: warp 3 fills one while the other is worked on.
struct Item { int q0, h, b, hk, nb_lo, n_it; int2 every; };      // n_it: key tiles, from nb_lo on (-1: no more work); inside `every` no row masks anything
struct Work {
    uint64_t full[2], empty[2], asked;
    __align__(16) uint4 answer;
    __align__(16) Item item[2];
};
__device__ __forceinline__ void init_work(Work& w, int readers) {      // readers of a slot: loads, products, softmax warps
    for (int s = 0; s < 2; ++s) { mbar_init(&w.full[s], 1); mbar_init(&w.empty[s], readers); }
    mbar_init(&w.asked, 1);
}
// Warp 3.  seen: [2][128] in shared memory for the rows' ranges, where the intervals are to be worked out (and, from the first head, noted for the backward pass); null: they are read from the notes.
template <class A>
__device__ __forceinline__ void hand_out(Work& w, int2 (*seen)[BM], const A& a, int group, volatile int* abort_flag, int* err, int code) {
    const int lane = threadIdx.x & 31, n_qb = (a.Tq + BM - 1) / BM;
    for (int it = 0;; ++it) {
        const int slot = it & 1;
        if (!wait_warp(&w.empty[slot], ((it >> 1) & 1) ^ 1, abort_flag, err, code)) return;
        int index = blockIdx.x;
        if (it > 0) {                                             // not before there is room: what a CTA has asked for no other one can take
            if (lane == 0) ask_work(&w.answer, &w.asked);
            __syncwarp();
            if (!wait_warp(&w.asked, (it - 1) & 1, abort_flag, err, code + 1)) return;
            index = work_of(&w.answer);
            __syncwarp();
        }
        Item x;
        x.n_it = -1;
        if (index >= 0) {
            const TileOf tile = longest_first(index, n_qb, a.B * a.Hq, group);
            const int qb = n_qb - 1 - tile.rank;
            x.h = tile.pair % a.Hq, x.b = tile.pair / a.Hq, x.hk = x.h / (a.Hq / a.Hkv), x.q0 = qb * BM;
            int4* note = a.x.tiles + (long long)x.b * n_qb + qb;
            int4 t;
            if (seen != nullptr) {
                t = make_int4(0x7fffffff, 0, 0, 0x7fffffff);     // {union, intersection}: empty rows add nothing to the first and leave none of the second
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = x.q0 + lane + 32 * e;
                    const int2 r = row < a.Tq ? visible_range(a, x.b, row) : make_int2(0, 0);
                    seen[slot][lane + 32 * e] = r;
                    if (row >= a.Tq) continue;
                    if (r.x < r.y) t = make_int4(min(t.x, r.x), max(t.y, r.y), max(t.z, r.x), min(t.w, r.y));
                    else t.z = 0x7fffffff, t.w = 0;
                }
                t.x = __reduce_min_sync(0xffffffffu, t.x);
                t.y = __reduce_max_sync(0xffffffffu, t.y);
                t.z = __reduce_max_sync(0xffffffffu, t.z);
                t.w = __reduce_min_sync(0xffffffffu, t.w);
                if (x.h == 0 && lane == 0) *note = t;
            } else t = __ldg(note);
            x.nb_lo = min(t.x, t.y) / BN;
            x.n_it = max((t.y + BN - 1) / BN - x.nb_lo, 0);
            x.every = make_int2(t.z, t.w);
        }
        __syncwarp();
        if (lane == 0) {
            w.item[slot] = x;
            mbar_arrive(&w.full[slot]);
        }
        __syncwarp();
        if (x.n_it < 0) return;
    }
}
// All softmax warps: do they all want to go on?  (A barrier; what it decides is the same for all.)
__device__ __forceinline__ bool all_softmax(bool ok) {
    uint32_t r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.and.pred q, 9, 512, p;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(r) : "r"((uint32_t)ok) : "memory");
    return r != 0;
}

// ---- products --------------------------------------------------------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int h, int row, int b) {
#pragma unroll
    for (int kb = 0; kb < D / 64; ++kb) tma_load_4d(dst + kb * BLK, map, bar, kb * 64, h, row, b);
}
// [128 x 128] = A B^T over D, both tiles K-major
template <int D, class F>
__device__ __forceinline__ void score_product(uint32_t tmem_d, const uint8_t* A, const uint8_t* B) {
    if (!elect_one()) return;
    const uint32_t al = desc_lo<false>(s32(A)), bl = desc_lo<false>(s32(B));
#pragma unroll
    for (int kk = 0; kk < D / UMMA_K; ++kk) {
        const uint32_t off = ((kk / 4) * BLK + (kk % 4) * 32) >> 4;
        umma_ss(tmem_d, al + off, bl + off, idesc_of<F, false, 128>(), kk > 0);
    }
}
// [128 x D] (+)= A B over 128: A in tensor memory as the warps left it (16 packed columns at the beginning of every part's 32), B's rows are K
template <int D, class F>
__device__ __forceinline__ void grad_product(uint32_t tmem_d, uint32_t tmem_a, const uint8_t* B, bool add) {
    if (!elect_one()) return;
    const uint32_t bl = ((s32(B) >> 4) & 0x3FFFu) | ((uint32_t)(BLK >> 4) << 16);
#pragma unroll
    for (int kk = 0; kk < 128 / UMMA_K; ++kk)
        umma_ts(tmem_d, tmem_a + kk / 2 * 32 + kk % 2 * 8, bl + ((kk * 2048) >> 4), idesc_of<F, true, D>(), add || kk > 0);
}
// The same with 64 queries for B, and over 64 queries.  QB: bytes between the 64-column blocks of B
template <int D, class F, int QB>
__device__ __forceinline__ void half_product(uint32_t tmem_d, const uint8_t* A, const uint8_t* B) {
    if (!elect_one()) return;
    const uint32_t al = desc_lo<false>(s32(A)), bl = desc_lo<false>(s32(B));
#pragma unroll
    for (int kk = 0; kk < D / UMMA_K; ++kk)
        umma_ss(tmem_d, al + (((kk / 4) * BLK + (kk % 4) * 32) >> 4), bl + (((kk / 4) * QB + (kk % 4) * 32) >> 4), idesc_of<F, false, 64>(), kk > 0);
}
template <int D, class F, int QB>
__device__ __forceinline__ void half_grad(uint32_t tmem_d, uint32_t tmem_a, const uint8_t* B, bool add) {
    if (!elect_one()) return;
    const uint32_t bl = ((s32(B) >> 4) & 0x3FFFu) | ((uint32_t)(QB >> 4) << 16);
#pragma unroll
    for (int kk = 0; kk < 64 / UMMA_K; ++kk)
        umma_ts(tmem_d, tmem_a + kk / 2 * 32 + kk % 2 * 8, bl + ((kk * 2048) >> 4), idesc_of<F, true, D>(), add || kk > 0);
}
// this thread's 32 columns of an operand, over scores that it has read
__device__ __forceinline__ void hand_over(uint32_t taddr, const uint32_t (&v)[16], uint64_t* bar) {
    tmem_st16(taddr, v);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ uint32_t tmem_alloc_512(uint32_t* slot) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(s32(slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    return 0;
}
__device__ __forceinline__ void tmem_free_512(uint32_t base) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(512u) : "memory");
}

// ---- forward ---------------------------------------------------------------------------------------------------------------------------
//   warp 0      loads: Q (two buffers) per tile of queries, K and V of 128 keys through rings of four (D 128: two) and two stages
//   warps 1, 2  products of the softmax groups: S = Q K^T, then O += P V
//   warp 3      the next tile of queries
//   warps 4-19  two softmax groups of eight, on alternating key tiles (the first one is always group 0's, so that results do not depend on which CTA took what), each with its own
//               maximum, sum and output, and stages of the rings; two warps share 32 rows
// Tensor memory: 2 x 128 columns of scores, 2 x D of outputs.
template <int D>
struct __align__(1024) SmemFwd {
    static constexpr int KS = D == 64 ? 4 : 2;                // half of them for each group
    uint8_t q[2][BM * D * 2];                                 // and, once its products are done, the output on its way to memory
    uint8_t k[KS][BN * D * 2], v[2][BN * D * 2];
    uint64_t q_full[2], q_empty[2], k_full[KS], k_empty[KS], v_full[2], v_empty[2], s_full[2], p_ready[2], pv_done[2];
    Work work;
    float mx[2][2][2][BM];                                    // [parity of the group's tile][group][half of the columns]
    float ls[2][2][2][BM], ms[2][2][BM];                      // sums and maxima at the end, [parity of the tile of queries][group]
    int2 seen[2][BM];                                         // [slot]: the rows' visible keys
    __align__(1024) uint8_t low[BM * D];
    uint32_t tmem_base;
    int abort_flag;
};

// N units of 16 bytes of a row, from unit `at` on, where a tensor map that swizzles rows of W bytes (64 or 128) expects them
template <int W, int N>
__device__ __forceinline__ void stage_units(uint8_t* tile, int row, int at, const uint32_t (&y)[4 * N]) {
    const int key = row * W / 128 & (W / 16 - 1);
#pragma unroll
    for (int u = 0; u < N; ++u)
        *reinterpret_cast<uint4*>(tile + row * W + ((at + u ^ key) << 4)) = make_uint4(y[4 * u], y[4 * u + 1], y[4 * u + 2], y[4 * u + 3]);
}
// 32 rows x OW columns of a warp (lane = row) through 32 x OW x 2 bytes of shared memory to rows of `d` numbers: a store then covers whole pieces of rows, not 16 bytes of 32 rows.
template <int OW>
__device__ __forceinline__ void rows_out(uint8_t* stage, const uint32_t (&y)[OW / 2], bf16* out, long long row_stride, int rows, int cols) {
    constexpr int U = OW / 8, RPI = 32 / U;                   // 16-byte units of a row; rows of a store
    const int lane = threadIdx.x & 31, key = lane * U / 8 & (U - 1);
#pragma unroll
    for (int u = 0; u < U; ++u)
        *reinterpret_cast<uint4*>(stage + lane * OW * 2 + ((u ^ key) << 4)) = make_uint4(y[4 * u], y[4 * u + 1], y[4 * u + 2], y[4 * u + 3]);
    __syncwarp();
    const int u = lane % U;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int r = i * RPI + lane / U;
        const uint4 z = *reinterpret_cast<const uint4*>(stage + r * OW * 2 + ((u ^ (r * U / 8 & (U - 1))) << 4));
        if (r < rows && u * 8 < cols) *reinterpret_cast<uint4*>(out + r * row_stride + u * 8) = z;
    }
    __syncwarp();
}

template <int D, class F>
__global__ void __launch_bounds__(THREADS, 1)
scored_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmL, const Args a, int group) {
    extern __shared__ uint8_t smem_raw[];
    SmemFwd<D>& sm = *reinterpret_cast<SmemFwd<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int KS = SmemFwd<D>::KS, DK = D / 64;
    constexpr uint32_t O_COL = 2 * BN;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;
    int* err = a.err;
    if (threadIdx.x == 0) {
        for (int s = 0; s < KS; ++s) { mbar_init(&sm.k_full[s], 1); mbar_init(&sm.k_empty[s], 1); }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.q_full[s], 1); mbar_init(&sm.q_empty[s], 4);
            mbar_init(&sm.v_full[s], 1); mbar_init(&sm.v_empty[s], 1);
            mbar_init(&sm.s_full[s], 1); mbar_init(&sm.pv_done[s], 1);
            mbar_init(&sm.p_ready[s], 8);
        }
        init_work(sm.work, 1 + 2 + 16);
        sm.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_512(&sm.tmem_base);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = uniform(sm.tmem_base);

    // qi counts the tiles of queries that see something, c a group's key tiles of all of them
    if (warp == 0) {
        if (lane == 0) {
            int c0 = 0, c1 = 0;
            for (int it = 0, qi = 0;; ++it) {
                const int slot = it & 1;
                if (!wait_for(&sm.work.full[slot], (it >> 1) & 1, abort_flag, err, 0x21000 | slot)) break;
                const Item w = sm.work.item[slot];
                if (w.n_it < 0) break;
                mbar_arrive(&sm.work.empty[slot]);
                if (w.n_it == 0) continue;
                const int qs = qi & 1;
                if (!wait_for(&sm.q_empty[qs], ((qi >> 1) & 1) ^ 1, abort_flag, err, 0x21010 | qs)) break;
                mbar_expect_tx(&sm.q_full[qs], BM * D * 2);
                load_tile<D>(sm.q[qs], &tmQ, &sm.q_full[qs], w.h, w.q0, w.b);
                bool ok = true;
                for (int j = 0; j < w.n_it; ++j) {
                    const int s = j & 1, c = s == 0 ? c0++ : c1++, sk = c % (KS / 2) * 2 + s, key0 = (w.nb_lo + j) * BN;
                    ok = wait_for(&sm.k_empty[sk], ((c / (KS / 2)) & 1) ^ 1, abort_flag, err, 0x21020 | sk);
                    if (!ok) break;
                    mbar_expect_tx(&sm.k_full[sk], BN * D * 2);
                    load_tile<D>(sm.k[sk], &tmK, &sm.k_full[sk], w.hk, key0, w.b);
                    ok = wait_for(&sm.v_empty[s], (c & 1) ^ 1, abort_flag, err, 0x21030 | s);
                    if (!ok) break;
                    mbar_expect_tx(&sm.v_full[s], BN * D * 2);
                    // MN-major operand: per 64 keys, D / 64 boxes of {64 d, 64 keys} (8 KiB each)
#pragma unroll
                    for (int kk = 0; kk < BN / 64; ++kk)
#pragma unroll
                        for (int nb = 0; nb < DK; ++nb)
                            tma_load_4d(sm.v[s] + (kk * DK + nb) * 8192, &tmV, &sm.v_full[s], nb * 64, w.hk, key0 + kk * 64, w.b);
                }
                if (!ok) break;
                ++qi;
            }
        }
    } else if (warp == 1 || warp == 2) {
        const int g = warp - 1;
        constexpr uint32_t idesc_s = idesc_of<F, false, BN>(), idesc_o = idesc_of<F, true, D>();
        bool ok = true;
        for (int it = 0, qi = 0, c = 0; ok; ++it) {
            const int slot = it & 1;
            ok = wait_warp(&sm.work.full[slot], (it >> 1) & 1, abort_flag, err, 0x22000 | slot);
            const int n_it = uniform(sm.work.item[slot].n_it);
            if (!ok || n_it < 0) break;
            if (lane == 0) mbar_arrive(&sm.work.empty[slot]);
            __syncwarp();
            if (n_it == 0) continue;
            const int qs = qi & 1;
            for (int j = g; ok && j < n_it; j += 2, ++c) {
                const int sk = c % (KS / 2) * 2 + g;
                const uint32_t ph = c & 1;
                const bool first = j == g;
                // the scores go over the group's last P: its product has to complete
                ok = (!first || wait_warp(&sm.q_full[qs], (qi >> 1) & 1, abort_flag, err, 0x22010 | qs)) &&
                     wait_warp(&sm.k_full[sk], (c / (KS / 2)) & 1, abort_flag, err, 0x22020 | sk) &&
                     (c == 0 || wait_warp(&sm.pv_done[g], ph ^ 1, abort_flag, err, 0x22030));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t ql = desc_lo<false>(s32(sm.q[qs])), kl = desc_lo<false>(s32(sm.k[sk]));
#pragma unroll
                    for (int kk = 0; kk < D / UMMA_K; ++kk) {
                        const uint32_t off = ((kk / 4) * (BM * 128) + (kk % 4) * 32) >> 4;
                        umma_ss(tmem_base + g * BN, ql + off, kl + off, idesc_s, kk > 0);
                    }
                    umma_commit(&sm.k_empty[sk]);
                    umma_commit(&sm.s_full[g]);
                }
                // (the first product of a tile of queries goes over the output of the one before, which the softmax warps have all read ahead of these weights)
                ok = wait_warp(&sm.v_full[g], ph, abort_flag, err, 0x22040 | g) && wait_warp(&sm.p_ready[g], ph, abort_flag, err, 0x22050 | g);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t vl = desc_lo<true>(s32(sm.v[g]));
#pragma unroll
                    for (int kk = 0; kk < BN / UMMA_K; ++kk) {
                        // every half of the columns left its 32 columns of P at its beginning
                        const uint32_t boff = ((kk / 4) * (DK * 8192) + (kk % 4) * 2048) >> 4;
                        umma_ts(tmem_base + O_COL + g * D, tmem_base + g * BN + kk / 4 * 64 + kk % 4 * 8, vl + boff, idesc_o, !first || kk > 0);
                    }
                    umma_commit(&sm.v_empty[g]);
                    umma_commit(&sm.pv_done[g]);
                }
            }
            ++qi;
        }
    } else if (warp == 3) {
        hand_out(sm.work, sm.seen, a, group, abort_flag, err, 0x23000);
    } else {
        const int qd = warp & 3, quarter = (warp - 4) >> 2, grp = quarter >> 1, part = quarter & 1;
        const int r = qd * 32 + lane;                         // query row inside the tile
        const uint32_t lane_addr = tmem_base + ((uint32_t)(qd * 32) << 16);
        const uint32_t s_addr = lane_addr + grp * BN + part * 64, o_addr = lane_addr + O_COL + grp * D + part * (D / 2);
        constexpr int OW = D / 4;
        bool ok = true;                                       // after a wait that ran out only the barriers are kept up with
        // (What the loop over key tiles does not need at every turn is left in shared memory: registers are few.)
        int done[2] = {0, 0};                                 // key tiles of the groups so far
        int owed = -1;                                        // (quarter 0) buffer of Q from which rows are still on their way
        auto settle = [&]() {
            if (owed < 0) return;
            if (lane == 0) {
                tma_store_wait_read();
                mbar_arrive(&sm.q_empty[owed]);
            }
            __syncwarp();
            owed = -1;
        };
        for (int it = 0, qi = 0;; ++it) {
            const int slot = it & 1;
            if (ok) ok = wait_warp(&sm.work.full[slot], (it >> 1) & 1, abort_flag, err, 0x24000 | slot);
            if (!all_softmax(ok)) break;
            const int n_it = sm.work.item[slot].n_it;
            if (n_it < 0) break;
            float m = -INFINITY, l = 0.f;
            const ScoreOf so = score_of<F>(a.scale, a.x, sm.work.item[slot].h);
            const float sc = so.unit;
            for (int j = grp, c = grp == 0 ? done[0] : done[1]; j < n_it; j += 2, ++c) {
                if (ok) ok = wait_warp(&sm.s_full[grp], c & 1, abort_flag, err, 0x24010 | grp);
                const volatile Item& w = sm.work.item[slot];
                const int tile_key0 = (w.nb_lo + j) * BN, key0 = tile_key0 + part * 64;
                const bool need_mask = tile_key0 < w.every.x || tile_key0 + BN > w.every.y;
                tc_fence_after();
                // The scores are read twice, 32 at a time, and stay in tensor memory while the maximum is looked for: 64 of them and what a bias or a cap needs did not fit into 96
                // registers (8192 queries with slopes 453 -> 367 us, plain scores 305 -> 300 us).
                uint32_t v[32];
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int col = 0; col < 64; col += 32) {
                    tmem_ld32(s_addr + col, v);
                    tmem_ld_wait();
                    scored<F>(v, so, a.x, (float)(key0 + col - a.q_offset - w.q0 - r));
                    if (need_mask) {
                        const int2 range = sm.seen[slot][r];
                        const int hi = range.y - 1 - key0 - col, lo = range.x - 1 - key0 - col;
                        if (__any_sync(0xffffffffu, hi < 31 || lo >= 0)) {                           // most blocks of 32 x 32 in a masked tile are visible
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i > hi || i <= lo) v[i] = 0xff800000u;                           // -inf
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < 32; i += 8) mx4[e] = max3(mx4[e], __uint_as_float(v[i + e]), __uint_as_float(v[i + e + 4]));
                    if (F::SCORE != SCORE_PLAIN || need_mask) tmem_st32(s_addr + col, v);
                }
                tmem_st_wait();
                float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                sm.mx[c & 1][grp][part][r] = mx;
                asm volatile("bar.sync %0, 64;" :: "r"(1 + grp * 4 + qd) : "memory");
                if (!ok) continue;
                mx = fmaxf(mx, sm.mx[c & 1][grp][part ^ 1][r]);
                // Both halves of a row see the same numbers and decide alike.  The maximum is followed exactly, so that the largest weight is one, without a rounding: with weights up to
                // 2^8 above one, or capped scores (whose exponentials fit without a maximum) as they are, dq and dk of rows with one large weight were off by 0.0027 and 0.0034, not 0.0025.
                // (Forward, 8192 queries in packed documents, 16 heads of 128: 111 us exactly and up to 2^8 behind, 105 without; a batch with prefixes of 3 x 1531: 83 / 79 us.)
                const bool grow = mx > m;                     // also the first visible key of the row (m = -inf)
                const bool scaled = grow && m != -INFINITY;
                const float corr = scaled ? exp2f((m - mx) * sc) : 1.f;
                if (grow) m = mx;
                l *= corr;
                if (__any_sync(0xffffffffu, scaled)) {        // not at the group's first tile; these scores were issued behind the last product of the group
                    ok = wait_warp(&sm.pv_done[grp], (c & 1) ^ 1, abort_flag, err, 0x24020 | grp);
                    if (!ok) continue;
                    tc_fence_after();
#pragma unroll
                    for (int col = 0; col < D / 2; col += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_addr + col, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                        tmem_st16(o_addr + col, o);
                    }
                }
                const float nm = m == -INFINITY ? 0.f : -m * sc;
                const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
                float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
                // The product takes the weights in 16 bits, as its operands have to be (half a step of each, in no common direction); the sum, in 32 bits, takes them as they were.
#pragma unroll
                for (int col = 0; col < 64; col += 32) {
                    uint32_t p[16];
                    tmem_ld32(s_addr + col, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float2 x01 = __ffma2_rn(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sc2, nm2);
                        const float2 x23 = __ffma2_rn(make_float2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), sc2, nm2);
                        const float p0 = exp2f(x01.x), p1 = exp2f(x01.y), p2 = exp2f(x23.x), p3 = exp2f(x23.y);
                        sum0 = __fadd2_rn(sum0, make_float2(p0, p1));
                        sum1 = __fadd2_rn(sum1, make_float2(p2, p3));
                        p[i >> 1] = pack16<F>(p0, p1);
                        p[(i >> 1) + 1] = pack16<F>(p2, p3);
                    }
                    tmem_st16(s_addr + (col >> 1), p);          // over scores that have been read
                }
                l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_ready[grp]);
            }
            settle();
            const Item w = sm.work.item[slot];
            const int row = w.q0 + r, d = a.x.d;
            const long long out0 = (((long long)w.b * a.Tq + w.q0 + qd * 32) * a.Hq + w.h) * d + quarter * OW, row_stride = (long long)a.Hq * d;
            const int rows = min(32, a.Tq - w.q0 - qd * 32), cols = d - quarter * OW;
            float* lse = a.lse + ((long long)w.b * a.Hq + w.h) * a.Tq + row;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.work.empty[slot]);
            if (n_it == 0) {                                  // nothing to see: zeros
                if (row < a.Tq) {
                    for (int c = 0; c < OW && c < cols; c += 8) *reinterpret_cast<uint4*>(a.out + out0 + lane * row_stride + c) = make_uint4(0, 0, 0, 0);
                    const int wide = (d + 15) & ~15;
                    if (a.x.low != nullptr)
                        for (int c = quarter * OW; c < (quarter + 1) * OW && c < wide; c += 16)
                            *reinterpret_cast<uint4*>(a.x.low + (((long long)w.b * a.Tq + row) * a.Hq + w.h) * wide + c) = make_uint4(0, 0, 0, 0);
                    if (quarter == 0) *lse = -INFINITY;
                }
                continue;
            }
            // join the groups: every warp takes a quarter of the columns of both outputs
            const int par = qi & 1;
            sm.ls[par][grp][part][r] = l;
            if (part == 0) sm.ms[par][grp][r] = m;
            asm volatile("bar.sync 10, 512;" ::: "memory");       // behind it at most the last product of each group is outstanding
            const float mm = fmaxf(sm.ms[par][0][r], sm.ms[par][1][r]);
            float wg[2];
            l = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float mg = sm.ms[par][g][r];
                wg[g] = mg == -INFINITY ? 0.f : exp2f((mg - mm) * sc);
                l += wg[g] * (sm.ls[par][g][0][r] + sm.ls[par][g][1][r]);
            }
            float o[OW];
#pragma unroll
            for (int i = 0; i < OW; ++i) o[i] = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (n_it <= g) continue;
                if (ok) ok = wait_warp(&sm.pv_done[g], (done[g] + (n_it - g - 1) / 2) & 1, abort_flag, err, 0x24030 | g);     // the group's last tile
                if (!ok) break;
                tc_fence_after();
                uint32_t x[OW];
                tmem_ld<OW>(lane_addr + O_COL + g * D + quarter * OW, x);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < OW; ++i) o[i] += wg[g] * __uint_as_float(x[i]);
            }
            tc_fence_before();                                // ahead of the next weights, behind which the outputs are written again
            if (ok) {
                const float inv = l > 0.f ? 1.f / l : 0.f;
                uint32_t y[OW / 2];
#pragma unroll
                for (int c = 0; c < OW; c += 2) y[c / 2] = pack16<F>(o[c] * inv, o[c + 1] * inv);
                // Both groups' products of this tile are done: the rows go through Q's buffer, by bulk copies, which go on while the warps turn to the next tile.  The four warps of 32 rows
                // join theirs: copies of 128 bytes a row are three times as fast as of 64 and 32.
                uint8_t* stage = sm.q[qi & 1];
                if constexpr (D == 128) stage_units<128, 4>(stage + (quarter >> 1) * BLK, r, (quarter & 1) * 4, y);
                else stage_units<128, 2>(stage, r, quarter * 2, y);
                if (a.x.low != nullptr) {
                    uint32_t z[OW / 4];
#pragma unroll
                    for (int c = 0; c < OW; c += 4) z[c / 4] = residues<F>(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv, y[c / 2], y[c / 2 + 1]);
                    stage_units<D, OW / 16>(sm.low, r, quarter * (OW / 16), z);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            asm volatile("bar.sync %0, 128;" :: "r"(11 + qd) : "memory");
            if (quarter == 0) {
                if (ok && lane == 0 && rows > 0) {
#pragma unroll
                    for (int kb = 0; kb < D / 64; ++kb)
                        if (kb * 64 < d) tma_store_4d(&tmO, sm.q[qi & 1] + kb * BLK + qd * 4096, kb * 64, w.h, w.q0 + qd * 32, w.b);
                    if (a.x.low != nullptr) tma_store_4d(&tmL, sm.low + qd * 32 * D, 0, w.h, w.q0 + qd * 32, w.b);
                    tma_store_commit();
                }
                const float unit = F::SCORE == SCORE_PLAIN ? a.scale : F::SCORE == SCORE_BIAS ? 1.f / LOG2E : a.x.cap;
                if (row < a.Tq) *lse = l > 0.f ? mm * unit + logf(l) : -INFINITY;
                owed = qi & 1;
            }
            done[0] += (n_it + 1) / 2;
            done[1] += n_it / 2;
            ++qi;
        }
        if (lane == 0) tma_store_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free_512(tmem_base);
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------------
// Two kernels that recompute the scores, on tiles of 128 queries x 128 keys, as in flash_attn_tc.cu; a thread holds 32 columns of a row.
//   dq       warp 1 issues S = Q K^T and dP = dO V^T, the softmax warps make dS of them (in 16 bits over S), dQ += dS K.  Persistent, as the forward kernel.  Its rows go out through dO's
//            buffer: direct stores of 16 bytes of 32 rows filled the load / store pipe for 2000 cycles, behind which other warps' waits on barriers queued too.
//   dk / dv  a CTA has 128 keys of a key head and goes through some of its query heads and, for each, the query tiles that see one of its keys:
//            S^T = K Q^T, dP^T = V dO^T, P^T and dS^T over them, dV += P^T dO, dK += dS^T Q.  In two halves of 64 queries, eight softmax warps each, half a turn apart: while one makes its
//            weights the other makes its gradients, and their products and the next scores run meanwhile.  (Against all warps in step:
//            documents of 4096, capped, 393 -> 336 us, a batch with prefixes 127 -> 116 us; uncapped 128-wide heads 254 -> 263 us by themselves, 642 -> 630 us with all kernels in a graph.)

// The weights' exponents and (SCORE_CAP) the derivative of the cap, from 32 scores; dist: distance of the first column
template <class F>
__device__ __forceinline__ void derive(uint32_t (&v)[32], float2 (&p)[16], const ScoreOf& so, const Ranges& x, float dist) {
    if constexpr (F::SCORE == SCORE_CAP) {
        tanh_of(v, so.a);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 t = make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
            p[i] = __ffma2_rn(make_float2(-t.x, -t.y), t, make_float2(1.f, 1.f));
        }
        if (x.slopes != nullptr) biased(v, 1.f, so.sl, dist);
    } else scored<F>(v, so, x, dist);
}

template <int D>
struct __align__(1024) SmemDq {
    uint8_t q[BM * D * 2], g[BM * D * 2], k[3][BM * D * 2], v[2][BM * D * 2];      // K: read by a tile's first and last product; g in the end: dq on its way to memory
    uint64_t q_full, q_empty, g_full, g_empty, k_full[3], k_empty[3], v_full[2], v_empty[2], s_full[2], dp_full, ds_ready, dq_done, all_done;
    Work work;
    uint32_t tmem_base;
    int abort_flag;
};

template <int D, class F>
__global__ void __launch_bounds__(THREADS, 1)
scored_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const BwdArgs a, int group) {
    extern __shared__ uint8_t smem_raw[];
    SmemDq<D>& sm = *reinterpret_cast<SmemDq<D>*>(smem_raw);
    if ((s32(smem_raw) & 1023u) != 0) {                                       // with 128-wide heads the tiles fill the shared memory
        if (threadIdx.x == 0) atomicCAS(a.err, 0, 0x25001);
        return;
    }
    constexpr uint32_t DP = 256, DQ = 384;                                    // two buffers of scores in front
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;
    int* err = a.err;
    if (threadIdx.x == 0) {
        mbar_init(&sm.q_full, 1); mbar_init(&sm.q_empty, 1); mbar_init(&sm.g_full, 1); mbar_init(&sm.g_empty, 16);
        for (int s = 0; s < 3; ++s) { mbar_init(&sm.k_full[s], 1); mbar_init(&sm.k_empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&sm.v_full[s], 1); mbar_init(&sm.v_empty[s], 1); mbar_init(&sm.s_full[s], 1); }
        mbar_init(&sm.dp_full, 1); mbar_init(&sm.ds_ready, 16); mbar_init(&sm.dq_done, 1); mbar_init(&sm.all_done, 1);
        init_work(sm.work, 1 + 1 + 16);
        sm.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_512(&sm.tmem_base);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = uniform(sm.tmem_base);

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int it = 0, qi = 0, n = 0; ok; ++it) {
                const int slot = it & 1;
                ok = wait_for(&sm.work.full[slot], (it >> 1) & 1, abort_flag, err, 0x25010 | slot);
                if (!ok) break;
                const Item w = sm.work.item[slot];
                if (w.n_it < 0) break;
                mbar_arrive(&sm.work.empty[slot]);
                if (w.n_it == 0) continue;
                for (int j = 0; ok && j < w.n_it; ++j, ++n) {
                    const int s = n & 1, s3 = n % 3, key0 = (w.nb_lo + j) * BN;
                    ok = wait_for(&sm.k_empty[s3], ((n / 3) & 1) ^ 1, abort_flag, err, 0x25020 | s3);
                    if (!ok) break;
                    mbar_expect_tx(&sm.k_full[s3], BM * D * 2);
                    load_tile<D>(sm.k[s3], &tmK, &sm.k_full[s3], w.hk, key0, w.b);
                    if (j == 0) {
                        ok = wait_for(&sm.q_empty, (qi & 1) ^ 1, abort_flag, err, 0x25030);
                        if (!ok) break;
                        mbar_expect_tx(&sm.q_full, BM * D * 2);
                        load_tile<D>(sm.q, &tmQ, &sm.q_full, w.h, w.q0, w.b);
                        ok = wait_for(&sm.g_empty, (qi & 1) ^ 1, abort_flag, err, 0x25031);
                        if (!ok) break;
                        mbar_expect_tx(&sm.g_full, BM * D * 2);
                        load_tile<D>(sm.g, &tmG, &sm.g_full, w.h, w.q0, w.b);
                    }
                    ok = wait_for(&sm.v_empty[s], ((n >> 1) & 1) ^ 1, abort_flag, err, 0x25040 | s);
                    if (!ok) break;
                    mbar_expect_tx(&sm.v_full[s], BM * D * 2);
                    load_tile<D>(sm.v[s], &tmV, &sm.v_full[s], w.hk, key0, w.b);
                }
                ++qi;
            }
        }
    } else if (warp == 1) {
        int last = 0;
        auto scores = [&](int n) -> bool {
            const int s = n & 1, s3 = n % 3;
            if (!wait_warp(&sm.k_full[s3], (n / 3) & 1, abort_flag, err, 0x25100 | s3)) return false;
            tc_fence_after();
            score_product<D, F>(tmem_base + s * 128, sm.q, sm.k[s3]);
            if (elect_one()) {
                umma_commit(&sm.s_full[s]);
                if (n + 1 == last) umma_commit(&sm.q_empty);              // the next Q may come: only scores read it
            }
            return true;
        };
        auto dprobs = [&](int n) -> bool {
            const int s = n & 1;
            if (!wait_warp(&sm.v_full[s], (n >> 1) & 1, abort_flag, err, 0x25110 | s)) return false;
            tc_fence_after();
            score_product<D, F>(tmem_base + DP, sm.g, sm.v[s]);
            if (elect_one()) {
                umma_commit(&sm.v_empty[s]);
                umma_commit(&sm.dp_full);
            }
            return true;
        };
        bool ok = true;
        for (int it = 0, qi = 0, base = 0; ok; ++it) {
            const int slot = it & 1;
            ok = wait_warp(&sm.work.full[slot], (it >> 1) & 1, abort_flag, err, 0x25120 | slot);
            const int n_it = uniform(sm.work.item[slot].n_it);
            if (!ok || n_it < 0) break;
            if (lane == 0) mbar_arrive(&sm.work.empty[slot]);
            __syncwarp();
            if (n_it == 0) continue;
            last = base + n_it;
            ok = wait_warp(&sm.q_full, qi & 1, abort_flag, err, 0x25130) && scores(base) && wait_warp(&sm.g_full, qi & 1, abort_flag, err, 0x25131) && dprobs(base) &&
                 (n_it < 2 || scores(base + 1));
            for (int n = base; ok && n < last; ++n) {
                if (!wait_warp(&sm.ds_ready, n & 1, abort_flag, err, 0x25140)) { ok = false; break; }
                if (n + 1 < last && !dprobs(n + 1)) { ok = false; break; }
                tc_fence_after();
                grad_product<D, F>(tmem_base + DQ, tmem_base + (n & 1) * 128, sm.k[n % 3], n > base);
                if (elect_one()) {
                    umma_commit(&sm.k_empty[n % 3]);
                    umma_commit(&sm.dq_done);
                    if (n + 1 == last) umma_commit(&sm.all_done);
                }
                // the next scores of this buffer go over dS_n: the product that reads it has to complete.  (Waited for at every tile, so that no phase is passed over.)
                ok = wait_warp(&sm.dq_done, n & 1, abort_flag, err, 0x25150) && (n + 2 >= last || scores(n + 2));
            }
            base = last;
            ++qi;
        }
    } else if (warp == 3) {
        hand_out(sm.work, nullptr, a, group, abort_flag, err, 0x25160);
    } else if (warp >= 4) {
        const int qd = warp & 3, part = (warp - 4) >> 2;
        const int r = qd * 32 + lane;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(qd * 32) << 16);
        constexpr int OW = D / SPLIT;
        bool ok = true;
        for (int it = 0, qi = 0, base = 0;; ++it) {
            const int slot = it & 1;
            if (ok) ok = wait_warp(&sm.work.full[slot], (it >> 1) & 1, abort_flag, err, 0x25200 | slot);
            if (!all_softmax(ok)) break;
            const Item w = sm.work.item[slot];
            __syncwarp();
            if (w.n_it < 0) break;
            if (lane == 0) mbar_arrive(&sm.work.empty[slot]);
            const int row = w.q0 + r, qi_at = a.q_offset + row, last = base + w.n_it, d = a.x.d;
            const long long row_stride = (long long)a.Hq * d;
            bf16* out = a.dq + (((long long)w.b * a.Tq + w.q0 + qd * 32) * a.Hq + w.h) * d + part * OW;      // of the warp's first row
            if (w.n_it == 0) {
                if (row < a.Tq)
                    for (int c = 0; c < OW && part * OW + c < d; c += 8) *reinterpret_cast<uint4*>(out + lane * row_stride + c) = make_uint4(0, 0, 0, 0);
                continue;
            }
            const ScoreOf so = score_of<F>(a.scale, a.x, w.h);
            const float sc = so.unit;
            const long long stat = ((long long)w.b * a.Hq + w.h) * a.Tq + row;
            float lse2 = row < a.Tq ? a.lse[stat] : INFINITY, dl = row < a.Tq ? a.delta[stat] : 0.f;
            int2 range = row < a.Tq ? visible_range(a, w.b, row) : make_int2(0, 0);
            for (int n = base; ok && n < last; ++n) {
                const int s = n & 1;
                const int tile_key0 = (w.nb_lo + n - base) * BN, key0 = tile_key0 + part * 32;
                const bool need_mask = tile_key0 < w.every.x || tile_key0 + BN > w.every.y;
                ok = wait_warp(&sm.s_full[s], (n >> 1) & 1, abort_flag, err, 0x25210 | s);
                if (!ok) break;
                tc_fence_after();
                if (n == base) {                                             // the row's numbers have been on their way while the products ran
                    asm volatile("" : "+f"(lse2), "+f"(dl), "+r"(range.x), "+r"(range.y));
                    lse2 = lse2 == -INFINITY ? INFINITY : lse2 * LOG2E;      // a row that sees nothing: its weights are zero
                }
                uint32_t v[32];
                float2 p[16];
                tmem_ld32(lane_addr + s * 128 + part * 32, v);
                tmem_ld_wait();
                derive<F>(v, p, so, a.x, (float)(key0 - qi_at));
                if (need_mask && __any_sync(0xffffffffu, key0 < range.x || key0 + 32 > range.y)) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (key0 + i < range.x || key0 + i >= range.y) v[i] = 0xff800000u;       // -inf -> p = 0
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), make_float2(sc, sc), make_float2(-lse2, -lse2));
                    const float2 e = make_float2(exp2f(x.x), exp2f(x.y));
                    p[i] = F::SCORE == SCORE_CAP ? __fmul2_rn(p[i], e) : e;
                    asm volatile("" : "+f"(p[i].x), "+f"(p[i].y));                                 // here, not behind the wait
                }
                ok = wait_warp(&sm.dp_full, n & 1, abort_flag, err, 0x25220);
                if (!ok) break;
                tc_fence_after();
                tmem_ld32(lane_addr + DP + part * 32, v);
                tmem_ld_wait();
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {                                                   // the softmax scale is applied to dQ at the end
                    const float2 x = __fmul2_rn(p[i], __fadd2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), make_float2(-dl, -dl)));
                    pk[i] = pack16<F>(x.x, x.y);
                }
                hand_over(lane_addr + s * 128 + part * 32, pk, &sm.ds_ready);
            }
            if (ok) ok = wait_warp(&sm.all_done, qi & 1, abort_flag, err, 0x25230);
            tc_fence_after();
            if (ok) {
                uint32_t v[OW], y[OW / 2];
                tmem_ld<OW>(lane_addr + DQ + part * OW, v);
                tmem_ld_wait();
                tc_fence_before();                                                               // ahead of the next weights, behind which the accumulator is written again
#pragma unroll
                for (int c = 0; c < OW; c += 2) y[c / 2] = pack16<F>(a.scale * __uint_as_float(v[c]), a.scale * __uint_as_float(v[c + 1]));
                rows_out<OW>(sm.g + (warp - 4) * 32 * OW * 2, y, out, row_stride, min(32, a.Tq - w.q0 - qd * 32), d - part * OW);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                         // ahead of the next dO in this buffer
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.g_empty);
            base = last;
            ++qi;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free_512(tmem_base);
    }
}

template <int D>
struct __align__(1024) SmemDkv {
    static constexpr int QS = 4;                                             // half tiles of Q
    uint8_t k[BM * D * 2], v[BM * D * 2], q[QS][64 * D * 2], g[2][BM * D * 2];        // at the end q: the other CTA's part of the sum, g: dk and dv on their way to memory
    float lse2[2][BM], delta[2][BM];                                         // of the looped queries
    int first[2][BM], stop[2][BM];
    int2 every[2][4];                                                        // keys that 32 of them all see
    uint16_t list[MAX_TILES];                                                // query tiles that see a key of this tile
    uint64_t kv_full, q_full[QS], q_empty[QS], stat_full[2], stat_empty[2], g_full[2], g_empty[2];
    uint64_t s_full[2], dp_full[2], p_ready[2], ds_ready[2], dv_done[2], dk_done[2], all_done;      // [half of the queries]
    uint32_t tmem_base;
    int abort_flag, listed;
};

// `heads`: query heads that this CTA takes; a cluster of Hq / Hkv / heads CTAs shares a tile of keys.
template <int D, class F>
__global__ void __launch_bounds__(THREADS, 1)
scored_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const BwdArgs a, int group, int heads) {
    extern __shared__ uint8_t smem_raw[];
    SmemDkv<D>& sm = *reinterpret_cast<SmemDkv<D>*>(smem_raw);
    if ((s32(smem_raw) & 1023u) != 0) {                                       // (the same for all CTAs of a cluster)
        if (threadIdx.x == 0) atomicCAS(a.err, 0, 0x26001);
        return;
    }
    constexpr uint32_t ST = 0, DP = 128, DV = 256, DKC = 384;
    constexpr int QS = SmemDkv<D>::QS;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rep = a.Hq / a.Hkv, share = rep / heads, rank = blockIdx.x % share;
    const TileOf t = longest_first(blockIdx.x / share, (a.Tk + BM - 1) / BM, a.B * a.Hkv, group);
    const int kb_tile = t.rank, hk = t.pair % a.Hkv, b = t.pair / a.Hkv, h0 = hk * rep + rank * heads;      // early key tiles are seen by the most queries
    const int k0 = kb_tile * BM;
    volatile int* abort_flag = &sm.abort_flag;
    int* err = a.err;
    if (warp == 3) {                                                         // otherwise idle: lists the query tiles in order
        const int n_qb = (a.Tq + BM - 1) / BM, k1 = min(k0 + BM, a.Tk);
        int n = 0;
        for (int t0 = 0; t0 < n_qb; t0 += 32) {
            const int4 r = t0 + lane < n_qb ? __ldg(a.x.tiles + (long long)b * n_qb + t0 + lane) : make_int4(0, 0, 0, 0);
            const bool sees = r.x < k1 && r.y > k0;
            const uint32_t who = __ballot_sync(0xffffffffu, sees);
            if (sees) sm.list[n + __popc(who & ((1u << lane) - 1))] = (uint16_t)(t0 + lane);
            n += __popc(who);
        }
        if (lane == 0) sm.listed = n;
    }
    if (threadIdx.x == 0) {
        mbar_init(&sm.kv_full, 1);
        for (int s = 0; s < QS; ++s) { mbar_init(&sm.q_full[s], 1); mbar_init(&sm.q_empty[s], 1); }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.stat_full[s], 1); mbar_init(&sm.stat_empty[s], 1);
            mbar_init(&sm.g_full[s], 1); mbar_init(&sm.g_empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.s_full[s], 1); mbar_init(&sm.dp_full[s], 1);
            mbar_init(&sm.p_ready[s], 8); mbar_init(&sm.ds_ready[s], 8);
            mbar_init(&sm.dv_done[s], 1); mbar_init(&sm.dk_done[s], 1);
        }
        mbar_init(&sm.all_done, 1);
        sm.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(&sm.kv_full, 2 * BM * D * 2);                          // on their way while the tensor memory is fetched and the list made
        load_tile<D>(sm.k, &tmK, &sm.kv_full, hk, k0, b);
        load_tile<D>(sm.v, &tmV, &sm.kv_full, hk, k0, b);
    }
    if (warp == 1) tmem_alloc_512(&sm.tmem_base);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = uniform(sm.tmem_base);
    const int ni = uniform(sm.listed), n_it = ni * heads;
    bool alive = true;

    if (warp == 0) {
        if (lane == 0) {
            for (int it = 0; it < n_it; ++it) {
                const int s = it & 1, h = h0 + it / ni, q0 = sm.list[it % ni] * BM;
                auto half_q = [&](int half) -> bool {
                    const int n = 2 * it + half, sq = n % QS;
                    if (!wait_for(&sm.q_empty[sq], ((n / QS) & 1) ^ 1, abort_flag, err, 0x26100 | sq)) return false;
                    mbar_expect_tx(&sm.q_full[sq], 64 * D * 2);
#pragma unroll
                    for (int kb = 0; kb < D / 64; ++kb) tma_load_4d(sm.q[sq] + kb * 8192, &tmQ, &sm.q_full[sq], kb * 64, h, q0 + half * 64, b);
                    return true;
                };
                if (!half_q(0)) break;                            // in the order in which the buffers get free
                if (!wait_for(&sm.g_empty[s], ((it >> 1) & 1) ^ 1, abort_flag, err, 0x26120 | s)) break;
                mbar_expect_tx(&sm.g_full[s], BM * D * 2);
                load_tile<D>(sm.g[s], &tmG, &sm.g_full[s], h, q0, b);
                if (!half_q(1)) break;
            }
        }
    } else if (warp == 1) {
        bool ok = wait_warp(&sm.kv_full, 0, abort_flag, err, 0x26200);
        if (n_it > 0) {
            auto scores = [&](int it, int half) -> bool {
                const int n = 2 * it + half, sq = n % QS;
                if (!wait_warp(&sm.q_full[sq], (n / QS) & 1, abort_flag, err, 0x26300 | sq)) return false;
                tc_fence_after();
                half_product<D, F, 8192>(tmem_base + ST + half * 64, sm.k, sm.q[sq]);
                if (elect_one()) umma_commit(&sm.s_full[half]);
                return true;
            };
            auto dprobs = [&](int it, int half) -> bool {
                if (!wait_warp(&sm.g_full[it & 1], (it >> 1) & 1, abort_flag, err, 0x26310 | (it & 1))) return false;
                tc_fence_after();
                half_product<D, F, BLK>(tmem_base + DP + half * 64, sm.v, sm.g[it & 1] + half * 8192);
                if (elect_one()) umma_commit(&sm.dp_full[half]);
                return true;
            };
            auto grad_v = [&](int it, int half) -> bool {                                         // dV += P^T dO
                if (!wait_warp(&sm.p_ready[half], it & 1, abort_flag, err, 0x26400 | half)) return false;
                tc_fence_after();
                half_grad<D, F, BLK>(tmem_base + DV, tmem_base + ST + half * 64, sm.g[it & 1] + half * 8192, it > 0 || half > 0);
                if (elect_one()) umma_commit(&sm.dv_done[half]);
                if (half == 1 && elect_one()) umma_commit(&sm.g_empty[it & 1]);
                return true;
            };
            auto grad_k = [&](int it, int half) -> bool {                                         // dK += dS^T Q
                if (!wait_warp(&sm.ds_ready[half], it & 1, abort_flag, err, 0x26410 | half)) return false;
                tc_fence_after();
                const int sq = (2 * it + half) % QS;
                half_grad<D, F, 8192>(tmem_base + DKC, tmem_base + DP + half * 64, sm.q[sq], it > 0 || half > 0);
                if (elect_one()) umma_commit(&sm.dk_done[half]);
                if (elect_one()) umma_commit(&sm.q_empty[sq]);
                if (half == 1 && elect_one()) umma_commit(&sm.stat_empty[it & 1]);
                return true;
            };
            // the next scores go over P^T, the next dP^T over dS^T: the products that read them have to complete (waited for at every tile, so that no phase is passed over)
            auto free_p = [&](int it, int half) { return wait_warp(&sm.dv_done[half], it & 1, abort_flag, err, 0x26600 | half); };
            auto free_ds = [&](int it, int half) { return wait_warp(&sm.dk_done[half], it & 1, abort_flag, err, 0x26610 | half); };
            ok = ok && scores(0, 0) && dprobs(0, 0) && scores(0, 1) && dprobs(0, 1);
            for (int it = 0; ok && it < n_it; ++it) {
                const bool more = it + 1 < n_it;
                // the first half's weights and the second half's gradients of the tile before
                ok = grad_v(it, 0) && (it == 0 || grad_k(it - 1, 1)) && free_p(it, 0) && (!more || scores(it + 1, 0)) && (it == 0 || (free_ds(it - 1, 1) && dprobs(it, 1)));
                // the second half's weights and the first half's gradients
                ok = ok && grad_v(it, 1) && grad_k(it, 0) && free_p(it, 1) && (!more || scores(it + 1, 1)) && free_ds(it, 0) && (!more || dprobs(it + 1, 0));
            }
            if (ok && grad_k(n_it - 1, 1) && elect_one()) umma_commit(&sm.all_done);
        }
    } else if (warp == 2) {                                      // log-sum-exp, delta and range of the looped queries
        for (int it = 0; it < n_it; ++it) {
            const int s = it & 1;
            const int h = h0 + it / ni, q0 = sm.list[it % ni] * BM;
            const long long row = ((long long)b * a.Hq + h) * a.Tq;
            float x[4], y[4];
            int2 range[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int q = q0 + lane + 32 * e;
                x[e] = q < a.Tq ? __ldg(a.lse + row + q) * LOG2E : INFINITY;
                y[e] = q < a.Tq ? __ldg(a.delta + row + q) : 0.f;
                if (x[e] == -INFINITY) x[e] = INFINITY;          // a row that sees nothing: its weights are zero
                range[e] = q < a.Tq ? visible_range(a, b, q) : make_int2(0, 0);
            }
            if (!wait_warp(&sm.stat_empty[s], ((it >> 1) & 1) ^ 1, abort_flag, err, 0x26110 | s)) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sm.lse2[s][lane + 32 * e] = x[e]; sm.delta[s][lane + 32 * e] = y[e];
                sm.first[s][lane + 32 * e] = range[e].x; sm.stop[s][lane + 32 * e] = range[e].y;
                const int lo = __reduce_max_sync(0xffffffffu, range[e].x), hi = __reduce_min_sync(0xffffffffu, range[e].y);
                if (lane == 0) sm.every[s][e] = make_int2(lo, hi);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.stat_full[s]);
        }
    } else if (warp >= 4) {
        const int qd = warp & 3, part = (warp - 4) >> 2, half = part >> 1;
        const int r = qd * 32 + lane;                            // key row inside the tile
        const int key = k0 + r;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(qd * 32) << 16);
        ScoreOf so = score_of<F>(a.scale, a.x, h0);
        const float sc = so.unit;
        for (int it = 0, at = 0, h = h0; it < n_it; ++it) {
            const int s = it & 1, tile_q0 = sm.list[at] * BM;
            if (!wait_warp(&sm.stat_full[s], (it >> 1) & 1, abort_flag, err, 0x26510 | s)) { alive = false; break; }
            if (!wait_warp(&sm.s_full[half], it & 1, abort_flag, err, 0x26500 | half)) { alive = false; break; }
            tc_fence_after();
            uint32_t v[32], pk[16];
            float2 p[16];
            tmem_ld32(lane_addr + ST + part * 32, v);
            tmem_ld_wait();
            derive<F>(v, p, so, a.x, (float)(a.q_offset + tile_q0 + part * 32 - key));
            const int2 every = sm.every[s][part];
            if (k0 + qd * 32 < every.x || k0 + qd * 32 + 32 > every.y) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const int4 lo = *reinterpret_cast<const int4*>(&sm.first[s][part * 32 + i]), hi = *reinterpret_cast<const int4*>(&sm.stop[s][part * 32 + i]);
                    if (key < lo.x || key >= hi.x) v[i] = 0xff800000u;
                    if (key < lo.y || key >= hi.y) v[i + 1] = 0xff800000u;
                    if (key < lo.z || key >= hi.z) v[i + 2] = 0xff800000u;
                    if (key < lo.w || key >= hi.w) v[i + 3] = 0xff800000u;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float4 l2 = *reinterpret_cast<const float4*>(&sm.lse2[s][part * 32 + 2 * i]);
                const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), make_float2(sc, sc), make_float2(-l2.x, -l2.y));
                const float2 y = __ffma2_rn(make_float2(__uint_as_float(v[2 * i + 2]), __uint_as_float(v[2 * i + 3])), make_float2(sc, sc), make_float2(-l2.z, -l2.w));
                const float2 ex = make_float2(exp2f(x.x), exp2f(x.y)), ey = make_float2(exp2f(y.x), exp2f(y.y));
                pk[i] = pack16<F>(ex.x, ex.y);
                pk[i + 1] = pack16<F>(ey.x, ey.y);
                p[i] = F::SCORE == SCORE_CAP ? __fmul2_rn(p[i], ex) : ex;
                p[i + 1] = F::SCORE == SCORE_CAP ? __fmul2_rn(p[i + 1], ey) : ey;
            }
            hand_over(lane_addr + ST + part * 32, pk, &sm.p_ready[half]);
            if (!wait_warp(&sm.dp_full[half], it & 1, abort_flag, err, 0x26520 | half)) { alive = false; break; }
            tc_fence_after();
            tmem_ld32(lane_addr + DP + part * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; i += 2) {                                                   // scale applied to dK at the end
                const float4 dl = *reinterpret_cast<const float4*>(&sm.delta[s][part * 32 + 2 * i]);
                const float2 x = __fmul2_rn(p[i], __fadd2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), make_float2(-dl.x, -dl.y)));
                const float2 y = __fmul2_rn(p[i + 1], __fadd2_rn(make_float2(__uint_as_float(v[2 * i + 2]), __uint_as_float(v[2 * i + 3])), make_float2(-dl.z, -dl.w)));
                pk[i] = pack16<F>(x.x, x.y);
                pk[i + 1] = pack16<F>(y.x, y.y);
            }
            hand_over(lane_addr + DP + part * 32, pk, &sm.ds_ready[half]);
            if (++at == ni) {                                                                   // the next head
                at = 0;
                if (F::SCORE != SCORE_PLAIN && it + 1 < n_it) so = score_of<F>(a.scale, a.x, ++h);
            }
        }
        if (alive && n_it > 0) alive = wait_warp(&sm.all_done, 0, abort_flag, err, 0x26700);        // covers dV, which was issued before dK
        tc_fence_after();
    }
    // Two CTAs that share a tile of keys: the first one finishes dv, the second one dk.  Each warp leaves its part of the other sum in the other CTA's shared memory, where its counterpart
    // there, which holds the same rows and columns, adds it to its own.
    cg::cluster_group cl = cg::this_cluster();
    constexpr int OW = D / SPLIT;
    constexpr uint32_t NAN16 = 0x7fff7fffu;                                                     // in both types: a wait ran out (keys that no query sees get zeros)
    const uint32_t sums_at = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + ((warp - 4) >> 2) * OW;
    float4* given = reinterpret_cast<float4*>(sm.q[0]) + (threadIdx.x - 128);                   // [unit of 4 columns][thread]
    if (share > 1) {
        cl.sync();                                                                              // both CTAs' products have read their tiles
        if (warp >= 4) {
            float4* theirs = cl.map_shared_rank(given, rank ^ 1);
            uint32_t v[OW];
            tmem_ld<OW>(sums_at + (rank == 0 ? DKC : DV), v);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < OW; c += 4)
                theirs[c / 4 * 512] = alive ? make_float4(__uint_as_float(v[c]), __uint_as_float(v[c + 1]), __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]))
                                            : make_float4(NAN, NAN, NAN, NAN);
        }
        cl.sync();
    }
    if (warp >= 4) {
        const int row0 = k0 + (warp & 3) * 32, col0 = ((warp - 4) >> 2) * OW, d = a.x.d;
        const long long at = (((long long)b * a.Tk + row0) * a.Hkv + hk) * d + col0;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if (share > 1 && rank != x) continue;
            uint32_t v[OW], y[OW / 2];
            tmem_ld<OW>(sums_at + (x == 0 ? DV : DKC), v);
            tmem_ld_wait();
            const float f = x == 0 ? 1.f : a.scale;
#pragma unroll
            for (int c = 0; c < OW; c += 4) {
                float4 z = make_float4(__uint_as_float(v[c]), __uint_as_float(v[c + 1]), __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
                if (share > 1) {
                    const float4 o = given[c / 4 * 512];
                    z.x += o.x; z.y += o.y; z.z += o.z; z.w += o.w;
                }
                y[c / 2] = n_it == 0 ? 0u : alive ? pack16<F>(f * z.x, f * z.y) : NAN16;
                y[c / 2 + 1] = n_it == 0 ? 0u : alive ? pack16<F>(f * z.z, f * z.w) : NAN16;
            }
            rows_out<OW>(sm.g[0] + (warp - 4) * 32 * OW * 2, y, (x == 0 ? a.dv : a.dk) + at, (long long)a.Hkv * d, min(32, a.Tk - row0), d - col0);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free_512(tmem_base);
    }
}

// delta[b,h,t] = sum_d dO[b,t,h,d] O[b,t,h,d], O with its residue.  Bound by reading the tensors once: D / 8 lanes take a row 16 bytes at a time, and a thread
// asks for its pieces of four rows before it uses the first (a warp per row with 4-byte loads had too little in flight).
template <int D, class F>
__global__ void __launch_bounds__(256) scored_delta_kernel(const bf16* __restrict__ o, const int8_t* __restrict__ low, const bf16* __restrict__ d_o,
                                                          float* __restrict__ delta, int Tq, int Hq, int d) {
    constexpr int LANES = D / 8, PER = 256 / LANES, U = 4;       // lanes of a row, rows of a block at a time
    const int l = threadIdx.x % LANES, rows = Tq * Hq;           // of a sequence: below 2^31 (64-bit divisions for every row cost more than the sums)
    const int blocks = (rows + PER * U - 1) / (PER * U), b = blockIdx.x / blocks, row0 = (blockIdx.x - b * blocks) * (PER * U) + threadIdx.x / LANES;
    uint4 x[U], y[U];
    uint2 z[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        x[u] = y[u] = make_uint4(0, 0, 0, 0), z[u] = make_uint2(0, 0);
        if (l * 8 >= d) continue;
        const long long row = (long long)b * rows + min(row0 + u * PER, rows - 1), at = row * d + l * 8;
        x[u] = *reinterpret_cast<const uint4*>(o + at);
        y[u] = *reinterpret_cast<const uint4*>(d_o + at);
        z[u] = *reinterpret_cast<const uint2*>(low + row * ((d + 15) & ~15) + l * 8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int row = row0 + u * PER;
        float s = 0.f;
        const uint32_t* xs = reinterpret_cast<const uint32_t*>(&x[u]);
        const uint32_t* ys = reinterpret_cast<const uint32_t*>(&y[u]);
        const int8_t* zs = reinterpret_cast<const int8_t*>(&z[u]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 p = unpack16<F>(xs[e]), g = unpack16<F>(ys[e]);
            s += with_residue<F>(p.x, zs[2 * e]) * g.x;
            s += with_residue<F>(p.y, zs[2 * e + 1]) * g.y;
        }
#pragma unroll
        for (int w = LANES / 2; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        if (l == 0 && row < rows) {
            const int t = row / Hq, h = row - t * Hq;
            delta[((long long)b * Hq + h) * Tq + t] = s;
        }
    }
}

// ---- launches: strides in elements (batch, token, head); 16-byte aligned bases, strides multiples of 8 ---------------------------
// Contiguous [B, T, H, d] bytes: boxes of 32 rows of D
template <int D>
static int make_map_low(CUtensorMap* map, const void* ptr, int B, int T, int H, int d) {
    EncodeTiledFn enc = get_encode();
    if (enc == nullptr) return -10;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
    const cuuint64_t strides[3] = {(cuuint64_t)d, (cuuint64_t)d * H, (cuuint64_t)d * H * T};
    const cuuint32_t box[4] = {D, 1, 32, 1}, estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : -11;
}
template <int D, class F>
static int launch_fwd(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const Args& a, cudaStream_t st) {
    const int d = a.x.d;
    CUtensorMap mq, mk, mv;
    int rc = make_map_4d(&mq, q, a.B, a.Tq, a.Hq, d, qs[0], qs[1], qs[2], BM);
    if (rc) return rc;
    rc = make_map_4d(&mk, k, a.B, a.Tk, a.Hkv, d, ks[0], ks[1], ks[2], BN);
    if (rc) return rc;
    rc = make_map_4d(&mv, v, a.B, a.Tk, a.Hkv, d, vs[0], vs[1], vs[2], 64);
    if (rc) return rc;
    CUtensorMap mo, ml;
    rc = make_map_4d(&mo, a.out, a.B, a.Tq, a.Hq, d, (long long)a.Tq * a.Hq * d, (long long)a.Hq * d, d, 32);
    if (rc) return rc;
    const int wide = (d + 15) & ~15;
    rc = a.x.low != nullptr ? make_map_low<D>(&ml, a.x.low, a.B, a.Tq, a.Hq, wide) : 0;
    if (rc) return rc;
    if (a.x.low == nullptr) ml = mo;                             // not read
    const unsigned grid = (unsigned)((a.Tq + BM - 1) / BM) * a.Hq * a.B;
    const size_t smem = sizeof(SmemFwd<D>) + 1024;
    rc = (int)cudaFuncSetAttribute(scored_fwd_kernel<D, F>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (rc) return rc;
    scored_fwd_kernel<D, F><<<grid, THREADS, smem, st>>>(mq, mk, mv, mo, ml, a, pairs_in_l2(a.B * a.Hq, a.Tk, D, a.Hq / a.Hkv));
    return (int)cudaGetLastError();
}

// CTAs that share a tile of keys: two, each with half of the query heads, where those can be halved.  Two short ones leave less of a tail than a long one, but a CTA has its fixed costs.
// Measured, 16 over 4 heads of 128, 8192 tokens, dk / dv kernel at one / two: documents of 4096 271 / 273 us, 1024 120 / 112 us, 256 60 / 75 us; of uneven lengths, 1024 on average, 169 / 145 us.
// Both passes together: documents of 700 on average 428 / 386 us, a batch with prefixes 301 / 286 us, one document of 8192 with slopes 667 / 657 us.  Four were slower than two everywhere.
static int key_share(int rep) { return rep % 2 == 0 ? 2 : 1; }

// o, d_o: contiguous [B,Tq,Hq,d]; delta: scratch [B,Hq,Tq]; writes dq, dk, dv.
template <int D, class F>
static int launch_bwd(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const void* o,
                      const void* d_o, float* delta, BwdArgs a, cudaStream_t st) {
    const int d = a.x.d;
    a.delta = delta;
    const long long gs[3] = {(long long)a.Tq * a.Hq * d, (long long)a.Hq * d, (long long)d};
    CUtensorMap mq, mqh, mg, mk, mv;
    int rc = 0;
    rc |= make_map_4d(&mq, q, a.B, a.Tq, a.Hq, d, qs[0], qs[1], qs[2], BM);
    rc |= make_map_4d(&mqh, q, a.B, a.Tq, a.Hq, d, qs[0], qs[1], qs[2], BM / 2);
    rc |= make_map_4d(&mg, d_o, a.B, a.Tq, a.Hq, d, gs[0], gs[1], gs[2], BM);
    rc |= make_map_4d(&mk, k, a.B, a.Tk, a.Hkv, d, ks[0], ks[1], ks[2], BM);
    rc |= make_map_4d(&mv, v, a.B, a.Tk, a.Hkv, d, vs[0], vs[1], vs[2], BM);
    if (rc) return -11;
    constexpr int per_block = 4 * 256 / (D / 8);
    scored_delta_kernel<D, F><<<(unsigned)((a.Tq * a.Hq + per_block - 1) / per_block) * a.B, 256, 0, st>>>((const bf16*)o, a.x.low, (const bf16*)d_o, delta, a.Tq, a.Hq, d);
    constexpr int dq_smem = sizeof(SmemDq<D>), dkv_smem = sizeof(SmemDkv<D>);
    rc = (int)cudaFuncSetAttribute(scored_dq_kernel<D, F>, cudaFuncAttributeMaxDynamicSharedMemorySize, dq_smem);
    if (rc) return rc;
    rc = (int)cudaFuncSetAttribute(scored_dkv_kernel<D, F>, cudaFuncAttributeMaxDynamicSharedMemorySize, dkv_smem);
    if (rc) return rc;
    scored_dq_kernel<D, F><<<(unsigned)((a.Tq + BM - 1) / BM) * a.Hq * a.B, THREADS, dq_smem, st>>>(
        mq, mg, mk, mv, a, pairs_in_l2(a.B * a.Hq, a.Tk, D, a.Hq / a.Hkv));
    rc = (int)cudaGetLastError();
    if (rc) return rc;
    const int rep = a.Hq / a.Hkv, share = key_share(rep);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.Tk + BM - 1) / BM) * a.Hkv * a.B * share);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = dkv_smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = share;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = share > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, scored_dkv_kernel<D, F>, mqh, mg, mk, mv, a, pairs_in_l2(a.B * a.Hkv, a.Tq, D, 1), rep / share);
    return (int)cudaGetLastError();
}

template <class F>
static int fwd_by_width(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const Args& a, cudaStream_t st) {
    return a.x.d <= 64 ? launch_fwd<64, F>(q, qs, k, ks, v, vs, a, st) : launch_fwd<128, F>(q, qs, k, ks, v, vs, a, st);
}
template <class F>
static int bwd_by_width(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const void* o, const void* d_o, float* delta,
                        const BwdArgs& a, cudaStream_t st) {
    return a.x.d <= 64 ? launch_bwd<64, F>(q, qs, k, ks, v, vs, o, d_o, delta, a, st) : launch_bwd<128, F>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
}
static bool scored_args_ok(const Ranges& x, int B, int Tq, int Tk, int Hq, int Hkv) {
    return B > 0 && Tq > 0 && Tk > 0 && Hkv > 0 && Hq % Hkv == 0 && x.d > 0 && x.d <= 128 && x.d % 8 == 0 && x.tiles != nullptr &&
           (Tq + BM - 1) / BM <= MAX_TILES && Hq < 1024;               // (below 2^30 rows of a sequence)
}
template <bool H>
static int scored_fwd(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const Args& a, cudaStream_t st) {
    if (!scored_args_ok(a.x, a.B, a.Tq, a.Tk, a.Hq, a.Hkv)) return -1;
    if (a.x.cap > 0.f) return fwd_by_width<Form<SCORE_CAP, H>>(q, qs, k, ks, v, vs, a, st);
    if (a.x.slopes != nullptr) return fwd_by_width<Form<SCORE_BIAS, H>>(q, qs, k, ks, v, vs, a, st);
    return fwd_by_width<Form<SCORE_PLAIN, H>>(q, qs, k, ks, v, vs, a, st);
}
template <bool H>
static int scored_bwd(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const void* o, const void* d_o, float* delta,
                      const BwdArgs& a, cudaStream_t st) {
    if (!scored_args_ok(a.x, a.B, a.Tq, a.Tk, a.Hq, a.Hkv) || a.x.low == nullptr) return -1;
    if (a.x.cap > 0.f) return bwd_by_width<Form<SCORE_CAP, H>>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
    if (a.x.slopes != nullptr) return bwd_by_width<Form<SCORE_BIAS, H>>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
    return bwd_by_width<Form<SCORE_PLAIN, H>>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
}

}  // namespace fatc
}  // namespace lmoe
