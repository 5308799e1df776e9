// Attention of one new token per request over a paged cache, bf16 and fp16, heads of up to 128:
//   x_j = cap tanh(scale q k_j / cap) - slope_h (n - 1 - j),   o = sum_j softmax_j(x_j) v_j   over the keys  max(0, n - window) <= j < n
// where n = lengths[b] counts the new token, whose key and value the kernel takes from k_new / v_new and stores at their place in the cache.
//
// Bound by reading the visible rows of K and V once.  The query heads of a key head share its rows: 16 of them are the M of mma.sync (fp32 FMAs would need
// 1.4 times the GPU's rate for 8 heads), so the tensor cores have four times the work that the formula asks for and are still idle for most of the time.
// A CTA of four warps takes one key head and a range of keys; a warp takes every fourth group of 16 keys and has a ring of three groups of its own that TMA fills
// (128-byte swizzle, one lane issues), so no warp waits for another one until the end.  The operands come out of the ring by ldmatrix: K as it lies, V transposed.
// Maxima lag by up to 2^8: unless a score runs ahead of that, which one vote tells, nothing is exchanged between lanes and nothing rescaled.
// Weights in bf16 have their rounding's remainder as a second operand, with up to 8 query heads in the rows of the products that no head has: it takes the output's error from 0.0024 (of 300
// keys) to that of its own rounding, 0.0017, and at most 0.3 us (1 x 300 keys 5.4 / 5.7 us, 64 x 8192 191 / 191 us).
// Rows of a group that are hidden (behind the last key, in front of the window) are masked, and their values set to zero in the ring, so that nothing stale meets a weight of zero;
// a page number outside the pool is outside the tensor map and reads as zeros.
// A NaN score raises no maximum, so what has seen nothing is told by its sum of zero, not by its maximum: a head that sees NaN gives NaN.
//
// The keys of a request are shared by up to 8 CTAs of a cluster, which join their maxima, sums and outputs in distributed shared memory; long contexts with few heads take
// more CTAs, which leave their parts in fp32 for a second launch.  (First form, cp.async into the rings by all lanes, byte permutes instead of transposing loads and always two launches:
// 766 instructions a group and 257 us at 64 requests of up to 8192 keys, 8 key heads of 128, against 190 for the bytes alone.)
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "attn_math.cuh"
#include "flash_tc_utils.cuh"
#include "mma_utils.cuh"
#include "paged_step.cuh"
#include "tanh_cap.cuh"

namespace lmoe {
namespace paged {
namespace cg = cooperative_groups;

constexpr int WARPS = 4, STAGES = 3, MAX_CLUSTER = 8;
constexpr float LOG2E = 1.4426950408889634f, LAG = 8.f;

template <bool HALF> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (HALF) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
}
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }      // zero: nothing seen
// What rounding two numbers to bf16 took away, rounded itself
__device__ __forceinline__ uint32_t rest(float x, float y, uint32_t rounded) {
    return pack2<false>(x - __uint_as_float(rounded << 16), y - __uint_as_float(rounded & 0xffff0000u));
}
template <bool HALF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// DP: head size as laid out in shared memory, 64 or 128; HR: 1 with up to 8 query heads per key head (rows 8 - 15 of the products are empty), else 2.
// The pointers are read behind pdl_wait by plain loads: the kernel may start while the one before it runs.
template <bool HALF, int DP, int HR>
__global__ void __launch_bounds__(WARPS * 32, 2) paged_step_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
    constexpr int BOXES = DP / 64, BOX = GROUP * 128, HALF_STAGE = BOXES * BOX, STAGE = 2 * HALF_STAGE;      // bytes; a box is 16 rows of 64 numbers
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[WARPS][STAGES];
    __shared__ float part_m[WARPS][16], part_l[WARPS][16], cta_m[16], cta_l[16];
    __shared__ int abort_flag, drain_flag, chosen, lens[WARPS * 32];     // lens: beside the rings, whose bulk copies no fence keeps behind ordinary accesses
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int qpg = a.H / a.G, tiles = (qpg + 8 * HR - 1) / (8 * HR);
    int b = blockIdx.z;
    const int hk = blockIdx.y / tiles, tile = blockIdx.y % tiles, split = blockIdx.x;
    const int h0 = hk * qpg + tile * 8 * HR, nh = min(8 * HR, hk * qpg + qpg - h0);
    if (threadIdx.x == 0) abort_flag = drain_flag = 0;
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) tc::mbar_init(&full[w][s], 1);
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
        for (int i = 0; i < a.B; ++i) rank += lens[i] > mine || (lens[i] == mine && i < threadIdx.x);
        if (threadIdx.x < a.B && rank == blockIdx.z) chosen = threadIdx.x;
        __syncthreads();
        b = chosen;
    }
    const Share sh = share_of(a, b);
    const int beg = sh.first + split * sh.per, end = min(sh.last, beg + sh.per);
    if (threadIdx.x == 0 && split == 0 && blockIdx.y == 0 && a.lengths[b] != sh.len) atomicCAS(a.err, 0, 0x11000);
    if (beg >= end && a.splits > MAX_CLUSTER) return;                  // (a cluster's CTAs all stay, and one of them writes zeros where there is nothing to see)

    unsigned char* ring = smem + w * STAGES * STAGE;
    const int n_mine = beg + w < end ? (end - beg - w + WARPS - 1) / WARPS : 0;              // groups beg + w, beg + w + WARPS, ...
    int pages_ahead = 0, bad = 0;                                      // a lane's page number; a bit per stage whose page is none
    auto group_page = [&](int gi) -> int { return a.table[b * a.table_ld + gi * GROUP / a.page]; };
    auto issue = [&](int j) {
        if (j >= n_mine) return;
        const int gi = beg + w + j * WARPS, st = j % STAGES;
        if ((j & 31) == 0) pages_ahead = j + lane < n_mine ? group_page(gi + lane * WARPS) : 0;
        const int page = __shfl_sync(0xffffffffu, pages_ahead, j & 31), row = gi * GROUP % a.page;
        const bool there = page >= 0 && page < a.pages;
        bad = there ? bad & ~(1 << st) : bad | 1 << st;
        if (lane == 0) {
            if (!there) atomicCAS(a.err, 0, 0x12000);
            unsigned char* at = ring + st * STAGE;
            tc::mbar_expect_tx(&full[w][st], STAGE);
#pragma unroll
            for (int c = 0; c < BOXES; ++c) fatc::tma_load_4d(at + c * BOX, &tmK, &full[w][st], c * 64, hk, row, there ? page : a.pages);
#pragma unroll
            for (int c = 0; c < BOXES; ++c) fatc::tma_load_4d(at + HALF_STAGE + c * BOX, &tmV, &full[w][st], c * 64, hk, row, there ? page : a.pages);
        }
    };
#pragma unroll
    for (int j = 0; j < STAGES - 1; ++j) issue(j);

    // the new token's row into the cache: one CTA has the group that it belongs to
    const int fresh = a.k_new != nullptr && sh.len > 0 ? sh.len - 1 : -1;
    const bf16 *kn = a.k_new + b * a.n_b + hk * a.n_h, *vn = a.v_new + b * a.m_b + hk * a.m_h;
    constexpr int UNITS = DP / 8;
    if (fresh >= 0 && tile == 0 && sh.last - 1 >= beg && sh.last - 1 < end && threadIdx.x < 2 * UNITS && threadIdx.x % UNITS * 8 < a.D) {
        const int page = group_page(fresh / GROUP), u = threadIdx.x % UNITS;
        if (page >= 0 && page < a.pages) {
            const bool val = threadIdx.x >= UNITS;
            bf16* to = val ? a.v + page * a.v_page + fresh % a.page * a.v_row + hk * a.v_head : a.k + page * a.k_page + fresh % a.page * a.k_row + hk * a.k_head;
            *reinterpret_cast<uint4*>(to + u * 8) = *reinterpret_cast<const uint4*>((val ? vn : kn) + u * 8);
        }
    }

    // queries: rows g and g + 8 of the A operand
    uint32_t qa[HR][DP / 16][2];
    float slope[HR];
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        const bool there = g + 8 * i < nh;
        const bf16* q = a.q + b * a.q_b + (h0 + g + 8 * i) * a.q_h + 2 * t;
        slope[i] = there && a.slopes != nullptr ? a.slopes[h0 + g + 8 * i] * LOG2E : 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x) qa[i][kk][x] = there && kk * 16 + 8 * x < a.D ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8 * x) : 0u;
    }
    const float pre = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E, cap = a.cap * LOG2E, unit = a.cap > 0.f ? cap : pre;
    float m[HR], l[HR], o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < HR; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 8; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;
    // ldmatrix: lane's row of 128 bytes and its 16-byte units, which lie at (unit ^ (row & 7))
    int k_at[2], v_at[4];
#pragma unroll
    for (int c = 0; c < 2; ++c) k_at[c] = (lane & 7) * 128 + (((4 * c + (lane >> 3)) ^ (lane & 7)) << 4);
#pragma unroll
    for (int c = 0; c < 4; ++c) v_at[c] = ((lane & 7) + 8 * (lane >> 3 & 1)) * 128 + (((2 * c + (lane >> 4)) ^ (lane & 7)) << 4);

    bool alive = true;
    int j = 0;
    for (; j < n_mine; ++j) {
        const int st = j % STAGES, key0 = (beg + w + j * WARPS) * GROUP;
        const bool hidden = bad >> st & 1;
        issue(j + STAGES - 1);                                         // into the stage that was read last
        alive = fatc::mbar_wait_warp(&full[w][st], j / STAGES & 1, &abort_flag, a.err, 0x14000 | st);
        if (!alive) break;
        unsigned char *K = ring + st * STAGE, *V = K + HALF_STAGE;
        const bool edge = hidden || key0 < sh.lo || key0 + GROUP > sh.len || (fresh >= key0 && fresh < key0 + GROUP);
        if (edge) {                                                    // hidden rows get values of zero, the new token's row comes from where it is
            for (int i = lane; i < GROUP * UNITS; i += 32) {
                const int r = i / UNITS, u = i % UNITS, key = key0 + r;
                const int at = u / 8 * BOX + r * 128 + ((u % 8 ^ (r & 7)) << 4);
                if (hidden || key < sh.lo || key >= sh.len) *reinterpret_cast<uint4*>(V + at) = make_uint4(0, 0, 0, 0);
                else if (key == fresh) {
                    const bool in = u * 8 < a.D;
                    *reinterpret_cast<uint4*>(K + at) = in ? *reinterpret_cast<const uint4*>(kn + u * 8) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(V + at) = in ? *reinterpret_cast<const uint4*>(vn + u * 8) : make_uint4(0, 0, 0, 0);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // ahead of the next copy into this stage
            __syncwarp();
        }
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int c = 0; c < 2 * BOXES; ++c) {
                uint32_t kb[4];
                ldsm_x4(kb, K + c / 2 * BOX + n * 1024 + k_at[c & 1]);
                mma<HALF>(s[n], qa[0][2 * c][0], HR == 2 ? qa[HR - 1][2 * c][0] : 0u, qa[0][2 * c][1], HR == 2 ? qa[HR - 1][2 * c][1] : 0u, kb[0], kb[1]);
                mma<HALF>(s[n], qa[0][2 * c + 1][0], HR == 2 ? qa[HR - 1][2 * c + 1][0] : 0u, qa[0][2 * c + 1][1], HR == 2 ? qa[HR - 1][2 * c + 1][1] : 0u, kb[2], kb[3]);
            }
        }
        auto seen = [&](int e) -> bool {
            const int key = key0 + 8 * (e >> 1) + 2 * t + (e & 1);
            return !hidden && key >= sh.lo && key < sh.len;
        };
        float x[HR][4];
        bool ahead = false;
#pragma unroll
        for (int i = 0; i < HR; ++i) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(s[e >> 1][2 * i + (e & 1)]);
            if (a.cap > 0.f) fatc::tanh_each(v, pre);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y = __uint_as_float(v[e]) * unit;
                if (a.slopes != nullptr) y -= slope[i] * (float)(sh.len - 1 - (key0 + 8 * (e >> 1) + 2 * t + (e & 1)));
                x[i][e] = y;
            }
            if (edge) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!seen(e)) x[i][e] = -INFINITY;
            }
            ahead |= fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])) > m[i] + LAG;
        }
        if (__any_sync(0xffffffffu, ahead)) {                          // the first visible keys too
            float corr[HR];
#pragma unroll
            for (int i = 0; i < HR; ++i) {
                float mx = fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                mx = fmaxf(mx, m[i]);
                corr[i] = m[i] == -INFINITY ? 1.f : ex2(m[i] - mx);    // nothing has been summed up in front of the first one
                m[i] = mx;
                l[i] *= corr[i];
            }
#pragma unroll
            for (int e = 0; e < DP / 8; ++e) {
                o[e][0] *= corr[0]; o[e][1] *= corr[0];
                o[e][2] *= corr[HR - 1]; o[e][3] *= corr[HR - 1];
            }
        }
        uint32_t p[2][2] = {{0, 0}, {0, 0}}, low[2][2];                // [rows g, g + 8][keys 2 t, 2 t + 8]; low: what their rounding took away
#pragma unroll
        for (int i = 0; i < HR; ++i) {
            const float base = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = ex2(x[i][e] - base);
            l[i] += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
            p[i][0] = pack2<HALF>(x[i][0], x[i][1]);
            p[i][1] = pack2<HALF>(x[i][2], x[i][3]);
            if constexpr (!HALF) low[i][0] = rest(x[i][0], x[i][1], p[i][0]), low[i][1] = rest(x[i][2], x[i][3], p[i][1]);
        }
        if constexpr (!HALF && HR == 1) p[1][0] = low[0][0], p[1][1] = low[0][1];       // in the rows that no head has
#pragma unroll
        for (int c = 0; c < 4 * BOXES; ++c) {
            uint32_t vb[4];
            ldsm_x4_t(vb, V + c / 4 * BOX + v_at[c & 3]);
            mma<HALF>(o[2 * c], p[0][0], p[1][0], p[0][1], p[1][1], vb[0], vb[1]);
            mma<HALF>(o[2 * c + 1], p[0][0], p[1][0], p[0][1], p[1][1], vb[2], vb[3]);
            if constexpr (!HALF && HR == 2) {
                mma<HALF>(o[2 * c], low[0][0], low[1][0], low[0][1], low[1][1], vb[0], vb[1]);
                mma<HALF>(o[2 * c + 1], low[0][0], low[1][0], low[0][1], low[1][1], vb[2], vb[3]);
            }
        }
        __syncwarp();                                                  // the stage is read; the next issue() fills it
    }
    if (!alive)                                                        // after a wait that ran out: copies in flight, again within a limit
        for (int i = j; i < min(j + STAGES, n_mine); ++i) fatc::mbar_wait_suspend(&full[w][i % STAGES], i / STAGES & 1, &drain_flag, a.err, 0x14010);

    // the warps' parts meet in shared memory
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) part_m[w][g + 8 * i] = m[i], part_l[w][g + 8 * i] = l[i];
    }
    __syncthreads();
    constexpr int LD = DP + 4;
    float* O = reinterpret_cast<float*>(smem);                         // [WARPS][8 HR][LD], over the rings
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        float top = part_m[0][g + 8 * i];
#pragma unroll
        for (int y = 1; y < WARPS; ++y) top = fmaxf(top, part_m[y][g + 8 * i]);
        const float f = m[i] == -INFINITY ? 0.f : ex2(m[i] - top);
#pragma unroll
        for (int e = 0; e < DP / 8; ++e)
            *reinterpret_cast<float2*>(O + (w * 8 * HR + g + 8 * i) * LD + e * 8 + 2 * t) =
                !HALF && HR == 1 ? make_float2(f * (o[e][0] + o[e][2]), f * (o[e][1] + o[e][3])) : make_float2(f * o[e][2 * i], f * o[e][2 * i + 1]);
    }
    if (threadIdx.x < 8 * HR) {
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
    for (int i = threadIdx.x; i < nh * (DP / 4); i += WARPS * 32) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        float4 y = load4(O + r * LD + d);
#pragma unroll
        for (int c = 1; c < WARPS; ++c) {
            const float4 z = load4(O + (c * 8 * HR + r) * LD + d);
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        const long long bh = (long long)b * a.H + h0 + r;
        if (cluster) store4(O + r * LD + d, y);
        else if (d >= a.D) continue;
        else if (a.splits == 1) {
            const float inv = inverse(cta_l[r]);
            *reinterpret_cast<uint2*>(a.out + bh * a.D + d) = make_uint2(pack2<HALF>(y.x * inv, y.y * inv), pack2<HALF>(y.z * inv, y.w * inv));
        } else {
            store4(a.part + (bh * a.splits + split) * a.D + d, y);
            if (d == 0) *reinterpret_cast<float2*>(a.ml + (bh * a.splits + split) * 2) = make_float2(cta_m[r], cta_l[r]);
        }
    }
    if (!cluster) return;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (int i = split * WARPS * 32 + threadIdx.x; i < nh * (DP / 4); i += a.splits * WARPS * 32) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        if (d >= a.D) continue;
        float ms[MAX_CLUSTER], ls[MAX_CLUSTER], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
            ms[c] = c < a.splits ? *cl.map_shared_rank(&cta_m[r], c) : -INFINITY;
            ls[c] = c < a.splits ? *cl.map_shared_rank(&cta_l[r], c) : 0.f;
            top = fmaxf(top, ms[c]);
        }
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
            if (ls[c] == 0.f) continue;
            const float f = ex2(ms[c] - top);
            const float4 z = load4(cl.map_shared_rank(O + r * LD + d, c));
            sum += f * ls[c];
            y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
        }
        const float inv = inverse(sum);
        *reinterpret_cast<uint2*>(a.out + ((long long)b * a.H + h0 + r) * a.D + d) = make_uint2(pack2<HALF>(y.x * inv, y.y * inv), pack2<HALF>(y.z * inv, y.w * inv));
    }
    cl.sync();                                                         // the other CTAs have read this one's part
}

// The parts of a request's CTAs: a block per (request, query head), a warp per part, a lane per four numbers.
constexpr int JOIN_WARPS = 8;
template <bool HALF>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(Args a) {
    __shared__ float4 O[JOIN_WARPS][32];
    __shared__ float L[JOIN_WARPS];
    pdl_wait();
    const int bh = blockIdx.x, b = bh / a.H, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Share sh = share_of(a, b);
    const int n = (sh.last - sh.first + sh.per - 1) / sh.per;
    const float* ml = a.ml + (long long)bh * a.splits * 2;
    const float* part = a.part + (long long)bh * a.splits * a.D + lane * 4;
    const bool mine = lane * 4 < a.D;
    float top = -INFINITY;                                             // of all parts, first: then no part waits for the one before it
    for (int s = lane; s < n; s += 32) top = fmaxf(top, ml[2 * s]);
    top = warp_max(top);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = w; s < n; s += JOIN_WARPS) {
        const float2 x = *reinterpret_cast<const float2*>(ml + 2 * s);
        const float4 y = mine ? load4(part + (long long)s * a.D) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float f = x.x == -INFINITY ? 0.f : ex2(x.x - top);
        l += x.y * f;
        o.x += y.x * f; o.y += y.y * f; o.z += y.z * f; o.w += y.w * f;
    }
    O[w][lane] = o;
    if (lane == 0) L[w] = l;
    __syncthreads();
    if (w > 0) return;
    float sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < JOIN_WARPS; ++x) {
        const float4 y = O[x][lane];
        sum += L[x];
        o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
    }
    const float inv = inverse(sum);
    if (mine) *reinterpret_cast<uint2*>(a.out + (long long)bh * a.D + lane * 4) = make_uint2(pack2<HALF>(o.x * inv, o.y * inv), pack2<HALF>(o.z * inv, o.w * inv));
}

template <bool HALF, int DP, int HR>
static int launch(const Args& a, cudaStream_t st) {
    constexpr int smem = WARPS * STAGES * 2 * GROUP * DP * 2 + 1024;
    static_assert(smem - 1024 >= WARPS * 8 * HR * (DP + 4) * 4, "the warps' outputs over the rings");
    CUtensorMap mk, mv;
    int rc = fatc::make_map_4d(&mk, a.k, a.pages, a.page, a.G, a.D, a.k_page, a.k_row, a.k_head, GROUP);
    if (rc) return rc;
    rc = fatc::make_map_4d(&mv, a.v, a.pages, a.page, a.G, a.D, a.v_page, a.v_row, a.v_head, GROUP);
    if (rc) return rc;
    rc = (int)cudaFuncSetAttribute(paged_step_kernel<HALF, DP, HR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc) return rc;
    const int tiles = (a.H / a.G + 8 * HR - 1) / (8 * HR);
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
    cudaLaunchKernelEx(&cfg, paged_step_kernel<HALF, DP, HR>, mk, mv, a);
    rc = (int)cudaGetLastError();
    if (rc || a.splits <= MAX_CLUSTER) return rc;
    return launch_early(paged_join_kernel<HALF>, (int64_t)a.B * a.H, JOIN_WARPS * 32, st, a);
}
template <bool HALF, int DP>
static int by_heads(const Args& a, cudaStream_t st) { return a.H / a.G <= 8 ? launch<HALF, DP, 1>(a, st) : launch<HALF, DP, 2>(a, st); }

}  // namespace paged
}  // namespace lmoe

// half: fp16, else bf16.  All strides in elements, positive multiples of 8; bases 16-byte aligned; D a multiple of 8 up to 128; page a multiple of 16.
LMOE_API int lmoe_paged_step(const lmoe::paged::Args* ap, int half, cudaStream_t st) {
    using namespace lmoe::paged;
    const Args& a = *ap;
    if (a.B <= 0 || a.B > 65535 || a.G <= 0 || a.H % a.G != 0 || a.D <= 0 || a.D > 128 || a.D % 8 != 0 || a.page <= 0 || a.page % GROUP != 0 || a.pages <= 0 ||
        a.splits < 1 || (a.sorted && a.B > WARPS * 32) || a.table_n < 0 || (long long)a.table_n * a.page > 0x7fffffff - GROUP || (long long)a.G * ((a.H / a.G + 7) / 8) > 65535 ||
        (a.splits > MAX_CLUSTER && (a.part == nullptr || a.ml == nullptr))) return -1;
    if (half) return a.D <= 64 ? by_heads<true, 64>(a, st) : by_heads<true, 128>(a, st);
    return a.D <= 64 ? by_heads<false, 64>(a, st) : by_heads<false, 128>(a, st);
}
