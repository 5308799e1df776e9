// Attention of one new token per request over a paged cache, bf16 and fp16, heads of up to 128:
//   x_j = cap tanh(scale q k_j / cap) - slope_h (n - 1 - j),   o = sum_j softmax_j(x_j) v_j   over the keys  max(0, n - window) <= j < n
// where n = lengths[b] counts the new token, whose key and value the kernel takes from k_new / v_new and stores at their place in the cache.
//
// Bound by reading the visible rows of K and V once.  The query heads of a key head share its rows: 16 of them are the M of mma.sync (fp32 FMAs would need
// 1.4 times the GPU's rate for 8 heads), so the tensor cores have four times the work that the formula asks for and are still idle for most of the time.
// A CTA of four warps takes one key head and a range of keys; a warp takes every fourth group of 16 keys and has a ring of its own that cp.async
// fills, so no warp waits for another one until the end.  Both operands come out of shared memory by 16-byte reads without ldmatrix:
//   S = Q K^T     the order of the head dimension inside a product is free: thread t of a quad holds the 8 numbers 32 c + 8 t ..., of its query and of its key
//   O += P V      so is the order of the columns: column g of product e is number 64 c + 8 g + e; pairs of keys are put together by byte permutes
// The units of 16 bytes lie at (unit ^ 4 (row & 1)) for K and (unit ^ 2 (row / 2 & 3)) for V, which keeps both reads free of bank conflicts.
// Maxima lag by up to 2^8 as in the prompt kernel, so rescaling is rare.  Long contexts are split over CTAs that leave their maximum, sum and output in
// fp32; a second launch joins them.  Hidden rows of a group (behind the last key, in front of the window, on a page that is none) are filled with zeros instead of being
// read, so nothing stale reaches a product.
#include <cuda_fp16.h>

#include "attn_math.cuh"
#include "mma_utils.cuh"
#include "paged_step.cuh"

namespace lmoe {
namespace paged {

constexpr int WARPS = 4, STAGES = 3;
constexpr float LOG2E = 1.4426950408889634f, LAG = 8.f;

template <bool HALF> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (HALF) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
}
template <bool HALF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// DP: head size as laid out in shared memory, 64 or 128; HR: 1 with up to 8 query heads per key head (rows 8 - 15 of the products are empty), else 2
template <bool HALF, int DP, int HR>
__global__ void __launch_bounds__(WARPS * 32, 2) paged_step_kernel(const Args a) {
    constexpr int UNITS = DP / 8, STAGE = 2 * GROUP * DP * 2, NC = DP / 32, NV = DP / 64;      // units of 16 bytes in a row; bytes of a stage
    constexpr int RI = 32 / UNITS;                                     // rows that a warp fills with one cp.async
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float part_m[WARPS][16], part_l[WARPS][16];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int qpg = a.H / a.G, tiles = (qpg + 8 * HR - 1) / (8 * HR);
    const int b = blockIdx.z, hk = blockIdx.y / tiles, tile = blockIdx.y % tiles, split = blockIdx.x;
    const int h0 = hk * qpg + tile * 8 * HR, nh = min(8 * HR, hk * qpg + qpg - h0);
    const Share sh = share_of(a, b);
    const int beg = sh.first + split * sh.per, end = min(sh.last, beg + sh.per);
    if (threadIdx.x == 0 && split == 0 && blockIdx.y == 0 && __ldg(a.lengths + b) != sh.len) atomicCAS(a.err, 0, 0xb100);
    if (beg >= end && a.splits > 1) return;                            // (one CTA per request writes zeros where there is nothing to see)

    unsigned char* ring = smem + w * STAGES * STAGE;
    const int n_mine = beg + w < end ? (end - beg - w + WARPS - 1) / WARPS : 0;              // groups beg + w, beg + w + WARPS, ...
    const int u = lane % UNITS, r0 = lane / UNITS;
    int pages_ahead = 0, bad = 0;                                      // a lane's page number; a bit per stage whose page is none
    auto group_page = [&](int gi) -> int { return __ldg(a.table + b * a.table_ld + gi * GROUP / a.page); };
    auto issue = [&](int j) {
        if (j < n_mine) {
            const int gi = beg + w + j * WARPS;
            if ((j & 31) == 0) pages_ahead = j + lane < n_mine ? group_page(gi + lane * WARPS) : 0;
            const int page = __shfl_sync(0xffffffffu, pages_ahead, j & 31), st = j % STAGES;
            const bool there = page >= 0 && page < a.pages;
            if (there) bad &= ~(1 << st);
            else {
                bad |= 1 << st;
                if (lane == 0) atomicCAS(a.err, 0, 0xb200);
            }
            const int row = gi * GROUP % a.page;
            const bf16* kp = a.k + (long long)page * a.k_page + row * a.k_row + hk * a.k_head + u * 8;
            const bf16* vp = a.v + (long long)page * a.v_page + row * a.v_row + hk * a.v_head + u * 8;
            unsigned char* at = ring + st * STAGE;
#pragma unroll
            for (int i = 0; i < GROUP / RI; ++i) {
                const int r = r0 + i * RI, key = gi * GROUP + r;
                const bool fill = there && key >= sh.lo && key < sh.len && u * 8 < a.D, fresh = a.k_new != nullptr && key == sh.len - 1;
                const bf16* ks = fresh ? a.k_new + b * a.n_b + hk * a.n_h + u * 8 : kp + r * a.k_row;
                const bf16* vs = fresh ? a.v_new + b * a.m_b + hk * a.m_h + u * 8 : vp + r * a.v_row;
                cp_async16(at + r * DP * 2 + ((u ^ ((r & 1) << 2)) << 4), fill ? ks : a.q, fill);
                cp_async16(at + (GROUP + r) * DP * 2 + ((u ^ ((r >> 1 & 3) << 1)) << 4), fill ? vs : a.q, fill);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < STAGES - 1; ++j) issue(j);

    // the new token's row into the cache: one CTA has the group that it belongs to
    if (a.k_new != nullptr && tile == 0 && sh.len > 0 && sh.last - 1 >= beg && sh.last - 1 < end && threadIdx.x < 2 * UNITS && u * 8 < a.D) {
        const int key = sh.len - 1, page = group_page(key / GROUP);
        const bool val = threadIdx.x >= UNITS;
        if (page >= 0 && page < a.pages) {
            const bf16* from = val ? a.v_new + b * a.m_b + hk * a.m_h : a.k_new + b * a.n_b + hk * a.n_h;
            bf16* to = val ? a.v + page * a.v_page + key % a.page * a.v_row + hk * a.v_head : a.k + page * a.k_page + key % a.page * a.k_row + hk * a.k_head;
            *reinterpret_cast<uint4*>(to + u * 8) = *reinterpret_cast<const uint4*>(from + u * 8);
        }
    }

    // queries: rows g and g + 8 of the A operand, in the order of the head dimension that the keys are read in
    uint4 qa[HR][NC];
    float slope[HR];
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        const bool there = g + 8 * i < nh;
        slope[i] = there && a.slopes != nullptr ? __ldg(a.slopes + h0 + g + 8 * i) * LOG2E : 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            qa[i][c] = there && c * 32 + t * 8 < a.D ? __ldg(reinterpret_cast<const uint4*>(a.q + b * a.q_b + (h0 + g + 8 * i) * a.q_h + c * 32 + t * 8))
                                                     : make_uint4(0, 0, 0, 0);
    }
    const float pre = a.cap > 0.f ? a.scale / a.cap * 2.f * LOG2E : a.scale * LOG2E, cap = a.cap * LOG2E;
    float m[HR], l[HR], o[8 * NV][4];
#pragma unroll
    for (int i = 0; i < HR; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 8 * NV; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;

    for (int j = 0; j < n_mine; ++j) {
        const int gi = beg + w + j * WARPS, st = j % STAGES, key0 = gi * GROUP;
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        const bool hidden = bad >> st & 1;                             // before issue() may set it for the stage's next group
        issue(j + STAGES - 1);
        const unsigned char* K = ring + st * STAGE;
        const unsigned char* V = K + GROUP * DP * 2;
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
            const int r = 8 * n + g;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const uint4 kb = *reinterpret_cast<const uint4*>(K + r * DP * 2 + (((c * 4 + t) ^ ((r & 1) << 2)) << 4));
                const uint4 q0 = qa[0][c], q1 = HR == 2 ? qa[HR - 1][c] : make_uint4(0, 0, 0, 0);
                mma<HALF>(s[n], q0.x, q1.x, q0.y, q1.y, kb.x, kb.y);
                mma<HALF>(s[n], q0.z, q1.z, q0.w, q1.w, kb.z, kb.w);
            }
        }
        uint32_t p[2][2] = {{0, 0}, {0, 0}};                           // [rows g, g + 8][keys 2 t, 2 t + 8]
        float corr[HR];
        bool rescale = false;
#pragma unroll
        for (int i = 0; i < HR; ++i) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = key0 + 8 * (e >> 1) + 2 * t + (e & 1);
                float y = s[e >> 1][2 * i + (e & 1)] * pre;
                if (a.cap > 0.f) y = cap * (1.f - 2.f * rcp(ex2(y) + 1.f));
                y -= slope[i] * (float)(sh.len - 1 - key);
                x[e] = hidden || key < sh.lo || key >= sh.len ? -INFINITY : y;
            }
            float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const bool grow = mx > m[i] + LAG;                         // the first visible key too
            corr[i] = grow && m[i] != -INFINITY ? ex2(m[i] - mx) : 1.f;
            rescale |= corr[i] != 1.f;
            if (grow) m[i] = mx;
            const float base = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = ex2(x[e] - base);
            l[i] = l[i] * corr[i] + ((x[0] + x[1]) + (x[2] + x[3]));
            p[i][0] = pack2<HALF>(x[0], x[1]);
            p[i][1] = pack2<HALF>(x[2], x[3]);
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int e = 0; e < 8 * NV; ++e) {
                o[e][0] *= corr[0]; o[e][1] *= corr[0];
                o[e][2] *= corr[HR - 1]; o[e][3] *= corr[HR - 1];
            }
        }
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {                              // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
                const int r = 2 * t + (i & 1) + 8 * (i >> 1);
                v[i] = *reinterpret_cast<const uint4*>(V + r * DP * 2 + (((c * 8 + g) ^ ((r >> 1 & 3) << 1)) << 4));
            }
            const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&v[0]);
            const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&v[1]);
            const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&v[2]);
            const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&v[3]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t pick = e & 1 ? 0x7632 : 0x5410;
                mma<HALF>(o[c * 8 + e], p[0][0], p[1][0], p[0][1], p[1][1], __byte_perm(v0[e >> 1], v1[e >> 1], pick), __byte_perm(v2[e >> 1], v3[e >> 1], pick));
            }
        }
        __syncwarp();                                                  // the stage is read; the next issue() may fill it
    }
    cp_async_wait<0>();
    pdl_trigger();

    // the warps' parts meet in shared memory
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) part_m[w][g + 8 * i] = m[i], part_l[w][g + 8 * i] = l[i];
    }
    __syncthreads();
    float* O = reinterpret_cast<float*>(smem);                         // [WARPS][8 HR][DP], over the rings
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        float top = part_m[0][g + 8 * i];
#pragma unroll
        for (int x = 1; x < WARPS; ++x) top = fmaxf(top, part_m[x][g + 8 * i]);
        const float f = m[i] == -INFINITY ? 0.f : ex2(m[i] - top);
#pragma unroll
        for (int e = 0; e < 8 * NV; ++e) {
            float* row = O + (w * 8 * HR + g + 8 * i) * DP + (e >> 3) * 64 + (e & 7);
            row[2 * t * 8] = f * o[e][2 * i];
            row[(2 * t + 1) * 8] = f * o[e][2 * i + 1];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * (DP / 4); i += WARPS * 32) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        if (d >= a.D) continue;
        float top = part_m[0][r], sum = 0.f;
#pragma unroll
        for (int x = 1; x < WARPS; ++x) top = fmaxf(top, part_m[x][r]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < WARPS; ++x) {
            const float4 z = load4(O + (x * 8 * HR + r) * DP + d);
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            sum += part_m[x][r] == -INFINITY ? 0.f : part_l[x][r] * ex2(part_m[x][r] - top);
        }
        const long long bh = (long long)b * a.H + h0 + r;
        if (a.splits == 1) {
            const float inv = sum > 0.f ? 1.f / sum : 0.f;
            *reinterpret_cast<uint2*>(a.out + bh * a.D + d) = make_uint2(pack2<HALF>(y.x * inv, y.y * inv), pack2<HALF>(y.z * inv, y.w * inv));
        } else {
            store4(a.part + (bh * a.splits + split) * a.D + d, y);
            if (d == 0) *reinterpret_cast<float2*>(a.ml + (bh * a.splits + split) * 2) = make_float2(top, sum);
        }
    }
}

// The parts of a request's CTAs: a block per (request, query head), a warp per part, a lane per four numbers.
constexpr int JOIN_WARPS = 8;
template <bool HALF>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(Args a) {
    __shared__ float4 O[JOIN_WARPS][32];
    __shared__ float M[JOIN_WARPS], L[JOIN_WARPS];
    pdl_wait();
    const int bh = blockIdx.x, b = bh / a.H, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Share sh = share_of(a, b);
    const int n = (sh.last - sh.first + sh.per - 1) / sh.per;
    const float* ml = a.ml + (long long)bh * a.splits * 2;
    const float* part = a.part + (long long)bh * a.splits * a.D + lane * 4;
    const bool mine = lane * 4 < a.D;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = w; s < n; s += JOIN_WARPS) {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(ml + 2 * s));
        const float4 y = mine ? __ldcg(reinterpret_cast<const float4*>(part + (long long)s * a.D)) : o;
        const float top = fmaxf(m, x.x);
        if (top == -INFINITY) continue;
        const float f = ex2(m - top), z = ex2(x.x - top);
        m = top;
        l = l * f + x.y * z;
        o.x = o.x * f + y.x * z; o.y = o.y * f + y.y * z; o.z = o.z * f + y.z * z; o.w = o.w * f + y.w * z;
    }
    O[w][lane] = o;
    if (lane == 0) M[w] = m, L[w] = l;
    __syncthreads();
    if (w > 0) return;
    float top = M[0];
#pragma unroll
    for (int x = 1; x < JOIN_WARPS; ++x) top = fmaxf(top, M[x]);
    float sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < JOIN_WARPS; ++x) {
        const float f = M[x] == -INFINITY ? 0.f : ex2(M[x] - top);
        const float4 y = O[x][lane];
        sum += f * L[x];
        o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    if (mine) *reinterpret_cast<uint2*>(a.out + (long long)bh * a.D + lane * 4) = make_uint2(pack2<HALF>(o.x * inv, o.y * inv), pack2<HALF>(o.z * inv, o.w * inv));
}

template <bool HALF, int DP, int HR>
static int launch(const Args& a, cudaStream_t st) {
    constexpr int smem = WARPS * STAGES * 2 * GROUP * DP * 2;
    static_assert(smem >= WARPS * 8 * HR * DP * 4, "the warps' outputs over the rings");
    int rc = (int)cudaFuncSetAttribute(paged_step_kernel<HALF, DP, HR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc) return rc;
    const int tiles = (a.H / a.G + 8 * HR - 1) / (8 * HR);
    paged_step_kernel<HALF, DP, HR><<<dim3(a.splits, a.G * tiles, a.B), WARPS * 32, smem, st>>>(a);
    rc = (int)cudaGetLastError();
    if (rc || a.splits == 1) return rc;
    return launch_early(paged_join_kernel<HALF>, (int64_t)a.B * a.H, JOIN_WARPS * 32, st, a);
}
template <bool HALF, int DP>
static int by_heads(const Args& a, cudaStream_t st) { return a.H / a.G <= 8 ? launch<HALF, DP, 1>(a, st) : launch<HALF, DP, 2>(a, st); }

}  // namespace paged
}  // namespace lmoe

// half: fp16, else bf16.  All strides in elements, multiples of 8; bases 16-byte aligned; D a multiple of 8 up to 128; page a multiple of 16.
LMOE_API int lmoe_paged_step(const lmoe::paged::Args* ap, int half, cudaStream_t st) {
    using namespace lmoe::paged;
    const Args& a = *ap;
    if (a.B <= 0 || a.B > 65535 || a.G <= 0 || a.H % a.G != 0 || a.D <= 0 || a.D > 128 || a.D % 8 != 0 || a.page <= 0 || a.page % GROUP != 0 || a.splits < 1 ||
        a.table_n < 0 || (long long)a.table_n * a.page > 0x7fffffff - GROUP || (long long)a.G * ((a.H / a.G + 7) / 8) > 65535 ||
        (a.splits > 1 && (a.part == nullptr || a.ml == nullptr))) return -1;
    if (half) return a.D <= 64 ? by_heads<true, 64>(a, st) : by_heads<true, 128>(a, st);
    return a.D <= 64 ? by_heads<false, 64>(a, st) : by_heads<false, 128>(a, st);
}
