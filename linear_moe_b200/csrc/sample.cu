// The next token of every request out of its logits and one random number:
//   w_i = exp((x_i - max) / temperature);  tokens in the order of falling logits, equal ones by their number; a token is kept while fewer than k come before it, what comes before it is below p of the
//   whole, and w_i >= min_p;  the token drawn is the first one, in the order of their numbers, up to which the kept weights exceed u times their sum.
//
// Sums of floating-point weights depend on their order, and so would the token next to a border.  So a weight is a whole number, 2^44 w rounded, from an exponential in 64 bits (a table of 32 powers of two
// and a polynomial of degree 5 behind it, good to 2^-47; Tang, "Table-driven implementation of the exponential function", 1989), and all sums are exact: the same token however a row is shared out.
//
// A row is one cluster's: each CTA reads its part of the logits once and keeps it in shared memory where that holds it.  Then, if anything is cut off: a histogram over the weights' logarithms (16 bins
// for a factor of two) with the number and the weight of each bin's tokens tells the bin in which the cut lies; histograms over the numbers inside of it tell the logit, and the equal ones are counted
// by their numbers.  Last, the kept weights are summed up per thread, and a scan finds the thread, and the token, that the random number falls to.
//
// One row of 32000 logits 16 us, 17 rows of 50257 with settings of their own 24, 128 rows of 128256 in fp32 with top-p 165 (the logits alone take 10 at the copy rate).  Of the 60000
// cycles of such a row's CTAs (four waves of two per SM) 8000 to 13000 are the loads, 9000 the exponentials of the histogram (some 60 instructions each), 6000 its atomics, 2000 what is kept (without a cut, where all of it is: 10000), and
// about half are barriers of the cluster, five or six of them with what lies between, and the searches over bins.  The first form, a CTA per 65536 logits with branches around its
// exponentials, took 68, 96 and 273.  CTAs of 768 threads, which leaves 40 registers and spills, take 22, 31 and 182 where 512 threads take 18, 27 and 162 (replayed from a graph).
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "common.cuh"

namespace lmoe {
namespace sample {
namespace cg = cooperative_groups;

struct Args {
    const void* logits;                                // [B, V], rows of `ld`
    const float* draw;                                 // [B]
    const float *temperature, *top_p, *min_p;          // [B] or null: the one below for all
    const int* top_k;
    long long* token;                                  // [B]
    float* logp;                                       // [B]
    long long ld;
    int B, V, parts, len;                              // CTAs of a row, logits of each
    int k;
    float t, p, least;
};

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 768, PER_OCTAVE = 16, MAX_PARTS = 8, SUB_BITS = 9;
constexpr int BITS = 44;                               // of a weight of one: 2^19 of them stay below 2^63
typedef unsigned long long u64;

// Logits go as whole numbers of their own width, in the logits' order: NaN is minus infinity, zeros are equal.
template <typename T> struct Key { typedef uint16_t N; static constexpr uint32_t SIGN = 0x8000u, ONES = 0xffffu; };
template <> struct Key<float> { typedef uint32_t N; static constexpr uint32_t SIGN = 0x80000000u, ONES = 0xffffffffu; };
template <typename T> __device__ __forceinline__ uint32_t infinity();
template <> __device__ __forceinline__ uint32_t infinity<float>() { return 0x7f800000u; }
template <> __device__ __forceinline__ uint32_t infinity<bf16>() { return 0x7f80u; }
template <> __device__ __forceinline__ uint32_t infinity<__half>() { return 0x7c00u; }
template <typename T> __device__ __forceinline__ uint32_t lowest() { return Key<T>::ONES ^ (Key<T>::SIGN | infinity<T>()); }      // minus infinity's
template <typename T> __device__ __forceinline__ uint32_t key_of_bits(uint32_t b) {
    const uint32_t size = b & ~Key<T>::SIGN, key = size == 0 ? Key<T>::SIGN : b & Key<T>::SIGN ? b ^ Key<T>::ONES : b | Key<T>::SIGN;
    return size > infinity<T>() ? lowest<T>() : key;
}
template <typename T> __device__ __forceinline__ float value_of(uint32_t key) {
    const uint32_t b = key & Key<T>::SIGN ? key ^ Key<T>::SIGN : key ^ Key<T>::ONES;
    if constexpr (sizeof(T) == 4) return __uint_as_float(b);
    else if constexpr (std::is_same<T, bf16>::value) return __uint_as_float(b << 16);
    else return __half2float(__ushort_as_half((unsigned short)b));
}
// The key at or below a number in 32 bits, and at or above it
template <typename T> __device__ __forceinline__ uint32_t key_down(float x) {
    if constexpr (sizeof(T) == 4) return key_of_bits<T>(__float_as_uint(x));
    else if constexpr (std::is_same<T, bf16>::value) return key_of_bits<T>(__bfloat16_as_ushort(__float2bfloat16_rd(x)));
    else return key_of_bits<T>(__half_as_ushort(__float2half_rd(x)));
}
template <typename T> __device__ __forceinline__ uint32_t key_up(float x) {
    if constexpr (sizeof(T) == 4) return key_of_bits<T>(__float_as_uint(x));
    else if constexpr (std::is_same<T, bf16>::value) return key_of_bits<T>(__bfloat16_as_ushort(__float2bfloat16_ru(x)));
    else return key_of_bits<T>(__half_as_ushort(__float2half_ru(x)));
}

// 2^(i / 32)
__constant__ double POWERS[32] = {1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951,
    1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965, 1.681792830507429, 1.718619298122478,
    1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};

struct Scale { uint32_t top; double max, c; };         // the largest logit, log2(e) / temperature
// 2^44 exp((x - max) / temperature), rounded, and its bin.  (No branches, so that several go on side by side: with them a pass over 16000 logits took 28000 cycles.)
template <typename T> __device__ __forceinline__ u64 weight(uint32_t key, const Scale& s, const double* powers, int& bin) {
    double y = ((double)value_of<T>(key) - s.max) * s.c;
    y = key == lowest<T>() ? -64.0 : key == s.top ? 0.0 : fmax(y, -64.0);      // (infinities, whose differences and products may be NaN)
    const double magic = 6755399441055744.0;           // 1.5 2^52: what is added to it is rounded to a whole number in its lower bits
    const double shifted = fma(y, 32.0, magic);
    const int n = (int)__double_as_longlong(shifted);
    const double f = fma(shifted - magic, -0.03125, y) * 0.6931471805599453;      // up to ln 2 / 64
    const double e = fma(f, fma(f, fma(f, fma(f, fma(f, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0);
    const double power = __longlong_as_double(__double_as_longlong(powers[n & 31]) + ((long long)(BITS + (n >> 5)) << 52));
    bin = min(-n >> 1, BINS - 1);
    return (u64)(__double_as_longlong(fma(power, e, magic)) - 0x4338000000000000ll);
}
template <typename T> __device__ __forceinline__ u64 weight(uint32_t key, const Scale& s, const double* powers) {
    int bin;
    return weight<T>(key, s, powers, bin);
}

struct Bins { uint32_t count[BINS], part[3][BINS]; };  // weights in three parts of 15 bits, whose sums over a CTA's logits 32 bits hold
__device__ __forceinline__ u64 mass_of(const Bins& h, int bin) { return (u64)h.part[0][bin] + ((u64)h.part[1][bin] << 15) + ((u64)h.part[2][bin] << 30); }
constexpr int COARSE = BINS / 32;
static_assert(COARSE <= 32, "a lane for 32 bins");
struct Shared {
    Bins bins[2];
    // of 32 bins together, read by the others, who may still be at it when this CTA has gone on to its next level: two sets in turn, as of the bins
    u64 coarse_mass[2][COARSE], all_mass[MAX_PARTS][32];
    uint32_t coarse_count[2][COARSE], all_count[MAX_PARTS][32];
    double powers[32];
    uint32_t count[WARPS];
    u64 mass[WARPS];
    uint32_t top;                                      // this CTA's, read by the others
    u64 above[WARPS];                                  // per warp: weight of the tokens above the edge, and how many lie on it
    uint32_t on_edge[WARPS];
    int found, chosen;
    uint32_t at_count, total_count;
    u64 at_mass, total_mass;
    uint32_t tied;                                     // of the chosen warp: tokens on the edge, and weight, ahead of it
    u64 ahead;
};

__device__ __forceinline__ u64 up_to(u64 v) {          // inclusive over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += x;
    }
    return v;
}
__device__ __forceinline__ uint32_t up_to(uint32_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += x;
    }
    return v;
}
// What comes before this thread, and in all; a barrier at the beginning and one inside.
template <typename N> __device__ __forceinline__ N before(N v, N* warps, N& all) {
    const N in = up_to(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 31) warps[threadIdx.x >> 5] = in;
    __syncthreads();
    N sum = 0, ahead = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const N x = warps[w];
        if (w < (int)(threadIdx.x >> 5)) ahead += x;
        sum += x;
    }
    all = sum;
    return ahead + in - v;
}

// Keys of four neighbours in shared memory, or out of the logits (aligned, or some of them)
__device__ __forceinline__ void four_keys(const uint32_t* p, uint32_t (&k)[4]) { const uint4 y = *reinterpret_cast<const uint4*>(p); k[0] = y.x, k[1] = y.y, k[2] = y.z, k[3] = y.w; }
__device__ __forceinline__ void four_keys(const uint16_t* p, uint32_t (&k)[4]) {
    const uint2 y = *reinterpret_cast<const uint2*>(p);
    k[0] = y.x & 0xffffu, k[1] = y.x >> 16, k[2] = y.y & 0xffffu, k[3] = y.y >> 16;
}

template <typename T, bool HELD>                       // HELD: the part of a row lies in shared memory
__global__ void __launch_bounds__(THREADS) sample_kernel(const Args a) {
    extern __shared__ __align__(16) unsigned char held[];
    __shared__ Shared sm;
    cg::cluster_group cl = cg::this_cluster();
    const int b = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = rank * a.len, n = max(0, min(a.len, a.V - first));
    typedef typename Key<T>::N N;
    const N* row = (const N*)a.logits + b * a.ld + first;
    N* mine = reinterpret_cast<N*>(held);
    if (tid < 32) sm.powers[tid] = POWERS[tid];
    for (int i = tid; i < (int)(sizeof(Bins) / 4); i += THREADS) reinterpret_cast<uint32_t*>(&sm.bins[0])[i] = 0;

    const float temperature = a.temperature != nullptr ? a.temperature[b] : a.t, top_p = a.top_p != nullptr ? a.top_p[b] : a.p, min_p = a.min_p != nullptr ? a.min_p[b] : a.least;
    const bool greedy = !(temperature > 0.f);
    int k = a.top_k != nullptr ? a.top_k[b] : a.k;
    if (greedy) k = 1;
    if (k <= 0 || k > a.V) k = a.V;
    const bool by_mass = top_p < 1.f && k > 1, cut = by_mass || k < a.V;

    // the part, and the largest logit
    constexpr int E = 16 / sizeof(T);
    const bool wide = reinterpret_cast<uintptr_t>(row) % 16 == 0;
    const int padded = (n + 127) & ~127;               // (a.len is a multiple of 128)
    uint32_t top = 0;
    if (wide) {
#pragma unroll 4
        for (int i = tid * E; i + E <= n; i += THREADS * E) {
            uint4 raw = *reinterpret_cast<const uint4*>(row + i);
            N* keys = reinterpret_cast<N*>(&raw);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t key = key_of_bits<T>(keys[e]);
                keys[e] = (N)key;
                top = max(top, key);
            }
            if constexpr (HELD) *reinterpret_cast<uint4*>(mine + i) = raw;
        }
    }
#pragma unroll 4
    for (int i = (wide ? n / E * E : 0) + tid; i < n; i += THREADS) {
        const uint32_t key = key_of_bits<T>(row[i]);
        if constexpr (HELD) mine[i] = (N)key;
        top = max(top, key);
    }
    if constexpr (HELD)
        for (int i = n + tid; i < padded; i += THREADS) mine[i] = (N)lowest<T>();
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) sm.count[warp] = top;
    __syncthreads();
    if (tid == 0) {
        uint32_t y = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) y = max(y, sm.count[w]);
        sm.top = y;
    }
    cl.sync();
    uint32_t top_key = 0;
    for (int r = 0; r < a.parts; ++r) top_key = max(top_key, *cl.map_shared_rank(&sm.top, r));
    top_key = max(top_key, lowest<T>());               // (a CTA without logits has none)
    Scale s;
    s.top = top_key;
    s.max = value_of<T>(top_key);
    s.c = greedy ? 1.0 : 1.4426950408889634 / (double)temperature;
    auto four = [&](int i, uint32_t (&k)[4]) {         // logits i .. i + 3 of the part; behind the last one minus infinity, which weighs nothing
        if constexpr (HELD) four_keys(mine + i, k);
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = i + e < n ? key_of_bits<T>(row[i + e]) : lowest<T>();
        }
    };

    // The logit that the cut lies at: tokens with keys above `edge` are kept, and `ties` of those equal to it.  First its bin (16 of them for a factor of two in weight), then its key among those of the bin.
    uint32_t edge = 0, ties = 0;
    int turn = 0;
    if (cut && k == 1) edge = top_key, ties = 1;
    else if (cut) {
        uint32_t lo = lowest<T>(), hi = top_key;       // around the keys of the bin
        int shift = 0, chosen = 0;
        uint32_t ahead = 0;                            // tokens, and weight, above the edge
        u64 ahead_mass = 0, limit = ~0ull;             // a token is kept if less than the limit comes before it
        for (int level = 0;; ++level, turn ^= 1) {
            Bins& h = sm.bins[turn];
            uint32_t all = 0;
            for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
                uint32_t key[4];
                four(i, key);
                bool any = level == 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) any |= key[e] - lo <= hi - lo;
                if (!any) continue;
                u64 w[4];
                int of[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = weight<T>(key[e], s, sm.powers, of[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (w[e] == 0 || (level > 0 && (of[e] != chosen || key[e] - lo > hi - lo))) continue;      // (of no weight: never drawn)
                    const int bin = level == 0 ? of[e] : (int)((hi - key[e]) >> shift);
                    atomicAdd(&h.count[bin], 1u);
                    if (by_mass)
#pragma unroll
                        for (int j = 0; j < 3; ++j) {
                            const uint32_t y = (uint32_t)(w[e] >> (15 * j)) & 0x7fffu;
                            if (y) atomicAdd(&h.part[j][bin], y);
                        }
                }
            }
            __syncthreads();
            // The CTAs' bins: sums of 32 neighbours first, which tell the 32 that have to be read.  (All bins of all CTAs: 98 KB a CTA through the cluster's network, 12000 cycles.)
            for (int c = warp; c < COARSE; c += WARPS) {
                uint32_t count = h.count[32 * c + lane];
                u64 mass = mass_of(h, 32 * c + lane);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    count += __shfl_xor_sync(0xffffffffu, count, o);
                    mass += __shfl_xor_sync(0xffffffffu, mass, o);
                }
                if (lane == 0) sm.coarse_count[turn][c] = count, sm.coarse_mass[turn][c] = mass;
            }
            cl.sync();
            for (int i = tid; i < (int)(sizeof(Bins) / 4); i += THREADS) reinterpret_cast<uint32_t*>(&sm.bins[turn ^ 1])[i] = 0;
            uint32_t from_count = ahead;
            u64 from_mass = ahead_mass;
            int bin = 0;
#pragma unroll
            for (int step = 0; step < 2; ++step) {     // the 32 bins, then the bin
                if (warp < a.parts) {
                    const Shared* o = cl.map_shared_rank(&sm, warp);
                    const bool there = step == 1 || lane < COARSE;
                    sm.all_count[warp][lane] = !there ? 0 : step ? o->bins[turn].count[bin + lane] : o->coarse_count[turn][lane];
                    sm.all_mass[warp][lane] = !there || !by_mass ? 0 : step ? mass_of(o->bins[turn], bin + lane) : o->coarse_mass[turn][lane];
                }
                __syncthreads();
                if (warp == 0) {
                    uint32_t count = 0;
                    u64 mass = 0;
                    for (int r = 0; r < a.parts; ++r) count += sm.all_count[r][lane], mass += sm.all_mass[r][lane];
                    const uint32_t c1 = up_to(count);
                    const u64 m1 = up_to(mass), whole = __shfl_sync(0xffffffffu, m1, 31);
                    if (level == 0 && step == 0 && by_mass) limit = top_p > 0.f ? max(1ull, (u64)ceil((double)top_p * (double)whole)) : 1ull;
                    const uint32_t c = from_count + c1 - count;
                    const u64 m = from_mass + m1 - mass;
                    const uint32_t good = __ballot_sync(0xffffffffu, count > 0 && c < (uint32_t)k && m < limit);
                    const int last = 31 - __clz(good);
                    if (lane == max(last, 0)) sm.found = last, sm.at_count = c, sm.at_mass = m;
                    if (lane == 31) sm.total_count = c1, sm.total_mass = limit;
                }
                __syncthreads();
                if (sm.found < 0) { bin = -1; break; }
                bin = step ? bin + sm.found : 32 * sm.found;
                from_count = sm.at_count, from_mass = sm.at_mass;
                if (step == 0) all = sm.total_count;
                limit = sm.total_mass;
                __syncthreads();
            }
            if (bin < 0) break;                        // nothing above minus infinity
            if (level == 0 && !by_mass && all <= (uint32_t)k) break;      // no more tokens than k
            ahead = from_count;
            ahead_mass = from_mass;
            if (level == 0) {
                chosen = bin;
                // The bin's logits, and some beside them: 16 y lies between -bin - 3/4 and -bin + 1/4, up to the roundings of 32 bits.  (An endless or vanishing temperature: all logits.)
                const float slope = (float)fmin(s.c * PER_OCTAVE, 1e30), top_value = (float)s.max;
                if (slope > 1e-20f && slope < 1e20f && fabsf(top_value) < 1e30f) {
                    const float up = top_value - ((float)bin - 0.25f) / slope, down = top_value - ((float)bin + 0.75f) / slope, slack = 1e-6f * (fabsf(top_value) + fabsf(up) + fabsf(down));
                    hi = min(hi, key_up<T>(up + slack));
                    if (bin < BINS - 1) lo = max(lo, key_down<T>(down - slack));
                }
            } else {
                hi -= (uint32_t)bin << shift;
                lo = max(lo, hi - ((1u << shift) - 1));
            }
            if (level > 0 && lo == hi) {
                edge = lo;
                const u64 w = weight<T>(edge, s, sm.powers);
                ties = (uint32_t)k - ahead;
                if (by_mass) ties = (uint32_t)min((u64)ties, (limit - ahead_mass + w - 1) / w);
                break;
            }
            shift = max(0, 32 - __clz(hi - lo) - SUB_BITS);
        }
    }

    // Kept weight: a warp takes a segment of the part, in order.  Tokens on the edge weigh the same, so their number is enough.
    const u64 least = min_p > 0.f ? (u64)ceil((double)min_p * (double)(1ull << BITS)) : 0ull;
    auto kept = [&](uint32_t key) -> u64 {             // of a token above the edge
        const u64 w = weight<T>(key, s, sm.powers);
        return key > edge && (w >= least || key == top_key) ? w : 0;      // the largest ones stay whatever min_p
    };
    u64 edge_weight = 0;
    if (edge != 0) {
        edge_weight = weight<T>(edge, s, sm.powers);
        if (edge_weight < least && edge != top_key) edge_weight = 0;
    }
    const int seg = (padded / 128 + WARPS - 1) / WARPS * 128, from = min(padded, warp * seg), to = min(padded, from + seg);
    u64 sum = 0;
    uint32_t on = 0;
    for (int i = from + 4 * lane; i < to; i += 128) {
        uint32_t key[4];
        four(i, key);
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= key[e] > edge, on += key[e] == edge;      // (an edge of 0 is no key)
        if (!any) continue;
        u64 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = kept(key[e]);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        on += __shfl_xor_sync(0xffffffffu, on, o);
    }
    if (lane == 0) sm.above[warp] = sum, sm.on_edge[warp] = on;
    if (tid == 0) sm.chosen = -1;
    cl.sync();
    // the segments of all CTAs, in order: a thread each
    const bool one = tid < a.parts * WARPS;
    const u64 above = one ? *cl.map_shared_rank(&sm.above[tid % WARPS], tid / WARPS) : 0;
    const uint32_t edges = one ? *cl.map_shared_rank(&sm.on_edge[tid % WARPS], tid / WARPS) : 0;
    uint32_t all_edges;
    u64 whole;
    const uint32_t tied = before(edges, sm.count, all_edges);
    const u64 weight_here = above + edge_weight * (tied >= ties ? 0u : min(edges, ties - tied));
    const u64 ahead = before(weight_here, sm.mass, whole);
    const double u = (double)a.draw[b];
    u64 goal = u > 0.0 ? (u64)(u * (double)whole) : 0ull;      // the token up to which the weights exceed it
    if (whole > 0 && goal >= whole) goal = whole - 1;
    if (one && tid / WARPS == rank && ahead <= goal && goal < ahead + weight_here) {
        sm.chosen = tid % WARPS;
        sm.tied = tied;
        sm.ahead = ahead;
    }
    __syncthreads();
    if (warp == sm.chosen) {
        u64 sofar = sm.ahead;
        uint32_t rank_on = sm.tied;
        for (int i0 = from; i0 < to; i0 += 128) {
            const int i = i0 + 4 * lane;
            uint32_t key[4];
            four(i, key);
            u64 w[4], own = 0;
            uint32_t mark = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = kept(key[e]);
                mark += key[e] == edge;
            }
            const uint32_t marks = up_to(mark);
            uint32_t mine_on = rank_on + marks - mark;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (key[e] == edge && mine_on++ < ties) w[e] = edge_weight;
                own += w[e];
            }
            const u64 upto = up_to(own);
            rank_on += __shfl_sync(0xffffffffu, marks, 31);
            const bool hit = sofar + upto - own <= goal && goal < sofar + upto;
            if (hit) {
                u64 y = sofar + upto - own;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (y <= goal && goal < y + w[e]) {
                        a.token[b] = first + i + e;
                        a.logp[b] = (float)log((double)w[e] / (double)whole);
                    }
                    y += w[e];
                }
            }
            if (__any_sync(0xffffffffu, hit)) break;
            sofar += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (whole == 0 && rank == 0 && tid == 0) a.token[b] = 0, a.logp[b] = -INFINITY;       // a row of nothing but minus infinity
    cl.sync();                                         // the others have read this one's sums
}

constexpr int MOST_HELD = 192 * 1024;                       // bytes of a part in shared memory, at most
static_assert(sizeof(Shared) + MOST_HELD <= 227 * 1024, "a CTA's shared memory");
template <typename T>
static int launch(const Args& a, cudaStream_t st) {
    const long long bytes = (long long)a.len * sizeof(T);
    const bool held = bytes <= MOST_HELD;
    auto kernel = held ? sample_kernel<T, true> : sample_kernel<T, false>;
    if (held) {                                        // (the same for every call: it belongs to the kernel, and another thread may be between this and its launch)
        const int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_HELD);
        if (rc) return rc;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.parts, a.B);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = held ? (size_t)bytes : 0;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, a);
    return (int)cudaGetLastError();
}

}  // namespace sample
}  // namespace lmoe

// type: 0 fp32, 1 bf16, 2 fp16.
LMOE_API int lmoe_sample(const lmoe::sample::Args* ap, int type, cudaStream_t st) {
    using namespace lmoe::sample;
    const Args& a = *ap;
    if (a.B <= 0 || a.B > 65535 || a.V <= 0 || a.V > 1 << 19 || a.parts < 1 || a.parts > MAX_PARTS || a.len <= 0 || a.len > 1 << 16 || a.len % 128 != 0 || (long long)a.parts * a.len < a.V) return -1;
    return type == 0 ? launch<float>(a, st) : type == 1 ? launch<lmoe::bf16>(a, st) : launch<__half>(a, st);
}
