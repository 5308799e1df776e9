// One step of a beam search.
//
// Selection: the best n of  s_b + x_bt - lse_b  over the beams b and the vocabulary t of every prompt, ties to the lowest b V + t.  Bound by reading the logits once.
// What is compared: inside a beam the logits; between beams 64-bit scores whose log-sums carry the error of sums of 32-bit exponentials (some 1e-7; equal rows have equal ones), so
// candidates of different beams closer than that can come in either order.
//   beam_parts_kernel   a CTA goes through a part of one beam's logits, 4096 at a time in registers, with the next ones on their way: their maximum and sum of exponentials, and their n
//                       best.  The threads' maxima of the first chunk give a bound that n logits reach and few others do; those go to shared memory, their n-th best
//                       is the bound of the chunks behind, and in the end each candidate finds its rank by counting.  Where too many reach the bound a closer one is searched, and where
//                       many are equal the n best are taken out one by one.
//   beam_join_kernel    a CTA per prompt does the same with the parts' candidates.  Candidates of different beams can lie next to one another, so their scores are
//                       compared in 64 bits and rounded once.
// Inside a beam the order of the logits is the order of the scores, so no part needs another one's sum.
// NaN counts as minus infinity.
//
// Reordering: rows of many tensors gathered by one launch (states of the beams that go on; pages that a beam may no longer share).
#include <cuda_fp16.h>

#include "common.cuh"

namespace lmoe {
namespace beam {

struct Args {
    const void* logits;                   // [N, K, V], unit stride along V
    const float* scores;                  // [N, K]
    float* out;                           // [N, n]
    long long *beam, *token;              // [N, n]
    float *key, *top;                     // scratch: [N K, parts, n] candidates' logits, [N K, parts] maxima,
    int* at;                              //          [N K, parts, n] their tokens,
    double* sum;                          //          [N K, parts] sums
    long long s_n, s_k, c_n, c_k;         // strides of logits and of scores
    int N, K, V, n, parts, length;        // length: numbers of a part, a multiple of 8
};

constexpr int THREADS = 256, PER = 16, CHUNK = THREADS * PER, HOLD = 1024, MOST = 128;      // MOST: largest n; HOLD: candidates that fit shared memory
constexpr int MANY = 512;                                    // candidates from which on a closer bound is worth its search

template <typename T> __device__ __forceinline__ float number(T x);
template <> __device__ __forceinline__ float number(float x) { return x; }
template <> __device__ __forceinline__ float number(bf16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float number(__half x) { return __half2float(x); }

// Candidates in shared memory: keys and places (negative: none).  Better: larger key, or the lower place.
template <typename Key, int BLOCK> struct Pool {
    Key key[HOLD];
    int at[HOLD];
    Key last[BLOCK];                          // (one by one) a thread's best
    int bound[BLOCK / 32], some[2][BLOCK / 32];
    int count;
};
template <typename Key> __device__ __forceinline__ bool better(Key a, int ia, Key b, int ib) { return a > b || (a == b && ia < ib); }
// fp32 numbers in the order of signed integers, and back
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i ^ (i >> 31 & 0x7fffffff);
}
__device__ __forceinline__ long long ordered64(double x) {
    const long long i = __double_as_longlong(x);
    return i ^ (i >> 63 & 0x7fffffffffffffffLL);
}
__device__ __forceinline__ double number64_of(long long i) { return __longlong_as_double(i ^ (i >> 63 & 0x7fffffffffffffffLL)); }
__device__ __forceinline__ float number_of(int i) { return __int_as_float(i ^ (i >> 31 & 0x7fffffff)); }

// Where more than MANY keys reach the first bound: the largest bound that n keys reach, by halving, then its keys into shared memory.  Keys are read from memory again: out of line, this
// costs the usual path no registers.  hi: one above the largest.
template <typename Key, int BLOCK, typename Keys>
__device__ __noinline__ int closer(Pool<Key, BLOCK>& sm, int n, int lo, int most, const Keys ks) {
    constexpr int W = BLOCK / 32;
    const int t = threadIdx.x;
    long long low = lo, hi = (long long)most + 1;            // n keys or more reach low, fewer than n reach hi
    for (int step = 0; hi - low > 1; ++step) {
        const int mid = (int)((low + hi) >> 1);
        int c = 0;
        for (int i = t; i < ks.count; i += BLOCK) c += ks.place(i) >= 0 && ordered(ks.near(i)) >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (t % 32 == 0) sm.some[step & 1][t >> 5] = c;
        __syncthreads();
        c = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) c += sm.some[step & 1][i];
        if (c >= n) low = mid;
        else hi = mid;
    }
    __syncthreads();                                         // the count so far has been read
    if (t == 0) sm.count = 0;
    __syncthreads();
    for (int i = t; i < ks.count; i += BLOCK)
        if (ks.place(i) >= 0 && ordered(ks.near(i)) >= (int)low) {
            const int c = atomicAdd(&sm.count, 1);
            if (c < HOLD) sm.key[c] = ks.key(i), sm.at[c] = ks.place(i);
        }
    __syncthreads();
    return sm.count;
}
template <typename Key> struct Top;                          // a key above all and one below all
template <> struct Top<float> {
    static __device__ float value() { return INFINITY; }
    static __device__ float none() { return -INFINITY; }
};
template <> struct Top<long long> {
    static __device__ long long value() { return 0x7fffffffffffffffLL; }
    static __device__ long long none() { return -0x7fffffffffffffffLL - 1; }
};
// Many equal keys: one after the other, each the best of those behind the last.
template <typename Key, int BLOCK, typename Keys, typename Put>
__device__ __noinline__ void one_by_one(Pool<Key, BLOCK>& sm, int n, const Keys ks, const Put put) {
    const int t = threadIdx.x;
    Key last = Top<Key>::value();
    int last_at = -1;
    for (int r = 0; r < n; ++r) {
        Key bk = Top<Key>::none();
        int ba = 0x7fffffff;
        for (int i = t; i < ks.count; i += BLOCK) {
            const Key x = ks.key(i);
            const int at = ks.place(i);
            if (at >= 0 && (x < last || (x == last && at > last_at)) && better<Key>(x, at, bk, ba)) bk = x, ba = at;
        }
        __syncthreads();                                     // the winner of the round before has been read
        sm.last[t] = bk;
        sm.at[t] = ba;
        __syncthreads();
        for (int s = BLOCK / 2; s > 0; s >>= 1) {
            if (t < s && better<Key>(sm.last[t + s], sm.at[t + s], sm.last[t], sm.at[t])) sm.last[t] = sm.last[t + s], sm.at[t] = sm.at[t + s];
            __syncthreads();
        }
        last = sm.last[0], last_at = sm.at[0];
        if (t == 0) put(r, last, last_at);
    }
}

// A bound that at least n keys reach, and an empty pool: with w warps that have candidates, the n / w-th largest of the threads' maxima in each of them, the smallest of these.
// best: the thread's largest key (minus infinity: none; rounding to fp32 keeps the order).  The whole block calls it.
template <typename Key, int BLOCK>
__device__ __forceinline__ float first_bound(Pool<Key, BLOCK>& sm, int n, float best) {
    const int t = threadIdx.x, lane = t & 31;
    int v = ordered(best), top = 0x80000000;
    const int first = __reduce_max_sync(0xffffffffu, v), none = ordered(-INFINITY);
    if (t == 0) sm.count = 0;
    const int warps = __syncthreads_count(lane == 0 && first != none), rounds = (n + warps - 1) / max(warps, 1);
    for (int r = 0; r < min(rounds, 33); ++r) {              // (of 32 maxima the 33rd is below all)
        top = r == 0 ? first : __reduce_max_sync(0xffffffffu, v);
        if (lane == __ffs(__ballot_sync(0xffffffffu, v == top)) - 1) v = 0x80000000;
    }
    if (lane == 0) sm.bound[t >> 5] = first != none ? max(top, none) : 0x7fffffff;
    __syncthreads();
    int bound = sm.bound[0];
#pragma unroll
    for (int i = 1; i < BLOCK / 32; ++i) bound = min(bound, sm.bound[i]);
    return warps == 0 ? -INFINITY : number_of(bound);
}
// The n best of the pool's candidates (all keys from `bound` on, none above `most`), in order, given to put(rank, key, place); of `total` candidates that there are, also in memory (ks),
// min(n, total) are given.  The whole block calls it.
template <typename Key, int BLOCK, typename Keys, typename Put>
__device__ __forceinline__ void best_of(Pool<Key, BLOCK>& sm, int n, int total, float bound, float most, const Keys ks, const Put put) {
    const int t = threadIdx.x;
    __syncthreads();
    int count = sm.count;
    if (count > MANY && total > n && bound < most) count = closer<Key, BLOCK>(sm, n, ordered(bound), ordered(most), ks);
    if (count > HOLD) return one_by_one<Key, BLOCK>(sm, min(n, total), ks, put);
    for (int c = t; c < count; c += BLOCK) {
        const Key x = sm.key[c];
        const int at = sm.at[c];
        int r = 0;
        for (int i = 0; i < count; ++i) r += better<Key>(sm.key[i], sm.at[i], x, at);
        if (r < n) put(r, x, at);
    }
}
// The largest number of the block's threads' ones.
template <int BLOCK> __device__ __forceinline__ float block_top(float x, float* red) {
    x = warp_max(x);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < BLOCK / 32; ++i) x = fmaxf(x, red[i]);
    return x;
}
template <typename Key, int BLOCK> __device__ __forceinline__ void keep(Pool<Key, BLOCK>& sm, Key k, int at) {
    const int c = atomicAdd(&sm.count, 1);
    if (c < HOLD) sm.key[c] = k, sm.at[c] = at;
}

template <typename T> __device__ __forceinline__ T nothing();
template <> __device__ __forceinline__ float nothing() { return -INFINITY; }
template <> __device__ __forceinline__ bf16 nothing() { return __ushort_as_bfloat16(0xff80); }
template <> __device__ __forceinline__ __half nothing() { return __ushort_as_half(0xfc00); }
template <typename T> struct PartKeys {                      // the tokens [lo, lo + count) of a row
    const T* x;
    int lo, count;
    __device__ float key(int i) const { return fmaxf(number<T>(x[lo + i]), -INFINITY); }
    __device__ float near(int i) const { return key(i); }
    __device__ int place(int i) const { return lo + i; }
};
struct PartPut {
    float* key;
    int* at;
    __device__ void operator()(int r, float k, int p) const { key[r] = k; at[r] = p; }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 4) beam_parts_kernel(Args a) {
    constexpr int VN = 16 / sizeof(T), VECS = PER / VN, W = sizeof(T) == 4 ? 4 : 5;       // numbers and 32-bit words of a vector, the latter with one more where numbers straddle words
    __shared__ Pool<float, THREADS> sm;
    __shared__ float red[THREADS / 32];
    __shared__ double sums[THREADS / 32];
    __shared__ float closer_bound;
    const int row = blockIdx.y, part = blockIdx.x, t = threadIdx.x, w = t >> 5, lane = t & 31;
    const T* x = (const T*)a.logits + row / a.K * a.s_n + row % a.K * a.s_k;
    // Which thread sums up which tokens does not depend on where the row begins: equal rows have equal sums, to the bit, and their candidates tie.
    const bool whole = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    const int odd = sizeof(T) == 2 ? (int)(reinterpret_cast<uintptr_t>(x) >> 1 & 1) : 0;      // the row begins in the middle of a word
    const int lo = part * a.length, hi = min(lo + a.length, a.V), total = max(hi - lo, 0), chunks = (a.length + CHUNK - 1) / CHUNK;
    const long long slot = (long long)row * a.parts + part;
    const PartPut put{a.key + slot * a.n, a.at + slot * a.n};
    auto load = [&](int c, uint32_t (&raw)[VECS][W]) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int at = lo + c * CHUNK + (i * THREADS + t) * VN;
            raw[i][W - 1] = 0;
            if (whole && at + VN <= hi) {
                const uint4 y = __ldcs(reinterpret_cast<const uint4*>(x + at));
                raw[i][0] = y.x; raw[i][1] = y.y; raw[i][2] = y.z; raw[i][3] = y.w;
            } else if (!whole && at >= odd && at + VN <= hi && at + VN + odd <= a.V) {           // the words that hold them, none of them outside the row
                const uint32_t* y = reinterpret_cast<const uint32_t*>(x + at - odd);
#pragma unroll
                for (int k = 0; k < 4; ++k) raw[i][k] = y[k];
                if (odd) raw[i][W - 1] = y[W - 1];
            } else {
                T y[VN];
#pragma unroll
                for (int e = 0; e < VN; ++e) y[e] = at + e < hi ? x[at + e] : nothing<T>();
                uint32_t last = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t word;
                    memcpy(&word, y + k * (VN / 4), 4);
                    raw[i][k] = odd ? __funnelshift_r(last, word, 16) : word;
                    last = word;
                }
                if (odd) raw[i][W - 1] = last >> 16;
            }
        }
    };
    uint32_t raw[VECS][W];
    load(0, raw);
    float top = -INFINITY, s = 0.f, bound = -INFINITY;       // the thread's largest logit so far, its sum in units of that
    for (int c = 0; c < chunks; ++c) {
        float v[PER];
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            T y[VN];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t word = W == 5 ? __funnelshift_r(raw[i][k], raw[i][W == 5 ? k + 1 : k], odd * 16) : raw[i][k];
                memcpy(y + k * (VN / 4), &word, 4);
            }
#pragma unroll
            for (int e = 0; e < VN; ++e) v[i * VN + e] = fmaxf(number<T>(y[e]), -INFINITY);      // NaN -> -inf
        }
        if (c + 1 < chunks) load(c + 1, raw);                // on its way while this chunk is looked at
        float best = v[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = fmaxf(best, v[i]);
        if (best > top) {
            s *= top == -INFINITY ? 0.f : __expf(top - best);
            top = best;
        }
        if (top != -INFINITY)
#pragma unroll
            for (int i = 0; i < PER; i += 4) s += (__expf(v[i] - top) + __expf(v[i + 1] - top)) + (__expf(v[i + 2] - top) + __expf(v[i + 3] - top));
        if (c == 0) bound = first_bound<float, THREADS>(sm, a.n, best);
        if (best >= bound) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (v[i] >= bound) {
                    const int p = lo + c * CHUNK + (i / VN * THREADS + t) * VN + i % VN;
                    if (p < hi) keep(sm, v[i], p);
                }
        }
        if (c == 0 && chunks > 1) {                          // what the chunks behind this one have to reach: its own n-th best
            __syncthreads();
            const int count = sm.count;
            if (t == 0) closer_bound = bound;
            __syncthreads();
            if (count <= HOLD)
                for (int i = t; i < count; i += THREADS) {
                    int r = 0;
                    for (int j = 0; j < count; ++j) r += better<float>(sm.key[j], sm.at[j], sm.key[i], sm.at[i]);
                    if (r == a.n - 1) closer_bound = sm.key[i];
                }
            __syncthreads();
            bound = closer_bound;
        }
    }
    pdl_trigger();
    const float most = block_top<THREADS>(top, red);
    s = top == -INFINITY ? 0.f : s * __expf(top - most);
    s = warp_sum(s);
    if (lane == 0) sums[w] = (double)s;
    for (int r = total + t; r < a.n; r += THREADS) put.at[r] = -1;            // fewer tokens than candidates
    best_of<float, THREADS>(sm, a.n, total, bound, most, PartKeys<T>{x, lo, total}, put);
    if (t == 0) {                                            // behind best_of's barriers
        double d = 0.;
        for (int i = 0; i < THREADS / 32; ++i) d += sums[i];
        a.top[slot] = most;
        a.sum[slot] = d;
    }
}

// The parts' candidates of a prompt, with their scores in 64 bits (as integers of the same order: the ranks are counted with integer comparisons).
struct JoinKeys {
    const float* logit;
    const int* token;
    const double* add;
    const float* tops;
    int per_beam, V, count;
    __device__ double score(float x, int c) const {
        const int b = c / per_beam;
        const double k = ((double)x - tops[b]) + add[b];
        return k == k ? k : -INFINITY;
    }
    __device__ long long key(int c) const { return ordered64(score(logit[c], c)); }
    __device__ float near(int c) const { return (float)score(logit[c], c); }
    __device__ int place(int c) const { return token[c] < 0 ? -1 : c / per_beam * V + token[c]; }
};
struct JoinPut {
    float* out;
    long long *beam, *token;
    int V;
    __device__ void operator()(int r, long long k, int p) const { out[r] = (float)number64_of(k); beam[r] = p / V; token[r] = p % V; }
};
constexpr int JOIN = 512, CANDS = 8;                         // candidates that a thread holds at a time
__global__ void __launch_bounds__(JOIN) beam_join_kernel(Args a) {
    __shared__ Pool<long long, JOIN> sm;
    __shared__ double add[MOST];                             // s_b - log of the sum in units of the largest logit, which the candidates are measured from too:
    __shared__ float tops[MOST];                             // logits of the type's lowest value would lose the rest
    __shared__ __align__(16) float heads[JOIN];
    __shared__ float red[JOIN / 32], head_bound;
    pdl_wait();
    const int prompt = blockIdx.x, t = threadIdx.x, w = t >> 5, lane = t & 31;
    const int per_beam = a.parts * a.n, all = a.K * per_beam, lists = a.K * a.parts;
    const long long c0 = (long long)prompt * all, o0 = (long long)prompt * a.n;
    const JoinKeys ks{a.key + c0, a.at + c0, add, tops, per_beam, a.V, all};
    float logit[CANDS];
    int token[CANDS];
#pragma unroll
    for (int i = 0; i < CANDS; ++i) {
        const int c = t + i * JOIN;
        logit[i] = c < all ? ks.logit[c] : -INFINITY;
        token[i] = c < all ? ks.token[c] : -1;
    }
    for (int b = w; b < a.K; b += JOIN / 32) {
        const long long r0 = ((long long)prompt * a.K + b) * a.parts;
        float top = -INFINITY;
        for (int i = lane; i < a.parts; i += 32) top = fmaxf(top, a.top[r0 + i]);
        top = warp_max(top);
        double s = 0.;
        if (top != -INFINITY)
            for (int i = lane; i < a.parts; i += 32) s += a.sum[r0 + i] * (double)__expf(a.top[r0 + i] - top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
            add[b] = top == -INFINITY ? -INFINITY : (double)a.scores[prompt * a.c_n + b * a.c_k] - log(s);
            tops[b] = top == -INFINITY ? 0.f : top;
        }
    }
    if (t == 0) sm.count = 0;
    __syncthreads();
    // A bound that n candidates reach: the n-th largest of the parts' best ones (their first `deep` each), if these are few enough to be counted
    const int deep = (a.n + lists - 1) / lists, m = lists * deep;
    double k[CANDS], best = -INFINITY;
#pragma unroll
    for (int i = 0; i < CANDS; ++i) {
        k[i] = token[i] >= 0 ? ks.score(logit[i], t + i * JOIN) : -INFINITY;
        best = fmax(best, k[i]);
    }
    float bound;
    if (m <= JOIN) {
        const int c = t / deep * a.n + t % deep;
        const float mine = t < m && ks.token[c] >= 0 ? ks.near(c) : -INFINITY;
        heads[t] = mine;
        __syncthreads();
        int r = 0;
        for (int i = 0; i < m; i += 4) {
            const float4 y = load4(heads + i);
            r += better<float>(y.x, i, mine, t) + better<float>(y.y, i + 1, mine, t) + better<float>(y.z, i + 2, mine, t) + better<float>(y.w, i + 3, mine, t);
        }
        if (t < m && r == a.n - 1) head_bound = mine;        // (behind the m-th are only minus infinities of higher places)
        __syncthreads();
        bound = head_bound;
    } else {
        for (int c = t + CANDS * JOIN; c < all; c += JOIN)
            if (ks.token[c] >= 0) best = fmax(best, (double)ks.near(c));
        bound = first_bound<long long, JOIN>(sm, a.n, (float)best);
    }
    // candidates beyond the held ones (larger vocabularies, wider beams) are read again
#pragma unroll
    for (int i = 0; i < CANDS; ++i)
        if (token[i] >= 0 && (float)k[i] >= bound) keep(sm, ordered64(k[i]), (t + i * JOIN) / per_beam * a.V + token[i]);
    for (int c = t + CANDS * JOIN; c < all; c += JOIN)
        if (ks.token[c] >= 0 && ks.near(c) >= bound) {
            best = fmax(best, (double)ks.near(c));
            keep(sm, ks.key(c), ks.place(c));
        }
    const float most = block_top<JOIN>((float)best, red);
    best_of<long long, JOIN>(sm, a.n, 0x7fffffff, bound, most, ks, JoinPut{a.out + o0, a.beam + o0, a.token + o0, a.V});
}

template <typename T>
static int select(const Args& a, cudaStream_t st) {
    beam_parts_kernel<T><<<dim3(a.parts, a.N * a.K), THREADS, 0, st>>>(a);
    const int rc = (int)cudaGetLastError();
    return rc ? rc : launch_early(beam_join_kernel, a.N, JOIN, st, a);
}

// ---- rows of many tensors -----------------------------------------------------------------------------------------------------------
constexpr int TENSORS = 64;
struct Rows {
    const void* src[TENSORS];
    void* dst[TENSORS];
    long long bytes[TENSORS], rows[TENSORS];                 // of a row; rows of src (and of dst, where `to` is given)
    const long long *from, *to;                              // [count]; to null: 0, 1, ...
    long long count;
    int tensors;
    int* err;
};
constexpr int SLAB = 32768;                                 // bytes of a row that a CTA takes
template <typename V>
__device__ __forceinline__ void copy_as(const char* src, char* dst, long long n) {
    const V* s = reinterpret_cast<const V*>(src);
    V* d = reinterpret_cast<V*>(dst);
    const long long m = n / (long long)sizeof(V);
    constexpr int U = 4;
    for (long long i = threadIdx.x; i < m; i += U * THREADS) {
        V x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * THREADS < m) x[u] = s[i + u * THREADS];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * THREADS < m) d[i + u * THREADS] = x[u];
    }
}
__global__ void __launch_bounds__(THREADS) copy_rows_kernel(const __grid_constant__ Rows a) {
    const int k = blockIdx.z;
    const long long off = (long long)blockIdx.x * SLAB, n = min(a.bytes[k] - off, (long long)SLAB);
    if (n <= 0) return;
    for (long long r = blockIdx.y; r < a.count; r += gridDim.y) {
        const long long from = __ldg(a.from + r), to = a.to != nullptr ? __ldg(a.to + r) : r;
        if (from < 0 || from >= a.rows[k] || (a.to != nullptr && (to < 0 || to >= a.rows[k]))) {
            if (threadIdx.x == 0) atomicCAS(a.err, 0, 0x13000);
            continue;
        }
        const char* s = (const char*)a.src[k] + from * a.bytes[k] + off;
        char* d = (char*)a.dst[k] + to * a.bytes[k] + off;
        const uintptr_t all = reinterpret_cast<uintptr_t>(s) | reinterpret_cast<uintptr_t>(d) | (uintptr_t)n;
        if (all % 16 == 0) copy_as<uint4>(s, d, n);
        else if (all % 4 == 0) copy_as<uint32_t>(s, d, n);
        else if (all % 2 == 0) copy_as<uint16_t>(s, d, n);
        else copy_as<uint8_t>(s, d, n);
    }
}

}  // namespace beam
}  // namespace lmoe

// type of the logits: 0 fp32, 1 bf16, 2 fp16
LMOE_API int lmoe_beam_select(const lmoe::beam::Args* ap, int type, cudaStream_t st) {
    using namespace lmoe::beam;
    const Args& a = *ap;
    if (a.N <= 0 || a.K <= 0 || a.K > MOST || a.V <= 0 || a.n <= 0 || a.n > MOST || (long long)a.N * a.K > 65535 || (long long)a.K * a.V > 0x7fffffff - 4 * CHUNK ||
        (long long)a.K * a.V < a.n || a.length <= 0 || a.length % 8 != 0 ||
        (long long)a.parts * a.length < a.V || (long long)a.K * a.parts * a.n > 0x7fffffff) return -1;
    return type == 0 ? select<float>(a, st) : type == 1 ? select<lmoe::bf16>(a, st) : select<__half>(a, st);
}

LMOE_API int lmoe_copy_rows(const lmoe::beam::Rows* ap, cudaStream_t st) {
    using namespace lmoe::beam;
    const Rows& a = *ap;
    if (a.tensors < 1 || a.tensors > TENSORS || a.count < 1) return -1;
    long long most = 1;
    for (int i = 0; i < a.tensors; ++i) most = a.bytes[i] > most ? a.bytes[i] : most;
    const long long chunks = (most + SLAB - 1) / SLAB;
    if (chunks > 0x7fffffff) return -1;
    copy_rows_kernel<<<dim3((unsigned)chunks, (unsigned)(a.count < 65535 ? a.count : 65535), a.tensors), THREADS, 0, st>>>(a);
    return (int)cudaGetLastError();
}
