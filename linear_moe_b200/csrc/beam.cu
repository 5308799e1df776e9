// One step of a beam search.
//
// Selection: the best n of  s_b + x_bt - lse_b  over the beams b and the vocabulary t of every prompt, ties to the lowest b V + t.  Bound by reading the logits once.
//   beam_parts_kernel   a CTA holds 4096 logits of one beam in registers: their maximum and sum of exponentials, and their n best.  The n-th largest of the
//                       256 threads' maxima is a bound that at least n logits reach and few others do; those go to shared memory, and each finds its rank by counting.
//                       Where too many reach it (equal logits) the n best are taken out one by one instead.
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
    int N, K, V, n, parts;
};

constexpr int THREADS = 256, PER = 16, PART = THREADS * PER, HOLD = 1024, MOST = 128;      // MOST: largest n; HOLD: candidates that fit shared memory

template <typename T> __device__ __forceinline__ float number(T x);
template <> __device__ __forceinline__ float number(float x) { return x; }
template <> __device__ __forceinline__ float number(bf16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float number(__half x) { return __half2float(x); }

// Candidates in shared memory: keys and places (negative: none).  Better: larger key, or the lower place.
template <typename Key> struct Pool {
    Key key[HOLD];
    int at[HOLD];
    Key tmax[THREADS];
    Key bound;
    int count;
    int winner;
};
template <typename Key> __device__ __forceinline__ bool better(Key a, int ia, Key b, int ib) { return a > b || (a == b && ia < ib); }

// The n best of every thread's `mine` candidates (key(i), place(i)), in order, given to put(rank, key, place); `total` of them are real, and at least min(n, total) are given.
// best: the thread's largest key (minus infinity: none).  The whole block calls it.
template <typename Key, int BLOCK, typename KeyOf, typename PlaceOf, typename Put>
__device__ __forceinline__ void best_of(Pool<Key>& sm, int n, int total, int mine, Key best, KeyOf key, PlaceOf place, Put put) {
    const int t = threadIdx.x;
    sm.tmax[t] = best;
    if (t == 0) sm.count = 0;
    __syncthreads();
    // the n-th largest of the maxima (with fewer real candidates than threads: minus infinity lets all pass)
    int rank = 0;
    for (int i = 0; i < BLOCK; ++i) rank += better<Key>(sm.tmax[i], i, best, t);
    if (rank == min(n, BLOCK) - 1) sm.bound = n <= BLOCK ? best : (Key)-INFINITY;
    __syncthreads();
    const Key bound = sm.bound;
    for (int i = 0; i < mine; ++i)
        if (place(i) >= 0 && key(i) >= bound) {
            const int c = atomicAdd(&sm.count, 1);
            if (c < HOLD) sm.key[c] = key(i), sm.at[c] = place(i);
        }
    __syncthreads();
    const int count = sm.count;
    if (count <= HOLD) {
        for (int c = t; c < count; c += BLOCK) {
            const Key x = sm.key[c];
            const int at = sm.at[c];
            int r = 0;
            for (int i = 0; i < count; ++i) r += better<Key>(sm.key[i], sm.at[i], x, at);
            if (r < n) put(r, x, at);
        }
        return;
    }
    // many equal keys: one after the other, each the best of those behind the last
    Key last = (Key)INFINITY;
    int last_at = -1;
    for (int r = 0; r < min(n, total); ++r) {
        Key bk = (Key)-INFINITY;
        int ba = 0x7fffffff;
        for (int i = 0; i < mine; ++i) {
            const Key x = key(i);
            const int at = place(i);
            if (at >= 0 && (x < last || (x == last && at > last_at)) && better<Key>(x, at, bk, ba)) bk = x, ba = at;
        }
        __syncthreads();                                     // the winner of the round before has been read
        sm.tmax[t] = bk;
        sm.at[t] = ba;
        __syncthreads();
        for (int s = BLOCK / 2; s > 0; s >>= 1) {
            if (t < s && better<Key>(sm.tmax[t + s], sm.at[t + s], sm.tmax[t], sm.at[t])) sm.tmax[t] = sm.tmax[t + s], sm.at[t] = sm.at[t + s];
            __syncthreads();
        }
        last = sm.tmax[0], last_at = sm.at[0];
        if (t == 0) put(r, last, last_at);
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) beam_parts_kernel(Args a) {
    constexpr int VN = 16 / sizeof(T);
    __shared__ Pool<float> sm;
    __shared__ float red[THREADS / 32];
    __shared__ double dred[THREADS / 32];
    const int row = blockIdx.y, part = blockIdx.x, t = threadIdx.x, w = t >> 5, lane = t & 31;
    const T* x = (const T*)a.logits + row / a.K * a.s_n + row % a.K * a.s_k;
    // vectors lie on 16-byte boundaries: the part begins up to VN - 1 numbers early, and those belong to nobody
    const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int base = part * PART - skew;                     // token of the part's first number
    const int lo = max(base, 0), hi = min(base + PART, a.V);
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER / VN; ++i) {
        const int at = base + (i * THREADS + t) * VN;
        if (at >= lo && at + VN <= hi) {
            const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(x + at));
            const T* p = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int e = 0; e < VN; ++e) v[i * VN + e] = fmaxf(number<T>(p[e]), -INFINITY);      // NaN -> -inf
        } else {
#pragma unroll
            for (int e = 0; e < VN; ++e) v[i * VN + e] = at + e >= lo && at + e < hi ? fmaxf(number<T>(x[at + e]), -INFINITY) : -INFINITY;
        }
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
    const float mine = top;
    top = warp_max(top);
    if (lane == 0) red[w] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) top = fmaxf(top, red[i]);
    float s = 0.f;
    const float unit = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < PER; i += 4) s += (__expf(v[i] - unit) + __expf(v[i + 1] - unit)) + (__expf(v[i + 2] - unit) + __expf(v[i + 3] - unit));
    s = warp_sum(s);
    if (lane == 0) dred[w] = (double)s;
    __syncthreads();
    const long long slot = (long long)row * a.parts + part;
    if (t == 0) {
        double d = 0.;
        for (int i = 0; i < THREADS / 32; ++i) d += dred[i];
        a.top[slot] = top;
        a.sum[slot] = d;
    }
    const int total = max(hi - lo, 0);
    float* key = a.key + slot * a.n;
    int* at = a.at + slot * a.n;
    for (int r = total + t; r < a.n; r += THREADS) at[r] = -1;            // fewer tokens than candidates
    best_of<float, THREADS>(
        sm, a.n, total, PER, mine, [&](int i) { return v[i]; },
        [&](int i) {
            const int p = base + (i / VN * THREADS + t) * VN + i % VN;
            return p >= lo && p < hi ? p : -1;
        },
        [&](int r, float k, int p) { key[r] = k; at[r] = p; });
}

constexpr int JOIN = 256;
__global__ void __launch_bounds__(JOIN) beam_join_kernel(Args a) {
    __shared__ Pool<double> sm;
    __shared__ double add[MOST];                             // s_b - log of the sum in units of the largest logit, which the candidates are measured from too:
    __shared__ float tops[MOST];                             // logits of the type's lowest value would lose the rest
    pdl_wait();
    const int prompt = blockIdx.x, t = threadIdx.x, w = t >> 5, lane = t & 31;
    for (int b = w; b < a.K; b += JOIN / 32) {
        const long long r0 = ((long long)prompt * a.K + b) * a.parts;
        float top = -INFINITY;
        for (int i = lane; i < a.parts; i += 32) top = fmaxf(top, __ldcg(a.top + r0 + i));
        top = warp_max(top);
        double s = 0.;
        if (top != -INFINITY)
            for (int i = lane; i < a.parts; i += 32) s += __ldcg(a.sum + r0 + i) * exp((double)(__ldcg(a.top + r0 + i) - top));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
            add[b] = top == -INFINITY ? -INFINITY : (double)a.scores[prompt * a.c_n + b * a.c_k] - log(s);
            tops[b] = top == -INFINITY ? 0.f : top;
        }
    }
    __syncthreads();
    const int per_beam = a.parts * a.n, all = a.K * per_beam, mine = t < all ? (all - t + JOIN - 1) / JOIN : 0;
    const long long c0 = (long long)prompt * all;
    auto key = [&](int i) -> double {
        const int c = t + i * JOIN;
        const double k = ((double)__ldcg(a.key + c0 + c) - tops[c / per_beam]) + add[c / per_beam];
        return k == k ? k : -INFINITY;
    };
    auto place = [&](int i) -> int {
        const int c = t + i * JOIN, p = __ldcg(a.at + c0 + c);
        return p < 0 ? -1 : c / per_beam * a.V + p;
    };
    double best = -INFINITY;
    for (int i = 0; i < mine; ++i)
        if (place(i) >= 0) best = fmax(best, key(i));
    best_of<double, JOIN>(sm, a.n, a.n, mine, best, key, place, [&](int r, double k, int p) {
        const long long o = (long long)prompt * a.n + r;
        a.out[o] = (float)k;
        a.beam[o] = p / a.V;
        a.token[o] = p % a.V;
    });
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
constexpr int CHUNK = 32768;                                 // bytes of a row that a CTA takes
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
    const long long off = (long long)blockIdx.x * CHUNK, n = min(a.bytes[k] - off, (long long)CHUNK);
    if (n <= 0) return;
    for (long long r = blockIdx.y; r < a.count; r += gridDim.y) {
        const long long from = __ldg(a.from + r), to = a.to != nullptr ? __ldg(a.to + r) : r;
        if (from < 0 || from >= a.rows[k] || (a.to != nullptr && (to < 0 || to >= a.rows[k]))) {
            if (threadIdx.x == 0) atomicCAS(a.err, 0, 0xb300);
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
    if (a.N <= 0 || a.K <= 0 || a.K > MOST || a.V <= 0 || a.n <= 0 || a.n > MOST || (long long)a.N * a.K > 65535 || (long long)a.K * a.V > 0x7fffffff ||
        (long long)a.K * a.V < a.n || (long long)a.parts * PART < (long long)a.V + 7 || (long long)a.K * a.parts * a.n > 0x7fffffff) return -1;
    return type == 0 ? select<float>(a, st) : type == 1 ? select<lmoe::bf16>(a, st) : select<__half>(a, st);
}

LMOE_API int lmoe_copy_rows(const lmoe::beam::Rows* ap, cudaStream_t st) {
    using namespace lmoe::beam;
    const Rows& a = *ap;
    if (a.tensors < 1 || a.tensors > TENSORS || a.count < 1) return -1;
    long long most = 1;
    for (int i = 0; i < a.tensors; ++i) most = a.bytes[i] > most ? a.bytes[i] : most;
    const long long chunks = (most + CHUNK - 1) / CHUNK;
    if (chunks > 0x7fffffff) return -1;
    copy_rows_kernel<<<dim3((unsigned)chunks, (unsigned)(a.count < 65535 ? a.count : 65535), a.tensors), THREADS, 0, st>>>(a);
    return (int)cudaGetLastError();
}
