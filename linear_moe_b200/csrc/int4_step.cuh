// Arguments of the one-token attention kernels over a paged cache of 4 bits a number, and how a request's keys are shared out.
#pragma once
#include "int4_cache.cuh"

namespace lmoe {
namespace int4 {

struct StepArgs {
    const void* q;                        // [B, H, D]
    const unsigned char *k, *v;           // [pages, G, page bytes] twice
    void* out;                            // [B, H, D]
    float *part, *ml;                     // [B, H, splits, D], averages, and [B, H, splits, 2]: (maximum in units of log 2, sum); more parts than a cluster joins
    const float* slopes;                  // [H] or null
    const int *table, *lengths;           // [B, table_n], [B]
    long long q_b, q_h, table_ld;
    int B, H, G, D, page, pages, table_n, window, splits;
    int q_rows;                           // queries on 16-byte boundaries
    int sorted;                           // more CTAs than fit at once: the longest requests come first
    float scale, cap;                     // cap 0: none
    int* err;
};

constexpr int GROUP = 16, MIN_GROUPS = 8;               // keys of a group; groups that a CTA has at least when a request is split

// The groups of 16 keys that a request's CTAs share: CTA s has [first + s per, first + (s + 1) per) of [first, last), from 64-key boundaries on.
struct Share { int len, lo, first, last, per; };
__device__ __forceinline__ Share share_of(const StepArgs& a, int b) {
    Share s;
    s.len = min(max(a.lengths[b], 0), a.table_n * a.page);
    s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
    s.first = s.lo / (4 * GROUP) * 4;
    s.last = (s.len + GROUP - 1) / GROUP;
    s.per = max(MIN_GROUPS, ((s.last - s.first + a.splits - 1) / a.splits + 3) & ~3);
    if (a.splits == 1) s.per = max(s.last - s.first, 0);
    return s;
}

inline bool fits(const StepArgs& a) {
    return a.B > 0 && a.B <= 65535 && a.G > 0 && a.H > 0 && a.H % a.G == 0 && a.D > 0 && a.D <= 256 && a.D % UNIT == 0 && a.page > 0 && a.page <= 65536 && a.page % GROUP == 0 && a.pages >= 0 && a.table_n >= 0 &&
           (long long)a.table_n * a.page <= 0x7fffffff - 4096 && a.splits >= 1;
}

}  // namespace int4
}  // namespace lmoe
