// Arguments of the one-token attention kernels over a paged cache, and how a request's keys are shared out.
#pragma once
#include "common.cuh"

namespace lmoe {
namespace paged {

struct Args {
    const bf16 *q, *k_new, *v_new;        // [B, H, D], [B, G, D] (k_new null: the token's row is in the cache already)
    bf16 *k, *v, *out;                    // [pages, page, G, D] twice, [B, H, D]
    float *part, *ml;                     // [B, H, splits, D], [B, H, splits, 2]: (maximum in units of log 2, sum); splits > 1
    const float* slopes;                  // [H] or null
    const int *table, *lengths;           // [B, table_n], [B]
    long long q_b, q_h, n_b, n_h, m_b, m_h, k_page, k_row, k_head, v_page, v_row, v_head, table_ld;      // n: k_new, m: v_new
    int B, H, G, D, page, pages, table_n, window, splits;
    int sorted;                           // more CTAs than fit at once: the longest requests come first
    float scale, cap;                     // cap 0: none
    int* err;
};

constexpr int GROUP = 16, MIN_GROUPS = 8;               // keys of a group; groups that a CTA has at least when a request is split

// The groups of 16 keys that a request's CTAs share: CTA s has [first + s per, first + (s + 1) per) of [first, last).
struct Share { int len, lo, first, last, per; };
__device__ __forceinline__ Share share_of(const Args& a, int b) {
    Share s;
    const int n = a.lengths[b], most = a.table_n * a.page;
    s.len = min(max(n, 0), most);
    s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
    s.first = s.lo / GROUP;
    s.last = (s.len + GROUP - 1) / GROUP;
    s.per = max(MIN_GROUPS, (s.last - s.first + a.splits - 1) / a.splits);
    if (a.splits == 1) s.per = s.last - s.first;
    return s;
}

}  // namespace paged
}  // namespace lmoe
