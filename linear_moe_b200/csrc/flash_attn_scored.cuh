// Entry points of the `Scored` forms of flash_attn_tc.cuh for one type (defined once per type, so that the types compile side by side).
// Heads of d (a multiple of 8 up to 128); ap->x.tiles [B, ceil(Tq / 128)] is written by the forward and read by the backward pass.
#pragma once
#include "flash_attn_tc.cuh"

namespace lmoe {
namespace fatc {
static bool scored_args_ok(const Ranges& x, int B, int Tq, int Tk, int Hq, int Hkv) {
    return B > 0 && Tq > 0 && Tk > 0 && Hkv > 0 && Hq % Hkv == 0 && x.d > 0 && x.d <= 128 && x.d % 8 == 0 && x.tiles != nullptr &&
           (Tq + BM - 1) / BM <= MAX_TILES;
}
template <bool H>
static int scored_fwd_any(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const Args& a, cudaStream_t st) {
    if (!scored_args_ok(a.x, a.B, a.Tq, a.Tk, a.Hq, a.Hkv)) return -1;
    if (a.x.cap > 0.f) return scored_fwd<SCORE_CAP, H>(q, qs, k, ks, v, vs, a, st);
    if (a.x.slopes != nullptr) return scored_fwd<SCORE_BIAS, H>(q, qs, k, ks, v, vs, a, st);
    return scored_fwd<SCORE_PLAIN, H>(q, qs, k, ks, v, vs, a, st);
}
template <bool H>
static int scored_bwd_any(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const void* o,
                          const void* d_o, float* delta, const BwdArgs& a, cudaStream_t st) {
    if (!scored_args_ok(a.x, a.B, a.Tq, a.Tk, a.Hq, a.Hkv) || a.x.low == nullptr) return -1;
    if (a.x.cap > 0.f) return scored_bwd<SCORE_CAP, H>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
    if (a.x.slopes != nullptr) return scored_bwd<SCORE_BIAS, H>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
    return scored_bwd<SCORE_PLAIN, H>(q, qs, k, ks, v, vs, o, d_o, delta, a, st);
}
}  // namespace fatc
}  // namespace lmoe
