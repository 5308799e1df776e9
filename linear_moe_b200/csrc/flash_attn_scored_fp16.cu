// Attention with key ranges, capped scores and a bias by distance over fp16: see flash_attn_scored.cuh.  (A source per type, so that they compile side by side.)
#include "flash_attn_scored.cuh"

using namespace lmoe::fatc;

// q [B,Tq,Hq,d], k / v [B,Tk,Hkv,d] with element strides; ap->x.tiles [B, ceil(Tq / 128)] is written by the forward and read by the backward pass.
LMOE_API int lmoe_scored_attn_fwd_fp16(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const Args* ap,
                                 cudaStream_t st) {
    return scored_fwd<true>(q, qs, k, ks, v, vs, *ap, st);
}
LMOE_API int lmoe_scored_attn_bwd_fp16(const void* q, const long long* qs, const void* k, const long long* ks, const void* v, const long long* vs, const void* o,
                                 const void* d_o, float* delta, const BwdArgs* ap, cudaStream_t st) {
    return scored_bwd<true>(q, qs, k, ks, v, vs, o, d_o, delta, *ap, st);
}
