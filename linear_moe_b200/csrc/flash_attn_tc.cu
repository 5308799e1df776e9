// Causal attention over bf16, heads of 64 and 128: the kernels of flash_attn_tc.cuh without ranges, cap and bias.
#include "flash_attn_tc.cuh"

using namespace lmoe::fatc;

// q [B,Tq,Hq,D], k/v [B,Tk,Hkv,D] bf16 with element strides (batch, token, head); 16-byte aligned bases, strides % 8 == 0.
LMOE_API int lmoe_flash_attn_fwd_tc(const void* q, const long long* qs, const void* k, const long long* ks, const void* v,
                                    const long long* vs, const Args* ap, int D, cudaStream_t st) {
    if (D == 128) return launch_fwd<128, Plain>(q, qs, k, ks, v, vs, *ap, st);
    if (D == 64) return launch_fwd<64, Plain>(q, qs, k, ks, v, vs, *ap, st);
    return -1;
}

// Backward of lmoe_flash_attn_fwd_tc.  o, d_o: contiguous [B,Tq,Hq,D]; delta is scratch [B,Hq,Tq]; writes dq, dk, dv.
LMOE_API int lmoe_flash_attn_bwd_tc(const void* q, const long long* qs, const void* k, const long long* ks, const void* v,
                                    const long long* vs, const void* o, const void* d_o, float* delta, const BwdArgs* ap, int D,
                                    cudaStream_t st) {
    if (D == 128) return launch_bwd<128, Plain>(q, qs, k, ks, v, vs, o, d_o, delta, *ap, st);
    if (D == 64) return launch_bwd<64, Plain>(q, qs, k, ks, v, vs, o, d_o, delta, *ap, st);
    return -1;
}
