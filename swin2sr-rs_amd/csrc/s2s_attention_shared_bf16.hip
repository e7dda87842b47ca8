// s2s_attention_shared_bf16.hip - the attention kernels of s2s_attention.h for steps over keys that a batch shares, for bf16 arrays.
#include "s2s_attention.h"

hipError_t launch_both_attention_bf16(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const attn::Cut &c, bool own_wk,
                                      int align, hipStream_t st) {
    return attn::launch_both_type<bfloat_t>(a, own, shared, c, own_wk, align, st);
}
