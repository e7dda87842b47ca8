// s2s_attention_shared_f16.hip - the attention kernels of s2s_attention.h for steps over keys that a batch shares, for f16 arrays.
#include "s2s_attention.h"

hipError_t launch_both_attention_f16(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const attn::Cut &c, bool own_wk,
                                      int align, hipStream_t st) {
    return attn::launch_both_type<half_t>(a, own, shared, c, own_wk, align, st);
}
