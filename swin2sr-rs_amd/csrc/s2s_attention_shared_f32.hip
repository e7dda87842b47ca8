// s2s_attention_shared_f32.hip - the attention kernels of s2s_attention.h for steps over keys that a batch shares, for f32 arrays.
#include "s2s_attention.h"

hipError_t launch_both_attention_f32(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const attn::Cut &c, bool own_wk,
                                      int align, hipStream_t st) {
    return attn::launch_both_type<float>(a, own, shared, c, own_wk, align, st);
}
