// s2s_attention_shared_f32.hip - the attention kernels of s2s_attention.h over keys that a batch shares, for f32 arrays.
#include "s2s_attention.h"

hipError_t launch_shared_attention_f32(const AttnOpArgs &s, const AttnLaunch &L, const attn::Cut &c, int align, const AttnOpArgs &own,
                                        const AttnLaunch &J, hipStream_t st) {
    return attn::launch_shared_type<float>(s, L, c, align, own, J, st);
}
