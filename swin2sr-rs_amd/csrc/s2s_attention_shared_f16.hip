// s2s_attention_shared_f16.hip - the attention kernels of s2s_attention.h over keys that a batch shares, for f16 arrays.
#include "s2s_attention.h"

hipError_t launch_shared_attention_f16(const AttnOpArgs &s, const AttnLaunch &L, const attn::Cut &c, int align, const AttnOpArgs &own,
                                        const AttnLaunch &J, hipStream_t st) {
    return attn::launch_shared_type<half_t>(s, L, c, align, own, J, st);
}
