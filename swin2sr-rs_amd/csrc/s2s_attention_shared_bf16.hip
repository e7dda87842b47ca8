// s2s_attention_shared_bf16.hip - the attention kernels of s2s_attention.h over keys that a batch shares, for bf16 arrays.
#include "s2s_attention.h"

hipError_t launch_shared_attention_bf16(const AttnOpArgs &s, const AttnLaunch &L, const attn::Cut &c, int align, const AttnOpArgs &own,
                                        const AttnLaunch &J, hipStream_t st) {
    return attn::launch_shared_type<bfloat_t>(s, L, c, align, own, J, st);
}
