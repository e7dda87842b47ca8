// s2s_attention_whole_bf16.hip - the attention kernels of s2s_attention.h over shared keys and an entry's own, for bf16 arrays.
#include "s2s_attention.h"

hipError_t launch_whole_attention_bf16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st) {
    return attn::launch_type<bfloat_t, attn::WHOLE>(a, L, c, align, st);
}
