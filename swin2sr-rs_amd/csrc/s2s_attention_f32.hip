// s2s_attention_f32.hip - the attention kernels of s2s_attention.h for f32 arrays.
#include "s2s_attention.h"

hipError_t launch_attention_f32(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st) {
    return attn::launch_type<float>(a, L, c, align, st);
}
