// s2s_attention_window_f16.hip - the attention kernels of s2s_attention.h with a sliding window, for f16 arrays.
#include "s2s_attention.h"

hipError_t launch_window_attention_f16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st) {
    return attn::launch_type<half_t, attn::WINDOW>(a, L, c, align, st);
}
