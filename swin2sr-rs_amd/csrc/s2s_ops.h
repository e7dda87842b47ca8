// s2s_ops.h - argument blocks and launchers of the transformer operators
// (s2s_attention.hip, s2s_ops.hip). s2s_ops_api.cpp checks a call and fills
// these; strides are in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <type_traits>

struct Strides {
    long long b, t, h;
};

struct AttnOpArgs {
    int batch, nq, nk, hq, hk, group, width;
    int causal;
    float scale, cap;
    const void *q, *k, *v;
    void *out;
    Strides sq, sk, sv, so;
    const int *q_lens, *k_lens, *prefix;
    const int *q_docs, *k_docs;
    long long q_docs_b, k_docs_b;
    const int *q_pos, *k_pos;
    long long q_pos_b, k_pos_b;
    const float *slopes, *table;
    int table_size;
    int window, sinks;  // window 0: none
    // keys that the batch shares, ahead of each entry's own, and each entry's part of them
    const void *shared_k, *shared_v;
    Strides shared_sk, shared_sv;  // (b counts for nothing)
    const int *shared_lens;
    int shared_nk;
};

struct RotaryArrays {
    int batch, tokens, hq, hk, width, axes, pairs;
    int adjacent;
    const void *q, *k;
    void *qo, *ko;
    Strides sq, sk, sqo, sko;
    const int *pos;
    long long pos_b;
    const int *lens;
};

// The turns of P pairs at most.
template <int P>
struct RotaryTurns {
    unsigned long long freq[P];  // 2^64 turns per position, negated for the inverse
    unsigned char axis[P];
};

struct RotaryArgs : RotaryArrays, RotaryTurns<128> {};

// Rotary positions behind a norm of every head.
struct HeadNorm {
    const float *qw, *kw;
    long long qw_head, kw_head;  // the weights' head strides (0: one row for all heads)
    float offset, eps;
};
struct NormRotaryArgs : HeadNorm {
    RotaryArgs r;
};

struct RmsNormArgs {
    long long rows;
    int cols, group, groups;  // group: columns per scale
    const void *x, *res;
    void *sum, *out;
    long long xs, rs, ss, os;
    const float *weight;
    float offset, eps;
    float *scales;
};

// ---- element types -----------------------------------------------------------
typedef _Float16 half_t;
typedef __bf16 bfloat_t;

// N elements, accessed as one where their address is a multiple of A of them
template <typename T, int N, int A = N>
struct alignas(sizeof(T) * A) VecOf {
    T e[N];
};

// Enqueues a kernel and returns that launch's own error: hipGetLastError would return any
// earlier one that the caller has not taken.
template <typename... P>
hipError_t enqueue(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, std::common_type_t<P>... args) {
    void *ptrs[] = {&args...};
    return hipLaunchKernel((const void *)kernel, grid, block, ptrs, lds, st);
}

size_t attn_op_workspace(int dtype, const AttnOpArgs &a);
hipError_t launch_attention_op(int dtype, const AttnOpArgs &a, void *ws, hipStream_t st);
size_t shared_attn_op_workspace(int dtype, const AttnOpArgs &a);
hipError_t launch_shared_attention_op(int dtype, const AttnOpArgs &a, void *ws, hipStream_t st);
hipError_t launch_rotary_op(int dtype, const RotaryArgs &a, hipStream_t st);
hipError_t launch_norm_rotary_op(int dtype, const NormRotaryArgs &a, hipStream_t st);
hipError_t launch_rms_norm_op(int dtype, bool e4m3, const RmsNormArgs &a, hipStream_t st);
