// s2s_attention.hip - attention over token arrays of any layout: capped scores,
// biases by distance, document, causal and prefix masks, grouped heads.
#include <algorithm>
#include <cmath>

#include "s2s_device.h"
#include "s2s_kernels.h"
#include "s2s_ops.h"

namespace {

// One wave per query row: 64 keys at a time, a lane per key for the scores,
// then a lane per channel for the products with v.
template <typename T>
__global__ __launch_bounds__(64) void k_attn_row(AttnOpArgs a) {
    const int lane = threadIdx.x;
    const long long id = blockIdx.x;
    const int h = (int)(id % a.hq), i = (int)(id / a.hq % a.nq), b = (int)(id / a.hq / a.nq);
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    const int kl = a.k_lens ? min(max(a.k_lens[b], 0), a.nk) : a.nk;
    if (i >= ql) return;
    const int at = kl - ql + i;
    int lim = kl;
    if (a.causal) lim = min(kl, max(at + 1, a.prefix ? a.prefix[b] : 0));
    const T *q = (const T *)a.q + b * a.sq.b + i * a.sq.t + h * a.sq.h;
    const T *k = (const T *)a.k + b * a.sk.b + (h / a.group) * a.sk.h;
    const T *v = (const T *)a.v + b * a.sv.b + (h / a.group) * a.sv.h;
    const int doc = a.q_docs ? a.q_docs[b * a.q_docs_b + i] : 0;
    if (a.q_docs && doc < 0) lim = 0;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j0 = 0; j0 < lim; j0 += 64) {
        const int j = j0 + lane;
        bool ok = j < lim;
        if (ok && a.q_docs) ok = a.k_docs[b * a.k_docs_b + j] == doc;
        float s = -INFINITY;
        if (ok) {
            s = 0.f;
            for (int d = 0; d < a.width; ++d) s = fmaf((float)q[d], (float)k[j * a.sk.t + d], s);
            s *= a.scale;
            if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
            const int dist = a.q_pos ? a.q_pos[b * a.q_pos_b + i] - a.k_pos[b * a.k_pos_b + j] : at - j;
            if (a.slopes) s -= a.slopes[h] * fabsf((float)dist);
            if (a.table) {
                const int half = a.table_size / 2;
                s += a.table[(long long)h * a.table_size + min(max(dist, -half), half) + half];
            }
        }
        float top = s;
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
        const float mn = fmaxf(m, top);
        const float p = mn == -INFINITY ? 0.f : expf(s - mn), f = mn == -INFINITY ? 0.f : expf(m - mn);
        m = mn;
        l = l * f + p;
        o0 *= f;
        o1 *= f;
        for (int x = 0; x < min(64, lim - j0); ++x) {
            const float px = __shfl(p, x);
            if (!__shfl((int)ok, x)) continue;
            const T *vr = v + (j0 + x) * a.sv.t;
            if (lane < a.width) o0 = fmaf(px, (float)vr[lane], o0);
            if (lane + 64 < a.width) o1 = fmaf(px, (float)vr[lane + 64], o1);
        }
    }
    for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
    const float r = l > 0.f || l != l ? 1.f / l : 0.f;
    T *out = (T *)a.out + b * a.so.b + i * a.so.t + h * a.so.h;
    if (lane < a.width) out[lane] = (T)(o0 * r);
    if (lane + 64 < a.width) out[lane + 64] = (T)(o1 * r);
}

template <typename T>
hipError_t attention_type(const AttnOpArgs &a, void *, hipStream_t st) {
    const long long n = (long long)a.batch * a.hq * a.nq;
    if (n > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_row<T>), dim3((unsigned)n), dim3(64), 0, st, a);
    return hipGetLastError();
}

}  // namespace

size_t attn_op_workspace(int, const AttnOpArgs &) { return 0; }

hipError_t launch_attention_op(int dtype, const AttnOpArgs &a, void *ws, hipStream_t st) {
    switch (dtype) {
        case 0: return attention_type<float>(a, ws, st);
        case 1: return attention_type<half_t>(a, ws, st);
        case 2: return attention_type<bfloat_t>(a, ws, st);
    }
    return hipErrorInvalidValue;
}
