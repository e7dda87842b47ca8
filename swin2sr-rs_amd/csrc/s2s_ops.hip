// s2s_ops.hip - rotary positions with several axes, and the root-mean-square
// norm with the residual's addition and an e4m3 output. Both are bound by HBM:
// every element is read once and written once.
#include <algorithm>
#include <cmath>

#include "s2s_device.h"
#include "s2s_kernels.h"
#include "s2s_ops.h"

namespace {

// ---- rotary ------------------------------------------------------------------

// sin and cos of a whole turn times f / 2^64. The angle arrives in turns as a
// 64-bit fraction (position times frequency, the product wrapping modulo one
// turn by itself, exact for any int32 position up to the frequency's last
// bit), so no reduction loses bits however far the position is. The nearest
// quarter turn is split off in integers; what is left, within an eighth of a
// turn, goes through the Taylor polynomials of sin and cos (their next terms,
// y^11 / 11! and y^12 / 12! at y = pi / 4, are 1.8e-9 and 1.1e-10).
__device__ __forceinline__ void sincos_turns(unsigned long long f, float &s, float &c) {
    const unsigned u = (unsigned)(f >> 32) + 0x20000000u;
    const int r = (int)(u & 0x3fffffffu) - 0x20000000;
    const float y = (float)r * 1.4629180792671596e-09f;  // 2 pi / 2^32
    const float z = y * y;
    float a = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    a = fmaf(z, a, 8.3333333e-3f);
    a = fmaf(z, a, -1.6666667e-1f);
    const float sn = fmaf(y * z, a, y);
    float b = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    b = fmaf(z, b, -1.3888889e-3f);
    b = fmaf(z, b, 4.1666667e-2f);
    b = fmaf(z, b, -0.5f);
    const float cs = fmaf(z, b, 1.0f);
    const unsigned q = u >> 30;
    const float ss = (q & 1) ? cs : sn, cc = (q & 1) ? sn : cs;
    s = (q & 2) ? -ss : ss;
    c = ((q + 1) & 2) ? -cc : cc;
}

// One thread: V pairs of one token (their angles once) in the heads h0, h0 + hs,
// ... of q and of k, or V of the channels that are copied. Neighbouring threads
// take neighbouring pairs of a token, then the next token, so that a wave reads
// whole rows; heads are split over gridDim.y until the launch fills the chip.
template <typename T, bool ADJ, int V, bool ALIGNED = true>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs a, int per_token) {
    typedef VecOf<T, ADJ ? 2 * V : V, ALIGNED ? (ADJ ? 2 * V : V) : 1> Vec;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long tok = id / per_token;
    const int g = (int)(id - tok * per_token);
    if (tok >= (long long)a.batch * a.tokens) return;
    const int b = (int)(tok / a.tokens), t = (int)(tok - (long long)b * a.tokens);
    if (a.lens && t >= a.lens[b]) return;
    const T *q = (const T *)a.q + b * a.sq.b + t * a.sq.t;
    T *qo = (T *)a.qo + b * a.sqo.b + t * a.sqo.t;
    const T *k = (const T *)a.k + b * a.sk.b + t * a.sk.t;
    T *ko = (T *)a.ko + b * a.sko.b + t * a.sko.t;
    const int heads = a.hq + a.hk, rot = a.pairs / V;
    if (g < rot) {
        float sn[V], cs[V];
        const int *pos = a.pos + b * a.pos_b + (long long)t * a.axes;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int p = g * V + i;
            sincos_turns((unsigned long long)(long long)pos[a.axis[p]] * a.freq[p], sn[i], cs[i]);
        }
        const int c0 = ADJ ? g * 2 * V : g * V, c1 = ADJ ? c0 + 1 : c0 + a.pairs;
#pragma unroll 4
        for (int h = blockIdx.y; h < heads; h += gridDim.y) {
            const bool isq = h < a.hq;
            const T *src = isq ? q + h * a.sq.h : k + (h - a.hq) * a.sk.h;
            T *dst = isq ? qo + h * a.sqo.h : ko + (h - a.hq) * a.sko.h;
            Vec x = *(const Vec *)(src + c0);
            if (ADJ) {
                Vec o;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float u = (float)x.e[2 * i], w = (float)x.e[2 * i + 1];
                    o.e[2 * i] = (T)fmaf(u, cs[i], -w * sn[i]);
                    o.e[2 * i + 1] = (T)fmaf(u, sn[i], w * cs[i]);
                }
                *(Vec *)(dst + c0) = o;
            } else {
                Vec y = *(const Vec *)(src + c1), o, r;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float u = (float)x.e[i], w = (float)y.e[i];
                    o.e[i] = (T)fmaf(u, cs[i], -w * sn[i]);
                    r.e[i] = (T)fmaf(u, sn[i], w * cs[i]);
                }
                *(Vec *)(dst + c0) = o;
                *(Vec *)(dst + c1) = r;
            }
        }
    } else {
        typedef VecOf<T, V> Part;
        const int c = 2 * a.pairs + (g - rot) * V;
        for (int h = blockIdx.y; h < heads; h += gridDim.y) {
            const bool isq = h < a.hq;
            const T *src = isq ? q + h * a.sq.h : k + (h - a.hq) * a.sk.h;
            T *dst = isq ? qo + h * a.sqo.h : ko + (h - a.hq) * a.sko.h;
            *(Part *)(dst + c) = *(const Part *)(src + c);
        }
    }
}

// The largest power of two, in elements and up to 16 bytes, that the array's
// address and strides are multiples of.
int aligned_elements(const void *p, const Strides &s, int size) {
    unsigned long long m = (unsigned long long)(uintptr_t)p | 16;
    m |= (unsigned long long)(s.b * size) | (unsigned long long)(s.t * size) | (unsigned long long)(s.h * size);
    return (int)((m & (~m + 1)) / size);
}

template <typename T, bool ADJ>
hipError_t rotary_of(const RotaryArgs &a, hipStream_t st) {
    const int size = sizeof(T);
    int w = std::min(aligned_elements(a.q, a.sq, size), aligned_elements(a.qo, a.sqo, size));
    if (a.hk) w = std::min(w, std::min(aligned_elements(a.k, a.sk, size), aligned_elements(a.ko, a.sko, size)));
    // V pairs a thread: what one access of 16 bytes holds, where the arrays and
    // the pair and channel counts allow it
    int v = ADJ ? w / 2 : w;
    while (v > 1 && (a.pairs % v || (a.width - 2 * a.pairs) % v)) v /= 2;
    v = std::max(v, 1);
    const int per_token = (a.pairs + a.width - 2 * a.pairs) / v;
    const long long items = (long long)a.batch * a.tokens * per_token, blocks = (items + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    // threads enough for 8 waves on every SIMD, before heads are looped over
    const long long want = (long long)cu_count() * 2048;
    const int hs = (int)std::max(1LL, std::min((long long)(a.hq + a.hk), want / std::max(1LL, blocks * 256)));
    const dim3 grid((unsigned)blocks, (unsigned)hs);
    switch (v) {
        case 8:
            if constexpr (!ADJ && sizeof(T) == 2) {
                hipLaunchKernelGGL((k_rotary<T, ADJ, 8>), grid, dim3(256), 0, st, a, per_token);
                break;
            }
            return hipErrorInvalidValue;
        case 4:
            if constexpr (!(ADJ && sizeof(T) == 4)) {
                hipLaunchKernelGGL((k_rotary<T, ADJ, 4>), grid, dim3(256), 0, st, a, per_token);
                break;
            }
            return hipErrorInvalidValue;
        case 2:
            hipLaunchKernelGGL((k_rotary<T, ADJ, 2>), grid, dim3(256), 0, st, a, per_token);
            break;
        default:
            if (ADJ && w < 2)
                hipLaunchKernelGGL((k_rotary<T, ADJ, 1, false>), grid, dim3(256), 0, st, a, per_token);
            else
                hipLaunchKernelGGL((k_rotary<T, ADJ, 1>), grid, dim3(256), 0, st, a, per_token);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t rotary_type(const RotaryArgs &a, hipStream_t st) {
    return a.adjacent ? rotary_of<T, true>(a, st) : rotary_of<T, false>(a, st);
}

// ---- root-mean-square norm ------------------------------------------------------

__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    float w = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
    return half_sum(v + w);
}

// The nearest e4m3 (OCP, ties to even) of v clamped to +-448; NaN stays NaN.
__device__ __forceinline__ unsigned char to_e4m3(float v) {
    v = v > 448.f ? 448.f : (v < -448.f ? -448.f : v);
    return (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

// The largest magnitude of a row or group; NaN where one is among them (a
// maximum would drop it, and with it the only sign that the scale is void).
__device__ __forceinline__ float nan_max(float m, float v) {
    return v > m || v != v ? v : m;
}

__device__ __forceinline__ float e4m3_scale(float top) {
    const float s = top / 448.f;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// A workgroup per row, any width and alignment: the row is read for the sum of
// squares and again for the output (and for the scales), from the caches the
// second time where it fits.
template <typename T, bool E4M3>
__global__ __launch_bounds__(256) void k_rms_norm_rows(RmsNormArgs a) {
    const long long row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.xs;
    const T *res = a.res ? (const T *)a.res + row * a.rs : nullptr;
    T *sum = a.sum ? (T *)a.sum + row * a.ss : nullptr;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ float part[4];
    float ss = 0.f;
    for (int c = tid; c < a.cols; c += 256) {
        const float h = (float)x[c] + (res ? (float)res[c] : 0.f);
        ss = fmaf(h, h, ss);
    }
    ss = wave_sum(ss);
    if (lane == 0) part[wave] = ss;
    __syncthreads();
    const float mean = ((part[0] + part[1]) + (part[2] + part[3])) / (float)a.cols;
    const float inv = 1.0f / sqrtf(mean + a.eps);
    auto value = [&](int c) {
        const float h = (float)x[c] + (res ? (float)res[c] : 0.f);
        return h * inv * (a.weight[c] + a.offset);
    };
    if constexpr (!E4M3) {
        T *out = (T *)a.out + row * a.os;
        for (int c = tid; c < a.cols; c += 256) {
            const float h = (float)x[c] + (res ? (float)res[c] : 0.f);
            if (sum) sum[c] = (T)h;
            out[c] = (T)(h * inv * (a.weight[c] + a.offset));
        }
    } else {
        unsigned char *out = (unsigned char *)a.out + row * a.os;
        float *scales = a.scales + row * a.groups;
        if (a.groups == 1) {
            float top = 0.f;
            for (int c = tid; c < a.cols; c += 256) top = nan_max(top, fabsf(value(c)));
            __syncthreads();
#pragma unroll
            for (int m = 1; m < 64; m *= 2) top = nan_max(top, __shfl_xor(top, m));
            if (lane == 0) part[wave] = top;
            __syncthreads();
            top = nan_max(nan_max(part[0], part[1]), nan_max(part[2], part[3]));
            const float s = e4m3_scale(top);
            if (tid == 0) scales[0] = s;
            for (int c = tid; c < a.cols; c += 256) out[c] = to_e4m3(value(c) / s);
        } else {
            for (int g = wave; g < a.groups; g += 4) {  // a wave per group
                const int c0 = g * a.group, c1 = min(a.cols, c0 + a.group);
                float top = 0.f;
                for (int c = c0 + lane; c < c1; c += 64) top = nan_max(top, fabsf(value(c)));
#pragma unroll
                for (int m = 1; m < 64; m *= 2) top = nan_max(top, __shfl_xor(top, m));
                const float s = e4m3_scale(top);
                if (lane == 0) scales[g] = s;
                for (int c = c0 + lane; c < c1; c += 64) out[c] = to_e4m3(value(c) / s);
            }
        }
        // the sum last: it may lie where x or res did
        if (sum) {
            __syncthreads();
            for (int c = tid; c < a.cols; c += 256) sum[c] = (T)((float)x[c] + (res ? (float)res[c] : 0.f));
        }
    }
}

template <typename T>
hipError_t rms_type(bool e4m3, const RmsNormArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.rows);
    if (e4m3)
        hipLaunchKernelGGL((k_rms_norm_rows<T, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_rms_norm_rows<T, false>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary_op(int dtype, const RotaryArgs &a, hipStream_t st) {
    switch (dtype) {
        case 0: return rotary_type<float>(a, st);
        case 1: return rotary_type<half_t>(a, st);
        case 2: return rotary_type<bfloat_t>(a, st);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_rms_norm_op(int dtype, bool e4m3, const RmsNormArgs &a, hipStream_t st) {
    switch (dtype) {
        case 0: return rms_type<float>(e4m3, a, st);
        case 1: return rms_type<half_t>(e4m3, a, st);
        case 2: return rms_type<bfloat_t>(e4m3, a, st);
    }
    return hipErrorInvalidValue;
}
