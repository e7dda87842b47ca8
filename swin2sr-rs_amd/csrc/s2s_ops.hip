// s2s_ops.hip - rotary positions with several axes, the same behind a norm of each head, and the
// root-mean-square norm with the residual's addition and an e4m3 output. All are bound by HBM:
// every element is read once and written once. Measured on an MI355X, whose plain
// copy of 1 GiB makes 5.05 TB/s: rotary of 16384 tokens, 32 + 8 bf16 heads of 128, 64 us
// (5.2 TB/s); the norm of 16391 x 5120 bf16 with residual, sum and e4m3 groups of 128, 115 us
// (5.1 TB/s). Steps (4 rows, 32 tokens) take 4 to 5 us, a launch and two or three reads that
// wait for each other.
#include <algorithm>
#include <cmath>

#include "s2s_device.h"
#include "s2s_kernels.h"
#include "s2s_ops.h"

namespace {

__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    float w = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
    return half_sum(v + w);
}

// Over G neighbouring lanes (a power of two), every lane receiving the total.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (G >= 2) v = DPP_ADD(v, 0xB1);
    if constexpr (G >= 4) v = DPP_ADD(v, 0x4E);
    if constexpr (G >= 8) v = DPP_ADD(v, 0x141);
    if constexpr (G >= 16) v = DPP_ADD(v, 0x140);
    if constexpr (G >= 32) {
        float w = v;
        asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
        v += w;
    }
    if constexpr (G >= 64) v = half_sum(v);
    return v;
}

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

// A workgroup takes `tb` tokens of q and k. Their sines and cosines are made once, in
// LDS; then the threads walk the tokens' heads in memory order, a unit of V pairs (or of
// V channels that are copied) at a time, neighbours next to each other across heads, so
// that a wave's accesses are whole runs whatever the width. (A thread that kept its
// angles in registers and looped over heads touched a run per head: 45 us against 38 for
// 2 x 23400 tokens of 6 + 6 f32 heads of 30, of which every run is 120 bytes.)
template <typename T, bool ADJ, int V, bool ALIGNED = true>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs a, int tb, int per_head) {
    typedef VecOf<T, ADJ ? 2 * V : V, ALIGNED ? (ADJ ? 2 * V : V) : 1> Vec;
    typedef VecOf<T, V, ALIGNED ? V : 1> Part;
    extern __shared__ float2 turn[];  // [tb][pairs]
    const int tid = threadIdx.x, heads = a.hq + a.hk, rot = a.pairs / V;
    const long long tok0 = (long long)blockIdx.x * tb, all = (long long)a.batch * a.tokens;
    const int n_tok = (int)min((long long)tb, all - tok0);
    for (int i = tid; i < n_tok * a.pairs; i += 256) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        const long long b = (tok0 + t) / a.tokens, at = (tok0 + t) - b * a.tokens;
        const int pos = a.pos[b * a.pos_b + at * a.axes + a.axis[p]];
        float2 x;
        sincos_turns((unsigned long long)(long long)pos * a.freq[p], x.y, x.x);
        turn[i] = x;
    }
    __syncthreads();
    // unit (token t, head h, g) of this thread, and the step of 256 units
    const int dg = 256 % per_head, dh = 256 / per_head;
    int g = tid % per_head, h = tid / per_head, t = 0;
    while (h >= heads) h -= heads, ++t;
    while (t < n_tok) {
        const int b = (int)((tok0 + t) / a.tokens), at = (int)((tok0 + t) - (long long)b * a.tokens);
        if (!a.lens || at < a.lens[b]) {
            const bool isq = h < a.hq;
            const T *src = isq ? (const T *)a.q + b * a.sq.b + at * a.sq.t + h * a.sq.h
                               : (const T *)a.k + b * a.sk.b + at * a.sk.t + (h - a.hq) * a.sk.h;
            T *dst = isq ? (T *)a.qo + b * a.sqo.b + at * a.sqo.t + h * a.sqo.h
                         : (T *)a.ko + b * a.sko.b + at * a.sko.t + (h - a.hq) * a.sko.h;
            if (g < rot) {
                const float2 *cs = turn + t * a.pairs + g * V;
                const int c0 = ADJ ? g * 2 * V : g * V, c1 = ADJ ? c0 : c0 + a.pairs;
                Vec x = *(const Vec *)(src + c0), o;
                if (ADJ) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float u = (float)x.e[2 * i], w = (float)x.e[2 * i + 1];
                        o.e[2 * i] = (T)fmaf(u, cs[i].x, -w * cs[i].y);
                        o.e[2 * i + 1] = (T)fmaf(u, cs[i].y, w * cs[i].x);
                    }
                } else {
                    Vec y = *(const Vec *)(src + c1), r;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float u = (float)x.e[i], w = (float)y.e[i];
                        o.e[i] = (T)fmaf(u, cs[i].x, -w * cs[i].y);
                        r.e[i] = (T)fmaf(u, cs[i].y, w * cs[i].x);
                    }
                    *(Vec *)(dst + c1) = r;
                }
                *(Vec *)(dst + c0) = o;
            } else {
                const int c = 2 * a.pairs + (g - rot) * V;
                *(Part *)(dst + c) = *(const Part *)(src + c);
            }
        }
        g += dg, h += dh;
        if (g >= per_head) g -= per_head, ++h;
        while (h >= heads) h -= heads, ++t;
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
    const int per_head = (a.pairs + a.width - 2 * a.pairs) / v;
    // tokens per workgroup: a unit for every thread and 128 sines at least, since the threads past
    // them idle there; fewer where that leaves CUs without work. (16384 tokens, 32 + 8 bf16 heads of 128:
    // 64 us, 72 by 8 units a thread; 2 x 23400, 6 + 6 f32 heads of 30, whose tokens have 15 sines:
    // 38 and 37 us, 42 by a unit a thread alone. Reading a unit's channels ahead of the sines, 55 and 73.)
    const long long units = (long long)(a.hq + a.hk) * per_head, all = (long long)a.batch * a.tokens;
    const long long fill = std::max(1LL, all / (4LL * cu_count()));
    // (a launch holds less than 2^24 workgroups of 256: of 2^30 tokens 65 each, 66 KB of LDS at most)
    const int tb = (int)std::max({1LL, std::min({std::max((256 + units - 1) / units, (128LL + a.pairs - 1) / a.pairs), fill, 16LL}), all / 0xffffff + 1});
    const dim3 grid((unsigned)((all + tb - 1) / tb));
    const size_t lds = (size_t)tb * a.pairs * sizeof(float2);
    switch (v) {
        case 8:
            if constexpr (!ADJ && sizeof(T) == 2) return enqueue(k_rotary<T, ADJ, 8>, grid, dim3(256), lds, st, a, tb, per_head);
            return hipErrorInvalidValue;
        case 4:
            if constexpr (!(ADJ && sizeof(T) == 4)) return enqueue(k_rotary<T, ADJ, 4>, grid, dim3(256), lds, st, a, tb, per_head);
            return hipErrorInvalidValue;
        case 2: return enqueue(k_rotary<T, ADJ, 2>, grid, dim3(256), lds, st, a, tb, per_head);
    }
    if (ADJ && w < 2) return enqueue(k_rotary<T, ADJ, 1, false>, grid, dim3(256), lds, st, a, tb, per_head);
    return enqueue(k_rotary<T, ADJ, 1>, grid, dim3(256), lds, st, a, tb, per_head);
}

template <typename T>
hipError_t rotary_type(const RotaryArgs &a, hipStream_t st) {
    return a.adjacent ? rotary_of<T, true>(a, st) : rotary_of<T, false>(a, st);
}

// ---- root-mean-square norm ------------------------------------------------------

// The nearest e4m3 (OCP, ties to even) of v clamped to +-448; NaN stays NaN.
__device__ __forceinline__ unsigned char to_e4m3(float v) {
    v = v > 448.f ? 448.f : (v < -448.f ? -448.f : v);
    return (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

// Four codes in a word.
__device__ __forceinline__ unsigned to_e4m3x4(float a, float b, float c, float d) {
    auto clip = [](float v) { return v > 448.f ? 448.f : (v < -448.f ? -448.f : v); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(clip(a), clip(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(clip(c), clip(d), w, true);
    return (unsigned)w;
}

// The largest magnitude of a row or group; NaN where one is among them (a
// maximum would drop it, and with it the only sign that the scale is void).
__device__ __forceinline__ float nan_max(float m, float v) {
    return v > m || v != v ? v : m;
}

// What norms a row whose squares' sum passes an f32's range (FAR), or (with so small an eps) lies where
// its precision ends (NEAR): the sum is made again of the row times 2^-80 or 2^100, and that factor is
// multiplied in by itself, ahead of the reciprocal root for a NEAR row and behind it for a FAR one, since a
// product of the two is no normal number for rows of 2^-128 or 2^127 (and a small channel of a FAR row times 2^-80
// none either). 2^100 takes the smallest f32, 2^-149, to squares of 2^-98, and what is below the border, 2^-50, to 2^50.
constexpr float kFar = 0x1p127f, kNear = 0x1p-100f, kFarUnit = 0x1p-80f, kNearUnit = 0x1p100f;
struct Root {
    float inv, before = 1.f, after = 1.f;
    __device__ bool plain() const { return before * after == 1.f; }
    __device__ float of(float v) const { return v * before * inv * after; }
};

// 1 / sqrt(mean of n squares + eps) from the squares' sum. `again(factor)` makes the sum of the row
// times a factor; all threads of the row call it or none. (Squares of f16 lie within 2^-48
// and 2^34, and 2^24 of them within both ends.)
template <typename T, typename F>
__device__ __forceinline__ Root inverse_root(float ss, int n, float eps, const F &again) {
    constexpr bool F16 = std::is_same<T, half_t>::value;
    const bool far = !F16 && ss > kFar, near = !F16 && ss < kNear && eps < kNear;
    if (__builtin_expect(far || near, 0)) {
        const float f = far ? kFarUnit : kNearUnit;
        return {1.0f / sqrtf(again(f) / (float)n + eps * f * f), far ? 1.f : f, far ? f : 1.f};
    }
    return {1.0f / sqrtf(ss / (float)n + eps)};
}

__device__ __forceinline__ float e4m3_scale(float top) {
    const float s = top / 448.f;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// A workgroup per row at a time, any width and alignment: the row is read for the sum of
// squares and again for the output (and for the scales), from the caches the
// second time where it fits. (45412 x 177 f16 38 us, to e4m3 75; with its elements one by one
// in registers, 32 a thread, a row of 5121 took twice as long: 278 us for 16391 of them, 599 so.)
template <typename T, bool E4M3>
__global__ __launch_bounds__(256) void k_rms_norm_rows(RmsNormArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ float part[4];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.xs;
        const T *res = a.res ? (const T *)a.res + row * a.rs : nullptr;
        T *sum = a.sum ? (T *)a.sum + row * a.ss : nullptr;
        auto squares = [&](float f) {
            float ss = 0.f;
            for (int c = tid; c < a.cols; c += 256) {
                const float h = ((float)x[c] + (res ? (float)res[c] : 0.f)) * f;
                ss = fmaf(h, h, ss);
            }
            ss = wave_sum(ss);
            if (lane == 0) part[wave] = ss;
            __syncthreads();
            return (part[0] + part[1]) + (part[2] + part[3]);
        };
        const Root root = inverse_root<T>(squares(1.f), a.cols, a.eps, [&](float f) {
            __syncthreads();  // `part` has been read
            return squares(f);
        });
        auto value = [&](int c) {
            const float h = (float)x[c] + (res ? (float)res[c] : 0.f);
            return root.of(h) * (a.weight[c] + a.offset);
        };
        if constexpr (!E4M3) {
            T *out = (T *)a.out + row * a.os;
            for (int c = tid; c < a.cols; c += 256) {
                const float h = (float)x[c] + (res ? (float)res[c] : 0.f);
                if (sum) sum[c] = (T)h;
                out[c] = (T)(root.of(h) * (a.weight[c] + a.offset));
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
        __syncthreads();  // the words of `part` are free
    }
}

// The rows of a workgroup in registers: TPR threads a row (256 / TPR rows at once), NC
// chunks of V elements (16 or 8 bytes) a thread, so that x and the residual are read once and
// nothing is read again (rows read twice, k_rms_norm_rows: 493 us for the 16391 x 5120 above);
// the weights stay in registers over the rows that the workgroup walks. A group of the scales is a power of two of chunks, which neighbouring lanes hold.
template <typename T, bool E4M3, int V, int TPR, int NC>
__global__ __launch_bounds__(256) void k_rms_norm(RmsNormArgs a) {
    static_assert(V % 4 == 0, "codes are stored four and more at a time");
    typedef VecOf<T, V> Vec;
    const int tid = threadIdx.x, lane = tid & 63, r0 = tid / TPR, tr = tid % TPR;
    const int chunks = a.cols / V;
    __shared__ float part[2][4];
    float wt[NC][V];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = (n * TPR + tr) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) wt[n][e] = 0.f;
        if (c < a.cols) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 w = *(const float4 *)(a.weight + c + e);
                wt[n][e] = w.x + a.offset, wt[n][e + 1] = w.y + a.offset;
                wt[n][e + 2] = w.z + a.offset, wt[n][e + 3] = w.w + a.offset;
            }
        }
    }
    for (long long row = (long long)blockIdx.x * (256 / TPR) + r0;; row += (long long)gridDim.x * (256 / TPR)) {
        // (uniform in a wave, and in the workgroup where rows share it)
        if (row >= a.rows) break;
        const T *x = (const T *)a.x + row * a.xs;
        const T *res = a.res ? (const T *)a.res + row * a.rs : nullptr;
        float h[NC][V];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int i = n * TPR + tr;
            Vec u{}, v{};
            if (i < chunks) {
                u = *(const Vec *)(x + i * V);
                if (res) v = *(const Vec *)(res + i * V);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) h[n][e] = (float)u.e[e] + (float)v.e[e];
        }
        auto squares = [&](float f) {
            float ss = 0.f;
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) ss = fmaf(h[n][e] * f, h[n][e] * f, ss);
            return ss;
        };
        // part[0] is the squares' sum, part[1] the largest magnitude (e4m3): a barrier lies between a
        // row's last reading of either and the next row's writing, here the one behind the outputs, or
        // the one behind the largest magnitudes
        auto of_row = [&](float ss) {
            ss = wave_sum(ss);
            if constexpr (TPR == 256) {
                if (lane == 0) part[0][tid >> 6] = ss;
                __syncthreads();
                ss = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
            }
            return ss;
        };
        const float own = squares(1.f);
        if (a.sum) {
            T *sum = (T *)a.sum + row * a.ss;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const int i = n * TPR + tr;
                Vec u;
#pragma unroll
                for (int e = 0; e < V; ++e) u.e[e] = (T)h[n][e];
                if (i < chunks) *(Vec *)(sum + i * V) = u;
            }
        }
        const Root root = inverse_root<T>(of_row(own), a.cols, a.eps, [&](float f) {
            if constexpr (TPR == 256) __syncthreads();  // `part` has been read
            return of_row(squares(f));
        });
        float inv = root.inv;
        if (__builtin_expect(!root.plain(), 0)) {  // (all of the row)
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) h[n][e] = root.of(h[n][e]);
            inv = 1.f;
        }
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) h[n][e] = h[n][e] * inv * wt[n][e];
        if constexpr (!E4M3) {
            T *out = (T *)a.out + row * a.os;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const int i = n * TPR + tr;
                Vec u;
#pragma unroll
                for (int e = 0; e < V; ++e) u.e[e] = (T)h[n][e];
                if (i < chunks) *(Vec *)(out + i * V) = u;
            }
            if constexpr (TPR == 256) __syncthreads();
        } else {
            unsigned char *out = (unsigned char *)a.out + row * a.os;
            float *scales = a.scales + row * a.groups;
            float top[NC];
            const int gl = a.groups == 1 ? 64 : a.group / V;  // lanes of a group
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                top[n] = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) top[n] = nan_max(top[n], fabsf(h[n][e]));
            }
            if (a.groups == 1) {
#pragma unroll
                for (int n = 1; n < NC; ++n) top[0] = nan_max(top[0], top[n]);
            }
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (n && a.groups == 1) {
                    top[n] = top[0];
                    continue;
                }
#pragma unroll
                for (int m = 1; m < 64; m *= 2)
                    if (m < gl) top[n] = nan_max(top[n], __shfl_xor(top[n], m));
                if (a.groups == 1) {
                    if constexpr (TPR == 256) {
                        if (lane == 0) part[1][tid >> 6] = top[0];
                        __syncthreads();
                        top[0] = nan_max(nan_max(part[1][0], part[1][1]), nan_max(part[1][2], part[1][3]));
                    }
                }
            }
            if constexpr (TPR == 256)
                if (a.groups != 1) __syncthreads();
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const int i = n * TPR + tr;
                // h / s as h times 1 / s in two words: with the reciprocal's own rounding more values
                // land on the other side of a code's border (31925 x 720 bf16, groups of 64: 3.2e-5 of the
                // values away from a division's codes, 1.8e-5 so; no time)
                const float s = e4m3_scale(top[n]), r = 1.0f / s, low = r == 0.f ? 0.f : fmaf(-r, s, 1.f) * r;
                auto code_of = [&](float v) { return fmaf(v, r, v * low); };
                VecOf<unsigned, V / 4> code;
#pragma unroll
                for (int e = 0; e < V; e += 4) code.e[e / 4] = to_e4m3x4(code_of(h[n][e]), code_of(h[n][e + 1]), code_of(h[n][e + 2]), code_of(h[n][e + 3]));
                if (i < chunks) {
                    *(VecOf<unsigned, V / 4> *)(out + i * V) = code;
                    if (a.groups == 1 ? i == 0 : (lane & (gl - 1)) == 0) scales[a.groups == 1 ? 0 : i / gl] = s;
                }
            }
        }
    }
}

template <typename T, bool E4M3, int V, int TPR, int NC>
hipError_t rms_launch(const RmsNormArgs &a, hipStream_t st) {
    const long long blocks = (a.rows + 256 / TPR - 1) / (256 / TPR);
    // at most 32 workgroups a CU, which then walk their rows with the weights at hand (16391 x 5120
    // bf16 to e4m3: 117 us, 122 with 8, 120 with 64)
    const long long most = 32LL * cu_count();
    return enqueue(k_rms_norm<T, E4M3, V, TPR, NC>, dim3((unsigned)std::min(blocks, most)), dim3(256), 0, st, a);
}

// Whether rows of chunks of V elements can be taken: their places, their number, and the
// scales' groups, which are a power of two of chunks.
template <typename T, bool E4M3, int V>
bool rms_takes(const RmsNormArgs &a, int most) {
    auto fits = [](const void *p, long long stride, int size, int bytes) {
        return !p || ((uintptr_t)p % bytes == 0 && stride * size % bytes == 0);
    };
    constexpr int B = V * sizeof(T);
    const int gl = a.groups == 1 ? 1 : a.group / V;
    return a.cols % V == 0 && a.cols <= most * V && fits(a.x, a.xs, sizeof(T), B) && fits(a.res, a.rs, sizeof(T), B) &&
           fits(a.sum, a.ss, sizeof(T), B) && fits(a.out, a.os, E4M3 ? 1 : sizeof(T), E4M3 ? V : B) &&
           fits(a.weight, 0, 4, 16) && (!E4M3 || a.groups == 1 || (a.group % V == 0 && (gl & (gl - 1)) == 0 && gl <= 64));
}

template <typename T, bool E4M3>
hipError_t rms_type(const RmsNormArgs &a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int chunks = a.cols / V;
    if (rms_takes<T, E4M3, V>(a, 8 * 256)) {
        // a wave per row up to 2 chunks a lane (16384 x 1024 bf16 to e4m3: 22 us, 28 by a workgroup per
        // row), where there are rows for the chip (64 rows: 4.4 us, 3.4 by a workgroup each); 4 chunks
        // a lane (65536 x 2048: 183 us, 179 by a workgroup per row) gain nothing
        if (chunks <= 64) return rms_launch<T, E4M3, V, 64, 1>(a, st);
        if (chunks <= 128 && a.rows >= 4LL * cu_count()) return rms_launch<T, E4M3, V, 64, 2>(a, st);
        if (chunks <= 256) return rms_launch<T, E4M3, V, 256, 1>(a, st);
        if (chunks <= 512) return rms_launch<T, E4M3, V, 256, 2>(a, st);
        if (chunks <= 768) return rms_launch<T, E4M3, V, 256, 3>(a, st);
        if (chunks <= 1024) return rms_launch<T, E4M3, V, 256, 4>(a, st);
        return rms_launch<T, E4M3, V, 256, 8>(a, st);
    }
    // 16-bit rows of 8-byte multiples (180 or 60 columns): 45412 x 180 f16 to e4m3 21 us, 74 us by
    // rows read twice
    if constexpr (sizeof(T) == 2) {
        if (rms_takes<T, E4M3, 4>(a, 4 * 64)) {
            if (a.cols <= 4 * 64) return rms_launch<T, E4M3, 4, 64, 1>(a, st);
            return rms_launch<T, E4M3, 4, 64, 4>(a, st);
        }
    }
    return enqueue(k_rms_norm_rows<T, E4M3>, dim3((unsigned)std::min(a.rows, 1LL << 20)), dim3(256), 0, st, a);
}

// ---- norms of heads with the rotation ----------------------------------------------

// A wave per token and head, any width and alignment: the head is read for the sum of squares
// and, pair by pair, again for the output, with a pair's angle made where it is used. (16384 tokens of 32 + 8 bf16
// heads of 128: 388 us, 61 by the kernel below, which takes what it can.)
template <typename T>
__global__ __launch_bounds__(256) void k_norm_rotary_heads(NormRotaryArgs a) {
    const RotaryArgs &r = a.r;
    const int lane = threadIdx.x & 63, heads = r.hq + r.hk;
    const long long items = (long long)r.batch * r.tokens * heads;
    for (long long it = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += (long long)gridDim.x * 4) {
        const long long tok = it / heads;
        const int hh = (int)(it - tok * heads);
        const int b = (int)(tok / r.tokens), at = (int)(tok - (long long)b * r.tokens);
        if (r.lens && at >= r.lens[b]) continue;
        const bool isq = hh < r.hq;
        const int h = isq ? hh : hh - r.hq;
        const Strides &si = isq ? r.sq : r.sk, &so = isq ? r.sqo : r.sko;
        const T *x = (const T *)(isq ? r.q : r.k) + b * si.b + at * si.t + h * si.h;
        T *y = (T *)(isq ? r.qo : r.ko) + b * so.b + at * so.t + h * so.h;
        const float *w = isq ? a.qw + h * a.qw_head : a.kw + h * a.kw_head;
        const int *pos = r.pos + b * r.pos_b + (long long)at * r.axes;
        auto squares = [&](float f) {
            float ss = 0.f;
            for (int c = lane; c < r.width; c += 64) {
                const float v = (float)x[c] * f;
                ss = fmaf(v, v, ss);
            }
            return wave_sum(ss);
        };
        const Root root = inverse_root<T>(squares(1.f), r.width, a.eps, squares);
        auto value = [&](int c) { return root.of((float)x[c]) * (w[c] + a.offset); };
        for (int p = lane; p < r.pairs; p += 64) {
            const int c0 = r.adjacent ? 2 * p : p, c1 = r.adjacent ? c0 + 1 : c0 + r.pairs;
            const float u = value(c0), v = value(c1);
            float s, c;
            sincos_turns((unsigned long long)(long long)pos[r.axis[p]] * r.freq[p], s, c);
            y[c0] = (T)fmaf(u, c, -v * s);
            y[c1] = (T)fmaf(u, s, v * c);
        }
        for (int c = 2 * r.pairs + lane; c < r.width; c += 64) y[c] = (T)value(c);
    }
}

// One access of a VecOf at a 32-bit byte offset; past the resource zeros are read and nothing is written.
template <typename P>
__device__ __forceinline__ P buf_read(__amdgpu_buffer_rsrc_t r, int off) {
    if constexpr (sizeof(P) == 16) return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    else if constexpr (sizeof(P) == 8) return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    else if constexpr (sizeof(P) == 4) return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
    else return __builtin_bit_cast(P, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
}
template <typename P>
__device__ __forceinline__ void buf_write(__amdgpu_buffer_rsrc_t r, int off, P x) {
    if constexpr (sizeof(P) == 16) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, x), r, off, 0, 0);
    else if constexpr (sizeof(P) == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, x), r, off, 0, 0);
    else if constexpr (sizeof(P) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), r, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, x), r, off, 0, 0);
}

// How k_norm_rotary walks: the tokens of a workgroup, the units of a head, and for q and k the arrays'
// strides in units of V elements, with what the next batch entry's first token lies further on than
// the token behind this one's last.
struct NormRotaryWalk {
    int tb, per_head;
    struct Of {
        int in_t, in_h, in_b, out_t, out_h, out_b;
        unsigned by_heads;  // ceil(2^32 / heads)
    } of[2];
};

// A head in the registers of G lanes (a power of two): lane g holds V pairs, or V channels that are
// not turned, reads them once, and the squares' sum is made across the lanes. The sines of the
// workgroup's tokens are made once, in LDS. A wave takes 64 / G heads at a time, side by side in memory,
// first of q, then of k, so that what differs between the two is in scalar registers; the next heads are
// read while these are normed and turned. HBM bounds it: the 16384 tokens below take 61.4 us (5.5 TB/s, a part from the last-level
// cache), the f32 heads of 30 35.9 (3.8 TB/s: lanes of 8 bytes). Offsets are 32-bit ones from the workgroup's first token.
// (The turns as an argument of 64 or 128 pairs: a launch's time goes by its arguments' bytes.)
template <typename T, bool ADJ, int V, int G, bool EACH, int P>
__global__ __launch_bounds__(256) void k_norm_rotary(RotaryArrays r, HeadNorm a, NormRotaryWalk w, RotaryTurns<P> x) {
    typedef VecOf<T, V> Part;
    typedef VecOf<T, 2 * V> Both;
    constexpr int H = 64 / G, UNIT = V * (int)sizeof(T);  // heads a wave takes at a time
    // turns read ahead: two of short units (2 x 23400 tokens of 6 + 6 f32 heads of 30, 8 bytes a lane, 35.9 us; one 44.3,
    // three 37.2), one of 32 bytes a lane (16384 tokens of 32 + 8 bf16 heads of 128 61.4 us; two 62.8, three 66)
    constexpr int AHEAD = 2 * UNIT <= 16 ? 2 : 1;
    extern __shared__ float2 turn[];  // [tb][pairs]
    const int tid = threadIdx.x, lane = tid & 63, g = tid % G, rot = r.pairs / V;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned tok0 = blockIdx.x * (unsigned)w.tb, all = (unsigned)r.batch * (unsigned)r.tokens;  // (at most 2^30)
    const int n_tok = (int)min((unsigned)w.tb, all - tok0);
    const int b0 = (int)(tok0 / (unsigned)r.tokens), at0 = (int)(tok0 - (unsigned)b0 * r.tokens);
    const int cross = r.tokens - at0;  // tokens from here on are the next batch entry's (one at most: tb <= tokens)
    for (int i = tid; i < n_tok * r.pairs; i += 256) {
        const int t = (int)((unsigned)i / (unsigned)r.pairs), p = i - t * r.pairs;
        const int *pos = r.pos + (t < cross ? b0 * r.pos_b + (long long)(at0 + t) * r.axes : (b0 + 1) * r.pos_b + (long long)(t - cross) * r.axes);
        float2 c;
        sincos_turns((unsigned long long)(long long)pos[x.axis[p]] * x.freq[p], c.y, c.x);
        turn[i] = c;
    }
    // (lengths of any size, past the tokens or negative)
    const int len0 = r.lens ? min(min(max(r.lens[b0], 0), r.tokens) - at0, n_tok) : n_tok;
    const int len1 = r.lens && cross < n_tok ? min(min(max(r.lens[b0 + 1], 0), r.tokens) + cross, n_tok) : n_tok;
    // this lane's channels: two runs of V (ADJ: one of 2 V), or one of V that is not turned
    const bool turns = g < rot, there = g < w.per_head;
    const int u0 = !there ? 0 : turns ? (ADJ ? 2 : 1) * g : 2 * rot + (g - rot), u1 = turns ? (ADJ ? u0 + 1 : u0 + rot) : u0;
    const int c0 = u0 * V, c1 = u1 * V;
    const float mean = 1.f / (float)r.width;
    __syncthreads();
    auto walk = [&](const void *src, void *dst, const Strides &ss, const Strides &ds, const float *weight, long long weight_head, int heads,
                    const NormRotaryWalk::Of &o, int first) {
        // (the resources begin where the first token of either entry lies: the next one's may lie ahead of this one's)
        const int i_low = cross < n_tok ? min(cross * o.in_t + o.in_b, 0) : 0, o_low = cross < n_tok ? min(cross * o.out_t + o.out_b, 0) : 0;
        const auto in = buf_rsrc((const T *)src + b0 * ss.b + at0 * ss.t + (long long)i_low * V, BUF_MAX_BYTES);
        const auto out = buf_rsrc((const T *)dst + b0 * ds.b + at0 * ds.t + (long long)o_low * V, BUF_MAX_BYTES);
        const int end = (n_tok * heads + H - 1) / H;
        struct Item {
            int t, out;
            bool ok;
            Part x, y;
            Both z;
            float w[EACH ? 2 : 1][EACH ? V : 1];
        };
        float wt[2][V];
        auto weights = [&](const float *p, auto &to) {
            if constexpr (ADJ) {
                // one run of 2 V (of V channels that are not turned, its last ones where the head ends)
                const int back = min(c0, r.width - 2 * V);
                const auto z = *(const VecOf<float, 2 * V, 1> *)(p + back);
#pragma unroll
                for (int i = 0; i < V; ++i) to[0][i] = back == c0 ? z.e[i] : z.e[V + i], to[1][i] = z.e[V + i];
            } else {
                const auto x = *(const VecOf<float, V, 1> *)(p + c0), y = *(const VecOf<float, V, 1> *)(p + c1);
#pragma unroll
                for (int i = 0; i < V; ++i) to[0][i] = x.e[i], to[1][i] = y.e[i];
            }
        };
        auto read = [&](int n) {
            Item m;
            const int item = n * H + lane / G;
            m.t = heads == 1 ? item : (int)__umulhi((unsigned)item, o.by_heads);
            const int h = item - __mul24(m.t, heads), next = m.t < cross ? 0 : 1;
            m.ok = there && m.t < (next ? len1 : len0);
            const int at = __mul24(m.t, o.in_t) + __mul24(h, o.in_h) + (next ? o.in_b : 0) - i_low;
            m.out = __mul24(m.t, o.out_t) + __mul24(h, o.out_h) + (next ? o.out_b : 0) - o_low;
            const int i0 = m.ok ? (at + u0) * UNIT : BUF_OOB, i1 = m.ok && turns ? (at + u1) * UNIT : BUF_OOB;
            if constexpr (ADJ) {
                // (a lane of channels that are not turned reads V of them)
                m.z = buf_read<Both>(in, turns ? i0 : BUF_OOB);
                if (rot < w.per_head) m.x = buf_read<Part>(in, turns ? BUF_OOB : i0);
            } else {
                m.x = buf_read<Part>(in, i0);
                m.y = buf_read<Part>(in, i1);
            }
            if constexpr (EACH) weights(weight + (m.ok ? h : 0) * weight_head, m.w);
            return m;
        };
        if (first >= end) return;
        if constexpr (!EACH) {
            weights(weight, wt);
#pragma unroll
            for (int i = 0; i < V; ++i) wt[0][i] += a.offset, wt[1][i] += a.offset;
        }
        Item ahead[AHEAD];
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
            if (first + 4 * d < end) ahead[d] = read(first + 4 * d);
        for (int n = first; n < end; n += 4) {
            const Item m = ahead[0];
#pragma unroll
            for (int d = 1; d < AHEAD; ++d) ahead[d - 1] = ahead[d];
            if (n + 4 * AHEAD < end) ahead[AHEAD - 1] = read(n + 4 * AHEAD);
            float u[2][V];
            if constexpr (ADJ) {
#pragma unroll
                for (int i = 0; i < V; ++i) u[0][i] = (float)m.z.e[i], u[1][i] = (float)m.z.e[V + i];
                if (rot < w.per_head) {
#pragma unroll
                    for (int i = 0; i < V; ++i) u[0][i] = turns ? u[0][i] : (float)m.x.e[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) u[0][i] = (float)m.x.e[i], u[1][i] = (float)m.y.e[i];
            }
            auto squares = [&](float f) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float p = u[0][i] * f, q = u[1][i] * f;
                    ss = fmaf(p, p, fmaf(q, q, ss));
                }
                return lanes_sum<G>(ss);
            };
            const float ss = squares(1.f);
            float inv = __builtin_amdgcn_rsqf(fmaf(ss, mean, a.eps));
            // heads whose squares pass an f32's range, either way (as of a row of the norm)
            const bool far = ss > kFar, near = ss < kNear && a.eps < kNear;
            if (__builtin_expect(__any(far || near), 0)) {
                const float f = far ? kFarUnit : near ? kNearUnit : 1.f;
                const Root root = {__builtin_amdgcn_rsqf(fmaf(squares(f), mean, a.eps * f * f)), far ? 1.f : f, far ? f : 1.f};
#pragma unroll
                for (int i = 0; i < V; ++i) u[0][i] = root.of(u[0][i]), u[1][i] = root.of(u[1][i]);
                inv = 1.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float w0 = EACH ? m.w[0][EACH ? i : 0] + a.offset : wt[0][i], w1 = EACH ? m.w[EACH ? 1 : 0][EACH ? i : 0] + a.offset : wt[1][i];
                u[0][i] = u[0][i] * inv * w0, u[1][i] = u[1][i] * inv * w1;
            }
            const int o0 = m.ok ? (m.out + u0) * UNIT : BUF_OOB, o1 = m.ok && turns ? (m.out + u1) * UNIT : BUF_OOB;
            const float2 *cs = turn + (m.ok && turns ? __mul24(m.t, r.pairs) + g * V : 0);
            if constexpr (ADJ) {
                Both z;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float p = u[2 * i / V][2 * i % V], q = u[(2 * i + 1) / V][(2 * i + 1) % V];
                    z.e[2 * i] = (T)fmaf(p, cs[i].x, -q * cs[i].y);
                    z.e[2 * i + 1] = (T)fmaf(p, cs[i].y, q * cs[i].x);
                }
                buf_write(out, turns ? o0 : BUF_OOB, z);
                if (rot < w.per_head) {
                    Part x;
#pragma unroll
                    for (int i = 0; i < V; ++i) x.e[i] = (T)u[0][i];
                    buf_write(out, turns ? BUF_OOB : o0, x);
                }
            } else {
                Part x, y;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float c = cs[i].x, s = cs[i].y;
                    x.e[i] = (T)(turns ? fmaf(u[0][i], c, -u[1][i] * s) : u[0][i]);
                    y.e[i] = (T)fmaf(u[0][i], s, u[1][i] * c);
                }
                buf_write(out, o0, x);
                buf_write(out, o1, y);
            }
        }
    };
    walk(r.q, r.qo, r.sq, r.sqo, a.qw, a.qw_head, r.hq, w.of[0], wave);
    // (k's turns follow q's from wave to wave)
    if (r.hk) walk(r.k, r.ko, r.sk, r.sko, a.kw, a.kw_head, r.hk, w.of[1], (wave - (n_tok * r.hq + H - 1) / H) & 3);
}

template <typename T, bool ADJ, int V, int G, int P>
hipError_t norm_rotary_launch(const NormRotaryArgs &a, const NormRotaryWalk &w, hipStream_t st) {
    const long long all = (long long)a.r.batch * a.r.tokens;
    const dim3 grid((unsigned)((all + w.tb - 1) / w.tb));
    const size_t lds = (size_t)w.tb * a.r.pairs * sizeof(float2);
    RotaryTurns<P> x;
    std::copy_n(a.r.freq, P, x.freq);
    std::copy_n(a.r.axis, P, x.axis);
    // (where only one of q and k has a row of weights for each head, the other takes its one row for each)
    if (a.qw_head || a.kw_head) return enqueue(k_norm_rotary<T, ADJ, V, G, true, P>, grid, dim3(256), lds, st, a.r, a, w, x);
    return enqueue(k_norm_rotary<T, ADJ, V, G, false, P>, grid, dim3(256), lds, st, a.r, a, w, x);
}

template <typename T, bool ADJ, int V>
hipError_t norm_rotary_of(const NormRotaryArgs &a, const NormRotaryWalk &w, hipStream_t st) {
    if constexpr (V > 1) {
        if (a.r.pairs > 64) {  // over 64 / V lanes
            if constexpr (V == 8)
                if (w.per_head <= 16) return norm_rotary_launch<T, ADJ, V, 16, 128>(a, w, st);
            if constexpr (V >= 4)
                if (w.per_head <= 32) return norm_rotary_launch<T, ADJ, V, 32, 128>(a, w, st);
            return norm_rotary_launch<T, ADJ, V, 64, 128>(a, w, st);
        }
    }
    if (w.per_head <= 4) return norm_rotary_launch<T, ADJ, V, 4, 64>(a, w, st);
    if (w.per_head <= 8) return norm_rotary_launch<T, ADJ, V, 8, 64>(a, w, st);
    if (w.per_head <= 16) return norm_rotary_launch<T, ADJ, V, 16, 64>(a, w, st);
    if (w.per_head <= 32) return norm_rotary_launch<T, ADJ, V, 32, 64>(a, w, st);
    return norm_rotary_launch<T, ADJ, V, 64, 64>(a, w, st);
}

// Whether offsets of an array within a workgroup's tokens, and across an entry's end where another follows, are
// 32-bit ones. (65536 tokens of 32 + 8 + 8 bf16 heads of 128 in one array of 805 MB, one entry: 247 us; by a wave a
// head, as if an entry followed 805 MB back, 1539.)
bool norm_rotary_offsets(const Strides &s, int tb, int batch, int tokens, int heads, int width, int size, int unit, int &t, int &h, int &b) {
    const __int128 next = batch > 1 ? ((__int128)s.b - (__int128)tokens * s.t) * size : 0, most = BUF_MAX_BYTES / 4;
    if ((__int128)tb * s.t * size > most || (__int128)heads * s.h * size > most || next > most || next < -most || width * size > (1 << 20)) return false;
    // (factors of 24 bits)
    if (s.t / unit >= (1 << 23) || s.h / unit >= (1 << 23)) return false;
    t = (int)(s.t / unit), h = (int)(s.h / unit), b = (int)(next / (unit * size));
    return true;
}

template <typename T>
hipError_t norm_rotary_type(const NormRotaryArgs &a, hipStream_t st) {
    constexpr int size = sizeof(T);
    NormRotaryArgs c = a;
    RotaryArgs &r = c.r;
    // entries of one token without lengths are the tokens of one entry
    if (r.tokens == 1 && !r.lens && r.pos_b % r.axes == 0 && (r.pos_b == r.axes || r.batch == 1)) {
        r.tokens = r.batch, r.batch = 1;
        r.sq.t = r.sq.b, r.sk.t = r.sk.b, r.sqo.t = r.sqo.b, r.sko.t = r.sko.b;
        r.sq.b = r.sk.b = r.sqo.b = r.sko.b = r.pos_b = 0;
    }
    int v = std::min(aligned_elements(r.q, r.sq, size), aligned_elements(r.qo, r.sqo, size));
    if (r.hk) v = std::min(v, std::min(aligned_elements(r.k, r.sk, size), aligned_elements(r.ko, r.sko, size)));
    const int most = v;
    // V pairs a lane, as in k_rotary
    if (r.adjacent) v /= 2;
    while (v > 1 && (r.pairs % v || (r.width - 2 * r.pairs) % v)) v /= 2;
    // (adjacent pairs of odd addresses, and heads of more than a wave's lanes, element by element)
    NormRotaryWalk w{};
    bool fits = most >= (r.adjacent ? 2 : 1) && (r.width - r.pairs) / v <= 64;
    if (fits) {
        w.per_head = (r.width - r.pairs) / v;
        const long long all = (long long)r.batch * r.tokens, fill = std::max(1LL, all / (4LL * cu_count()));
        // tokens of 12 KB in all, fewer where that leaves CUs without work (16384 tokens, 32 + 8 bf16 heads
        // of 128, 10 KB each: 62.9 us, by two 65.3, by four 68; 2 x 23400, 6 + 6 f32 heads of 30, 1.4 KB each: 37.3
        // by eight, 73 by one, 39.4 by four and by sixteen)
        w.tb = (int)std::max(1LL, std::min({12288 / ((long long)(r.hq + r.hk) * r.width * size), fill, (long long)r.tokens}));
        fits = all / w.tb < (1 << 24) - 1 && w.tb * std::max(r.hq, r.hk) <= (1 << 15);  // (by_heads is exact that far)
        auto set = [&](int k, const Strides &in, const Strides &out, int heads) {
            NormRotaryWalk::Of &o = w.of[k];
            o.by_heads = (unsigned)(((1ULL << 32) + heads - 1) / heads);
            return norm_rotary_offsets(in, w.tb, r.batch, r.tokens, heads, r.width, size, v, o.in_t, o.in_h, o.in_b) &&
                   norm_rotary_offsets(out, w.tb, r.batch, r.tokens, heads, r.width, size, v, o.out_t, o.out_h, o.out_b);
        };
        fits = fits && set(0, r.sq, r.sqo, r.hq) && (!r.hk || set(1, r.sk, r.sko, r.hk));
    }
    if (fits) {
        if (r.adjacent) switch (v) {
                case 4:
                    if constexpr (size == 2) return norm_rotary_of<T, true, 4>(c, w, st);
                    break;
                case 2: return norm_rotary_of<T, true, 2>(c, w, st);
                case 1: return norm_rotary_of<T, true, 1>(c, w, st);
            }
        else switch (v) {
                case 8:
                    if constexpr (size == 2) return norm_rotary_of<T, false, 8>(c, w, st);
                    break;
                case 4: return norm_rotary_of<T, false, 4>(c, w, st);
                case 2: return norm_rotary_of<T, false, 2>(c, w, st);
                case 1: return norm_rotary_of<T, false, 1>(c, w, st);
            }
    }
    const long long items = (long long)a.r.batch * a.r.tokens * (a.r.hq + a.r.hk);
    return enqueue(k_norm_rotary_heads<T>, dim3((unsigned)std::min((items + 3) / 4, 1LL << 20)), dim3(256), 0, st, a);
}

}  // namespace

hipError_t launch_norm_rotary_op(int dtype, const NormRotaryArgs &a, hipStream_t st) {
    switch (dtype) {
        case 0: return norm_rotary_type<float>(a, st);
        case 1: return norm_rotary_type<half_t>(a, st);
        case 2: return norm_rotary_type<bfloat_t>(a, st);
    }
    return hipErrorInvalidValue;
}

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
        case 0: return e4m3 ? rms_type<float, true>(a, st) : rms_type<float, false>(a, st);
        case 1: return e4m3 ? rms_type<half_t, true>(a, st) : rms_type<half_t, false>(a, st);
        case 2: return e4m3 ? rms_type<bfloat_t, true>(a, st) : rms_type<bfloat_t, false>(a, st);
    }
    return hipErrorInvalidValue;
}
