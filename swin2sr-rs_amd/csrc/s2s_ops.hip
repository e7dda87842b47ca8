// s2s_ops.hip - rotary positions with several axes, and the root-mean-square
// norm with the residual's addition and an e4m3 output. Both are bound by HBM:
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

// 1 / sqrt(mean of n squares + eps) from the squares' sum. Where that lies past an f32's range, or
// (with so small an eps) where its precision ends, it is made again of the row times 2^-80 or
// 2^80: `again(factor)`, which all threads of the row call or none. (Squares of f16 lie within 2^-48
// and 2^34, and 2^24 of them within both ends.)
template <typename T, typename F>
__device__ __forceinline__ float inverse_root(float ss, int n, float eps, const F &again) {
    constexpr bool F16 = std::is_same<T, half_t>::value;
    const bool far = !F16 && ss > 0x1p127f, near = !F16 && ss < 0x1p-100f && eps < 0x1p-100f;
    if (__builtin_expect(far || near, 0)) {
        const float f = far ? 0x1p-80f : 0x1p80f;
        return f / sqrtf(again(f) / (float)n + eps * f * f);
    }
    return 1.0f / sqrtf(ss / (float)n + eps);
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
        const float inv = inverse_root<T>(squares(1.f), a.cols, a.eps, [&](float f) {
            __syncthreads();  // `part` has been read
            return squares(f);
        });
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
        const float inv = inverse_root<T>(of_row(own), a.cols, a.eps, [&](float f) {
            if constexpr (TPR == 256) __syncthreads();  // `part` has been read
            return of_row(squares(f));
        });
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
        case 0: return e4m3 ? rms_type<float, true>(a, st) : rms_type<float, false>(a, st);
        case 1: return e4m3 ? rms_type<half_t, true>(a, st) : rms_type<half_t, false>(a, st);
        case 2: return e4m3 ? rms_type<bfloat_t, true>(a, st) : rms_type<bfloat_t, false>(a, st);
    }
    return hipErrorInvalidValue;
}
