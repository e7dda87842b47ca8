// s2s_attention.h - the attention kernels of s2s_attention_*.hip, one file per
// element type (templates here), and what they share with the launcher.
//
// A query head h reads key head h / group, so the `group` heads of one key head
// and the query tokens are one axis of "columns": column c is token c / group,
// head c % group. A workgroup takes the columns of one (batch entry, key head)
// and walks the key tiles once, with the running maximum and sum of the softmax.
//
// Scores are made transposed, S^T = K Q^T on the 16x16 MFMAs: lane l holds
// column l % 16 and, in accumulator register i of key block kb, key 16 kb + 4 (l /
// 16) + i. A column's softmax is then within a lane but for two swaps across the
// four lane groups, and exp(S)^T is already in the B operand's layout of O^T =
// V^T P^T if the contraction's slots are numbered that way (32 slots: lane group
// q holds keys 4 q .. 4 q + 3 of two key blocks); V^T comes out of V's rows in LDS by
// the transposing LDS read (16-bit types) or by plain reads (f32, whose MFMA takes
// one key per lane group). Nothing of the scores passes through LDS or HBM.
#pragma once

#include <algorithm>
#include <cmath>

#include "s2s_device.h"
#include "s2s_kernels.h"
#include "s2s_ops.h"

// What a launch adds to the call's arguments.
struct AttnLaunch {
    int cols;       // group * nq
    int tiles;      // column tiles per (batch entry, key head)
    int splits;     // key ranges per column tile
    int vec;        // bytes of one element-wise access (unaligned arrays): 8, 4 or 2
    int out_vec;    // the output takes 4 elements at once
    float *part_o;  // splits > 1: [batch * hk][splits][cols][DP] unnormalised sums
    float *part_ml;  // [batch * hk][splits][cols][2]: reference and sum of the weights
    const int4 *meta;  // documents: [batch][key tiles] {smallest, largest id >= 0, smallest id, 0}
    int meta_tiles;
};

namespace attn {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
struct Type;
// V: 16 bytes of elements. kShift: weights are 2^kShift times e^(s - max), so that f16's
// smallest normal number, 2^-14, is 2^-24 of a row's largest weight and a long row of small
// weights is not lost below it. kLazy: how many powers of two a score may pass the
// reference before sums are rescaled (2^(kShift + kLazy) stays below f16's 65504).
template <>
struct Type<half_t> {
    typedef h8 V;
    static constexpr int kElems = 8;
    static constexpr float kShift = 10.f, kLazy = 5.f;
};
template <>
struct Type<bfloat_t> {
    typedef b8 V;
    static constexpr int kElems = 8;
    static constexpr float kShift = 0.f, kLazy = 8.f;
};
template <>
struct Type<float> {
    typedef f4v V;
    static constexpr int kElems = 4;
    static constexpr float kShift = 0.f, kLazy = 8.f;
};

__device__ __forceinline__ f4v mma(h8 a, h8 b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4v mma(b8 a, b8 b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// 16 channels of f32 as four products; slot q of product e is channel 4 q + e
__device__ __forceinline__ f4v mma(f4v a, f4v b, f4v c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = MFMA16(a[e], b[e], c);
    return c;
}

// Row r of a tile lies at r * CH chunks of 16 bytes (CH a power of two), its
// chunks permuted so that the 256 bytes a group of lanes reads at once lie in
// different banks. K: 16 rows' same chunk. V: the 32 bytes (f32: 64) that one
// 16-lane group reads of four rows (f32: that each of four rows 4 apart gives).
template <int CH>
__device__ __forceinline__ int k_slot(int r, int c) {
    constexpr int RPL = CH >= 16 ? 1 : 16 / CH, M = CH >= 16 ? 15 : CH - 1;
    return r * CH + (c ^ ((r / RPL) & M));
}
template <int CH, bool F32>
__device__ __forceinline__ int v_slot(int r, int c) {
    if constexpr (F32) {
        constexpr int M = CH >= 16 ? 3 : CH / 4 - 1;
        return r * CH + (c ^ (((r >> 2) & M) << 2));
    } else {
        constexpr int RPL = CH >= 16 ? 1 : 16 / CH, M = CH >= 16 ? 7 : CH / 2 - 1;
        return r * CH + (c ^ (((r / RPL) & M) << 1));
    }
}

// max and sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ void swap16(float &a, float &b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ float col_max(float x) {
    float y = x;
    swap16(x, y);
    return half_max(fmaxf(x, y));
}
__device__ __forceinline__ float col_sum(float x) {
    float y = x;
    swap16(x, y);
    return half_sum(x + y);
}

// 16 bytes of a row from channel c on, element by element in accesses of `vec`
// bytes; zeros from channel n on.
template <typename T>
__device__ __forceinline__ v4u load_chunk(const T *row, int c, int n, int vec) {
    constexpr int E = Type<T>::kElems;
    union {
        T e[E];
        unsigned d[4];
        unsigned long long l[2];
        v4u v;
    } u;
    u.v = v4u{0, 0, 0, 0};
    const int left = min(n - c, E);
    const T *p = row + c;
    if (vec == 8) {
        constexpr int S = 8 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (left >= (i + 1) * S) u.l[i] = *(const unsigned long long *)(p + i * S);
            else {
#pragma unroll
                for (int e = 0; e < S; ++e)
                    if (left > i * S + e) u.e[i * S + e] = p[i * S + e];
            }
    } else if (vec == 4) {
        constexpr int S = 4 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (left >= (i + 1) * S) u.d[i] = *(const unsigned *)(p + i * S);
            else if (S > 1 && left > i * S) u.e[i * S] = p[i * S];
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (left > e) u.e[e] = p[e];
    }
    return u.v;
}

// Whether any of 16 bytes' elements is an infinity or NaN.
__device__ __forceinline__ bool any_wild(h8 x) {
    const v4u u = __builtin_bit_cast(v4u, x);
    bool w = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (u[i] & 0x7c00u) == 0x7c00u || (u[i] & 0x7c000000u) == 0x7c000000u;
    return w;
}
__device__ __forceinline__ bool any_wild(b8 x) {
    const v4u u = __builtin_bit_cast(v4u, x);
    bool w = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (u[i] & 0x7f80u) == 0x7f80u || (u[i] & 0x7f800000u) == 0x7f800000u;
    return w;
}
__device__ __forceinline__ bool wild(float x) {
    return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u;
}
// (by value: __builtin_bit_cast of a vector's element reads element 0)
__device__ __forceinline__ bool any_wild(f4v x) { return wild(x[0]) || wild(x[1]) || wild(x[2]) || wild(x[3]); }

// One workgroup: 4 waves, the columns of one tile of a (batch entry, key head),
// one range of the keys.
//  WK false: wave w has columns 16 NB w .. + 16 NB of the tile's 64 NB, all keys.
//  WK true (at most 16 columns): every wave has all columns and a quarter of each
//  key tile (one block of 16 keys of 64); the four sums meet in LDS at the end.
// K and V tiles of TK keys are copied straight into LDS, two buffers each, the
// next tile in flight while one is computed. ALIGNED: rows of 16-byte multiples,
// copied by the DMA; otherwise through registers in narrower accesses.
template <typename T, int DP, int NB, bool WK, bool ALIGNED>
struct Kernel {
    typedef Type<T> Ty;
    typedef typename Ty::V Vec;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int E = Ty::kElems;
    static constexpr int TK = F32 && !WK ? 32 : 64;
    static constexpr int KB = WK ? 1 : TK / 16;          // key blocks per wave
    static constexpr int KS = DP / (4 * E);              // steps of four chunks
    static constexpr int DB = DP / 16;                   // channel blocks of the output
    static constexpr int CHD = DP / E;                   // chunks per row
    static constexpr int CH = CHD <= 4 ? 4 : CHD <= 8 ? 8 : CHD <= 16 ? 16 : 32;
    static constexpr int COLS = WK ? 16 : 64 * NB;       // columns per workgroup
    static constexpr int LOADS = TK * CH / 256;          // chunks per thread and tile
    static constexpr size_t kTile = (size_t)TK * CH * 16;
    static constexpr size_t kJoin = WK ? (size_t)4 * 16 * (DP + 4) * 4 : 0;
    static constexpr size_t kLds = 4 * kTile > kJoin ? 4 * kTile : kJoin;

    static __device__ void run(const AttnOpArgs &a, const AttnLaunch &L, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int n16 = lane & 15, q = lane >> 4;
        // tile-major, so that with a multiple of 8 (batch, key head) pairs one XCD
        // keeps a pair's keys in its L2, and the tiles with the most keys (the last
        // ones, under the causal mask) start first
        const int nbh = a.batch * a.hk;
        const int bh = blockIdx.x % nbh, rest = blockIdx.x / nbh;
        const int ct = L.tiles - 1 - rest % L.tiles, split = rest / L.tiles;
        const int b = bh / a.hk, kvh = bh - b * a.hk;
        const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
        const int kl = a.k_lens ? min(max(a.k_lens[b], 0), a.nk) : a.nk;
        const int c0 = ct * COLS;
        if (c0 >= ql * a.group) return;  // (the whole workgroup; ql * group <= 2^30)
        const int pre = a.prefix ? a.prefix[b] : 0;
        auto limit = [&](int i) { return a.causal ? min(kl, max(max(kl - ql + i + 1, pre), 0)) : kl; };

        // the columns of this lane
        const int wc0 = WK ? c0 : c0 + wave * 16 * NB;
        int tok[NB], lim[NB], doc[NB], at[NB];
        const float *tab[NB];
        float slope[NB];
        Vec qf[NB][KS];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int c = wc0 + nb * 16 + n16, i = c / a.group, h = kvh * a.group + (c - i * a.group);
            const bool ok = i < ql;
            tok[nb] = ok ? i : -1;
            lim[nb] = ok ? limit(i) : 0;
            doc[nb] = 0;
            if (a.q_docs && ok) {
                doc[nb] = a.q_docs[b * a.q_docs_b + i];
                if (doc[nb] < 0) lim[nb] = 0;
            }
            at[nb] = a.q_pos && ok ? a.q_pos[b * a.q_pos_b + i] : kl - ql + i;
            slope[nb] = a.slopes && ok ? a.slopes[h] * kLog2e : 0.f;
            tab[nb] = a.table ? a.table + (long long)(ok ? h : 0) * a.table_size : nullptr;
            const T *row = (const T *)a.q + b * a.sq.b + (long long)(ok ? i : 0) * a.sq.t + h * a.sq.h;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int c = (4 * ks + q) * E;
                v4u x = {0, 0, 0, 0};
                if (ok && c < a.width) {
                    if constexpr (ALIGNED) x = *(const v4u *)(row + c);
                    else x = load_chunk<T>(row, c, a.width, L.vec);
                }
                qf[nb][ks] = __builtin_bit_cast(Vec, x);
            }
        }
        // keys that any column of the workgroup (of the wave) may read, and that all may
        const int i_last = min(ql - 1, (c0 + COLS - 1) / a.group);
        const int wg_max = limit(i_last);
        const int w_first = min(ql - 1, wc0 / a.group), w_last = min(ql - 1, (wc0 + 16 * NB - 1) / a.group);
        const bool w_any = wc0 < ql * a.group;
        const int w_max = w_any ? limit(w_last) : 0, w_min = limit(w_first);
        // documents of the workgroup's columns
        int q_lo = 0, q_hi = 0, q_min = 0;
        if (a.q_docs) {
            q_lo = 0x7fffffff, q_hi = -1, q_min = 0x7fffffff;
            const int i_first = c0 / a.group;
            for (int i = i_first + lane; i <= i_last; i += 64) {
                const int d = a.q_docs[b * a.q_docs_b + i];
                q_min = min(q_min, d);
                if (d >= 0) q_lo = min(q_lo, d), q_hi = max(q_hi, d);
            }
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                q_lo = min(q_lo, __shfl_xor(q_lo, m));
                q_hi = max(q_hi, __shfl_xor(q_hi, m));
                q_min = min(q_min, __shfl_xor(q_min, m));
            }
            q_lo = __builtin_amdgcn_readfirstlane(q_lo);
            q_hi = __builtin_amdgcn_readfirstlane(q_hi);
            q_min = __builtin_amdgcn_readfirstlane(q_min);
        }
        const int nt = q_hi < 0 ? 0 : (wg_max + TK - 1) / TK;
        const int per = (nt + L.splits - 1) / L.splits;
        const int t_end = min(nt, (split + 1) * per);

        // the next tile from t on that holds a key some column's document has, and
        // whether all its keys and the columns are of one document
        unsigned long long live = 0, whole = 0;
        int live_at = -64;
        auto next = [&](int t) {
            if (!L.meta) return t;
            while (t < t_end) {
                if (t >= live_at + 64) {
                    live_at = t;
                    const int m = t + lane;
                    bool l = false, w = false;
                    if (m < t_end) {
                        const int4 x = L.meta[(long long)b * L.meta_tiles + m];
                        l = x.x <= q_hi && x.y >= q_lo;
                        w = x.z == x.y && q_min == q_hi && x.y == q_hi;
                    }
                    live = __ballot(l);
                    whole = __ballot(w);
                }
                const unsigned long long m = live >> (t - live_at);
                if (m) return t + (int)__builtin_ctzll(m);
                t = live_at + 64;
            }
            return t_end;
        };

        // copying a tile: this thread's chunks
        const T *kbase = (const T *)a.k + b * a.sk.b + kvh * a.sk.h;
        const T *vbase = (const T *)a.v + b * a.sv.b + kvh * a.sv.h;
        const int kst = (int)a.sk.t, vst = (int)a.sv.t;  // below 2^22
        auto stage = [&](int t, int buf) {
            char *kd = lds + buf * 2 * kTile, *vd = kd + kTile;
            const long long j0 = (long long)t * TK;
            const T *kp = kbase + j0 * kst, *vp = vbase + j0 * vst;
            const int left = kl - t * TK;
            if constexpr (ALIGNED) {
                const __amdgpu_buffer_rsrc_t kr = buf_rsrc(kp, BUF_MAX_BYTES), vr = buf_rsrc(vp, BUF_MAX_BYTES);
#pragma unroll
                for (int n = 0; n < LOADS; ++n) {
                    const int s = (n * 4 + wave) * 64 + lane, r = s / CH;
                    const int kc = k_slot<CH>(r, s & (CH - 1)) & (CH - 1), vc = v_slot<CH, F32>(r, s & (CH - 1)) & (CH - 1);
                    const bool ok = r < left;
                    dma16(kr, (float *)(kd + (size_t)(n * 4 + wave) * 1024),
                          ok && kc * E < a.width ? (r * kst + kc * E) * (int)sizeof(T) : BUF_OOB);
                    dma16(vr, (float *)(vd + (size_t)(n * 4 + wave) * 1024),
                          ok && vc * E < a.width ? (r * vst + vc * E) * (int)sizeof(T) : BUF_OOB);
                }
            } else {
                v4u x[2][LOADS];
#pragma unroll
                for (int n = 0; n < LOADS; ++n) {
                    const int s = n * 256 + tid, r = s / CH, c = s & (CH - 1);
                    x[0][n] = x[1][n] = v4u{0, 0, 0, 0};
                    if (r < left && c * E < a.width) {
                        x[0][n] = load_chunk<T>(kp + (long long)r * kst, c * E, a.width, L.vec);
                        x[1][n] = load_chunk<T>(vp + (long long)r * vst, c * E, a.width, L.vec);
                    }
                }
#pragma unroll
                for (int n = 0; n < LOADS; ++n) {
                    const int s = n * 256 + tid, r = s / CH, c = s & (CH - 1);
                    *(v4u *)(kd + k_slot<CH>(r, c) * 16) = x[0][n];
                    *(v4u *)(vd + v_slot<CH, F32>(r, c) * 16) = x[1][n];
                }
            }
        };

        f4v o[DB][NB];
        float m[NB], l[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb] = -INFINITY;
            l[nb] = 0.f;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db][nb] = f4v{0.f, 0.f, 0.f, 0.f};
        }
        const float c1 = a.cap > 0.f ? a.scale / a.cap * (2.f * kLog2e) : a.scale * kLog2e;
        const float capl = a.cap * kLog2e;
        const bool biased = a.slopes || a.table;

        int t = next(split * per), buf = 0;
        if (t < t_end) stage(t, 0);
        while (t < t_end) {
            const bool one_doc = !a.q_docs || (L.meta && ((whole >> (t - live_at)) & 1));
            const int tn = next(t + 1);
            if constexpr (ALIGNED) WAIT_VMCNT(0);
            lds_sync();
            if (tn < t_end) stage(tn, buf ^ 1);
            const int j0 = t * TK + (WK ? 16 * wave : 0);  // the wave's first key
            if (j0 < w_max) {
                const char *kd = lds + buf * 2 * kTile, *vd = kd + kTile;
                const bool full = j0 + 16 * KB <= w_min && one_doc && !a.table;
                tile(a, L, kd, vd, j0, b, kl, full, biased, c1, capl, lim, doc, at, slope, tab, qf, o, m, l);
            }
            t = tn;
            buf ^= 1;
        }

#pragma unroll
        for (int nb = 0; nb < NB; ++nb) l[nb] = col_sum(l[nb]);
        if constexpr (WK) {
            // the four waves' sums, rescaled to their largest reference
            __syncthreads();
            float *jo = (float *)lds + wave * 16 * (DP + 4), *jm = (float *)lds;
            float *mine = jo + n16 * (DP + 4);
#pragma unroll
            for (int db = 0; db < DB; ++db) *(f4v *)(mine + db * 16 + 4 * q) = o[db][0];
            if (q == 0) mine[DP] = m[0], mine[DP + 1] = l[0];
            __syncthreads();
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, jm[(w * 16 + n16) * (DP + 4) + DP]);
            float ls = 0.f, f[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float *p = jm + (w * 16 + n16) * (DP + 4) + DP;
                // a wave without keys has nothing to add (a NaN sum is passed on)
                f[w] = p[1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(p[0] - (top == -INFINITY ? 0.f : top));
                if (p[1] != p[1] && p[0] == -INFINITY) f[w] = 1.f;
                ls += p[1] == 0.f ? 0.f : f[w] * p[1];
            }
            m[0] = top;
            l[0] = ls;
            // wave w finishes channel blocks w, w + 4, ...
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                if ((db & 3) != wave) continue;
                f4v s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const f4v x = *(const f4v *)(jm + (w * 16 + n16) * (DP + 4) + db * 16 + 4 * q);
                    if (f[w] != 0.f) s += x * f[w];
                }
                o[db][0] = s;
            }
        }
        // out, or the sums of this key range
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if (tok[nb] < 0) continue;
            const int c = wc0 + nb * 16 + n16;
            if (L.splits > 1) {
                const long long row = ((long long)bh * L.splits + split) * L.cols + c;
                float *po = L.part_o + row * DP;
                if (q == 0 && (!WK || wave == 0)) {
                    L.part_ml[2 * row] = m[nb];
                    L.part_ml[2 * row + 1] = l[nb];
                }
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    if (!WK || (db & 3) == wave) *(f4v *)(po + db * 16 + 4 * q) = o[db][nb];
            } else {
                const int h = kvh * a.group + (c - tok[nb] * a.group);
                T *row = (T *)a.out + b * a.so.b + (long long)tok[nb] * a.so.t + h * a.so.h;
                const float r = l[nb] == 0.f ? 0.f : 1.f / l[nb];
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    if (WK && (db & 3) != wave) continue;
                    store(row, db * 16 + 4 * q, a.width, L.out_vec, o[db][nb] * r);
                }
            }
        }
    }

    static __device__ __forceinline__ void store(T *row, int c, int width, int vec, f4v x) {
        VecOf<T, 4> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.e[i] = (T)x[i];
        if (vec) {
            if (c < width) *(VecOf<T, 4> *)(row + c) = y;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < width) row[c + i] = y.e[i];
        }
    }

    // V^T's operand for channel block db: the keys of blocks 2 j and 2 j + 1 (f32: of
    // block j, one key per lane group and register). With WK the wave's one block.
    static __device__ __forceinline__ Vec v_operand(const char *vd, int j, int db, int lane) {
        const int n16 = lane & 15, q = lane >> 4, wave = threadIdx.x >> 6;
        if constexpr (F32) {
            f4v x;
            const int r0 = 16 * (WK ? wave : j) + 4 * q, c = 16 * db + n16;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = *(const float *)(vd + v_slot<CH, F32>(r0 + i, c >> 2) * 16 + (c & 3) * 4);
            return x;
        } else {
            const int r = 16 * (WK ? wave : 2 * j) + 4 * q + (n16 >> 2), c = 16 * db + 4 * (n16 & 3);
            union {
                s4 h[2];
                Vec v;
            } u;
            u.h[0] = read_tr(vd + v_slot<CH, F32>(r, c >> 3) * 16 + (c & 4) * 2);
            if constexpr (WK) u.h[1] = s4{0, 0, 0, 0};
            else u.h[1] = read_tr(vd + v_slot<CH, F32>(r + 16, c >> 3) * 16 + (c & 4) * 2);
            return u.v;
        }
    }
    static __device__ __forceinline__ s4 read_tr(const char *p) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p);
    }

    // The wave's keys of one tile: scores, softmax step, products with V.
    static __device__ __forceinline__ void tile(const AttnOpArgs &a, const AttnLaunch &L, const char *kd, const char *vd,
                                                int j0, int b, int kl, bool full, bool biased, float c1, float capl,
                                                const int *lim, const int *doc, const int *at, const float *slope,
                                                const float *const *tab, const Vec (*qf)[KS], f4v (*o)[NB], float *m,
                                                float *l) {
        const int lane = threadIdx.x & 63, n16 = lane & 15, q = lane >> 4, wave = threadIdx.x >> 6;
        f4v s[KB][NB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[kb][nb] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int r = 16 * (WK ? wave : kb) + n16;
                const Vec x = *(const Vec *)(kd + k_slot<CH>(r, 4 * ks + q) * 16);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[kb][nb] = mma(x, qf[nb][ks], s[kb][nb]);
            }
        // scores in powers of two
        if (a.cap > 0.f) {
            // cap tanh(z) = cap (1 - 2 / (e^2z + 1))
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = __builtin_amdgcn_exp2f(s[kb][nb][i] * c1);
                        s[kb][nb][i] = fmaf(-2.f * capl, __builtin_amdgcn_rcpf(e + 1.f), capl);
                    }
        } else {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[kb][nb] *= c1;
        }
        int kpos = 0, kdoc = 0;
        const int jl = j0 + min(lane, 16 * KB - 1);
        if (biased && a.k_pos) kpos = a.k_pos[b * a.k_pos_b + min(jl, kl - 1)];
        if (!full && a.k_docs) kdoc = a.k_docs[b * a.k_docs_b + min(jl, kl - 1)];
        if (biased) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int jr = 16 * kb + 4 * q + i;
                    const int kp = a.k_pos ? __shfl(kpos, jr) : j0 + jr;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const int dist = at[nb] - kp;
                        float x = s[kb][nb][i];
                        if (a.slopes) x = fmaf(-slope[nb], fabsf((float)dist), x);
                        if (a.table) x = add_bias(x, entry(a, tab[nb], dist));
                        // lowest values stay numbers, so that a row of them is even
                        s[kb][nb][i] = x < -1e30f && x != -INFINITY ? -1e30f : x;
                    }
                }
        }
        if (!full) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int jr = 16 * kb + 4 * q + i;
                    const int kdv = a.k_docs ? __shfl(kdoc, jr) : 0;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const bool ok = j0 + jr < lim[nb] && (!a.k_docs || kdv == doc[nb]);
                        if (!ok) s[kb][nb][i] = -INFINITY;
                    }
                }
        }
        // the running reference: rescaled only where a score passes it by 2^kLazy
        float top[NB];
        bool grow = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float x = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) x = fmaxf(x, s[kb][nb][i]);
            top[nb] = col_max(x);
            grow |= top[nb] > m[nb] + Ty::kLazy;
        }
        if (__any(grow)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float mn = fmaxf(m[nb], top[nb]);
                const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nb] - mn);
                m[nb] = mn;
                l[nb] *= f;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db][nb] *= f;
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float ref = (m[nb] == -INFINITY ? 0.f : m[nb]) - Ty::kShift;
            float sum = 0.f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(s[kb][nb][i] - ref);
                    s[kb][nb][i] = p;
                    sum += p;
                }
            l[nb] += sum;
        }
        // a masked key's weight is zero, and zero times an infinity is none: with such
        // values among a masked tile's v they are added key by key
        bool wildv = false;
        if (!full) {
#pragma unroll
            for (int j = 0; j < (F32 || WK ? KB : KB / 2); ++j)
#pragma unroll
                for (int db = 0; db < DB; ++db) wildv |= any_wild(v_operand(vd, j, db, lane));
            wildv = __any(wildv);
        }
        products(vd, lane, s, o, wildv);
        if (wildv) wild_products(a, vd, j0, b, kl, lim, doc, at, tab, o);
    }

    static __device__ __forceinline__ float entry(const AttnOpArgs &a, const float *tab, int dist) {
        const int half = a.table_size >> 1;
        return tab[min(max(dist, -half), half) + half];
    }
    // bias in powers of two; minus infinity takes the key out whatever its score
    static __device__ __forceinline__ float add_bias(float x, float bias) {
        return bias == -INFINITY ? -INFINITY : fmaxf(bias, -2e38f) * kLog2e + x;
    }

    static __device__ __forceinline__ void products(const char *vd, int lane, const f4v (*s)[NB], f4v (*o)[NB], bool clean) {
        constexpr int J = F32 || WK ? KB : KB / 2;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            Vec p[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                if constexpr (F32) p[nb] = s[j][nb];
                else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[nb][i] = (T)s[WK ? 0 : 2 * j][nb][i];
                        p[nb][4 + i] = WK ? (T)0.f : (T)s[WK ? 0 : 2 * j + 1][nb][i];
                    }
                }
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                Vec x = v_operand(vd, j, db, lane);
                if (clean) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (wild((float)x[e])) x[e] = (T)0.f;
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[db][nb] = mma(x, p[nb], o[db][nb]);
            }
        }
    }

    // The infinities and NaN of the tile's v, added to the columns that read their key.
    static __device__ __forceinline__ void wild_products(const AttnOpArgs &a, const char *vd, int j0, int b, int kl,
                                                      const int *lim, const int *doc, const int *at,
                                                      const float *const *tab, f4v (*o)[NB]) {
        const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6;
        for (int jr = 0; jr < 16 * KB; ++jr) {
            const int j = j0 + jr;
            if (j >= kl) break;
            const int r = (WK ? 16 * wave : 0) + jr;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                bool ok = j < lim[nb] && (!a.k_docs || a.k_docs[b * a.k_docs_b + j] == doc[nb]);
                if (ok && a.table)
                    ok = entry(a, tab[nb], at[nb] - (a.k_pos ? a.k_pos[b * a.k_pos_b + j] : j)) != -INFINITY;
                if (!ok) continue;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = 16 * db + 4 * q + i;
                        const float v = (float)*(const T *)(vd + v_slot<CH, F32>(r, c / E) * 16 + (c % E) * sizeof(T));
                        if (wild(v)) o[db][nb][i] += v;
                    }
            }
        }
    }
};

template <typename T, int DP, int NB, bool WK, bool ALIGNED>
__global__ __launch_bounds__(256, 2) void k_attn(AttnOpArgs a, AttnLaunch L) {
    extern __shared__ __align__(16) char lds[];
    Kernel<T, DP, NB, WK, ALIGNED>::run(a, L, lds);
}

// The key ranges' sums of one column: a wave per column, a lane per two channels.
template <typename T, int DP>
__global__ __launch_bounds__(256) void k_attn_join(AttnOpArgs a, AttnLaunch L) {
    const int lane = threadIdx.x & 63;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int c = (int)(id % L.cols);
    const long long bh = id / L.cols;
    const int b = (int)(bh / a.hk), kvh = (int)(bh - (long long)b * a.hk);
    if (b >= a.batch) return;
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    const int i = c / a.group;
    if (i >= ql) return;
    const long long row0 = bh * L.splits * L.cols + c;
    float top = -INFINITY;
    for (int s = 0; s < L.splits; ++s) top = fmaxf(top, L.part_ml[2 * (row0 + (long long)s * L.cols)]);
    if (top == -INFINITY) top = 0.f;
    float ls = 0.f, o0 = 0.f, o1 = 0.f;
    for (int s = 0; s < L.splits; ++s) {
        const long long row = row0 + (long long)s * L.cols;
        const float ms = L.part_ml[2 * row], l = L.part_ml[2 * row + 1];
        if (l == 0.f) continue;  // no key in this range
        const float f = ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ms - top);
        ls = fmaf(f, l, ls);
        const float *po = L.part_o + row * DP;
        if (lane < DP) o0 = fmaf(f, po[lane], o0);
        if (lane + 64 < DP) o1 = fmaf(f, po[lane + 64], o1);
    }
    const float r = ls == 0.f ? 0.f : 1.f / ls;
    const int h = kvh * a.group + (c - i * a.group);
    T *out = (T *)a.out + b * a.so.b + (long long)i * a.so.t + h * a.so.h;
    if (lane < a.width) out[lane] = (T)(o0 * r);
    if (lane + 64 < a.width) out[lane + 64] = (T)(o1 * r);
}

// How a call is cut, from its type and sizes alone (the workspace goes by it).
struct Cut {
    int dp, nb, tk;
    bool wk;
    int tiles, splits;
};

template <typename T, int DP, int NB, bool WK, bool ALIGNED>
hipError_t launch(const AttnOpArgs &a, const AttnLaunch &L, hipStream_t st) {
    typedef Kernel<T, DP, NB, WK, ALIGNED> K;
    const long long blocks = (long long)a.batch * a.hk * L.tiles * L.splits;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (K::kLds > 65536) {
        static_assert(K::kLds <= 163840, "LDS");
        const hipError_t e = hipFuncSetAttribute((const void *)k_attn<T, DP, NB, WK, ALIGNED>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)K::kLds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((k_attn<T, DP, NB, WK, ALIGNED>), dim3((unsigned)blocks), dim3(256), K::kLds, st, a, L);
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_width(const AttnOpArgs &a, const AttnLaunch &L, const Cut &c, bool aligned, hipStream_t st) {
    hipError_t e;
    if (c.wk) e = aligned ? launch<T, DP, 1, true, true>(a, L, st) : launch<T, DP, 1, true, false>(a, L, st);
    else if (c.nb == 1) e = aligned ? launch<T, DP, 1, false, true>(a, L, st) : launch<T, DP, 1, false, false>(a, L, st);
    else e = aligned ? launch<T, DP, 2, false, true>(a, L, st) : launch<T, DP, 2, false, false>(a, L, st);
    if (e != hipSuccess || L.splits == 1) return e;
    const long long rows = (long long)a.batch * a.hk * L.cols;
    hipLaunchKernelGGL((k_attn_join<T, DP>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, L);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const AttnOpArgs &a, const AttnLaunch &L, const Cut &c, bool aligned, hipStream_t st) {
    switch (c.dp) {
        case 32: return launch_width<T, 32>(a, L, c, aligned, st);
        case 64: return launch_width<T, 64>(a, L, c, aligned, st);
        case 96: return launch_width<T, 96>(a, L, c, aligned, st);
        default: return launch_width<T, 128>(a, L, c, aligned, st);
    }
}

}  // namespace attn

hipError_t launch_attention_f32(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, bool aligned, hipStream_t st);
hipError_t launch_attention_f16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, bool aligned, hipStream_t st);
hipError_t launch_attention_bf16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, bool aligned, hipStream_t st);
