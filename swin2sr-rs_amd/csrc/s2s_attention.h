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
//
// What bounds it, measured on an MI355X. Prompts: instructions, at the clock that power
// leaves: on 2 x 4096 causal bf16 tokens, 32 query and 8 key heads of 128, capped, the matrix
// cores are busy in 37% of the cycles and the other VALU instructions take 48%, at 2.04 GHz (341 us,
// 810 TFLOP/s of the pairs that the mask leaves); 12001 f16 tokens with slopes 38% and 43%, at 1.99
// GHz (680 us, 867 TFLOP/s); no LDS bank conflicts. (How far two waves of a SIMD could run the two at
// the same time is not known; fewer of either have made every kernel here faster.) Hence the tile's path
// counts its instructions: a polynomial for small capped scores, sums by MFMA, slopes in two
// operations, max by v_maximum3. (The maximum is looked for under a cap too: one reference for all
// of a call's rows, below the cap, gave 315 us, but left a row whose scores are all far below it
// weights of 2^-124, whose products with v are no normal numbers.) Steps: HBM (32
// sequences of up to 8192 keys, 8 x 128 bf16: 135 us, 5.07 TB/s). Small windows (1089
// of 64 f32 tokens, 6 heads of 30, table and bands): the 733 VALU and 584 scalar instructions of a
// wave for 16 columns, 79 us.
//
// With a sliding window (WINDOW) a column has a first key beside its last, and the key tiles between the sinks'
// and the workgroup's first window are passed over: 16391 causal bf16 tokens, 16 / 4 heads of 128, window 4096,
// 495 us (970 TFLOP/s), the next token of 32 sequences over 4096 keys 101 us (5.3 TB/s). Keys that a batch
// shares are walked by every entry's columns ahead of its own (WHOLE: 8 x 500 bf16 tokens behind 8191 shared keys, 32 / 8 heads
// of 128, 517 us, 1,070 TFLOP/s), or once by the columns of all entries (SHARED), in one launch with the entries' own
// keys (k_attn_both: 64 steps over 16384 and up to 1024 keys 66 us with the join, 80 in three launches).
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "s2s_device.h"
#include "s2s_kernels.h"
#include "s2s_ops.h"

constexpr float kAttnLog2e = 1.4426950408889634f;

// How a product q k becomes an exponent in powers of two.
struct AttnScore {
    float c1;    // without a cap: its factor; with one: 2 log2(e) / cap of scale q k
    float capl;  // cap in powers of two
    // cap tanh(z) for |z| <= 0.375 as x (p0 + p1 x^2 + p2 x^4 + p3 x^6) of the product x: tanh(z)
    // / z to 7e-8 (least squares, weights iterated towards equal ripple), three
    // fused operations where the exponential takes two transcendentals, and no
    // cancellation near zero. poly_max: the |x| that it holds for.
    float p0, p1, p2, p3, poly_max;
    float z;  // scale / cap
    bool general;  // a bias other than slopes by token distance
    void set(const AttnOpArgs &a) {
        // a negative or zero scale would turn masked minus infinities round: scores in
        // powers of two at once, with no slope
        general = a.table || a.k_pos || (!(a.cap > 0.f) && !(a.scale > 1e-30f));
        c1 = a.scale * kAttnLog2e;
        capl = a.cap * kAttnLog2e;
        p0 = p1 = p2 = p3 = z = 0.f;
        poly_max = -1.f;
        if (a.cap > 0.f) {
            z = a.scale / a.cap;
            const float w = z * z;
            c1 = z * (2.f * kAttnLog2e);
            // the coefficients and powers of x in the normal range
            if (std::fabs(z) > 1e-5f && std::fabs(z) < 1e5f && a.cap < 1e6f) {
                p0 = capl * z;
                p1 = p0 * w * -0.33332333f;
                p2 = p0 * w * w * 0.13289726f;
                p3 = p0 * w * w * w * -0.04848728f;
                poly_max = 0.375f / std::fabs(z);
            }
        }
    }
};

// n / d for 0 <= n < 2^31 by a multiplication: a division takes some twenty
// instructions, and the small launches do little else.
struct FastDiv {
    unsigned m;
    int s, d;
    void set(int by) {
        d = by;
        for (s = 0; (1LL << s) < by;) ++s;
        m = (unsigned)((((1ULL << s) - by) << 32) / by + 1);
    }
#ifdef __HIP_DEVICE_COMPILE__
    __device__ int of(int n) const { return (int)((__umulhi((unsigned)n, m) + (unsigned)n) >> s); }
#else
    int of(int n) const { return n / d; }
#endif
};

// What a launch adds to the call's arguments.
struct AttnLaunch {
    int cols;       // group * nq
    int tiles;      // column tiles per (batch entry, key head)
    int splits;     // key ranges per column tile
    int vec;        // bytes of one element-wise access (unaligned arrays): 8, 4 or 2
    int out_vec;    // elements that one store of the output takes: 4, 2 or 1
    // what a join reads, of one range too where it joins shared keys as well (else null without a second range):
    float *part_o;   // [batch * hk][splits][cols][DP] unnormalised sums
    float *part_ml;  // [batch * hk][splits][cols][2]: reference and sum of the weights
    const int4 *meta;  // documents: [batch][key tiles] {smallest, largest id >= 0, smallest id, 0}
    int meta_tiles;
    const int4 *col_docs;  // [batch][tiles] the same of a column tile's queries, and its key tiles
    const int *order;      // [batch][tiles] column tiles with the most key tiles first, or null
    int join;       // the ranges' sums are joined behind this launch
    int table_lds;  // the group's rows of the table fit LDS
    FastDiv by_pairs, by_tiles, by_hk, by_group, by_nq;
    // the ranges of the keys that the batch shares: their sums, number and columns (of all entries)
    float *shared_o, *shared_ml;
    int shared_splits, shared_cols;
    AttnScore score;
};

namespace attn {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = kAttnLog2e;

enum { CAP = 1, SLOPES = 2, ANY = 8, DOCS = 16, GENERAL = 32, WINDOW = 64, SHARED = 128, WHOLE = 256 };

template <typename T>
struct Type;
// V: 16 bytes of elements. kLazy: how many powers of two a score may pass the reference before
// sums are rescaled. kShift: weights are 2^kShift times e^(s - reference). For f16 10, so that its
// smallest normal number, 2^-14, is 2^-24 of a row's largest weight and a long row of small weights
// is not lost below it (2^(kShift + kLazy) stays below its 65504). For the types of f32's range
// -kLazy: no weight is above one, so that no product with a finite v passes what v has; a row's
// largest weight is 2^-8 at least, which leaves every v of 2^-118 (3e-36) and more its precision.
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
    static constexpr float kShift = -8.f, kLazy = 8.f;
};
template <>
struct Type<float> {
    typedef f4v V;
    static constexpr int kElems = 4;
    static constexpr float kShift = -8.f, kLazy = 8.f;
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

// A resource of less than 2^31 bytes (64 rows of 2^22 elements are 2^30 at most).
__device__ __forceinline__ v4u tile_rsrc(const void *p, int bytes) {
    const unsigned long long x = (unsigned long long)p;
    return v4u{(unsigned)x, (unsigned)(x >> 32) & 0xffffu, (unsigned)bytes, 0x00020000u};
}
// The direct copy of dma16 (16 or 4 bytes a lane to LDS address `to` + bytes * lane) as an
// instruction the compiler does not see through: it takes the transposing LDS
// read for a reader of whatever copy is in flight and waits for all of them in front
// of it, which leaves no copy in flight during the products. The kernel waits by
// itself, before the barrier that opens the tile. There is no result register; the
// wait states are those of a resource in scalar registers that a VALU instruction
// wrote.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved, and named as what it changes)
template <int BYTES>
__device__ __forceinline__ void tile_dma(v4u rsrc, unsigned to, int off) {
    static_assert(BYTES == 16 || BYTES == 4, "the copies' sizes");
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(to), "v"(off), "s"(rsrc)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                     :
                     : "s"(to), "v"(off), "s"(rsrc)
                     : "memory", "m0");
}
#pragma clang diagnostic pop

// LDS by byte address: a lane's address once per tile, what is constant in the
// instruction's offset.
typedef __attribute__((address_space(3))) char lds_t;
template <typename V>
__device__ __forceinline__ V lds_read(const lds_t *p, int off) {
    return *(const __attribute__((address_space(3))) V *)(p + off);
}
__device__ __forceinline__ s4 lds_read_tr(const lds_t *p, int off) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(p + off));
}
// The address itself, kept from being split into a loop-invariant part per use.
__device__ __forceinline__ const lds_t *opaque(const lds_t *p) {
    unsigned x = (unsigned)(size_t)p;
    asm volatile("" : "+v"(x));
    return (const lds_t *)(size_t)x;
}
__device__ __forceinline__ const lds_t *lds_xor(const lds_t *p, unsigned m) {
    return (const lds_t *)(size_t)((unsigned)(size_t)p ^ m);
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
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// The kernel's arguments, read again: what only the end of the kernel needs would
// otherwise take scalar registers through the loop.
struct AttnParams {
    AttnOpArgs a;
    AttnLaunch L[2];  // (the second only of a kernel that has two)
};
__device__ __forceinline__ const __attribute__((address_space(4))) AttnParams *late_params() {
    auto p = (const __attribute__((address_space(4))) AttnParams *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// The IEEE 754-2019 maximum (v_maximum3_f32), which passes a NaN on; fmaxf would quiet
// each operand first. A column with a NaN among its scores is NaN whatever its reference.
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
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

// Four channels of the output from c on, `vec` elements (4, 2, 1) a store.
    template <typename T>
__device__ __forceinline__ void store(T *row, int c, int width, int vec, f4v x) {
        VecOf<T, 4> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.e[i] = (T)x[i];
        if (vec == 4) {
            if (c < width) *(VecOf<T, 4> *)(row + c) = y;
        } else if (vec == 2) {
#pragma unroll
            for (int i = 0; i < 4; i += 2)
                if (c + i < width) *(VecOf<T, 2> *)(row + c + i) = VecOf<T, 2>{{y.e[i], y.e[i + 1]}};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < width) row[c + i] = y.e[i];
        }
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
//  MODE: CAP and SLOPES are known (0 to 3), or asked for in every tile (ANY); documents
//  (DOCS); or all of that and what AttnScore::general stands for (GENERAL); each with a
//  sliding window or without (WINDOW); or for the columns of all batch entries over keys that
//  they share (SHARED: the sums go to the ranges' join); or over those first, then over the
//  entry's own (WHOLE). Paths that a
//  kernel might take and does not cost it registers, spilled around its loop, and copies
//  where they meet.
// K and V tiles of TK keys are copied straight into LDS, two buffers each (three and four
// in flight gained nothing at any size and cost the loop 5 to 10%), the
// next tile in flight while one is computed. ALIGN: bytes of one copy by the DMA
// (16, or 4 for rows of 4-byte multiples), or 0: through registers, by elements.
template <typename T, int DP, int NB, bool WK, int ALIGN, int MODE>
struct Kernel {
    static constexpr bool WIN = MODE & WINDOW, SHARE = MODE & SHARED, ALL = MODE & WHOLE;
    static constexpr int KIND = MODE & ~(WINDOW | SHARED | WHOLE);
    static constexpr bool GEN = KIND == GENERAL, DOC = GEN || (KIND & DOCS), KNOWN = KIND < ANY;
    typedef Type<T> Ty;
    typedef typename Ty::V Vec;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr bool RETRY = WK && !F32;
    static constexpr int E = Ty::kElems;
    // keys per tile: 64, so that the barriers and the softmax's steps across lanes come half as often
    // (2048 f32 tokens, 64 wide, 147 us against 160 with 32; windows of 16 x 16, 57 and 73); 32 for f32 rows
    // over 64 wide, whose two buffers of 64 would fill 128 KB and leave a CU one workgroup
    static constexpr int TK = F32 && !WK && DP > 64 ? 32 : 64;
    static constexpr int KB = WK ? 1 : TK / 16;          // key blocks per wave
    static constexpr int KS = DP / (4 * E);              // steps of four chunks
    static constexpr int DB = DP / 16;                   // channel blocks of the output
    static constexpr int CHD = DP / E;                   // chunks per row
    static constexpr int CH = CHD <= 4 ? 4 : CHD <= 8 ? 8 : CHD <= 16 ? 16 : 32;
    static constexpr int COLS = WK ? 16 : 64 * NB;       // columns per workgroup
    static constexpr int LOADS = TK * CH / 256;          // chunks per thread and tile
    static constexpr int UNIT = ALIGN ? ALIGN : 16, SUB = 16 / UNIT;  // the copies' units, per chunk
    static constexpr size_t kTile = (size_t)TK * CH * 16;
    static constexpr size_t kJoin = WK ? (size_t)4 * 16 * (DP + 4) * 4 : 0;
    // two buffers of K and V (the join's sums afterwards), two of the keys' documents and
    // places, four flags, and the table's rows
    static constexpr int kIds = (int)(4 * kTile > kJoin ? 4 * kTile : kJoin), kPos = kIds + 512, kFlag = kPos + 512, kTab = kFlag + 16;
    static constexpr int kTabEntries = 2048;

    // What a tile needs that is the same for all of the workgroup.
    struct Uniform {
        const int *k_docs, *k_pos;  // of this batch entry, or null
        const float *table;
        int half;  // the table's middle
        const lds_t *tab0;  // the group's rows, in LDS
        int kl, sinks;
        bool capped, slopes, general, table_lds;
        AttnScore sc;
    };

    // (inlined into the kernel always: late_params has no meaning in a called function)
    // LAUNCH: which of the kernel's launches L is
    template <int LAUNCH = 0>
    static __device__ __forceinline__ void run(const AttnOpArgs &a, const AttnLaunch &L, int block, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = wave_of();
        const int n16 = lane & 15, q = lane >> 4;
        // tile-major, so that with a multiple of 8 (batch, key head) pairs one XCD
        // keeps a pair's keys in its L2, and the tiles with the most keys (the last
        // ones, under the causal mask) start first
        const int rest = L.by_pairs.of(block), bh = block - rest * (SHARE ? a.hk : a.batch * a.hk);
        const int split = L.by_tiles.of(rest), rank = rest - split * L.tiles;
        const int b = SHARE ? 0 : L.by_hk.of(bh), kvh = SHARE ? bh : bh - b * a.hk;
        const int ct = L.order ? L.order[b * L.tiles + rank] : L.tiles - 1 - rank;
        const int ql = SHARE ? a.batch * a.nq : a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
        int kl = !SHARE && a.k_lens ? min(max(a.k_lens[b], 0), a.nk) : a.nk;
        // the place of the first query among the keys
        int first = kl - ql;
        const int own = kl, mine = !ALL ? 0 : a.shared_lens ? min(max(a.shared_lens[b], 0), a.shared_nk) : a.shared_nk;
        if (ALL) first += mine, kl = mine;
        const int c0 = ct * COLS;
        if (c0 >= ql * a.group) return;  // (the whole workgroup; ql * group <= 2^30)
        const int pre = a.prefix ? a.prefix[b] : 0;
        auto limit = [&](int i) {
            if (WIN && !a.causal) return min(kl, max(first + i + a.window, 0));
            return a.causal ? min(kl, max(max(first + i + 1, pre), 0)) : kl;
        };
        // the first key of a query's window; before it lie only sinks that it reads
        auto start = [&](int i) { return WIN ? max(first + i + 1 - a.window, 0) : 0; };

        // the columns of this lane
        const int wc0 = WK ? c0 : c0 + wave * 16 * NB;
        int lim[NB], low[NB], doc[NB], at[NB];
        int tab[NB];  // the head's row of the table
        float slope[NB];
        Vec qf[NB][KS];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int c = wc0 + nb * 16 + n16, i = L.by_group.of(c), h = kvh * a.group + (c - i * a.group);
            bool ok = i < ql;
            const T *row;
            if constexpr (SHARE) {
                // the entry's lengths and the query's place behind its part of the shared keys
                const int e = ok ? L.by_nq.of(i) : 0, ie = i - e * a.nq;
                const int n = a.q_lens ? min(max(a.q_lens[e], 0), a.nq) : a.nq, own = a.k_lens ? min(max(a.k_lens[e], 0), a.nk) : a.nk;
                const int mine = a.shared_lens ? min(max(a.shared_lens[e], 0), a.shared_nk) : a.shared_nk;
                ok = ok && ie < n;
                at[nb] = mine + own - n + ie;
                lim[nb] = !ok ? -1 : a.causal ? min(mine, max(at[nb] + 1, 0)) : mine;
                low[nb] = doc[nb] = tab[nb] = 0;
                row = (const T *)a.q + e * a.sq.b + (long long)ie * a.sq.t + h * a.sq.h;
            } else {
                lim[nb] = ok ? limit(i) : 0;
                low[nb] = ok ? start(i) : 0;
                // (a column of no document computes what it may, and is zeroed at the end)
                doc[nb] = 0;
                if (DOC && a.q_docs && ok) doc[nb] = a.q_docs[b * a.q_docs_b + i];
                at[nb] = a.q_pos && ok ? a.q_pos[b * a.q_pos_b + i] : first + i;
                tab[nb] = ok ? (L.table_lds ? c - i * a.group : h) * a.table_size : 0;
                row = (const T *)a.q + b * a.sq.b + (long long)(ok ? i : 0) * a.sq.t + h * a.sq.h;
            }
            slope[nb] = a.slopes && ok ? slope_of(a.slopes[h]) : 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int c = (4 * ks + q) * E;
                v4u x = {0, 0, 0, 0};
                if (ok && c < a.width) {
                    if constexpr (ALIGN == 16) x = *(const v4u *)(row + c);
                    else x = load_chunk<T>(row, c, a.width, L.vec);
                }
                qf[nb][ks] = __builtin_bit_cast(Vec, x);
            }
        }
        const int *doc_keys = DOC && a.k_docs ? a.k_docs + b * a.k_docs_b : nullptr;
        const int *pos_keys = GEN && a.k_pos ? a.k_pos + b * a.k_pos_b : nullptr;
        // the sums of the weights: f32 per lane and key, over the lanes at the end; 16-bit types by
        // the matrix cores, of the rounded weights (a product with ones, half the additions' time)
        typedef typename std::conditional<F32, float, f4v>::type Sum;
        f4v o[DB][NB];
        float m[NB];
        Sum l[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb] = -INFINITY;
            l[nb] = Sum{};
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db][nb] = f4v{0.f, 0.f, 0.f, 0.f};
        }

        // this lane's first K and V addresses in a buffer: the others differ by a constant
        // or by the bits that count chunks (steps of K, channel blocks of V)
        const lds_t *base = (const lds_t *)lds;
        const lds_t *kl0 = base + k_slot<CH>((WK ? 16 * wave : 0) + n16, q) * 16;
        const int vr0 = (WK ? 16 * wave : 0) + 4 * q + (F32 ? 0 : n16 >> 2);
        const lds_t *vl0 = base + kTile + v_slot<CH, F32>(vr0, F32 ? n16 >> 2 : (n16 >> 1) & 1) * 16 +
                           (F32 ? (n16 & 3) * 4 : (n16 & 1) * 8);

        Uniform u;
        u.k_docs = doc_keys;
        u.k_pos = pos_keys;
        u.table = GEN ? a.table : nullptr;
        u.half = a.table_size >> 1;
        u.sinks = WIN ? a.sinks : 0;
        u.capped = a.cap > 0.f;
        u.slopes = a.slopes != nullptr;
        u.general = GEN && L.score.general;
        u.table_lds = GEN && L.table_lds;
        u.tab0 = base + kTab;
        u.sc = L.score;

        if (GEN && u.table_lds)
            for (int i = tid; i < a.group * a.table_size; i += 256)
                *(__attribute__((address_space(3))) float *)((lds_t *)lds + kTab + 4 * i) = a.table[kvh * a.group * a.table_size + i];

        // the keys' one part, or the shared ones' and the entry's own. (`careful`: all over again, below)
        bool careful = false;
        int shared_tiles = 0;
#pragma unroll 1
        for (int part = 0; part < (ALL ? 2 : 1); ++part) {
            if (ALL) {
                kl = part ? own : mine, first = (part ? own : mine + own) - ql;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const int i = L.by_group.of(wc0 + nb * 16 + n16);
                    lim[nb] = i < ql ? limit(i) : 0;
                    at[nb] = first + i;
                }
            }
            if ((ALL && part) || (RETRY && careful)) lds_sync();  // the buffers have been read
            // keys that any column of the workgroup (of the wave) may read, and that all may
            const int i_last = min(ql - 1, L.by_group.of(c0 + COLS - 1));
            int wg_max = 0, wg_min = 0;
            const int w_first = min(ql - 1, L.by_group.of(wc0)), w_last = min(ql - 1, L.by_group.of(wc0 + 16 * NB - 1));
            const bool w_any = wc0 < ql * a.group;
            int w_max = 0, w_min = 0, w_at = 0;  // (w_at: the first place among the wave's queries)
            if constexpr (SHARE) {
                // the limits in no order: over the wave's columns (those of no query aside), then the workgroup's
                w_min = w_at = 0x7fffffff;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    if (lim[nb] >= 0) w_max = max(w_max, lim[nb]), w_min = min(w_min, lim[nb]), w_at = min(w_at, at[nb]);
#pragma unroll
                for (int m = 1; m < 16; m *= 2) {
                    w_max = max(w_max, __shfl_xor(w_max, m));
                    w_min = min(w_min, __shfl_xor(w_min, m));
                    w_at = min(w_at, __shfl_xor(w_at, m));
                }
                w_max = __builtin_amdgcn_readfirstlane(w_max);
                w_min = __builtin_amdgcn_readfirstlane(w_min);
                w_at = __builtin_amdgcn_readfirstlane(w_at);
                w_at = w_at == 0x7fffffff ? 0 : w_at;
                if (lane == 0) ((int2 *)lds)[wave] = make_int2(w_max, w_min);
                __syncthreads();
                wg_min = 0x7fffffff;
                for (int w = 0; w < 4; ++w) wg_max = max(wg_max, ((int2 *)lds)[w].x), wg_min = min(wg_min, ((int2 *)lds)[w].y);
                __syncthreads();
                wg_max = __builtin_amdgcn_readfirstlane(wg_max);
                wg_min = __builtin_amdgcn_readfirstlane(wg_min);
                kl = wg_max;
            } else {
                wg_max = limit(i_last), wg_min = limit(L.by_group.of(c0));
                w_max = w_any ? limit(w_last) : 0, w_min = limit(w_first);
                w_at = first + w_first;
            }
            u.kl = kl;
            // what all columns' windows hold begins here, and what any holds
            // (in tiles: t_from, and the sinks' whole ones)
            const int w_low = start(w_first), t_from = WIN ? (start(i_last) + TK - 1) / TK : 0, t_whole = WIN ? a.sinks / TK : 0;
            // documents of the workgroup's columns and of the wave's, where key tiles can be passed
            // over
            int q_lo = 0, q_hi = 0, w_lo = 0, w_hi = 0;
            const bool summary = DOC && L.meta;
            if (summary) {
                const int4 x = L.col_docs[b * L.tiles + ct];
                q_lo = x.x, q_hi = x.y;
                w_lo = 0x7fffffff, w_hi = -1;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    if (lim[nb] > 0 && doc[nb] >= 0) w_lo = min(w_lo, doc[nb]), w_hi = max(w_hi, doc[nb]);
#pragma unroll
                for (int m = 1; m < 16; m *= 2) {
                    w_lo = min(w_lo, __shfl_xor(w_lo, m));
                    w_hi = max(w_hi, __shfl_xor(w_hi, m));
                }
                w_lo = __builtin_amdgcn_readfirstlane(w_lo);
                w_hi = __builtin_amdgcn_readfirstlane(w_hi);
            }
            const int nt = q_hi < 0 ? 0 : (wg_max + TK - 1) / TK;
            // under a window the tiles between the sinks' and its first one are passed over
            const int t_sinks = WIN ? min((a.sinks + TK - 1) / TK, nt) : 0;
            const int t_win = WIN ? max(t_sinks, min(start(L.by_group.of(c0)) / TK, nt)) : 0;
            const int live_tiles = nt - (t_win - t_sinks);
            // (of both parts: the own keys' tiles are counted behind the shared ones')
            const int ahead_tiles = ALL && part ? shared_tiles : 0;
            if (ALL && part == 0) shared_tiles = nt;
            const int all_tiles = ALL ? shared_tiles + (own + TK - 1) / TK : live_tiles;
            const int per = L.splits == 1 ? all_tiles : (all_tiles + L.splits - 1) / L.splits;
            auto tile_of = [&](int n) { return WIN && n >= t_sinks ? n + (t_win - t_sinks) : n; };
            const int t_end = min(nt, tile_of((split + 1) * per) - ahead_tiles), t_begin = max(tile_of(split * per) - ahead_tiles, 0);

            // the next tile from t on that holds a key some column's document has, and
            // whether all its keys and the columns are of one document
            unsigned long long live = 0, whole = 0;
            int live_at = -64, t_lo = 0, t_hi = 0, t_all = 0;
            auto next = [&](int t) {
                if (WIN && t >= t_sinks && t < t_win) t = t_win;
                if (!summary) return t;
                while (t < t_end) {
                    if (t >= live_at + 64) {
                        live_at = t;
                        const int m = t + lane;
                        bool l = false, w = false;
                        if (m < t_end) {
                            const int4 x = L.meta[(long long)b * L.meta_tiles + m];
                            t_lo = x.x, t_hi = x.y, t_all = x.z;
                            l = x.x <= q_hi && x.y >= q_lo;
                            w = x.z == x.y && q_lo == q_hi && x.y == q_hi;
                        }
                        live = __ballot(l);
                        whole = __ballot(w);
                    }
                    const unsigned long long m = live >> (t - live_at);
                    if (m) {
                        t += (int)__builtin_ctzll(m);
                        if (!WIN || t < t_sinks || t >= t_win) return t;
                        t = t_win;
                        continue;
                    }
                    t = live_at + 64;
                }
                return t_end;
            };

            // copying a tile: this thread's chunks. With the DMA a row past the keys lies
            // past the resource, which ends with the last row that is left (token strides are
            // no smaller than the width on this path), and reads as zeros, as does a
            // chunk past the width
            const bool shared_part = SHARE || (ALL && part == 0);
            const T *kp = shared_part ? (const T *)a.shared_k + kvh * a.shared_sk.h : (const T *)a.k + b * a.sk.b + kvh * a.sk.h;
            const T *vp = shared_part ? (const T *)a.shared_v + kvh * a.shared_sv.h : (const T *)a.v + b * a.sv.b + kvh * a.sv.h;
            const int kst = (int)(shared_part ? a.shared_sk.t : a.sk.t), vst = (int)(shared_part ? a.shared_sv.t : a.sv.t), kstep = TK * kst, vstep = TK * vst;  // (strides up to 2^22)
            // a wave's next units are STEP rows on; the permutations repeat every 16
            constexpr int ROW = CH * SUB, STEP = 256 / ROW, PER = STEP < 16 ? 16 / STEP : 1;
            int koff[PER], voff[PER];
#pragma unroll
            for (int p = 0; ALIGN && p < PER; ++p) {
                const int i = wave * 64 + lane, r = i / ROW + p * STEP, sl = i % ROW / SUB, sub = i % SUB * (E / SUB);
                const int kc = (k_slot<CH>(r, sl) & (CH - 1)) * E + sub, vc = (v_slot<CH, F32>(r, sl) & (CH - 1)) * E + sub;
                koff[p] = kc < a.width ? (r * kst + kc) * (int)sizeof(T) : 0x60000000;
                voff[p] = vc < a.width ? (r * vst + vc) * (int)sizeof(T) : 0x60000000;
            }
            const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(const lds_t *)lds);
            auto stage = [&](int t, int buf) {
                const int left = min(kl - t * TK, TK);
                if (DOC && doc_keys && wave == 0)
                    tile_dma<4>(tile_rsrc(doc_keys + t * TK, left * 4), lds0 + kIds + buf * 256, lane * 4);
                if (GEN && pos_keys && wave == 1)
                    tile_dma<4>(tile_rsrc(pos_keys + t * TK, left * 4), lds0 + kPos + buf * 256, lane * 4);
                if constexpr (ALIGN > 0) {
                    v4u kr = tile_rsrc(kp, ((left - 1) * kst + a.width) * (int)sizeof(T)),
                              vr = tile_rsrc(vp, ((left - 1) * vst + a.width) * (int)sizeof(T));
                    unsigned to = lds0 + buf * 2 * (unsigned)kTile + wave * 64 * UNIT;
                    if constexpr (ALL) {  // (uniform over the two parts too, which the compiler does not see)
#pragma unroll
                        for (int i = 0; i < 3; ++i) kr[i] = __builtin_amdgcn_readfirstlane(kr[i]), vr[i] = __builtin_amdgcn_readfirstlane(vr[i]);
                        to = __builtin_amdgcn_readfirstlane(to);
                    }
                    int ko[PER], vo[PER];
#pragma unroll
                    for (int p = 0; p < PER; ++p) {
                        ko[p] = koff[p], vo[p] = voff[p];
                        asm volatile("" : "+v"(ko[p]), "+v"(vo[p]));  // (sums formed here, not kept)
                    }
#pragma unroll
                    for (int n = 0; n < LOADS * SUB; ++n) {
                        tile_dma<UNIT>(kr, to + n * 256 * UNIT, ko[n % PER] + n / PER * (PER * STEP) * kst * (int)sizeof(T));
                        tile_dma<UNIT>(vr, to + (unsigned)kTile + n * 256 * UNIT, vo[n % PER] + n / PER * (PER * STEP) * vst * (int)sizeof(T));
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
                    char *kd = lds + buf * 2 * kTile, *vd = kd + kTile;
#pragma unroll
                    for (int n = 0; n < LOADS; ++n) {
                        const int s = n * 256 + tid, r = s / CH, c = s & (CH - 1);
                        *(v4u *)(kd + k_slot<CH>(r, c) * 16) = x[0][n];
                        *(v4u *)(vd + v_slot<CH, F32>(r, c) * 16) = x[1][n];
                    }
                }
            };

            // A found tile's documents: whether it and the workgroup's columns are of one, whether
            // the wave's columns have keys in it, and whether those are of one
            enum { ONE = 1, MINE = 2, SAME = 4 };
            auto documents = [&](int t) {
                if (!DOC || !doc_keys) return ONE | MINE | SAME;
                if (!summary || t >= t_end) return (int)MINE;
                const int at = t - live_at, lo = __builtin_amdgcn_readlane(t_lo, at), hi = __builtin_amdgcn_readlane(t_hi, at),
                          all = __builtin_amdgcn_readlane(t_all, at);
                return ((whole >> at) & 1 ? ONE : 0) | (lo <= w_hi && hi >= w_lo ? MINE : 0) |
                       (all == hi && w_lo == w_hi && hi == w_hi ? SAME : 0);
            };

            // the first two tiles set out together; then the next one's buffer is free when the one
            // before has been computed
            constexpr int W = 2 * LOADS * SUB;  // copies per thread and tile
            int t = next(t_begin), buf = 0, docs = documents(t);
            kp += (long long)t * kstep, vp += (long long)t * vstep;
            if (t < t_end) stage(t, 0);
            int tn = t < t_end ? next(t + 1) : t_end, docs_n = documents(tn);
            kp += (long long)(tn - t) * kstep, vp += (long long)(tn - t) * vstep;
            bool ahead = DOC && tn < t_end;
            if (ahead) stage(tn, 1);
            while (t < t_end) {
                if constexpr (ALIGN > 0) {
                    if (ahead) WAIT_VMCNT(W < 63 ? W : 63);
                    else WAIT_VMCNT(0);
                } else if (DOC) WAIT_VMCNT(0);
                lds_sync();
                if (!ahead && tn < t_end) stage(tn, buf ^ 1);
                ahead = false;
                const int at_buf = buf * 2 * (int)kTile;
                const bool inside = !WIN || t >= t_from || t < t_whole;
                if ((RETRY && careful) || !(t * TK + TK <= wg_min && (docs & ONE) && inside) || (GEN && u.table)) {
                    // a masked key's weight is zero, and zero times an infinity is none: with
                    // such values in the V of a tile that not every column reads whole, they are
                    // added by themselves to the columns that do read them, and taken out
                    lds_t *vd = (lds_t *)lds + at_buf + kTile;
                    auto *flag = (__attribute__((address_space(3))) int *)((lds_t *)lds + kFlag);
                    const bool w = __any(any_wild_chunk(vd));
                    if (lane == 0) flag[wave] = w;
                    lds_sync();
                    if (__builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3])) {
                        wild_products(u, vd, t * TK + (WK ? 16 * wave : 0), lim, low, doc, at, tab, o);
                        lds_sync();
                        remove_wild(vd);
                        lds_sync();
                    }
                }
                const int j0 = t * TK + (WK ? 16 * wave : 0);  // the wave's first key
                if (j0 < w_max && (docs & MINE) && (!WIN || j0 + 16 * KB > w_low || t < t_sinks)) {
                    const bool full = j0 + 16 * KB <= w_min && inside && (docs & SAME) && !(GEN && u.table);
                    tile(u, opaque(kl0 + at_buf), opaque(vl0 + at_buf), j0, full, j0 + 16 * KB <= w_at + 1, base + kIds + buf * 256 + (WK ? 64 * wave : 0), lim, low, doc, at, slope, tab, qf, o, m, l);
                }
                t = tn, docs = docs_n;
                buf ^= 1;
                if (t < t_end) {
                    tn = next(t + 1), docs_n = documents(tn);
                    kp += (long long)(tn - t) * kstep, vp += (long long)(tn - t) * vstep;
                }
            }
            // What the rounding of a weight left may be zero, and zero times an infinity is none: a sum that is
            // no number of weights that are is made again, with the infinities of v by themselves. (For the look: one query over
            // 131071 keys 20.9 -> 21.3 us, 32 of up to 8192 134.0 -> 134.5, in the join's own barriers 21.5 and 134.5.)
            if (RETRY && !careful && part == (ALL ? 1 : 0)) {
                bool none = false;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 4; ++i) none |= o[db][0][i] != o[db][0][i];
                auto *flag = (__attribute__((address_space(3))) int *)((lds_t *)lds + kFlag);
                lds_sync();
                if (lane == 0) flag[wave] = 0;
                if (__any(none && total_of(l[0]) == total_of(l[0])) && lane == 0) flag[wave] = 1;
                lds_sync();
                if (__builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3])) {
                    careful = true;
                    part = -1;
                    m[0] = -INFINITY, l[0] = Sum{};
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db][0] = f4v{0.f, 0.f, 0.f, 0.f};
                }
            }
        }

        float total[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if constexpr (F32) total[nb] = col_sum(l[nb]);
            else total[nb] = l[nb][0];
            if (DOC && doc[nb] < 0) {  // no document: no keys
                m[nb] = -INFINITY, total[nb] = 0.f;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db][nb] = f4v{0.f, 0.f, 0.f, 0.f};
            }
        }
        if constexpr (WK) {
            // the four waves' sums, rescaled to their largest reference
            __syncthreads();
            float *jo = (float *)lds + wave * 16 * (DP + 4), *jm = (float *)lds;
            float *mine = jo + n16 * (DP + 4);
#pragma unroll
            for (int db = 0; db < DB; ++db) *(f4v *)(mine + db * 16 + 4 * q) = o[db][0];
            if (q == 0) mine[DP] = m[0], mine[DP + 1] = total[0];
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
            total[0] = ls;
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
        const auto *late = late_params();
        const auto *launch = &late->L[LAUNCH];
        const int group = late->a.group, splits = launch->splits, width = late->a.width, vec = launch->out_vec;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int c = wc0 + nb * 16 + n16, i = (int)((__umulhi((unsigned)c, launch->by_group.m) + (unsigned)c) >> launch->by_group.s);
            if (SHARE ? lim[nb] < 0 : i >= ql) continue;
            if (SHARE || launch->part_o) {
                const long long row = ((long long)bh * splits + split) * launch->cols + c;
                float *po = launch->part_o + row * DP, *ml = launch->part_ml + 2 * row;
                if (q == 0 && (!WK || wave == 0)) ml[0] = m[nb], ml[1] = total[nb];
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    if (!WK || (db & 3) == wave) *(f4v *)(po + db * 16 + 4 * q) = o[db][nb];
            } else {
                const int h = kvh * group + (c - i * group);
                T *row = (T *)late->a.out + b * late->a.so.b + (long long)i * late->a.so.t + h * late->a.so.h;
                const float r = total[nb] == 0.f ? 0.f : 1.f / total[nb];
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    if (WK && (db & 3) != wave) continue;
                    store(row, db * 16 + 4 * q, width, vec, o[db][nb] * r);
                }
            }
        }
    }

    static __device__ __forceinline__ float total_of(float l) { return l; }
    static __device__ __forceinline__ float total_of(const f4v &l) { return l[0]; }

    // V^T's operand for channel block db (vl: the lane's address for it): the keys of
    // blocks 2 j and 2 j + 1 (f32: of block j, one key per lane group and register). With
    // WK the wave's one block, twice.
    static __device__ __forceinline__ Vec v_operand(const lds_t *vl, int j) {
        if constexpr (F32) {
            const int r = j * 16 * CH * 16;
            return f4v{lds_read<float>(vl, r), lds_read<float>(vl, r + CH * 16), lds_read<float>(vl, r + 2 * CH * 16),
                       lds_read<float>(vl, r + 3 * CH * 16)};
        } else {
            union {
                s4 h[2];
                Vec v;
            } u;
            u.h[0] = lds_read_tr(vl, j * 32 * CH * 16);
            if constexpr (WK) u.h[1] = u.h[0];
            else u.h[1] = lds_read_tr(vl, (j * 32 + 16) * CH * 16);
            return u.v;
        }
    }
    static __device__ __forceinline__ const lds_t *v_block(const lds_t *vl, int db) { return lds_xor(vl, db << (F32 ? 6 : 5)); }

    // The wave's keys of one tile: scores, softmax step, products with V.
    static __device__ __forceinline__ void tile(const Uniform &u, const lds_t *kl0, const lds_t *vl0, int j0,
                                                bool full, bool behind, const lds_t *ids, const int *lim, const int *low, const int *doc, const int *at, const float *slope, const int *tab,
                                                const Vec (*qf)[KS], f4v (*o)[NB], float *m,
                                                typename std::conditional<F32, float, f4v>::type *l) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
        // the table's entries on their way while the scores are made
        float bias[GEN ? KB : 1][4][GEN ? NB : 1];
        int place[GEN ? KB : 1][4];
        if (GEN && u.general) {
            if (u.k_pos) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const i4 x = lds_read<i4>(ids + (kPos - kIds) + 16 * q, 64 * kb);
#pragma unroll
                    for (int i = 0; i < 4; ++i) place[GEN ? kb : 0][i] = x[i];
                }
            } else {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) place[GEN ? kb : 0][i] = j0 + 16 * kb + 4 * q + i;
            }
            if (u.table) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            bias[GEN ? kb : 0][i][GEN ? nb : 0] = entry(u, tab[nb], at[nb] - place[GEN ? kb : 0][i]);
            }
        }
        f4v s[KB][NB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[kb][nb] = f4v{0.f, 0.f, 0.f, 0.f};
        const lds_t *kls[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kls[ks] = lds_xor(kl0, ks << 6);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const Vec x = lds_read<Vec>(kls[ks], kb * 16 * CH * 16);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[kb][nb] = mma(x, qf[nb][ks], s[kb][nb]);
            }
        // what is left of a score is a factor to powers of two, except where a cap or a
        // bias made it powers of two already
        const AttnScore &sc = u.sc;
        float unit = sc.c1;
        if (KNOWN ? (MODE & CAP) != 0 : u.capped) {
            float big = 0.f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    big = max3(big, fabsf(s[kb][nb][0]), fabsf(s[kb][nb][1]));
                    big = max3(big, fabsf(s[kb][nb][2]), fabsf(s[kb][nb][3]));
                }
            if (__any(!(big <= sc.poly_max))) {
                // cap tanh(z) = cap (1 - 2 / (e^2z + 1)), and the polynomial for the scores among
                // them that it holds for (the difference loses what z is smaller than one)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float t = s[kb][nb][i] * sc.z, w = t * t;
                            const float e = __builtin_amdgcn_exp2f(s[kb][nb][i] * sc.c1);
                            const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
                            const float near = t * fmaf(w, fmaf(w, fmaf(w, -0.04848728f, 0.13289726f), -0.33332333f), 1.f);
                            const float x = fabsf(t) <= 0.375f ? near : far;
                            s[kb][nb][i] = x * sc.capl;
                        }
            } else {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = s[kb][nb][i], w = x * x;
                            s[kb][nb][i] = x * fmaf(w, fmaf(w, fmaf(w, sc.p3, sc.p2), sc.p1), sc.p0);
                        }
            }
            unit = 1.f;
        }
        if (GEN && u.general) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[kb][nb][i] *= unit;
            if (u.slopes) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            s[kb][nb][i] = fmaf(-slope[nb], fabsf((float)(at[nb] - place[GEN ? kb : 0][i])), s[kb][nb][i]);
            }
            if (u.table) {
                // a bias of minus infinity takes the key out; lower values than -1e30 count as
                // that, so that a row of nothing but the type's lowest is even
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const float t = bias[GEN ? kb : 0][i][GEN ? nb : 0];
                            const float x = __builtin_elementwise_maximum(fmaf(t, kLog2e, s[kb][nb][i]), -1e30f);
                            s[kb][nb][i] = t == -INFINITY ? -INFINITY : x;
                        }
            }
            unit = 1.f;
        } else if (KNOWN ? (MODE & SLOPES) != 0 : u.slopes) {
            // distances of neighbours differ by what the register says; keys that all lie
            // behind the wave's queries, as under the causal mask, need no absolute value
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float d0 = (float)(at[nb] - j0 - 4 * q);
                if (behind) {
                    const float b0 = -slope[nb] * d0;
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[kb][nb][i] = fmaf(s[kb][nb][i], unit, fmaf(slope[nb], (float)(16 * kb + i), b0));
                } else {
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[kb][nb][i] = fmaf(s[kb][nb][i], unit, -slope[nb] * fabsf(d0 - (float)(16 * kb + i)));
                }
            }
            unit = 1.f;
        }
        if (!full) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const int n = lim[nb] - j0 - 4 * q;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * kb + i >= n) s[kb][nb][i] = -INFINITY;
                if (WIN) {
                    const int from = low[nb] - j0 - 4 * q, sinks = u.sinks - j0 - 4 * q;
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (16 * kb + i < from && 16 * kb + i >= sinks) s[kb][nb][i] = -INFINITY;
                }
            }
            if (DOC && u.k_docs) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const i4 x = lds_read<i4>(ids + 16 * q, 64 * kb);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            if (x[i] != doc[nb]) s[kb][nb][i] = -INFINITY;
                }
            }
        }
        // the running reference: rescaled only where a score passes it by 2^kLazy
        float top[NB];
        bool grow = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float x = s[0][nb][0];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) x = max3(max3(x, s[kb][nb][0], s[kb][nb][1]), s[kb][nb][2], s[kb][nb][3]);
            top[nb] = col_max(x) * unit;
            grow |= top[nb] > m[nb] + Ty::kLazy;
        }
        if (__any(grow)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float mn = fmaxf(m[nb], top[nb]);
                // (no reference yet: sums of zero, or infinities of v that stay)
                const float f = m[nb] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nb] - mn);
                m[nb] = mn;
                l[nb] *= f;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db][nb] *= f;
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float ref = Ty::kShift - (m[nb] == -INFINITY ? 0.f : m[nb]);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[kb][nb][i], unit, ref));
                    s[kb][nb][i] = p;
                    if (F32) sum[i] += p;
                }
            if constexpr (F32) l[nb] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        // the wave that multiplies goes first: the SIMD's other one then has its softmax to do beside it (8 x 500 tokens
        // behind 8191 shared keys 545 -> 517 us, a plane of f32 windows 258 -> 251, windows of a prompt as before;
        // the scores' products first too 530, 251, and theirs alone 536 and 260)
        if (KIND != MODE) __builtin_amdgcn_s_setprio(1);
        products(vl0, s, o, l);
        if (KIND != MODE) __builtin_amdgcn_s_setprio(0);
    }

    // A head's slope in powers of two, up to 10^20: its product with a distance, and the differences
    // of such products, are finite then (2^30 tokens are 1.5e29), and 10^20 between neighbours takes
    // all but a row's nearest keys out as well as more would. (NaN stays.)
    static __device__ __forceinline__ float slope_of(float x) {
        return (x > 1e20f ? 1e20f : x < -1e20f ? -1e20f : x) * kLog2e;
    }
    static __device__ __forceinline__ float entry(const Uniform &u, int tab, int dist) {
        const int i = tab + min(max(dist, -u.half), u.half) + u.half;
        return u.table_lds ? lds_read<float>(u.tab0 + 4 * i, 0) : u.table[i];
    }
    // O^T += V^T P^T, with P of 16-bit types rounded to the type: v's products would run at the rate of f32 otherwise. The
    // roundings of a row's weights, half a step each and independent, leave 1.2 to 1.4 times the error that the result's own
    // rounding makes (bf16 2.0e-3 to 2.3e-3 against 64 bits, 1.65e-3 with f32 weights). Where the waves split the keys what they
    // leave takes slots that are free. A product of its own for it over the keys that steps share (64 steps, 16384 bf16 keys: 1.65e-3 for
    // 2.30e-3) would cost 66 -> 69 us, and 3 to 13% at other sizes (64 steps over 16384 and 320 to 640 keys of their own 57 -> 64).
    static __device__ __forceinline__ void products(const lds_t *vl0, const f4v (*s)[NB], f4v (*o)[NB],
                                                    typename std::conditional<F32, float, f4v>::type *l) {
        constexpr int J = F32 || WK ? KB : KB / 2;
        Vec p[J][NB];
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                if constexpr (F32) p[j][nb] = s[j][nb];
                else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = s[WK ? 0 : 2 * j][nb][i];
                        const T hi = (T)x;
                        p[j][nb][i] = hi;
                        // with one block half the slots are free: what the rounding left of it
                        // (2^-17 of it then; the caches' reads take longer than the products)
                        p[j][nb][4 + i] = WK ? (T)(x - (float)hi) : (T)s[WK ? 0 : 2 * j + 1][nb][i];
                    }
                }
            }
        if constexpr (!F32) {
            Vec ones;
#pragma unroll
            for (int e = 0; e < E; ++e) ones[e] = (T)1.f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) l[nb] = mma(ones, p[j][nb], l[nb]);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const Vec x = v_operand(v_block(vl0, db), j);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[db][nb] = mma(x, p[j][nb], o[db][nb]);
            }
    }

    // Whether this thread's share of the tile's V (as it lies in LDS) holds an infinity or
    // NaN, and their removal.
    static __device__ __forceinline__ bool any_wild_chunk(const lds_t *vd) {
        bool w = false;
#pragma unroll
        for (int n = 0; n < LOADS; ++n) w |= any_wild(lds_read<Vec>(vd, (n * 256 + (int)threadIdx.x) * 16));
        return w;
    }
    static __device__ __forceinline__ void remove_wild(lds_t *vd) {
        for (int n = 0; n < LOADS * E; ++n) {
            auto *p = (__attribute__((address_space(3))) T *)(vd + (n * 256 + (int)threadIdx.x) * (int)sizeof(T));
            if (wild((float)*p)) *p = (T)0.f;
        }
    }

    // The infinities and NaN of the tile's v, added to the columns that read their key.
    static __device__ __forceinline__ void wild_products(const Uniform &u, const lds_t *vd, int j0, const int *lim, const int *low,
                                                         const int *doc, const int *at, const int *tab, f4v (*o)[NB]) {
        const int lane = threadIdx.x & 63, q = lane >> 4, wave = wave_of();
#pragma unroll 1
        for (int jr = 0; jr < 16 * KB; ++jr) {
            const int j = j0 + jr;
            if (j >= u.kl) break;
            const int r = (WK ? 16 * wave : 0) + jr;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                bool ok = j < lim[nb] && (!WIN || j >= low[nb] || j < u.sinks) && (!DOC || !u.k_docs || (u.k_docs[j] == doc[nb] && doc[nb] >= 0));
                if (GEN && ok && u.table) ok = entry(u, tab[nb], at[nb] - (u.k_pos ? u.k_pos[j] : j)) != -INFINITY;
                if (!ok) continue;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = 16 * db + 4 * q + i;
                        const float v = (float)lds_read<T>(vd, v_slot<CH, F32>(r, c / E) * 16 + (c % E) * (int)sizeof(T));
                        if (wild(v)) o[db][nb][i] += v;
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
    }
};

template <typename T, int DP, int NB, bool WK, int ALIGN, int MODE>
__global__ __launch_bounds__(256, 2) void k_attn(AttnOpArgs a, AttnLaunch L) {
    static_assert(sizeof(AttnOpArgs) % 8 == 0 && alignof(AttnLaunch) == 8, "late_params reads the two as one struct");
    extern __shared__ __align__(16) char lds[];
    Kernel<T, DP, NB, WK, ALIGN, MODE>::run(a, L, blockIdx.x, lds);
}

// The columns of all entries over the shared keys, `shared` workgroups, and each entry's few columns over its own keys
// in one launch: the first are bound by instructions, the second by HBM, and a CU takes both (64 steps over 16384 shared
// and 640 own keys, 32 / 8 bf16 heads of 128: 56 us with the join, 78 in a launch each). Of f32 heads over 64 wide a CU
// takes one workgroup of either, since the own keys' two buffers fill 128 KB and a launch has one size of LDS: 64 steps over 4096
// and 320 to 640 such keys 117 us, of 64 wide 52.
template <typename T, int DP, int NB, bool WK, int ALIGN, bool OWN_WK>
__global__ __launch_bounds__(256, 2) void k_attn_both(AttnOpArgs a, AttnLaunch own, AttnLaunch shared, int blocks) {
    extern __shared__ __align__(16) char lds[];
    if ((int)blockIdx.x < blocks) Kernel<T, DP, NB, WK, ALIGN, ANY | SHARED>::template run<1>(a, shared, blockIdx.x, lds);
    else Kernel<T, DP, 1, OWN_WK, ALIGN, ANY>::run(a, own, blockIdx.x - blocks, lds);
}

// The key ranges' sums of one column: a workgroup each, its threads over the ranges
// for their weights and then over (channel, every 256 / DP-th range), so that the
// reads of all ranges are in flight together.
// Where range s of a column has its sums: among its entry's own, or (SHARE) behind those
// among the shared keys'.
template <bool SHARE>
struct Ranges {
    const AttnLaunch &L;
    long long own, shared;
    __device__ Ranges(const AttnOpArgs &a, const AttnLaunch &L, int b, int kvh, int c)
        : L(L), own((long long)(b * a.hk + kvh) * L.splits * L.cols + c),
          shared(SHARE ? (long long)kvh * L.shared_splits * L.shared_cols + (long long)b * L.cols + c : 0) {}
    __device__ int count() const { return L.splits + (SHARE ? L.shared_splits : 0); }
    __device__ bool mine(int s) const { return !SHARE || s < L.splits; }
    __device__ long long row(int s) const { return mine(s) ? own + (long long)s * L.cols : shared + (long long)(s - L.splits) * L.shared_cols; }
    __device__ const float *ml(int s) const { return (mine(s) ? L.part_ml : L.shared_ml) + 2 * row(s); }
    template <int DP>
    __device__ const float *o(int s) const { return (mine(s) ? L.part_o : L.shared_o) + row(s) * DP; }
};

template <typename T, int DP, bool SHARE>
__global__ __launch_bounds__(256) void k_attn_join(AttnOpArgs a, AttnLaunch L) {
    constexpr int G = 256 / DP;
    const int tid = threadIdx.x;
    const int c = blockIdx.x % L.cols, bh = blockIdx.x / L.cols;
    const int b = bh / a.hk, kvh = bh - b * a.hk;
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    const int i = c / a.group;
    if (i >= ql) return;
    const Ranges<SHARE> at(a, L, b, kvh, c);
    const int count = at.count();
    __shared__ float weight[256], part[256], stat[8];
    float ms = -INFINITY, l = 0.f;
    if (tid < count) {
        const float *ml = at.ml(tid);
        ms = ml[0];
        l = ml[1];
    }
    // the first sums on their way while the weights are made
    constexpr int N = 16;
    const int d = tid % DP, g = tid / DP;
    float x[N];
    auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int s = s0 + k * G;
            x[k] = g < G && s < count ? at.template o<DP>(s)[d] : 0.f;
        }
    };
    load(g);
    float top = half_max(ms);
#pragma unroll
    for (int m = 1; m < 32; m *= 2) top = fmaxf(top, __shfl_xor(top, m));
    if ((tid & 63) == 0) stat[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(stat[0], stat[1]), fmaxf(stat[2], stat[3]));
    // a range without keys has weight zero; one whose sum is NaN passes it on
    const float f = l == 0.f ? 0.f : (ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ms - top));
    weight[tid] = f;
    float ls = l == 0.f ? 0.f : f * l;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) ls += __shfl_xor(ls, m);
    if ((tid & 63) == 0) stat[4 + (tid >> 6)] = ls;
    __syncthreads();
    ls = (stat[4] + stat[5]) + (stat[6] + stat[7]);
    float o = 0.f;
    for (int s0 = g; s0 < count; s0 += N * G) {
        if (s0 != g) load(s0);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int s = s0 + k * G;
            const float w = s < count ? weight[s] : 0.f;
            o += w == 0.f ? 0.f : w * x[k];
        }
    }
    part[tid] = o;
    __syncthreads();
    if (tid < a.width) {
        o = 0.f;
#pragma unroll
        for (int k = 0; k < G; ++k) o += part[k * DP + tid];
        const int h = kvh * a.group + (c - i * a.group);
        T *out = (T *)a.out + b * a.so.b + (long long)i * a.so.t + h * a.so.h;
        out[tid] = (T)(ls == 0.f ? 0.f : o / ls);
    }
}

// The same for up to kFewRanges ranges of many columns: four channels a thread, 256 / (DP / 4)
// columns a workgroup, all ranges' sums on their way at once.
constexpr int kFewRanges = 8;
template <typename T, int DP, bool SHARE>
__global__ __launch_bounds__(256) void k_attn_join_few(AttnOpArgs a, AttnLaunch L, int rows) {
    constexpr int R = DP / 4, N = 256 / R;
    const int tid = threadIdx.x, id = blockIdx.x * N + tid / R, d = tid % R * 4;
    if (tid >= N * R || id >= rows) return;
    const int bh = id / L.cols, c = id - bh * L.cols, b = L.by_hk.of(bh), kvh = bh - b * a.hk;
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    const int i = L.by_group.of(c);
    if (i >= ql) return;
    const Ranges<SHARE> at(a, L, b, kvh, c);
    const int count = at.count();
    f4v x[kFewRanges];
    float ms[kFewRanges], l[kFewRanges], top = -INFINITY;
#pragma unroll
    for (int s = 0; s < kFewRanges; ++s) {
        x[s] = f4v{0.f, 0.f, 0.f, 0.f};
        ms[s] = -INFINITY, l[s] = 0.f;
        if (s < count) {
            const float *ml = at.ml(s);
            ms[s] = ml[0], l[s] = ml[1];
            x[s] = *(const f4v *)(at.template o<DP>(s) + d);
        }
    }
#pragma unroll
    for (int s = 0; s < kFewRanges; ++s) top = fmaxf(top, ms[s]);
    float ls = 0.f;
    f4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kFewRanges; ++s) {
        // a range without keys has weight zero; one whose sum is NaN passes it on
        const float f = l[s] == 0.f ? 0.f : (ms[s] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ms[s] - top));
        ls += l[s] == 0.f ? 0.f : f * l[s];
        if (f != 0.f) o += x[s] * f;
    }
    const int h = kvh * a.group + (c - i * a.group);
    const float r = ls == 0.f ? 0.f : 1.f / ls;
    store((T *)a.out + b * a.so.b + (long long)i * a.so.t + h * a.so.h, d, a.width, L.out_vec, o * r);
}

// The same for up to kSomeRanges ranges, eight at a time, their weights first.
constexpr int kSomeRanges = 32;
template <typename T, int DP, bool SHARE>
__global__ __launch_bounds__(256) void k_attn_join_some(AttnOpArgs a, AttnLaunch L, int rows) {
    constexpr int R = DP / 4, N = 256 / R, W = 8;
    const int tid = threadIdx.x, slot = tid / R, lane = tid % R, id = blockIdx.x * N + slot;
    __shared__ float weight[N][kSomeRanges], total[N][kSomeRanges];
    const bool there = tid < N * R && id < rows;
    const int bh = there ? id / L.cols : 0, c = id - bh * L.cols, b = L.by_hk.of(bh), kvh = bh - b * a.hk;
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    const int i = there ? L.by_group.of(c) : 0;
    const bool ok = there && i < ql;
    const Ranges<SHARE> at(a, L, b, kvh, there ? c : 0);
    const int count = at.count();
    f4v x[W];
    auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] = ok && s0 + k < count ? *(const f4v *)(at.template o<DP>(s0 + k) + lane * 4) : f4v{0.f, 0.f, 0.f, 0.f};
    };
    if (ok)
        for (int s = lane; s < count; s += R) {
            const float *ml = at.ml(s);
            weight[slot][s] = ml[0], total[slot][s] = ml[1];
        }
    load(0);
    __syncthreads();
    if (!ok) return;
    float top = -INFINITY, ls = 0.f;
    for (int s = 0; s < count; ++s) top = fmaxf(top, weight[slot][s]);
    f4v o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < count; s0 += W) {
        if (s0) load(s0);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            if (s0 + k >= count) break;
            // a range without keys has weight zero; one whose sum is NaN passes it on
            const float m = weight[slot][s0 + k], l = total[slot][s0 + k];
            const float f = l == 0.f ? 0.f : (m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top));
            ls += l == 0.f ? 0.f : f * l;
            if (f != 0.f) o += x[k] * f;
        }
    }
    const int h = kvh * a.group + (c - i * a.group);
    const float r = ls == 0.f ? 0.f : 1.f / ls;
    store((T *)a.out + b * a.so.b + (long long)i * a.so.t + h * a.so.h, lane * 4, a.width, L.out_vec, o * r);
}

// How a call is cut.
struct Cut {
    int dp, nb, tk;
    bool wk;
    int tiles, splits;
};

template <typename T, int DP, int NB, bool WK, int ALIGN, int MODE>
hipError_t launch(const AttnOpArgs &a, const AttnLaunch &L, hipStream_t st) {
    typedef Kernel<T, DP, NB, WK, ALIGN, MODE> K;
    static_assert(K::kTab + 4 * K::kTabEntries <= 163840, "LDS");
    AttnLaunch M = L;
    M.table_lds = a.table && (long long)a.group * a.table_size <= K::kTabEntries;
    const size_t lds = K::kTab + (M.table_lds ? (size_t)a.group * a.table_size * 4 : 0);
    const long long blocks = (long long)a.batch * a.hk * L.tiles * L.splits;  // (below 2^24 by the entry's checks)
    return enqueue(k_attn<T, DP, NB, WK, ALIGN, MODE>, dim3((unsigned)blocks), dim3(256), lds, st, a, M);
}

// Arrays that are not of 16-byte multiples and general biases take the kernels of 16
// columns a wave. (W: WINDOW or 0)
template <typename T, int DP, bool WK, int W>
hipError_t launch_narrow(const AttnOpArgs &a, const AttnLaunch &L, int align, hipStream_t st) {
    if (align == 0) return launch<T, DP, 1, WK, 0, GENERAL | W>(a, L, st);
    if constexpr (W != 0)
        if (align < 16 && !L.score.general && !a.k_docs) return launch<T, DP, 1, WK, 4, ANY | W>(a, L, st);
    if (align < 16) return launch<T, DP, 1, WK, 4, GENERAL | W>(a, L, st);
    if (L.score.general) return launch<T, DP, 1, WK, 16, GENERAL | W>(a, L, st);
    if constexpr (W == 0 || W == WINDOW)
        if (a.k_docs) return launch<T, DP, 1, WK, 16, ANY | DOCS | W>(a, L, st);
    return launch<T, DP, 1, WK, 16, ANY | W>(a, L, st);
}

template <typename T, int DP, bool SHARE = false>
hipError_t join(const AttnOpArgs &a, const AttnLaunch &L, hipStream_t st) {
    const long long rows = (long long)a.batch * a.hk * L.cols;  // (few: the keys were split to fill the chip)
    // few ranges of many columns: 8 causal bf16 heads of 128 over 512, 1024 and 2048 tokens 15, 26
    // and 40 us against 21, 39 and 62 by a workgroup per column; 512 columns of 4 ranges (16 steps over
    // 1024 keys) 20.3 against 19.6
    constexpr int N = 256 / (DP / 4);
    if (L.splits + (SHARE ? L.shared_splits : 0) <= kFewRanges && rows >= 4 * cu_count())
        return enqueue(k_attn_join_few<T, DP, SHARE>, dim3((unsigned)((rows + N - 1) / N)), dim3(256), 0, st, a, L, (int)rows);
    // up to 32 ranges: 2048 columns of 9 ranges (64 steps over 16384 shared keys) 5.9 us, 8.0 by a workgroup a column
    if constexpr (SHARE)
        if (L.splits + L.shared_splits <= kSomeRanges && rows >= 4 * cu_count())
            return enqueue(k_attn_join_some<T, DP, SHARE>, dim3((unsigned)((rows + N - 1) / N)), dim3(256), 0, st, a, L, (int)rows);
    return enqueue(k_attn_join<T, DP, SHARE>, dim3((unsigned)rows), dim3(256), 0, st, a, L);
}

template <typename T, int DP, int W>
hipError_t launch_width(const AttnOpArgs &a, const AttnLaunch &L, const Cut &c, int align, hipStream_t st) {
    auto kernel = [&]() -> hipError_t {
        if (c.wk) return launch_narrow<T, DP, true, W>(a, L, align, st);
        if (c.nb == 1) return launch_narrow<T, DP, false, W>(a, L, align, st);
        if constexpr (W != 0)
            if (align < 16) return launch<T, DP, 2, false, 4, ANY | W>(a, L, st);
        if (a.k_docs) {  // (of narrow heads never: waves of 16 take them)
            if constexpr (W != WHOLE && DP > 64) return launch<T, DP, 2, false, 16, ANY | DOCS | W>(a, L, st);
            return hipErrorInvalidValue;
        }
        if (a.cap > 0.f)
            return a.slopes ? launch<T, DP, 2, false, 16, CAP | SLOPES | W>(a, L, st) : launch<T, DP, 2, false, 16, CAP | W>(a, L, st);
        return a.slopes ? launch<T, DP, 2, false, 16, SLOPES | W>(a, L, st) : launch<T, DP, 2, false, 16, W>(a, L, st);
    };
    const hipError_t e = kernel();
    return e != hipSuccess || !L.join ? e : join<T, DP>(a, L, st);
}

template <typename T, int W>
hipError_t launch_type(const AttnOpArgs &a, const AttnLaunch &L, const Cut &c, int align, hipStream_t st) {
    switch (c.dp) {
        case 32: return launch_width<T, 32, W>(a, L, c, align, st);
        case 64: return launch_width<T, 64, W>(a, L, c, align, st);
        case 96: return launch_width<T, 96, W>(a, L, c, align, st);
        default: return launch_width<T, 128, W>(a, L, c, align, st);
    }
}

// Both in one launch, and the join (c: how the shared keys are cut).
template <typename T, int DP, int NB, bool WK, int ALIGN, bool OWN_WK = true>
hipError_t launch_both(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, hipStream_t st) {
    typedef Kernel<T, DP, NB, WK, ALIGN, ANY | SHARED> S;
    typedef Kernel<T, DP, 1, OWN_WK, ALIGN, ANY> O;
    static_assert(std::max(S::kTab, O::kTab) <= 163840, "LDS");
    const int blocks = a.hk * shared.tiles * shared.splits;
    const long long all = blocks + (long long)a.batch * a.hk * own.tiles * own.splits;
    const hipError_t e = enqueue(k_attn_both<T, DP, NB, WK, ALIGN, OWN_WK>, dim3((unsigned)all), dim3(256), std::max(S::kTab, O::kTab), st, a, own, shared, blocks);
    return e != hipSuccess ? e : join<T, DP, true>(a, own, st);
}
template <typename T, int DP, int ALIGN>
hipError_t launch_both_align(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const Cut &c, bool own_wk, hipStream_t st) {
    if (!own_wk) return launch_both<T, DP, 2, false, ALIGN, false>(a, own, shared, st);
    if (c.wk) return launch_both<T, DP, 1, true, ALIGN>(a, own, shared, st);
    return c.nb == 1 ? launch_both<T, DP, 1, false, ALIGN>(a, own, shared, st) : launch_both<T, DP, 2, false, ALIGN>(a, own, shared, st);
}
template <typename T, int DP>
hipError_t launch_both_width(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const Cut &c, bool own_wk, int align, hipStream_t st) {
    return align < 16 ? launch_both_align<T, DP, 4>(a, own, shared, c, own_wk, st) : launch_both_align<T, DP, 16>(a, own, shared, c, own_wk, st);
}
template <typename T>
hipError_t launch_both_type(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const Cut &c, bool own_wk, int align, hipStream_t st) {
    switch (c.dp) {
        case 32: return launch_both_width<T, 32>(a, own, shared, c, own_wk, align, st);
        case 64: return launch_both_width<T, 64>(a, own, shared, c, own_wk, align, st);
        case 96: return launch_both_width<T, 96>(a, own, shared, c, own_wk, align, st);
        default: return launch_both_width<T, 128>(a, own, shared, c, own_wk, align, st);
    }
}

}  // namespace attn

hipError_t launch_attention_f32(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_attention_f16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_attention_bf16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_window_attention_f32(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_window_attention_f16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_window_attention_bf16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_whole_attention_f32(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_whole_attention_f16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_whole_attention_bf16(const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st);
hipError_t launch_both_attention_f32(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const attn::Cut &c, bool own_wk,
                                      int align, hipStream_t st);
hipError_t launch_both_attention_f16(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const attn::Cut &c, bool own_wk,
                                      int align, hipStream_t st);
hipError_t launch_both_attention_bf16(const AttnOpArgs &a, const AttnLaunch &own, const AttnLaunch &shared, const attn::Cut &c, bool own_wk,
                                      int align, hipStream_t st);
