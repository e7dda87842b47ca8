// s2s_attention.hip - the attention operator's launcher: how a call is cut over the
// chip, its workspace, and the documents' tile summary.
#include "s2s_attention.h"

namespace {

int round_up(int v, int m) { return (v + m - 1) / m * m; }

// Columns of at most 16 share one set of waves that split each key tile (f32 64 wide,
// one query of 8192 keys, 32 / 8 heads: 13.6 us against 18.8 by waves of 16 of which one works; 16-bit
// types are as fast either way, and keep what the weights' rounding leaves). More take waves
// of 16 columns, or of 32 where those give every CU two workgroups: a key tile's LDS reads then serve
// two products (2 x 4096 causal bf16, 32 / 8 heads: 128 wide 278 us against 366 by waves of 16,
// 64 wide 167 and 200; 2048 tokens of 16 / 4 heads, too few, 103 and 43). `narrow`: waves of 16 only.
// Where few columns leave CUs without work the keys are cut into ranges whose sums a second
// kernel joins, at most two workgroups a CU (four: nothing for one query, 32 us against 15 for 64
// sequences of 4 queries and 512 keys, by the join). Column tiles of more than one a CU and less than two
// are not cut, since the quotient is rounded down: 376 of them, 3000 f32 tokens of 8 heads of 32, take 91 us
// causal and 125 over all keys, 71 and 97 in two ranges; the same of bf16 heads of 128, 58 and 66 against
// 52 and 79. Ranges of four tiles at least; of two, and up to 16
// of one, for columns of at most 16, whose rows to join are few: one query of 32 / 8 bf16 heads of 128 over 512,
// 1024, 2048 and 4096 keys takes 9.1, 9.1, 9.9 and 10.5 us against 11.4 to 11.7, but over 256 keys
// 9.0 against 8.1 uncut; 64 queries of 8 sequences over 256 keys 20 against 9.5.
attn::Cut cut_of(int dtype, const AttnOpArgs &a, bool narrow) {
    attn::Cut c;
    const long long cols = (long long)a.group * a.nq, pairs = (long long)a.batch * a.hk;
    const int cus = cu_count();
    c.dp = round_up(std::max(a.width, 1), 32);
    c.wk = cols <= 16;
    c.nb = narrow || c.wk || cols <= 64 || (cols + 127) / 128 * pairs < 2 * cus ? 1 : 2;
    c.tk = dtype == 0 && !c.wk && c.dp > 64 ? 32 : 64;
    const int per = c.wk ? 16 : 64 * c.nb;
    c.tiles = (int)((cols + per - 1) / per);
    const long long blocks = std::max(1LL, pairs * c.tiles);
    long long nt = ((long long)a.nk + c.tk - 1) / c.tk;
    // of a window the tiles that a column tile's queries and the sinks lie in. (Whether a call has a prefix is not known when its
    // workspace is made. One past the window adds to a column tile's keys those of the queries behind it, which it then walks in
    // as many ranges as the window alone would have.)
    if (a.window) {
        nt = std::min(nt, ((long long)(a.causal ? 1 : 2) * a.window + per / a.group + c.tk) / c.tk + 1 + ((long long)a.sinks + c.tk - 1) / c.tk);
        // few tiles are not cut: a launch less (5 queries over windows of 128 of 700 keys, 8 f16 heads of 64, 8.7 us with
        // the host's call, 12.2 in ranges)
        if (c.wk && nt <= 6) nt = 1;
    }
    const long long ranges = c.wk && nt > 4 ? std::max({nt / 4, std::min(nt / 2, 32LL), std::min(nt, 16LL)}) : nt / 4;
    c.splits = (int)std::max(1LL, std::min({2LL * cus / blocks, ranges, 256LL}));
    return c;
}

int meta_tiles(const attn::Cut &c, const AttnOpArgs &a) { return (a.nk + c.tk - 1) / c.tk; }

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// {smallest id >= 0, largest, smallest of all} of a key tile's documents: a wave
// per tile.
__global__ __launch_bounds__(256) void k_doc_tiles(AttnOpArgs a, int tk, int tiles, int4 *meta) {
    const int lane = threadIdx.x & 63;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (long long)a.batch * tiles) return;
    const int b = (int)(id / tiles), t = (int)(id - (long long)b * tiles);
    const int kl = a.k_lens ? min(max(a.k_lens[b], 0), a.nk) : a.nk;
    const int j = t * tk + lane;
    int lo = 0x7fffffff, hi = -1, all = 0x7fffffff;
    if (lane < tk && j < kl) {
        all = a.k_docs[b * a.k_docs_b + j];
        if (all >= 0) lo = hi = all;
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        lo = min(lo, __shfl_xor(lo, m));
        hi = max(hi, __shfl_xor(hi, m));
        all = min(all, __shfl_xor(all, m));
    }
    if (lane == 0) meta[id] = make_int4(lo, hi, all, 0);
}

// The same of the queries of a column tile, and how many key tiles hold a document of
// theirs: a wave per column tile.
__global__ __launch_bounds__(256) void k_doc_columns(AttnOpArgs a, int tk, int key_tiles, int per, int tiles, const int4 *meta,
                                                     int4 *col) {
    const int lane = threadIdx.x & 63;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (long long)a.batch * tiles) return;
    const int b = (int)(id / tiles), t = (int)(id - (long long)b * tiles);
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    int lo = 0x7fffffff, hi = -1, all = 0x7fffffff;
    const int first = t * per / a.group, last = min(ql - 1, (t * per + per - 1) / a.group);
    for (int i = first + lane; i <= last; i += 64) {
        const int d = a.q_docs[b * a.q_docs_b + i];
        all = min(all, d);
        if (d >= 0) lo = min(lo, d), hi = max(hi, d);
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        lo = min(lo, __shfl_xor(lo, m));
        hi = max(hi, __shfl_xor(hi, m));
        all = min(all, __shfl_xor(all, m));
    }
    int live = 0;
    for (int k = lane; k < key_tiles; k += 64) {
        const int4 x = meta[(long long)b * key_tiles + k];
        live += x.x <= hi && x.y >= lo;
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) live += __shfl_xor(live, m);
    if (lane == 0) col[id] = make_int4(lo, hi, all, live);
}

// Column tiles by falling number of key tiles, to 256 steps: a workgroup per batch
// entry. (Tiles of one step come in any order; no result goes by it. Nine images of different sizes, 11003
// tokens: 120 us, 165 in the tokens' order.)
__global__ __launch_bounds__(256) void k_doc_order(int tiles, const int4 *col, int *order) {
    __shared__ int bin[256], most;
    const int tid = threadIdx.x;
    col += (long long)blockIdx.x * tiles, order += (long long)blockIdx.x * tiles;
    bin[tid] = 0;
    if (tid == 0) most = 1;
    __syncthreads();
    for (int t = tid; t < tiles; t += 256) atomicMax(&most, col[t].w);
    __syncthreads();
    const float step = 255.f / (float)most;
    auto of = [&](int t) { return 255 - min(255, (int)((float)col[t].w * step)); };
    for (int t = tid; t < tiles; t += 256) atomicAdd(&bin[of(t)], 1);
    __syncthreads();
    int n = bin[tid];  // its sum over the steps before
    for (int m = 1; m < 256; m *= 2) {
        __syncthreads();
        const int x = tid >= m ? bin[tid - m] : 0;
        __syncthreads();
        bin[tid] += x;
    }
    __syncthreads();
    n = bin[tid] - n;
    __syncthreads();
    bin[tid] = n;
    __syncthreads();
    for (int t = tid; t < tiles; t += 256) order[atomicAdd(&bin[of(t)], 1)] = t;
}

// The three above in one launch, a workgroup of 16 waves per batch entry, for up to 64 key and
// 64 column tiles: 16 lanes a tile for the ids, a wave per column tile for its live key tiles. (12 bf16
// heads of 64: 1000 tokens 29 us, 33 by the three; 3000 61 and 65; with more tiles one workgroup
// takes longer than the launches, 11003 tokens 161 and 158, 65536 885 and 750.)
constexpr int kDocTiles = 64;
__global__ __launch_bounds__(1024) void k_doc_all(AttnOpArgs a, int tk, int key_tiles, int per, int tiles, int4 *meta, int4 *col,
                                                  int *order) {
    __shared__ int2 keys[kDocTiles];
    __shared__ int4 cols[kDocTiles];
    __shared__ int bin[256], most;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = tid & 15, b = blockIdx.x;
    meta += (long long)b * key_tiles, col += (long long)b * tiles;
    const int kl = a.k_lens ? min(max(a.k_lens[b], 0), a.nk) : a.nk;
    const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.nq) : a.nq;
    const int *kd = a.k_docs + b * a.k_docs_b, *qd = a.q_docs + b * a.q_docs_b;
    // {smallest id >= 0, largest, smallest of all} of ids[first .. last], in all 16 lanes
    auto ids = [&](const int *p, int first, int last) {
        int lo = 0x7fffffff, hi = -1, all = 0x7fffffff;
        for (int i = first + sub; i <= last; i += 16) {
            const int d = p[i];
            all = min(all, d);
            if (d >= 0) lo = min(lo, d), hi = max(hi, d);
        }
#pragma unroll
        for (int m = 1; m < 16; m *= 2) {
            lo = min(lo, __shfl_xor(lo, m));
            hi = max(hi, __shfl_xor(hi, m));
            all = min(all, __shfl_xor(all, m));
        }
        return make_int4(lo, hi, all, 0);
    };
    const int t = tid >> 4;
    if (t < key_tiles) {
        const int4 x = ids(kd, t * tk, min(kl, t * tk + tk) - 1);
        if (sub == 0) meta[t] = x, keys[t] = make_int2(x.x, x.y);
    }
    if (t < tiles) {
        const int4 x = ids(qd, t * per / a.group, min(ql - 1, (t * per + per - 1) / a.group));
        if (sub == 0) cols[t] = x;
    }
    if (tid < 256) bin[tid] = 0;
    if (tid == 0) most = 1;
    __syncthreads();
    for (int t = wave; t < tiles; t += 16) {
        int4 x = cols[t];
        const int2 y = keys[min(lane, key_tiles - 1)];
        x.w = __popcll(__ballot(lane < key_tiles && y.x <= x.y && y.y >= x.x));
        if (lane == 0) col[t] = cols[t] = x, atomicMax(&most, x.w);
    }
    if (!order) return;  // (all of the workgroup)
    order += (long long)b * tiles;
    __syncthreads();
    const float step = 255.f / (float)most;
    auto of = [&](int t) { return 255 - min(255, (int)((float)cols[t].w * step)); };
    if (tid < tiles) atomicAdd(&bin[of(tid)], 1);
    __syncthreads();
    if (wave == 0) {  // four bins a lane to the sums before them
        int n[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = bin[4 * lane + i], sum += n[i];
        int before = sum;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            const int x = __shfl_up(before, m);
            if (lane >= m) before += x;
        }
        before -= sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) bin[4 * lane + i] = before, before += n[i];
    }
    __syncthreads();
    if (tid < tiles) order[atomicAdd(&bin[of(tid)], 1)] = tid;
}

// The largest power of two in bytes, up to 16, that an array's address, strides
// and width are multiples of.
int aligned_bytes(const void *p, const Strides &s, int width, int size) {
    unsigned long long m = (unsigned long long)(uintptr_t)p | (unsigned long long)((s.b | s.t | s.h) * size) | 16;
    m |= (unsigned long long)width * size;
    return (int)(m & (~m + 1));
}

}  // namespace

// The documents' summaries: of key tiles, of column tiles, the column tiles' order.
size_t doc_bytes(const attn::Cut &c, const AttnOpArgs &a) {
    return (size_t)a.batch * ((size_t)meta_tiles(c, a) + c.tiles) * sizeof(int4) + round16((size_t)a.batch * c.tiles * sizeof(int));
}

// The most that either cut of these sizes needs: which one runs goes by strides and
// biases too.
size_t attn_op_workspace(int dtype, const AttnOpArgs &a) {
    size_t most = 0;
    for (const bool narrow : {false, true}) {
        const attn::Cut c = cut_of(dtype, a, narrow);
        size_t n = doc_bytes(c, a);
        if (c.splits > 1) {
            const size_t rows = (size_t)a.batch * a.hk * c.splits * a.group * a.nq;
            n += rows * c.dp * 4 + rows * 8;
        }
        most = std::max(most, n);
    }
    return most;
}

namespace {

// The copies' size that a call's arrays allow: 16, or 4, or 0 for element by element.
int copies_of(const AttnOpArgs &a, int al) {
    // (rows that overlap have no end that the copies' resource could tell: by elements)
    return a.sk.t < a.width || a.sv.t < a.width ? 0 : al >= 16 ? 16 : al >= 4 ? 4 : 0;
}
int aligned_inputs(const AttnOpArgs &a, int size) {
    const int al = aligned_bytes(a.q, a.sq, a.width, size);
    return a.nk > 0 ? std::min(al, std::min(aligned_bytes(a.k, a.sk, a.width, size), aligned_bytes(a.v, a.sv, a.width, size))) : al;
}

hipError_t launch_of(int dtype, const AttnOpArgs &a, const AttnLaunch &L, const attn::Cut &c, int align, hipStream_t st) {
    if (a.window) switch (dtype) {
            case 0: return launch_window_attention_f32(a, L, c, align, st);
            case 1: return launch_window_attention_f16(a, L, c, align, st);
            case 2: return launch_window_attention_bf16(a, L, c, align, st);
        }
    switch (dtype) {
        case 0: return launch_attention_f32(a, L, c, align, st);
        case 1: return launch_attention_f16(a, L, c, align, st);
        case 2: return launch_attention_bf16(a, L, c, align, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attention_op(int dtype, const AttnOpArgs &a, void *ws, hipStream_t st) {
    const int size = dtype == 0 ? 4 : 2;
    AttnLaunch L{};
    L.score.set(a);
    const int al = aligned_inputs(a, size);
    L.vec = std::min(al, 8);
    L.out_vec = std::min(4, aligned_bytes(a.out, a.so, a.width, size) / size);
    const int align = copies_of(a, al);
    // Packed documents of narrow heads too: the fewer columns a workgroup has, the fewer lie
    // across two documents and mask both's tiles (nine images, 11003 tokens, 12 heads: 64
    // wide 153 us with waves of 32 and 127 with 16, 32 wide 132 and 105; 128 wide, 32 / 8
    // heads, where a wave of 16 reads LDS twice as often for its products, 369 and 483).
    const attn::Cut c = cut_of(dtype, a, (a.window && !a.k_docs ? align < 4 : align < 16) || L.score.general || (a.k_docs && a.width <= 64));
    L.cols = a.group * a.nq;
    L.tiles = c.tiles;
    L.splits = c.splits;
    char *w = (char *)ws;
    const int mt = meta_tiles(c, a);
    L.by_pairs.set(a.batch * a.hk);
    L.by_tiles.set(c.tiles);
    L.by_hk.set(a.hk);
    L.by_group.set(a.group);
    if (c.splits > 1) {
        const size_t rows = (size_t)a.batch * a.hk * c.splits * L.cols;
        L.part_o = (float *)(w + doc_bytes(c, a));
        L.part_ml = L.part_o + rows * c.dp;
        L.join = 1;
    }
    // a summary of few tiles would skip nothing
    if (a.k_docs && mt > 4) {
        int4 *meta = (int4 *)w, *col = meta + (size_t)a.batch * mt;
        int *order = (int *)(col + (size_t)a.batch * c.tiles);
        const int per = c.wk ? 16 : 64 * c.nb;
        L.meta = meta;
        L.meta_tiles = mt;
        L.col_docs = col;
        const long long nk = (long long)a.batch * mt, nc = (long long)a.batch * c.tiles;
        // documents of different sizes make column tiles of different work; the longest first
        if (c.tiles >= 8) L.order = order;
        hipError_t e;
        if (mt <= kDocTiles && c.tiles <= kDocTiles) {
            e = enqueue(k_doc_all, dim3((unsigned)a.batch), dim3(1024), 0, st, a, c.tk, mt, per, c.tiles, meta, col,
                        c.tiles >= 8 ? order : nullptr);
        } else {
            e = enqueue(k_doc_tiles, dim3((unsigned)((nk + 3) / 4)), dim3(256), 0, st, a, c.tk, mt, meta);
            if (e == hipSuccess)
                e = enqueue(k_doc_columns, dim3((unsigned)((nc + 3) / 4)), dim3(256), 0, st, a, c.tk, mt, per, c.tiles, meta, col);
            if (e == hipSuccess && c.tiles >= 8)
                e = enqueue(k_doc_order, dim3((unsigned)a.batch), dim3(256), 0, st, c.tiles, col, order);
        }
        if (e != hipSuccess) return e;
    }
    return launch_of(dtype, a, L, c, align, st);
}

// ---- a batch that shares a prefix ---------------------------------------------------

namespace {

// How the columns of all entries go over the shared keys, in one launch with the entries' own: ranges for one
// workgroup a CU, beside which it takes one of the own keys' (64 steps over 16384 shared keys, 640 own, 32 / 8 bf16
// heads of 128: 54 us, 67 with two and 87 with a half); waves of 32 columns from 257 columns a head on
// (200 steps over 8192 keys: 73 us against 86; 64 steps, 256 columns, over 4096 keys 46 against 41).
attn::Cut shared_cut(int dtype, const AttnOpArgs &a) {
    AttnOpArgs one = a;
    one.nq = a.batch * a.nq;
    one.batch = 1;
    one.nk = a.shared_nk;
    attn::Cut c = cut_of(dtype, one, true);
    const long long cols = (long long)one.nq * one.group, nt = ((long long)one.nk + c.tk - 1) / c.tk;
    if (cols > 256 || (long long)a.nq * a.group > 16) c.nb = 2, c.wk = false;
    const int per = c.wk ? 16 : 64 * c.nb;
    c.tiles = (int)((cols + per - 1) / per);
    c.splits = (int)std::max(1LL, std::min({cu_count() / std::max(1LL, (long long)c.tiles * a.hk), nt / 2, 128LL}));  // (the join takes 256 ranges)
    return c;
}
// How an entry's columns go over the shared keys and its own, as over keys of its own.
attn::Cut whole_cut(int dtype, const AttnOpArgs &a, bool narrow) {
    AttnOpArgs one = a;
    one.nk = a.shared_nk + a.nk;
    attn::Cut c = cut_of(dtype, one, narrow);
    // up to eight tiles one launch is faster than two (16 steps over 256 + 128 keys, 32 / 8 bf16 heads of 128, 11.1 us
    // uncut and 12.1 in ranges, and the host has one launch less)
    if (c.wk && one.nk <= 8 * c.tk) c.splits = 1;
    return c;
}
attn::Cut own_cut(int dtype, const AttnOpArgs &a) {
    attn::Cut c = cut_of(dtype, a, true);
    c.splits = std::min(c.splits, 128);
    return c;
}

size_t columns_of(const AttnOpArgs &a) { return (size_t)a.batch * a.nq * a.hq; }
size_t sums_bytes(const attn::Cut &c, const AttnOpArgs &a) { return round16(columns_of(a) * c.splits * ((size_t)c.dp * 4 + 8)); }

// Whether every column tile walks the shared keys by itself, and its entry's own behind them. For more than 32 columns
// an entry always, since the shared keys' sums of every range, written and read again, cost more than the keys
// (8 x 512 tokens behind 1024, 4096 and 16384 shared keys, 32 / 8 bf16 heads of 128: 98, 294 and 1077 us
// against 177, 379 and 1188; 16 x 16 tokens, 64 columns, 26, 31 and 60 behind 1024, 2048 and 8192, 29, 34 and 68; 64 x 9, 12 and 16
// tokens behind 8192 162, 162 and 175, 213, 216 and 221; 36 x 64 tokens of 6 f32 heads of 30 behind 1089 38.5 and 39.2. It is the slower way for
// f32 of fewer columns: 33 and 48 such tokens 36 and 37.5, 27 and 31; 16 x 40 of 8 heads of 128 behind 4096 154 and 117; but
// 64 x 40 of 64 behind 1024 83 and 91). 17 to 32,
// which leave the half of a tile of their own empty: of 16-bit types but for many keys times entries (16 x 8 tokens behind 1024
// and 8192 keys 20 and 52 us, 26 and 39 by the ranges), of f32, whose products take longer, never (16 x 24 tokens of 6
// heads of 30 behind 1024 and 8192 keys 23 and 83, 17 and 44). Steps over up to eight tiles.
bool goes_whole(int dtype, const AttnOpArgs &a, int tk, int align, bool general) {
    const long long cols = (long long)a.nq * a.group, tiles = ((long long)a.shared_nk + tk - 1) / tk;
    if (align == 0 || general || cols > 32) return true;
    if (cols > 16) return dtype != 0 && a.batch * a.hk * tiles < 48LL * cu_count();
    return (long long)a.shared_nk + a.nk <= 8 * tk;
}

}  // namespace

// The most that any way of these sizes needs: which one runs goes by strides and numbers too.
size_t shared_attn_op_workspace(int dtype, const AttnOpArgs &a) {
    const bool ranges = !goes_whole(dtype, a, cut_of(dtype, a, true).tk, 16, false);
    size_t most = ranges ? sums_bytes(own_cut(dtype, a), a) + sums_bytes(shared_cut(dtype, a), a) : 0;
    for (const bool narrow : {false, true}) {
        const attn::Cut c = whole_cut(dtype, a, narrow);
        if (c.splits > 1) most = std::max(most, sums_bytes(c, a));
    }
    return most;
}

hipError_t launch_shared_attention_op(int dtype, const AttnOpArgs &a, void *ws, hipStream_t st) {
    const int size = dtype == 0 ? 4 : 2;
    AttnOpArgs s = a;  // the shared keys as the keys
    s.k = a.shared_k, s.v = a.shared_v, s.sk = a.shared_sk, s.sv = a.shared_sv, s.nk = a.shared_nk;
    const int own_al = aligned_inputs(a, size), own_align = copies_of(a, own_al);
    const int shared_al = aligned_inputs(s, size), shared_align = copies_of(s, shared_al);
    AttnScore score;
    score.set(a);
    auto fill = [&](const attn::Cut &c, int al, float *sums) {
        AttnLaunch L{};
        L.score = score;
        L.vec = std::min(al, 8);
        L.out_vec = std::min(4, aligned_bytes(a.out, a.so, a.width, size) / size);
        L.cols = a.group * a.nq;
        L.tiles = c.tiles;
        L.splits = c.splits;
        L.by_pairs.set(a.batch * a.hk);
        L.by_tiles.set(c.tiles);
        L.by_hk.set(a.hk);
        L.by_group.set(a.group);
        L.by_nq.set(a.nq);
        L.part_o = sums;
        L.part_ml = sums + columns_of(a) * c.splits * c.dp;
        return L;
    };
    const int align = std::min(own_align, shared_align), al = std::min(own_al, shared_al);
    const attn::Cut wc = whole_cut(dtype, a, align < 4 || score.general);
    if (goes_whole(dtype, a, wc.tk, align, score.general)) {
        AttnLaunch L = fill(wc, al, (float *)ws);
        if (wc.splits > 1) L.join = 1;
        else L.part_o = L.part_ml = nullptr;
        switch (dtype) {
            case 0: return launch_whole_attention_f32(a, L, wc, align, st);
            case 1: return launch_whole_attention_f16(a, L, wc, align, st);
            case 2: return launch_whole_attention_bf16(a, L, wc, align, st);
        }
        return hipErrorInvalidValue;
    }
    const attn::Cut oc = own_cut(dtype, a), sc = shared_cut(dtype, a);
    AttnLaunch O = fill(oc, al, (float *)ws), S = fill(sc, al, (float *)((char *)ws + sums_bytes(oc, a)));
    S.cols = a.group * a.nq * a.batch;
    S.by_pairs.set(a.hk);
    O.shared_o = S.part_o;
    O.shared_ml = S.part_ml;
    O.shared_splits = sc.splits;
    O.shared_cols = S.cols;
    switch (dtype) {
        case 0: return launch_both_attention_f32(a, O, S, sc, oc.wk, align, st);
        case 1: return launch_both_attention_f16(a, O, S, sc, oc.wk, align, st);
        case 2: return launch_both_attention_bf16(a, O, S, sc, oc.wk, align, st);
    }
    return hipErrorInvalidValue;
}
