// s2s_ops_api.cpp - the transformer operators of include/swin2sr_hip.h: every
// check of a call's arguments, then one launcher (s2s_ops.h). Nothing here
// throws or allocates; a refused call has enqueued nothing.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "swin2sr_hip.h"
#include "s2s_kernels.h"
#include "s2s_ops.h"

namespace {

int refuse(const char *fmt, ...) __attribute__((format(printf, 1, 2)));
int refuse(const char *fmt, ...) {
    char m[320];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(m, sizeof m, fmt, ap);
    va_end(ap);
    return s2s_fail(m);
}

int refuse_hip(const char *op, const char *what, hipError_t e) {
    return refuse("%s: %s failed: %s%s", op, what, hipGetErrorString(e),
                  e == hipErrorOutOfMemory ? ": out of memory" : "");
}

// The stream's device made current for the call's launches, and the caller's
// restored.
struct OnDevice {
    int was = -1, dev = -1;
    hipError_t enter(hipStream_t st) {
        hipError_t e = hipGetDevice(&was);
        if (e != hipSuccess) return e;
        hipDevice_t d = was;
        if (st && (e = hipStreamGetDevice(st, &d)) != hipSuccess) return e;
        dev = d;
        return dev == was ? hipSuccess : hipSetDevice(dev);
    }
    ~OnDevice() {
        if (dev >= 0 && dev != was) (void)hipSetDevice(was);
    }
};

// Memory a kernel of this device may touch: its own, or page-locked host
// memory. Plain host pointers and other devices' memory would fault.
int check_memory(const char *op, const char *name, const void *p, int dev) {
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
        (void)hipGetLastError();
        return refuse("%s: %s is not device memory", op, name);
    }
    if (at.type == hipMemoryTypeUnregistered) return refuse("%s: %s is not device memory", op, name);
    if (at.type == hipMemoryTypeDevice && at.device != dev)
        return refuse("%s: %s is memory of device %d, the stream is of device %d", op, name, at.device, dev);
    return 0;
}

int type_size(int dtype) { return dtype == S2S_F32 ? 4 : 2; }

bool is_real_type(int dtype) { return dtype == S2S_F32 || dtype == S2S_F16 || dtype == S2S_BF16; }

// Strides are below 2^40 elements, so that no offset of these sizes wraps.
constexpr long long kMaxStride = 1LL << 40;

int check_tokens(const char *op, const char *name, const s2s_tokens &t, int dtype, int dev) {
    if (!t.data) return refuse("%s: %s is null", op, name);
    if ((uintptr_t)t.data % type_size(dtype))
        return refuse("%s: %s is not aligned to its elements", op, name);
    if (t.batch < 0 || t.token < 0 || t.head < 0 || t.batch > kMaxStride || t.token > kMaxStride ||
        t.head > kMaxStride)
        return refuse("%s: %s has a negative or impossible stride", op, name);
    return check_memory(op, name, t.data, dev);
}

// A written array's elements may not overlap: from the smallest stride up,
// each reaches past what the smaller ones span.
int check_written(const char *op, const char *name, const s2s_tokens &t, long long batch, long long tokens,
                  long long heads, long long width) {
    long long n[3] = {batch, tokens, heads}, s[3] = {t.batch, t.token, t.head};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2 - i; ++j)
            if (s[j] > s[j + 1]) {
                const long long a = s[j], b = n[j];
                s[j] = s[j + 1], n[j] = n[j + 1];
                s[j + 1] = a, n[j + 1] = b;
            }
    __int128 span = width;
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        if (s[i] < span) return refuse("%s: %s: written elements overlap", op, name);
        span += (__int128)(n[i] - 1) * s[i];
    }
    return 0;
}

int check_array(const char *op, const char *name, const void *p, size_t align, int dev) {
    if ((uintptr_t)p % align) return refuse("%s: %s is not aligned to its elements", op, name);
    return check_memory(op, name, p, dev);
}

// The strides the kernels go by: that of a dimension of one counts for nothing, so that it
// does not spoil the others' alignment either.
Strides strides(const s2s_tokens &t, int batch, int tokens, int heads) {
    return Strides{batch > 1 ? t.batch : 0, tokens > 1 ? t.token : 0, heads > 1 ? t.head : 0};
}

int attention_sizes(const char *op, const s2s_attention_args *a) {
    if (!is_real_type(a->dtype)) return refuse("%s: dtype %d is not f32, f16 or bf16", op, a->dtype);
    if (a->batch < 0 || a->q_tokens < 0 || a->k_tokens < 0)
        return refuse("%s: negative batch or token count", op);
    if (a->q_heads < 1 || a->k_heads < 1 || a->q_heads % a->k_heads)
        return refuse("%s: %d query heads are no multiple of %d key heads", op, a->q_heads, a->k_heads);
    if (a->width < 1 || a->width > 128) return refuse("%s: width %d is not in 1 to 128", op, a->width);
    // token counts and (query token, head of a group) pairs are ints in the kernels
    if (a->k_tokens > (1 << 30) || (long long)a->q_tokens * a->q_heads > (1LL << 30))
        return refuse("%s: over 2^30 tokens, or query tokens times heads", op);
    if ((long long)a->batch * a->k_heads > (1 << 20)) return refuse("%s: over 2^20 batch entries times key heads", op);
    // a workgroup takes 64 such pairs or more, of one batch entry and key head (a launch holds
    // 2^24 of them)
    const long long cols = (long long)a->q_tokens * (a->q_heads / a->k_heads);
    if ((long long)a->batch * a->k_heads * ((cols + 63) / 64) >= (1 << 24))
        return refuse("%s: over 2^30 query tokens times heads of the batch", op);
    return 0;
}

int window_sizes(const char *op, int window, int sinks) {
    if (window < 1 || window > (1 << 30)) return refuse("%s: a window of %d keys is not in 1 to 2^30", op, window);
    if (sinks < 0 || sinks > (1 << 30)) return refuse("%s: %d sinks are not in 0 to 2^30", op, sinks);
    return 0;
}

AttnOpArgs attention_args(const s2s_attention_args *a, int window = 0, int sinks = 0) {
    AttnOpArgs k{};
    k.window = window;
    k.sinks = sinks;
    k.batch = a->batch;
    k.nq = a->q_tokens;
    k.nk = a->k_tokens;
    k.hq = a->q_heads;
    k.hk = a->k_heads;
    k.group = a->q_heads / a->k_heads;
    k.width = a->width;
    k.causal = a->causal != 0;
    k.scale = a->scale;
    k.cap = a->cap;
    k.q = a->q.data;
    k.k = a->k.data;
    k.v = a->v.data;
    k.out = a->out.data;
    k.sq = strides(a->q, a->batch, a->q_tokens, a->q_heads);
    k.sk = strides(a->k, a->batch, a->k_tokens, a->k_heads);
    k.sv = strides(a->v, a->batch, a->k_tokens, a->k_heads);
    k.so = strides(a->out, a->batch, a->q_tokens, a->q_heads);
    if (a->k_tokens <= 1) k.sk.t = k.sv.t = a->width;  // (a tile's rows past the last do not overlap it)
    k.q_lens = a->q_lens;
    k.k_lens = a->k_lens;
    k.prefix = a->prefix;
    // (without keys the row is zeros whatever else is given)
    k.q_docs = a->k_tokens > 0 ? a->q_docs : nullptr;
    k.k_docs = a->k_tokens > 0 ? a->k_docs : nullptr;
    k.q_docs_b = a->q_docs_batch;
    k.k_docs_b = a->k_docs_batch;
    k.q_pos = a->k_tokens > 0 ? a->q_pos : nullptr;
    k.k_pos = a->k_tokens > 0 ? a->k_pos : nullptr;
    k.q_pos_b = a->q_pos_batch;
    k.k_pos_b = a->k_pos_batch;
    k.slopes = a->slopes;
    k.table = a->table;
    k.table_size = a->table_size;
    return k;
}

int shared_sizes(const char *op, const s2s_shared_attention_args *s) {
    const s2s_attention_args *a = &s->own;
    if (s->shared_tokens < 0) return refuse("%s: negative shared tokens", op);
    if ((long long)s->shared_tokens + a->k_tokens > (1 << 30)) return refuse("%s: over 2^30 shared and own tokens", op);
    // the columns of all entries are an int, and the join has one part of a workgroup for each
    if ((long long)a->batch * a->q_tokens * a->q_heads > (1 << 26))
        return refuse("%s: over 2^26 query tokens times heads of the batch", op);
    return 0;
}

AttnOpArgs shared_args(const s2s_shared_attention_args *s) {
    AttnOpArgs k = attention_args(&s->own);
    k.shared_k = s->shared_k.data;
    k.shared_v = s->shared_v.data;
    k.shared_sk = strides(s->shared_k, 1, s->shared_tokens, s->own.k_heads);
    k.shared_sv = strides(s->shared_v, 1, s->shared_tokens, s->own.k_heads);
    if (s->shared_tokens <= 1) k.shared_sk.t = k.shared_sv.t = s->own.width;
    k.shared_nk = s->shared_tokens;
    k.shared_lens = s->shared_lens;
    return k;
}

// A call whose sizes have been checked; window 0: none; `s`: the call whose own part `a` is, or null.
int attention_call(const char *op, const s2s_attention_args *a, int window, int sinks, const s2s_shared_attention_args *s,
                   void *workspace, uint64_t workspace_bytes, void *stream) {
    if (!std::isfinite(a->scale)) return refuse("%s: the scale is not finite", op);
    if (!(a->cap >= 0.f) || !std::isfinite(a->cap)) return refuse("%s: the cap is negative or not finite", op);
    if (a->cap > 0.f && a->cap < 1e-6f) return refuse("%s: a cap below 1e-6", op);
    // (their products with log2(e), and the quotient of the two, are finite)
    if (std::fabs(a->scale) > 1e30f) return refuse("%s: the scale is past 10^30", op);
    if (a->cap > 1e30f) return refuse("%s: the cap is past 10^30", op);
    if (a->prefix && !a->causal) return refuse("%s: a prefix without the causal mask", op);
    // (an array of no elements may have no address, or one that is nobody's)
    const bool keys = a->k_tokens > 0, some = keys && a->batch > 0 && a->q_tokens > 0;
    if (some && !a->q_docs != !a->k_docs) return refuse("%s: documents of queries and keys come together", op);
    if (some && !a->q_pos != !a->k_pos) return refuse("%s: positions of queries and keys come together", op);
    if (a->q_pos && !a->slopes && !a->table) return refuse("%s: positions without slopes or table", op);
    if (a->table && (a->table_size < 1 || a->table_size % 2 == 0 || a->table_size > (1 << 24)))
        return refuse("%s: a table of %d entries: an odd number up to 2^24 is wanted", op, a->table_size);
    if (a->table && (long long)a->q_heads * a->table_size > (1 << 30)) return refuse("%s: a table over 2^30 entries", op);
    if (a->q_docs_batch < 0 || a->k_docs_batch < 0 || a->q_pos_batch < 0 || a->k_pos_batch < 0 ||
        a->q_docs_batch > kMaxStride || a->k_docs_batch > kMaxStride || a->q_pos_batch > kMaxStride ||
        a->k_pos_batch > kMaxStride)
        return refuse("%s: a negative or impossible batch stride", op);
    // (a wave per key tile, of 32 keys at least, makes the documents' summary, four a workgroup, of which
    // a launch holds less than 2^24)
    if (a->k_docs && ((long long)a->batch * ((a->k_tokens + 31LL) / 32) + 3) / 4 >= (1 << 24))
        return refuse("%s: documents of over 2^31 keys of the batch", op);
    if (a->batch == 0 || a->q_tokens == 0) return 0;
    OnDevice on;
    const hipStream_t st = (hipStream_t)stream;
    hipError_t e = on.enter(st);
    if (e != hipSuccess) return refuse_hip(op, "the stream's device", e);
    if (int rc = check_tokens(op, "q", a->q, a->dtype, on.dev)) return rc;
    if (int rc = check_tokens(op, "out", a->out, a->dtype, on.dev)) return rc;
    if (int rc = check_written(op, "out", a->out, a->batch, a->q_tokens, a->q_heads, a->width)) return rc;
    if (keys) {
        if (int rc = check_tokens(op, "k", a->k, a->dtype, on.dev)) return rc;
        if (int rc = check_tokens(op, "v", a->v, a->dtype, on.dev)) return rc;
        // 64 tokens of a tile are reached by 32-bit byte offsets from its first
        if (a->k_tokens > 1 && (a->k.token > (1 << 22) || a->v.token > (1 << 22)))
            return refuse("%s: a token stride of k or v over 2^22 elements", op);
    }
    const bool shared = s && s->shared_tokens > 0;
    if (shared) {
        if (int rc = check_tokens(op, "shared_k", s->shared_k, a->dtype, on.dev)) return rc;
        if (int rc = check_tokens(op, "shared_v", s->shared_v, a->dtype, on.dev)) return rc;
        if (s->shared_tokens > 1 && (s->shared_k.token > (1 << 22) || s->shared_v.token > (1 << 22)))
            return refuse("%s: a token stride of shared_k or shared_v over 2^22 elements", op);
    }
    if (a->out.data == a->q.data || (keys && (a->out.data == a->k.data || a->out.data == a->v.data)) ||
        (shared && (a->out.data == s->shared_k.data || a->out.data == s->shared_v.data)))
        return refuse("%s: out is an input", op);
    const struct {
        const char *name;
        const void *p;
    } arrays[] = {{"q_lens", a->q_lens},
                  {"k_lens", a->k_lens},
                  {"prefix", a->prefix},
                  {"q_docs", a->q_docs},
                  {"k_docs", keys ? a->k_docs : nullptr},
                  {"q_pos", a->q_pos},
                  {"k_pos", keys ? a->k_pos : nullptr},
                  {"slopes", a->slopes},
                  {"table", a->table},
                  {"shared_lens", s ? s->shared_lens : nullptr}};
    for (const auto &x : arrays)
        if (x.p)
            if (int rc = check_array(op, x.name, x.p, 4, on.dev)) return rc;
    const AttnOpArgs k = s ? shared_args(s) : attention_args(a, window, sinks);
    const size_t need = s ? shared_attn_op_workspace(a->dtype, k) : attn_op_workspace(a->dtype, k);
    if (need) {
        if (!workspace || workspace_bytes < need)
            return refuse("%s: a workspace of %zu bytes is needed, %llu are given", op, need,
                          workspace ? (unsigned long long)workspace_bytes : 0ULL);
        if (int rc = check_array(op, "workspace", workspace, 16, on.dev)) return rc;
    }
    e = s ? launch_shared_attention_op(a->dtype, k, workspace, st) : launch_attention_op(a->dtype, k, workspace, st);
    return e == hipSuccess ? 0 : refuse_hip(op, "the launch", e);
}

// Rotary positions, behind a norm of the heads if `n` is not null (`a` is its part then).
int rotary_call(const char *op, const s2s_rotary_args *a, const s2s_norm_rotary_args *n, void *stream) {
    if (!is_real_type(a->dtype)) return refuse("%s: dtype %d is not f32, f16 or bf16", op, a->dtype);
    if (a->batch < 0 || a->tokens < 0 || a->q_heads < 1 || a->k_heads < 0)
        return refuse("%s: negative sizes, or no query head", op);
    if (a->width < 2 || a->width > 65536) return refuse("%s: width %d is not in 2 to 65536", op, a->width);
    if (a->axes < 1 || a->axes > 4) return refuse("%s: %d axes: 1 to 4 are wanted", op, a->axes);
    if (a->pairs < 1 || a->pairs > 128 || 2 * a->pairs > a->width)
        return refuse("%s: %d pairs: 1 to 128 that fit the width are wanted", op, a->pairs);
    if ((long long)a->batch * a->tokens > (1 << 30) || a->q_heads > 65535 || a->k_heads > 65535)
        return refuse("%s: over 2^30 tokens or 65535 heads", op);
    if (!a->inv_freq || !a->pair_axis) return refuse("%s: inv_freq or pair_axis is null", op);
    for (int i = 0; i < a->pairs; ++i) {
        if (!(std::fabs(a->inv_freq[i]) < 1048576.0)) return refuse("%s: inv_freq[%d] is not below 2^20", op, i);
        if (a->pair_axis[i] >= a->axes) return refuse("%s: pair_axis[%d] is no axis", op, i);
    }
    if (a->pos_batch < 0 || a->pos_batch > kMaxStride) return refuse("%s: a negative or impossible batch stride", op);
    if (n) {
        if (!(n->eps >= 0.f) || !std::isfinite(n->eps) || !std::isfinite(n->weight_offset))
            return refuse("%s: eps is negative, or eps or weight_offset not finite", op);
        if (n->q_weight_head < 0 || n->k_weight_head < 0 || n->q_weight_head > kMaxStride || n->k_weight_head > kMaxStride)
            return refuse("%s: a negative or impossible head stride of the weights", op);
    }
    if (a->batch == 0 || a->tokens == 0) return 0;
    if (a->k_heads > 0 && a->q_out.data && a->k_out.data == a->q_out.data)
        return refuse("%s: q_out and k_out are the same array", op);
    // (other workgroups may not have read the other input yet)
    if (a->k_heads > 0 && a->q_out.data && (a->q_out.data == a->k.data || a->k_out.data == a->q.data))
        return refuse("%s: q's output is k, or k's is q", op);
    OnDevice on;
    const hipStream_t st = (hipStream_t)stream;
    hipError_t e = on.enter(st);
    if (e != hipSuccess) return refuse_hip(op, "the stream's device", e);
    const bool has_k = a->k_heads > 0;
    if (int rc = check_tokens(op, "q", a->q, a->dtype, on.dev)) return rc;
    if (int rc = check_tokens(op, "q_out", a->q_out, a->dtype, on.dev)) return rc;
    if (int rc = check_written(op, "q_out", a->q_out, a->batch, a->tokens, a->q_heads, a->width)) return rc;
    if (has_k) {
        if (int rc = check_tokens(op, "k", a->k, a->dtype, on.dev)) return rc;
        if (int rc = check_tokens(op, "k_out", a->k_out, a->dtype, on.dev)) return rc;
        if (int rc = check_written(op, "k_out", a->k_out, a->batch, a->tokens, a->k_heads, a->width)) return rc;
    }
    auto same = [&](const s2s_tokens &x, const s2s_tokens &y, int heads) {
        const Strides s = strides(x, a->batch, a->tokens, heads), t = strides(y, a->batch, a->tokens, heads);
        return x.data != y.data || (s.b == t.b && s.t == t.t && s.h == t.h);
    };
    if (!same(a->q, a->q_out, a->q_heads) || (has_k && !same(a->k, a->k_out, a->k_heads)))
        return refuse("%s: in place, the output's strides must be the input's", op);
    if (!a->pos) return refuse("%s: pos is null", op);
    if (int rc = check_array(op, "pos", a->pos, 4, on.dev)) return rc;
    if (a->lens)
        if (int rc = check_array(op, "lens", a->lens, 4, on.dev)) return rc;
    if (n) {
        if (!n->q_weight || (has_k && !n->k_weight)) return refuse("%s: q_weight or k_weight is null", op);
        if (int rc = check_array(op, "q_weight", n->q_weight, 4, on.dev)) return rc;
        if (has_k)
            if (int rc = check_array(op, "k_weight", n->k_weight, 4, on.dev)) return rc;
    }
    NormRotaryArgs m{};
    RotaryArgs &k = m.r;
    k.batch = a->batch;
    k.tokens = a->tokens;
    k.hq = a->q_heads;
    k.hk = a->k_heads;
    k.width = a->width;
    k.axes = a->axes;
    k.pairs = a->pairs;
    k.adjacent = a->adjacent != 0;
    k.q = a->q.data;
    k.qo = a->q_out.data;
    k.sq = strides(a->q, a->batch, a->tokens, a->q_heads);
    k.sqo = strides(a->q_out, a->batch, a->tokens, a->q_heads);
    if (has_k) {
        k.k = a->k.data;
        k.ko = a->k_out.data;
        k.sk = strides(a->k, a->batch, a->tokens, a->k_heads);
        k.sko = strides(a->k_out, a->batch, a->tokens, a->k_heads);
    }
    k.pos = a->pos;
    k.pos_b = a->pos_batch;
    k.lens = a->lens;
    for (int i = 0; i < a->pairs; ++i) {
        // inv_freq / 2 pi turns, its fraction in 64 bits (long double: 64-bit significand)
        // inv_freq below 2^20 leaves whole turns that an int holds
        long double t = (long double)a->inv_freq[i] * 0.15915494309189533576888376337251436L;
        t -= (long double)(int)t;
        if (t < 0) t += 1.0L;
        const unsigned long long f = t >= 1.0L ? 0ULL : (unsigned long long)(t * 18446744073709551616.0L);
        k.freq[i] = a->inverse ? 0ULL - f : f;
        k.axis[i] = a->pair_axis[i];
    }
    if (n) {
        m.qw = n->q_weight;
        m.kw = n->k_weight;
        m.qw_head = a->q_heads > 1 ? n->q_weight_head : 0;
        m.kw_head = a->k_heads > 1 ? n->k_weight_head : 0;
        m.offset = n->weight_offset;
        m.eps = n->eps;
    }
    e = n ? launch_norm_rotary_op(a->dtype, m, st) : launch_rotary_op(a->dtype, k, st);
    return e == hipSuccess ? 0 : refuse_hip(op, "the launch", e);
}

}  // namespace

extern "C" {

int s2s_attention_workspace(const s2s_attention_args *a, uint64_t *bytes) {
    if (!a || !bytes) return refuse("s2s_attention_workspace: null argument");
    if (int rc = attention_sizes("s2s_attention_workspace", a)) return rc;
    *bytes = attn_op_workspace(a->dtype, attention_args(a));
    return 0;
}

int s2s_attention(const s2s_attention_args *a, void *workspace, uint64_t workspace_bytes, void *stream) {
    const char *op = "s2s_attention";
    if (!a) return refuse("%s: null argument", op);
    if (int rc = attention_sizes(op, a)) return rc;
    return attention_call(op, a, 0, 0, nullptr, workspace, workspace_bytes, stream);
}

int s2s_window_attention_workspace(const s2s_attention_args *a, int window, int sinks, uint64_t *bytes) {
    const char *op = "s2s_window_attention_workspace";
    if (!a || !bytes) return refuse("%s: null argument", op);
    if (int rc = attention_sizes(op, a)) return rc;
    if (int rc = window_sizes(op, window, sinks)) return rc;
    *bytes = attn_op_workspace(a->dtype, attention_args(a, window, sinks));
    return 0;
}

int s2s_window_attention(const s2s_attention_args *a, int window, int sinks, void *workspace, uint64_t workspace_bytes,
                         void *stream) {
    const char *op = "s2s_window_attention";
    if (!a) return refuse("%s: null argument", op);
    if (int rc = attention_sizes(op, a)) return rc;
    if (int rc = window_sizes(op, window, sinks)) return rc;
    // (a document's own first keys are not known)
    if (sinks > 0 && (a->q_docs || a->k_docs)) return refuse("%s: sinks with documents", op);
    return attention_call(op, a, window, sinks, nullptr, workspace, workspace_bytes, stream);
}

int s2s_shared_attention_workspace(const s2s_shared_attention_args *s, uint64_t *bytes) {
    const char *op = "s2s_shared_attention_workspace";
    if (!s || !bytes) return refuse("%s: null argument", op);
    if (int rc = attention_sizes(op, &s->own)) return rc;
    if (int rc = shared_sizes(op, s)) return rc;
    *bytes = shared_attn_op_workspace(s->own.dtype, shared_args(s));
    return 0;
}

int s2s_shared_attention(const s2s_shared_attention_args *s, void *workspace, uint64_t workspace_bytes, void *stream) {
    const char *op = "s2s_shared_attention";
    if (!s) return refuse("%s: null argument", op);
    const s2s_attention_args *a = &s->own;
    if (int rc = attention_sizes(op, a)) return rc;
    if (int rc = shared_sizes(op, s)) return rc;
    if (a->prefix || a->q_docs || a->k_docs || a->q_pos || a->k_pos || a->table)
        return refuse("%s: prefix, documents, positions and table are not taken", op);
    return attention_call(op, a, 0, 0, s, workspace, workspace_bytes, stream);
}

int s2s_rotary(const s2s_rotary_args *a, void *stream) {
    const char *op = "s2s_rotary";
    if (!a) return refuse("%s: null argument", op);
    return rotary_call(op, a, nullptr, stream);
}

int s2s_norm_rotary(const s2s_norm_rotary_args *a, void *stream) {
    const char *op = "s2s_norm_rotary";
    if (!a) return refuse("%s: null argument", op);
    return rotary_call(op, &a->rotary, a, stream);
}

int s2s_rms_norm(const s2s_rms_norm_args *a, void *stream) {
    const char *op = "s2s_rms_norm";
    if (!a) return refuse("%s: null argument", op);
    if (!is_real_type(a->dtype)) return refuse("%s: dtype %d is not f32, f16 or bf16", op, a->dtype);
    const bool q8 = a->out_dtype == S2S_E4M3;
    if (!q8 && a->out_dtype != a->dtype) return refuse("%s: out_dtype %d is neither dtype nor e4m3", op, a->out_dtype);
    if (a->rows < 0 || a->rows > (1LL << 31) - 1) return refuse("%s: %lld rows", op, (long long)a->rows);
    if (a->cols < 1 || a->cols > (1 << 24)) return refuse("%s: %d columns are not in 1 to 2^24", op, a->cols);
    if (!(a->eps >= 0.f) || !std::isfinite(a->eps) || !std::isfinite(a->weight_offset))
        return refuse("%s: eps is negative, or eps or weight_offset not finite", op);
    if (!q8 && (a->scales || a->group)) return refuse("%s: scales or a group without an e4m3 output", op);
    if (q8 && !a->scales && a->rows > 0) return refuse("%s: scales is null", op);
    if (a->group < 0 || a->group % 8) return refuse("%s: a group of %d is no multiple of 8", op, a->group);
    if (a->rows == 0) return 0;
    if (!a->x || !a->out || !a->weight) return refuse("%s: x, out or weight is null", op);
    OnDevice on;
    const hipStream_t st = (hipStream_t)stream;
    hipError_t e = on.enter(st);
    if (e != hipSuccess) return refuse_hip(op, "the stream's device", e);
    const size_t ts = type_size(a->dtype);
    const struct {
        const char *name;
        const void *p;
        long long stride;
        size_t align;
        bool written;
    } arrays[] = {{"x", a->x, a->x_stride, ts, false},
                  {"res", a->res, a->res_stride, ts, false},
                  {"sum", a->sum, a->sum_stride, ts, true},
                  {"out", a->out, a->out_stride, q8 ? 1 : ts, true}};
    for (const auto &x : arrays) {
        if (!x.p) continue;
        if (x.stride < 0 || x.stride > kMaxStride) return refuse("%s: %s has a negative or impossible stride", op, x.name);
        if (x.written && a->rows > 1 && x.stride < a->cols) return refuse("%s: %s: written elements overlap", op, x.name);
        if (int rc = check_array(op, x.name, x.p, x.align, on.dev)) return rc;
    }
    // in place: the same rows, or none
    for (int i = 2; i < 4; ++i)
        for (int j = 0; j < 2; ++j)
            if (arrays[i].p && arrays[i].p == arrays[j].p &&
                ((a->rows > 1 && arrays[i].stride != arrays[j].stride) || (i == 3 && q8)))
                return refuse("%s: %s is %s but not in its rows' places", op, arrays[i].name, arrays[j].name);
    if (a->sum && a->sum == a->out) return refuse("%s: sum and out are the same array", op);
    if (int rc = check_array(op, "weight", a->weight, 4, on.dev)) return rc;
    if (q8)
        if (int rc = check_array(op, "scales", a->scales, 4, on.dev)) return rc;
    RmsNormArgs k{};
    k.rows = a->rows;
    k.cols = a->cols;
    k.group = a->group > 0 && a->group < a->cols ? a->group : a->cols;
    k.groups = (a->cols + k.group - 1) / k.group;
    k.x = a->x;
    k.res = a->res;
    k.sum = a->sum;
    k.out = a->out;
    const bool many = a->rows > 1;  // (one row's stride counts for nothing)
    k.xs = many ? a->x_stride : 0;
    k.rs = many ? a->res_stride : 0;
    k.ss = many ? a->sum_stride : 0;
    k.os = many ? a->out_stride : 0;
    k.weight = a->weight;
    k.offset = a->weight_offset;
    k.eps = a->eps;
    k.scales = a->scales;
    e = launch_rms_norm_op(a->dtype, q8, k, st);
    return e == hipSuccess ? 0 : refuse_hip(op, "the launch", e);
}

}  // extern "C"
