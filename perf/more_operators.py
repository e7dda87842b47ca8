"""More transformer operators of the package (`ops`) as timed and checked cases.

Three that stand beside its attention, rotary positions and RMS norm:

  window       attention with a sliding window and a few first keys (sinks) that every query sees
  shared       attention of a batch whose entries all read one long prefix and each its own keys
  norm_rotary  q and k normed head by head and turned by their positions, in one pass

With `own` false, `run` computes them from elementary torch operations in 32 bits (angles in 64).
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    def window(name, dtype, batch, q_tokens, k_tokens, heads, kv_heads, width, layout, window, **more):
        c = dict(name=name, op="window", dtype=dtype, batch=batch, q_tokens=q_tokens, k_tokens=k_tokens, heads=heads,
                 kv_heads=kv_heads, width=width, layout=layout, window=window, sinks=0, cap=0.0, causal=True,
                 slopes=False, docs=0, ragged=False)
        c.update(more)
        return c

    def shared(name, dtype, batch, q_tokens, shared_tokens, k_tokens, heads, kv_heads, width, **more):
        c = dict(name=name, op="shared", dtype=dtype, batch=batch, q_tokens=q_tokens, shared_tokens=shared_tokens,
                 k_tokens=k_tokens, heads=heads, kv_heads=kv_heads, width=width, cap=0.0, causal=True, slopes=False,
                 ragged=False, part=False)
        c.update(more)
        return c

    return [
        # a few query tokens over a short sequence: the smallest call, latency alone
        window("window_few_f16", "f16", 1, 5, 700, 8, 8, 64, "cache", 128, sinks=4),
        # the next token of 32 sequences of different lengths, each over the last 4096 of its cache
        window("window_step_bf16", "bf16", 32, 1, 16384, 32, 8, 128, "cache", 4096, sinks=4, ragged=True),
        # one long odd prompt
        window("window_prompt_bf16", "bf16", 1, 16391, 16391, 16, 4, 128, "packed", 4096, sinks=4),
        # the tokens of a 128 x 128 plane, each seeing the eight rows around it, the width of this package's heads
        window("window_plane_f32", "f32", 1, 16384, 16384, 6, 6, 30, "packed", 1024, causal=False),
        # the next token of four sequences that share a short prefix
        shared("shared_few_f16", "f16", 4, 1, 333, 40, 8, 8, 64),
        # the next token of 64 sequences that began with the same document, with up to 1024 tokens of their own
        shared("shared_step_bf16", "bf16", 64, 1, 16384, 1024, 32, 8, 128, ragged=True),
        # eight continuations of one prompt, 500 new tokens each
        shared("shared_tail_bf16", "bf16", 8, 500, 8191, 500, 32, 8, 128),
        # 36 crops of 8 x 8 tokens that all read a coarse view of the whole image (33 x 33 tokens)
        shared("shared_crops_f32", "f32", 36, 64, 1089, 64, 6, 6, 30, causal=False),
        # the next token's q and k of 32 sequences
        dict(name="norm_rotary_step_bf16", op="norm_rotary", dtype="bf16", batch=32, tokens=1, heads=32, kv_heads=8,
             width=128, axes=3, pairs=64, adjacent=False, each=False),
        # the tokens of 13 frames of 45 x 40, the width of this package's heads, a weight for every head's channel
        dict(name="norm_rotary_video_f32", op="norm_rotary", dtype="f32", batch=2, tokens=23400, heads=6, kv_heads=6,
             width=30, axes=3, pairs=15, adjacent=True, each=True),
        # heads of which a half is turned, an odd number of tokens
        dict(name="norm_rotary_part_f16", op="norm_rotary", dtype="f16", batch=1, tokens=4099, heads=16, kv_heads=16,
             width=80, axes=2, pairs=20, adjacent=False, each=False),
        # the tokens of a large image's q and k
        dict(name="norm_rotary_image_bf16", op="norm_rotary", dtype="bf16", batch=1, tokens=16384, heads=32, kv_heads=8,
             width=128, axes=2, pairs=64, adjacent=False, each=False),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST = 16 * 16391 ** 2  # (head, query, key) triples of a case's batch
CACHE = 32 * 16384 * 8 * 128  # elements of k


def draw(rng):
    op = rng.choice(("window", "window", "shared", "shared", "norm_rotary"))
    dtype = rng.choice(("bf16", "f16", "bf16", "f32"))
    width = rng.choice((64, 128, 128, 96, 80, 32, 30, 10))
    kv = rng.choice((1, 2, 4, 6, 8))
    heads = kv * rng.choice((1, 1, 2, 4, 8)) if kv < 6 else kv * rng.choice((1, 2, 4))
    if op == "norm_rotary":
        tokens, batch = log_int(rng, 1, 30000), rng.choice((1, 1, 2, 7, 32))
        while batch * tokens * (heads + kv) * width > 16384 * 40 * 128:
            tokens, batch = max(1, tokens // 2), max(1, batch // 2)
        pairs = rng.choice((width // 2, width // 2, max(4, width // 4)))
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv, width=width,
                    axes=rng.randint(1, 4), pairs=pairs, adjacent=rng.random() < 0.5, each=rng.random() < 0.3)
    c = dict(op=op, dtype=dtype, batch=1, q_tokens=1, k_tokens=1, heads=heads, kv_heads=kv, width=width,
             cap=rng.choice((0.0, 0.0, 0.0, 50.0)), causal=True, slopes=rng.random() < 0.25, ragged=rng.random() < 0.5)
    step = rng.random() < 0.5
    if op == "window":
        c.update(layout="cache", window=log_int(rng, 8, 8192), sinks=rng.choice((0, 1, 4, 4, 16, 100)), docs=0)
        if step:
            c.update(batch=rng.choice((1, 2, 5, 16, 32)), q_tokens=rng.choice((1, 1, 1, 3, 4)))
            c["k_tokens"] = log_int(rng, 64, min(131072, CACHE // (c["batch"] * kv * width)))
        else:
            c["q_tokens"] = c["k_tokens"] = n = log_int(rng, 16, 12000)
            c.update(layout="packed", causal=rng.random() < 0.7)
            if rng.random() < 0.3:
                c.update(layout="cache", q_tokens=max(1, int(n * rng.uniform(0.1, 0.9))))
            elif c["sinks"] == 0 and rng.random() < 0.5:
                c.update(docs=rng.randint(2, 8), ragged=False)
            c["batch"] = max(1, min(rng.choice((1, 2, 3, 8)), MOST // (heads * c["q_tokens"] * n)))
        while c["batch"] * heads * c["q_tokens"] * c["k_tokens"] > MOST:
            c["q_tokens"], c["k_tokens"] = max(1, c["q_tokens"] // 2), max(1, c["k_tokens"] // 2)
        return c
    c.update(batch=rng.choice((2, 3, 8, 16, 64, 100)), causal=rng.random() < 0.8, part=rng.random() < 0.3)
    c["shared_tokens"] = log_int(rng, 16, 32768)
    if step:
        c["q_tokens"] = rng.choice((1, 1, 1, 2, 4))
        c["k_tokens"] = log_int(rng, 4, max(8, min(4096, CACHE // (c["batch"] * kv * width))))
    else:
        c["q_tokens"] = c["k_tokens"] = log_int(rng, 8, 2000)
    while c["batch"] * heads * c["q_tokens"] * (c["shared_tokens"] + c["k_tokens"]) > MOST // 4:
        c["batch"], c["shared_tokens"] = max(1, c["batch"] // 2), max(16, c["shared_tokens"] // 2)
        c["q_tokens"], c["k_tokens"] = max(1, c["q_tokens"] // 2), max(1, c["k_tokens"] // 2)
    return c


# ---- inputs ------------------------------------------------------------------------------------


def spread(n, total, least=0.25):
    """n lengths from least * total to total."""
    return [max(1, math.ceil(total * (least + (1 - least) * (i + 1) / n))) for i in range(n)]


def parts(n, total):
    """Document lengths 1 : 2 : ... : n of `total`; what is left over is padding."""
    unit = total / (n * (n + 1) / 2 + 0.25)
    return [max(1, int(unit * (i + 1))) for i in range(n)] if total >= n * (n + 1) else [max(1, total // n)] * min(n, total)


def lengths(case, order):
    got = spread(case["batch"], case["k_tokens"]) if case["ragged"] else [case["k_tokens"]] * case["batch"]
    order.shuffle(got)
    return got


def shared_lengths(case):
    """Where only parts of the prefix are read: none of it by the first entry, all of it by the last."""
    b, n = case["batch"], case["shared_tokens"]
    return [n * i // max(1, b - 1) for i in range(b)] if case["part"] else [n] * b


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    order = random.Random(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    st = {"case": case}
    b, d, heads, kv = case["batch"], case["width"], case["heads"], case["kv_heads"]
    if case["op"] == "norm_rotary":
        n, axes = case["tokens"], case["axes"]
        # one projection's output; its heads differ in size
        qkv = (normal(b, n, heads + 2 * kv, d) * torch.exp(normal(1, 1, heads + 2 * kv, 1))).to(t)
        st["q"], st["k"] = qkv[:, :, :heads], qkv[:, :, heads:heads + kv]
        st["q_out"], st["k_out"] = torch.empty(b, n, heads, d, device=DEV, dtype=t), torch.empty(b, n, kv, d, device=DEV, dtype=t)
        st["q_weight"] = 1 + 0.3 * (normal(heads, d) if case["each"] else normal(d))
        st["k_weight"] = 1 + 0.3 * (normal(kv, d) if case["each"] else normal(d))
        # coordinates on a grid, the first axis (time) far into a stream
        side = max(1, math.isqrt(n))
        i = torch.arange(n, device=DEV)
        grid = torch.stack([i // (side * side) + order.randint(0, 1 << 20), i // side % side, i % side, i % 7], 1)
        start = torch.tensor([order.randint(0, 4096) for _ in range(b)], device=DEV)
        st["pos"] = (grid[None, :, :axes] + start[:, None, None]).int().contiguous()
        share = [case["pairs"] // axes + (a < case["pairs"] % axes) for a in range(axes)]
        st["pair_axis"] = [a for a in range(axes) for _ in range(share[a])]
        st["inv_freq"] = [10000.0 ** (-i / share[a]) for a in range(axes) for i in range(share[a])]
        if own:
            st["plan"] = package().ops.NormRotary(st["inv_freq"], st["pair_axis"], eps=EPS, adjacent=case["adjacent"])
        else:
            st["axis_of"] = torch.tensor(st["pair_axis"], device=DEV)
            st["freq_of"] = torch.tensor(st["inv_freq"], device=DEV, dtype=torch.float64)
        return st
    nq, nk = case["q_tokens"], case["k_tokens"]
    if case["op"] == "window" and case["layout"] == "packed":
        # one projection's output, q, k and v of a token side by side
        qkv = normal(b, nq, heads + 2 * kv, d).to(t)
        st["q"], st["k"], st["v"] = qkv[:, :, :heads], qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:]
    else:
        # a cache with each head's tokens one behind the other
        st["q"] = normal(b, nq, heads, d).to(t)
        st["k"], st["v"] = (normal(b, kv, nk, d).to(t).transpose(1, 2) for _ in range(2))
    st["out"] = torch.zeros(b, nq, heads, d, device=DEV, dtype=t)
    st["scale"] = 1 / math.sqrt(d)
    more = st["more"] = {}
    if case["ragged"]:
        k_lens = lengths(case, order)
        more["k_lens"] = torch.tensor(k_lens, device=DEV, dtype=torch.int32)
        more["q_lens"] = more["k_lens"].clamp(max=nq)
    if case["slopes"]:
        more["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV) / heads)
    sizes = dict(scale=st["scale"], cap=case["cap"], causal=case["causal"])
    if case["op"] == "shared":
        n = case["shared_tokens"]
        st["shared_k"], st["shared_v"] = (normal(kv, n, d).to(t).transpose(0, 1) for _ in range(2))
        if case["part"]:
            more["shared_lens"] = torch.tensor(shared_lengths(case), device=DEV, dtype=torch.int32)
        if own:
            st["plan"] = package().ops.SharedAttention(case["dtype"], b, nq, n, nk, heads, kv, d, **sizes)
    else:
        if case["docs"]:
            ids = torch.full((b, nk), -1, dtype=torch.int32)
            for row in ids:
                at, lens = 0, parts(case["docs"], nk)
                order.shuffle(lens)
                for j, n in enumerate(lens):
                    row[at:at + n] = j
                    at += n
            more["q_docs"] = more["k_docs"] = ids.to(DEV)
        if own:
            st["plan"] = package().ops.Attention(case["dtype"], b, nq, nk, heads, kv, d, window=case["window"],
                                                 sinks=case["sinks"], **sizes)
    if own:
        st["workspace"] = torch.empty(st["plan"].workspace_bytes, device=DEV, dtype=torch.uint8)
    return st


def package():
    return importlib.import_module("swin2sr-rs_amd")


# ---- one pass ----------------------------------------------------------------------------------


def run(st):
    return {"window": run_window, "shared": run_shared, "norm_rotary": run_norm_rotary}[st["case"]["op"]](st)


def scores(q, k, scale, cap):
    """f32 [batch][heads][q_tokens][k_tokens] of q [batch][q_tokens][heads][width] and k [batch or 1][k_tokens][kv][width]."""
    b, nq, heads, d = q.shape
    kv = k.shape[2]
    rows = q.float().view(b, nq, kv, heads // kv, d).permute(0, 2, 3, 1, 4)
    if k.shape[0] == b:
        s = rows.reshape(b, kv, -1, d) @ k.float().permute(0, 2, 3, 1)
        s = s.view(b, heads, nq, -1)
    else:
        s = rows.transpose(0, 1).reshape(kv, -1, d) @ k[0].float().permute(1, 2, 0)
        s = s.view(kv, b, heads // kv, nq, -1).transpose(0, 1).reshape(b, heads, nq, -1)
    s = s.mul_(scale)
    if cap:
        s.div_(cap).tanh_().mul_(cap)
    return s


def weighted(p, v):
    """[batch][heads][q_tokens][width] of weights [batch][heads][q_tokens][k_tokens] and v [batch or 1][k_tokens][kv][width]."""
    b, heads, nq, nk = p.shape
    kv, d = v.shape[2], v.shape[3]
    if v.shape[0] == b:
        return (p.reshape(b, kv, -1, nk) @ v.float().transpose(1, 2)).view(b, heads, nq, d)
    o = p.view(b, kv, -1, nk).transpose(0, 1).reshape(kv, -1, nk) @ v[0].float().transpose(0, 1)
    return o.view(kv, b, heads // kv, nq, d).transpose(0, 1).reshape(b, heads, nq, d)


def places(q, nk, more):
    """Each query's place among its entry's keys, the keys' places, and which of the two are there."""
    i = torch.arange(q.shape[1], device=DEV)[None, :, None]
    j = torch.arange(nk, device=DEV)[None, None, :]
    kl = more["k_lens"][:, None, None] if "k_lens" in more else nk
    ql = more["q_lens"][:, None, None] if "q_lens" in more else q.shape[1]
    return i + (kl - ql), j, (j < kl) & (i < ql)


def run_window(st):
    c, q, k, v, more = st["case"], st["q"], st["k"], st["v"], st["more"]
    if own:
        st["plan"](q, k, v, st["out"], workspace=st["workspace"], stream=torch.cuda.current_stream().cuda_stream, **more)
        return st["out"]
    at, j, seen = places(q, k.shape[1], more)
    seen = seen & ((j > at - c["window"]) | (j < c["sinks"]))
    seen = seen & (j <= at if c["causal"] else j < at + c["window"])
    if "q_docs" in more:
        dq, dk = more["q_docs"][:, :, None], more["k_docs"][:, None, :]
        seen = seen & (dq == dk) & (dq >= 0)
    s = scores(q, k, st["scale"], c["cap"])
    if "slopes" in more:
        s.sub_(more["slopes"][None, :, None, None] * (at - j).abs().float()[:, None])
    s.masked_fill_(~seen[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    o = weighted(s, v) / total.clamp(min=1e-30)
    return o.transpose(1, 2).to(q.dtype).contiguous()


def run_shared(st):
    c, q, k, v, more = st["case"], st["q"], st["k"], st["v"], st["more"]
    if own:
        st["plan"](q, st["shared_k"], st["shared_v"], k, v, st["out"], workspace=st["workspace"],
                   stream=torch.cuda.current_stream().cuda_stream, **more)
        return st["out"]
    n = c["shared_tokens"]
    at, j, seen = places(q, k.shape[1], more)
    if c["causal"]:
        seen = seen & (j <= at)
    s2 = scores(q, k, st["scale"], c["cap"])
    first = torch.arange(n, device=DEV)[None, None, :]
    start = more["shared_lens"][:, None, None] if "shared_lens" in more else n
    place = at + start
    seen1 = (first < start) & (first <= place if c["causal"] else first >= 0)
    s1 = scores(q, st["shared_k"][None], st["scale"], c["cap"])
    if "slopes" in more:
        slopes = more["slopes"][None, :, None, None]
        s2.sub_(slopes * (at - j).abs().float()[:, None])
        s1.sub_(slopes * (place - first).abs().float()[:, None])
    s2.masked_fill_(~seen[:, None], -math.inf)
    s1.masked_fill_(~seen1[:, None], -math.inf)
    top = torch.maximum(s1.amax(-1, keepdim=True), s2.amax(-1, keepdim=True)).clamp(min=-1e30)
    s1.sub_(top).exp_()
    s2.sub_(top).exp_()
    total = s1.sum(-1, keepdim=True) + s2.sum(-1, keepdim=True)
    o = (weighted(s1, st["shared_v"][None]) + weighted(s2, v)) / total.clamp(min=1e-30)
    if "q_lens" in more:
        i = torch.arange(q.shape[1], device=DEV)[None, None, :, None]
        o.masked_fill_(i >= more["q_lens"][:, None, None, None], 0.0)
    return o.transpose(1, 2).to(q.dtype).contiguous()


def run_norm_rotary(st):
    c = st["case"]
    if own:
        st["plan"](st["q"], st["pos"], st["q_weight"], st["q_out"], k=st["k"], k_weight=st["k_weight"], k_out=st["k_out"],
                   stream=torch.cuda.current_stream().cuda_stream)
        return [st["q_out"], st["k_out"]]
    p = c["pairs"]
    angle = st["pos"][:, :, st["axis_of"]].double() * st["freq_of"]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    got = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        h = x.float()
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w
        if c["adjacent"]:
            a, b = h[..., 0:2 * p:2], h[..., 1:2 * p:2]
            y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = h[..., :p], h[..., p:2 * p]
            y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        got.append(torch.cat((y, h[..., 2 * p:]), -1).to(x.dtype))
    return got


# ---- what a pass cannot do without -------------------------------------------------------------


def seen_of(case, n):
    """(pairs, keys) of one sequence of n keys: how many (query, key) pairs of a head its masks leave, and how many keys any query sees."""
    m, w, s = min(n, case["q_tokens"]), case["window"], case["sinks"]
    at = torch.arange(n - m, n, dtype=torch.int64)
    low = (at - w + 1).clamp(min=0)
    end = at + 1 if case["causal"] else (at + w).clamp(max=n)
    sinks = torch.minimum(low, torch.full_like(low, s))
    first = n - m - w + 1
    return int((end - low + sinks).sum()), n - max(0, first - s) if first > 0 else n


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    b, d, heads, kv = case["batch"], case["width"], case["heads"], case["kv_heads"]
    if case["op"] == "norm_rotary":
        n = b * case["tokens"]
        return {"bytes": n * ((heads + kv) * d * 2 * size + 4 * case["axes"]),
                "flops": n * (heads + kv) * (4 * d + case["pairs"] * 6)}
    lens = lengths(case, random.Random(0))
    queries = sum(min(n, case["q_tokens"]) for n in lens)
    if case["op"] == "window":
        if case["docs"]:
            pairs = b * sum(seen_of(dict(case, q_tokens=n), n)[0] for n in parts(case["docs"], case["k_tokens"]))
            keys = b * case["k_tokens"]
        else:
            pairs, keys = (sum(x) for x in zip(*(seen_of(case, n) for n in lens)))
    else:
        first = shared_lengths(case)
        keys, pairs = sum(lens) + max(first), 0
        for n, s in zip(lens, first):
            m = min(n, case["q_tokens"])
            pairs += m * (n + s) - (m * (m - 1) // 2 if case["causal"] else 0)
    return {"bytes": size * d * (2 * queries * heads + 2 * keys * kv), "flops": 4 * d * heads * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return exact_norm_rotary(st) if case["op"] == "norm_rotary" else exact_attention(st)


def exact_attention(st):
    """Sequence by sequence and head by head, over all the keys that the sequence has, the shared ones in front."""
    c, more = st["case"], st["more"]
    out = torch.zeros(st["out"].shape, device=DEV, dtype=torch.float64)
    group = c["heads"] // c["kv_heads"]
    first = shared_lengths(c) if c["op"] == "shared" else [0] * c["batch"]
    for b in range(c["batch"]):
        n = int(more["k_lens"][b]) if "k_lens" in more else c["k_tokens"]
        m = int(more["q_lens"][b]) if "q_lens" in more else c["q_tokens"]
        s = first[b]
        dist = (torch.arange(m, device=DEV)[:, None] + (s + n - m)) - torch.arange(s + n, device=DEV)[None, :]
        hidden = dist < 0 if c["causal"] else torch.zeros_like(dist, dtype=torch.bool)
        if c["op"] == "window":
            hidden |= dist.abs() >= c["window"]
            if c["sinks"]:
                hidden[:, :c["sinks"]] = dist[:, :c["sinks"]] < 0 if c["causal"] else dist[:, :c["sinks"]] <= -c["window"]
        if "q_docs" in more:
            mine, theirs = more["q_docs"][b, :m, None], more["k_docs"][b, None, :n]
            hidden |= (mine != theirs) | (mine < 0)
        for h in range(c["heads"]):
            key, value = st["k"][b, :n, h // group].double(), st["v"][b, :n, h // group].double()
            if s:
                key = torch.cat((st["shared_k"][:s, h // group].double(), key))
                value = torch.cat((st["shared_v"][:s, h // group].double(), value))
            score = st["q"][b, :m, h].double() @ key.T * st["scale"]
            if c["cap"]:
                score = torch.tanh(score / c["cap"]) * c["cap"]
            if "slopes" in more:
                score = score - more["slopes"][h].double() * dist.abs()
            weight = torch.nan_to_num(torch.softmax(score.masked_fill_(hidden, -math.inf), 1), nan=0.0)
            out[b, :m, h] = weight @ value
    return out


def exact_norm_rotary(st):
    """Each pair of the normed head as a complex number times e^(i angle)."""
    c = st["case"]
    p = c["pairs"]
    angle = torch.stack([st["pos"][:, :, a].double() * f for a, f in zip(st["pair_axis"], st["inv_freq"])], -1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None, :]
    got = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.double()
        y = y / (y.pow(2).sum(3, keepdim=True) / c["width"] + EPS).sqrt() * w.double()
        one, two = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if c["adjacent"] else (slice(0, p), slice(p, 2 * p))
        z = torch.complex(y[..., one], y[..., two]) * turn
        y[..., one], y[..., two] = z.real, z.imag
        got.append(y)
    return got
