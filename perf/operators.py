"""The transformer operators of the package (`ops`) as timed and checked cases.

Three operators that a transformer over image tokens runs one after another:

  attention  softmax(bias + cap tanh(scale q k / cap)) v over views [batch][tokens][heads][width],
             with a bias by the distance of two positions (slopes, or a table), a document mask,
             a causal mask with a prefix that all may read, and lengths of a padded batch
  rotary     q and k turned by the angles of one to four coordinates (time, height, width)
  rms_norm   the residual's addition, the root-mean-square norm, and the result as it is or in
             e4m3 with a scale per group of columns

With `own` false, `run` computes them from elementary torch operations in 32 bits (angles in 64).
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    def attention(name, dtype, batch, q_tokens, k_tokens, heads, kv_heads, width, layout, **more):
        c = dict(name=name, op="attention", dtype=dtype, batch=batch, q_tokens=q_tokens, k_tokens=k_tokens,
                 heads=heads, kv_heads=kv_heads, width=width, layout=layout, cap=0.0, causal=False,
                 prefix=False, slopes=False, window=0, docs=0, ragged=False)
        c.update(more)
        return c

    return [
        # the 8 x 8 windows of a 264 x 264 plane, 6 heads of 30, with a bias by (dy, dx) and the
        # bands of a shifted plane as documents
        attention("windows_f32", "f32", 1089, 64, 64, 6, 6, 30, "packed", window=8, docs=-1),
        # a few query tokens over a short sequence: the smallest call, latency alone
        attention("few_f16", "f16", 1, 5, 77, 8, 8, 64, "cache", ragged=True),
        # nine images of different sizes packed one behind the other, each attending to itself
        attention("images_bf16", "bf16", 1, 11003, 11003, 12, 12, 64, "packed", docs=9),
        # two prompts with a prefix that all tokens read, capped scores
        attention("prompt_bf16", "bf16", 2, 4096, 4096, 32, 8, 128, "packed", causal=True, prefix=True, cap=50.0),
        # one long odd sequence, causal, with a bias that falls with the distance
        attention("long_f16", "f16", 1, 12001, 12001, 16, 4, 128, "packed", causal=True, slopes=True),
        # the next token of 32 sequences of different lengths, over their caches
        attention("step_bf16", "bf16", 32, 1, 8192, 32, 8, 128, "cache", causal=True, cap=50.0, ragged=True),
        # the next token of one very long sequence
        attention("step_long_f16", "f16", 1, 1, 131071, 16, 2, 64, "cache", causal=True, slopes=True),
        # the next token's q and k of 32 sequences
        dict(name="rotary_step_bf16", op="rotary", dtype="bf16", batch=32, tokens=1, heads=32, kv_heads=8,
             width=128, axes=3, pairs=64, adjacent=False, inverse=False),
        # the tokens of 13 frames of 45 x 40, the width of this package's heads
        dict(name="rotary_video_f32", op="rotary", dtype="f32", batch=2, tokens=23400, heads=6, kv_heads=6,
             width=30, axes=3, pairs=15, adjacent=True, inverse=False),
        # the tokens of a large image's q and k
        dict(name="rotary_image_bf16", op="rotary", dtype="bf16", batch=1, tokens=16384, heads=32, kv_heads=8,
             width=128, axes=2, pairs=64, adjacent=False, inverse=False),
        # four tokens of a step, 8-bit output with a scale per token
        dict(name="norm_step_bf16", op="rms_norm", dtype="bf16", rows=4, cols=4096, residual=True, out="e4m3", group=0),
        # the tokens of a long prompt, 8-bit output with a scale per 128 columns
        dict(name="norm_prompt_bf16", op="rms_norm", dtype="bf16", rows=16391, cols=5120, residual=True, out="e4m3",
             group=128),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "rotary", "rms_norm"))
    dtype = rng.choice(("bf16", "f16", "bf16", "f32"))
    if op == "rms_norm":
        cols = rng.choice((180, 60, 720, 1024, 4096, 5120, 8192, log_int(rng, 17, 8192)))
        out = rng.choice(("same", "same", "e4m3"))
        return dict(op=op, dtype=dtype, rows=log_int(rng, 1, min(100000, 80_000_000 // cols)), cols=cols,
                    residual=rng.random() < 0.7, out=out, group=rng.choice((0, 32, 64, 128)) if out == "e4m3" else 0)
    width = rng.choice((64, 128, 128, 96, 80, 32, 30, 10))
    kv = rng.choice((1, 2, 4, 6, 8))
    heads = kv * rng.choice((1, 1, 2, 4, 8)) if kv < 6 else kv * rng.choice((1, 2, 4))
    if op == "rotary":
        tokens, batch = log_int(rng, 1, 30000), rng.choice((1, 1, 2, 7, 32))
        while batch * tokens * (heads + kv) * width > 16384 * 40 * 128:
            tokens, batch = max(1, tokens // 2), max(1, batch // 2)
        pairs = rng.choice((width // 2, width // 2, max(4, width // 4)))
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv, width=width,
                    axes=rng.randint(1, 4), pairs=pairs, adjacent=rng.random() < 0.5, inverse=rng.random() < 0.25)
    c = dict(op=op, dtype=dtype, batch=1, q_tokens=1, k_tokens=1, heads=heads, kv_heads=kv, width=width,
             layout="packed", cap=rng.choice((0.0, 0.0, 30.0, 50.0)), causal=rng.random() < 0.6, prefix=False,
             slopes=rng.random() < 0.3, window=0, docs=0, ragged=rng.random() < 0.5)
    kind = rng.choice(("step", "step", "prompt", "prompt", "images", "windows"))
    if kind == "windows":
        c["window"] = rng.choice((8, 8, 16, 4))
        c.update(docs=-1, causal=False, slopes=False, ragged=False, batch=log_int(rng, 1, 1600) if c["window"] <= 8 else log_int(rng, 1, 120))
        c["q_tokens"] = c["k_tokens"] = c["window"] ** 2
    elif kind == "step":
        c.update(layout="cache", causal=True, batch=rng.choice((1, 2, 5, 16, 32)), q_tokens=rng.choice((1, 1, 1, 3, 4)))
        c["k_tokens"] = log_int(rng, 4, min(131072, 32 * 8192 * 8 * 128 // (c["batch"] * kv * width)))
    else:
        c["q_tokens"] = c["k_tokens"] = n = log_int(rng, 2, 8192)
        if kind == "prompt" and rng.random() < 0.3:
            c.update(layout="cache", q_tokens=max(1, int(n * rng.uniform(0.1, 0.9))))
        if kind == "images":
            c.update(docs=rng.randint(1, 12), causal=rng.random() < 0.2, ragged=False)
        c["prefix"] = c["causal"] and rng.random() < 0.4
        c["batch"] = max(1, min(rng.choice((1, 2, 3, 8)), 16 * 12001 ** 2 // (heads * c["q_tokens"] * n)))
    while c["batch"] * heads * c["q_tokens"] * c["k_tokens"] > 16 * 12001 ** 2:
        c["q_tokens"], c["k_tokens"] = max(1, c["q_tokens"] // 2), c["k_tokens"] // 2
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


def bands(count, side):
    """The masks of a square plane of `count` windows, shifted by half a window: the windows of the
    last row and column hold two bands each way."""
    across = max(1, math.isqrt(count))
    i = torch.arange(count)
    t = torch.arange(side)
    low = (t >= side - side // 2).long()
    y = torch.where(((i // across) == (count - 1) // across)[:, None], 1 + low[None, :], 0)
    x = torch.where(((i % across) == across - 1)[:, None], 1 + low[None, :], 0)
    return (3 * y[:, :, None] + x[:, None, :]).reshape(count, side * side).int()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    order = random.Random(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    st = {"case": case}
    if case["op"] == "rms_norm":
        rows, cols = case["rows"], case["cols"]
        st["x"] = (normal(rows, cols) * torch.exp(normal(rows, 1))).to(t)
        if case["residual"]:
            st["res"] = (3 * normal(rows, cols)).to(t)
            st["sum"] = torch.empty_like(st["res"])
        st["weight"] = 1 + 0.3 * normal(cols)
        groups = -(-cols // case["group"]) if case["group"] else 1
        st["out"] = torch.empty(rows, cols, device=DEV, dtype=torch.float8_e4m3fn if case["out"] == "e4m3" else t)
        st["scales"] = torch.empty(rows, groups, device=DEV) if case["out"] == "e4m3" else None
        return st
    b, d, heads, kv = case["batch"], case["width"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        n, axes = case["tokens"], case["axes"]
        qkv = normal(b, n, heads + 2 * kv, d).to(t)
        st["q"], st["k"] = qkv[:, :, :heads], qkv[:, :, heads:heads + kv]
        st["q_out"], st["k_out"] = torch.empty_like(st["q"]), torch.empty_like(st["k"])
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
            st["plan"] = package().ops.Rotary(st["inv_freq"], st["pair_axis"], adjacent=case["adjacent"],
                                              inverse=case["inverse"])
        else:
            st["axis_of"] = torch.tensor(st["pair_axis"], device=DEV)
            st["freq_of"] = torch.tensor(st["inv_freq"], device=DEV, dtype=torch.float64)
        return st
    nq, nk = case["q_tokens"], case["k_tokens"]
    if case["layout"] == "packed":
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
    if case["prefix"]:
        more["prefix"] = torch.tensor([order.randint(0, max(1, nk // 8)) for _ in range(b)], device=DEV, dtype=torch.int32)
    if case["slopes"]:
        more["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV) / heads)
    if case["window"]:
        w = case["window"]
        i = torch.arange(w * w, device=DEV)
        # the difference of two positions tells (dy, dx) apart
        pos = (i // w * (2 * w - 1) + i % w).int()
        more["q_pos"] = more["k_pos"] = pos
        more["table"] = 16 * torch.sigmoid(normal(heads, 2 * (w - 1) * 2 * w + 1))
    if case["docs"]:
        if case["docs"] > 0:
            ids = torch.full((b, nk), -1, dtype=torch.int32)
            for row in ids:
                at, sizes = 0, parts(case["docs"], nk)
                order.shuffle(sizes)
                for j, n in enumerate(sizes):
                    row[at:at + n] = j
                    at += n
        else:
            ids = bands(b, case["window"])
        more["q_docs"] = more["k_docs"] = ids.to(DEV)
    if own:
        st["plan"] = package().ops.Attention(case["dtype"], b, nq, nk, heads, kv, d, scale=st["scale"], cap=case["cap"],
                                             causal=case["causal"])
        st["workspace"] = torch.empty(st["plan"].workspace_bytes, device=DEV, dtype=torch.uint8)
    return st


def package():
    return importlib.import_module("swin2sr-rs_amd")


# ---- one pass ----------------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if op == "attention":
        return run_attention(st)
    return run_rotary(st) if op == "rotary" else run_rms_norm(st)


def run_attention(st):
    c, q, k, v, more = st["case"], st["q"], st["k"], st["v"], st["more"]
    if own:
        st["plan"](q, k, v, st["out"], workspace=st["workspace"], stream=torch.cuda.current_stream().cuda_stream, **more)
        return st["out"]
    b, nq, heads, d = q.shape
    nk, kv = k.shape[1], k.shape[2]
    i = torch.arange(nq, device=DEV)[None, :, None]
    j = torch.arange(nk, device=DEV)[None, None, :]
    kl = more["k_lens"][:, None, None] if "k_lens" in more else nk
    ql = more["q_lens"][:, None, None] if "q_lens" in more else nq
    at = i + (kl - ql)
    seen = (j < kl) & (i < ql)
    if c["causal"]:
        far = j <= at
        seen = seen & (far | (j < more["prefix"][:, None, None]) if "prefix" in more else far)
    if "q_docs" in more:
        dq, dk = more["q_docs"][:, :, None], more["k_docs"][:, None, :]
        seen = seen & (dq == dk) & (dq >= 0)
    s = q.float().view(b, nq, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d) @ k.float().permute(0, 2, 3, 1)
    s = s.view(b, heads, nq, nk).mul_(st["scale"])
    if c["cap"]:
        s.div_(c["cap"]).tanh_().mul_(c["cap"])
    if "table" in more or "slopes" in more:
        dist = more["q_pos"][None, :, None] - more["k_pos"][None, None, :] if "q_pos" in more else at - j
        if "slopes" in more:
            s.sub_(more["slopes"][None, :, None, None] * dist.abs().float()[:, None])
        if "table" in more:
            half = more["table"].shape[1] // 2
            s.add_(more["table"][:, (dist + half).clamp(0, 2 * half).long()].transpose(0, 1))
    s.masked_fill_(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = s.view(b, kv, -1, nk) @ v.float().transpose(1, 2)
    o = o.view(b, heads, nq, d) / total.clamp(min=1e-30)
    return o.transpose(1, 2).to(q.dtype).contiguous()


def run_rotary(st):
    c, q, k = st["case"], st["q"], st["k"]
    if own:
        st["plan"](q, st["pos"], st["q_out"], k, st["k_out"], stream=torch.cuda.current_stream().cuda_stream)
        return [st["q_out"], st["k_out"]]
    p, d = c["pairs"], c["width"]
    angle = st["pos"][:, :, st["axis_of"]].double() * st["freq_of"]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    if c["inverse"]:
        sin = -sin
    x = torch.cat((q, k), 2).float()
    if c["adjacent"]:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    y = torch.cat((y, x[..., 2 * p:]), -1).to(q.dtype)
    return [y[:, :, :c["heads"]].contiguous(), y[:, :, c["heads"]:].contiguous()]


EPS = 1e-6


def run_rms_norm(st):
    c, x = st["case"], st["x"]
    if own:
        package().ops.rms_norm(x, st["weight"], st["out"], eps=EPS, res=st.get("res"), sum=st.get("sum"),
                               scales=st["scales"], group=c["group"], stream=torch.cuda.current_stream().cuda_stream)
        return [t for t in (st["out"], st["scales"], st.get("sum")) if t is not None]
    h = x.float()
    more = []
    if c["residual"]:
        h = h + st["res"].float()
        more = [h.to(x.dtype)]
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * st["weight"]
    if c["out"] == "same":
        return [y.to(x.dtype)] + more
    rows, cols = y.shape
    group = c["group"] or cols
    y = torch.nn.functional.pad(y, (0, -cols % group)).view(rows, -1, group)
    scale = (y.abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126)
    code = (y / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(rows, -1)[:, :cols].contiguous()
    return [code, scale[:, :, 0]] + more


# ---- what a pass cannot do without -------------------------------------------------------------


def pairs_seen(case):
    """How many (query, key) pairs of one head the masks leave, over the batch; a prefix at its mean."""
    nq, nk, b = case["q_tokens"], case["k_tokens"], case["batch"]
    if case["docs"] > 0:
        one = [n * n for n in parts(case["docs"], nk)]
        return b * sum(one) / (2 if case["causal"] else 1)
    total = 0.0
    for n in lengths(case, random.Random(0)):
        m = min(n, nq)
        total += m * n - (m * (m - 1) / 2 if case["causal"] else 0)
        if case["prefix"]:
            total += min(nk / 16, m) ** 2 / 2
    return total


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rms_norm":
        n = case["rows"] * case["cols"]
        out = 1 if case["out"] == "e4m3" else size
        return {"bytes": n * (size * (3 if case["residual"] else 1) + out) + 4 * case["cols"], "flops": 6 * n}
    b, d, heads, kv = case["batch"], case["width"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        n = b * case["tokens"]
        return {"bytes": n * ((heads + kv) * d * 2 * size + 4 * case["axes"]), "flops": n * (heads + kv) * case["pairs"] * 6}
    keys = sum(lengths(case, random.Random(0)))
    queries = sum(min(n, case["q_tokens"]) for n in lengths(case, random.Random(0)))
    return {"bytes": size * d * (2 * queries * heads + 2 * keys * kv), "flops": 4 * d * heads * pairs_seen(case)}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": exact_attention, "rotary": exact_rotary, "rms_norm": exact_rms_norm}[case["op"]](st)


def exact_attention(st):
    """Sequence by sequence, over the keys that the sequence has."""
    c, more = st["case"], st["more"]
    out = torch.zeros(st["out"].shape, device=DEV, dtype=torch.float64)
    group = c["heads"] // c["kv_heads"]
    for b in range(c["batch"]):
        n = int(more["k_lens"][b]) if "k_lens" in more else c["k_tokens"]
        m = int(more["q_lens"][b]) if "q_lens" in more else c["q_tokens"]
        rows = torch.arange(m, device=DEV, dtype=torch.float64)[:, None] + (n - m)
        cols = torch.arange(n, device=DEV, dtype=torch.float64)[None, :]
        hidden = torch.zeros(m, n, device=DEV, dtype=torch.bool)
        if c["causal"]:
            hidden = cols > rows
            if "prefix" in more:
                hidden &= cols >= float(more["prefix"][b])
        if "q_docs" in more:
            mine, theirs = more["q_docs"][b, :m, None], more["k_docs"][b, None, :n]
            hidden = hidden | (mine != theirs) | (mine < 0)
        if "q_pos" in more:
            dist = (more["q_pos"][:m, None] - more["k_pos"][None, :n]).double()
        else:
            dist = rows - cols
        for h in range(c["heads"]):
            score = st["q"][b, :m, h].double() @ st["k"][b, :n, h // group].double().T * st["scale"]
            if c["cap"]:
                score = torch.tanh(score / c["cap"]) * c["cap"]
            if "slopes" in more:
                score = score - more["slopes"][h].double() * dist.abs()
            if "table" in more:
                reach = (c["window"] - 1) * 2 * c["window"]
                score = score + more["table"][h].double()[dist.clamp(-reach, reach).long() + reach]
            score = torch.where(hidden, -math.inf, score)
            weight = torch.nan_to_num(torch.softmax(score, 1), nan=0.0)
            out[b, :m, h] = weight @ st["v"][b, :n, h // group].double()
    return out


def exact_rotary(st):
    """Each pair as a complex number times e^(i angle)."""
    c = st["case"]
    p = c["pairs"]
    angle = torch.stack([st["pos"][:, :, a].double() * f for a, f in zip(st["pair_axis"], st["inv_freq"])], -1)
    turn = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)[:, :, None, :]
    got = []
    for x in (st["q"], st["k"]):
        y = x.double().clone()
        first, second = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if c["adjacent"] else (slice(0, p), slice(p, 2 * p))
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        got.append(y)
    return got


def exact_rms_norm(st):
    """The codes as the values that e4m3 has: to three bits behind the leading one, ties to even."""
    c = st["case"]
    h = st["x"].double() + (st["res"].double() if c["residual"] else 0)
    y = h / (h.pow(2).sum(1, keepdim=True) / c["cols"] + EPS).sqrt() * st["weight"].double()
    tail = [h] if c["residual"] else []
    if c["out"] == "same":
        return [y] + tail
    group = c["group"] or c["cols"]
    codes, scales = torch.empty_like(y), []
    for at in range(0, c["cols"], group):
        part = y[:, at:at + group]
        scale = (part.abs().max(1, keepdim=True).values / 448).clamp(min=2.0 ** -126)
        r = part / scale
        step = 2.0 ** (torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6))) - 3)
        codes[:, at:at + group] = (torch.round(r / step) * step).clamp(-448, 448)
        scales.append(scale)
    return [codes, torch.cat(scales, 1)] + tail
