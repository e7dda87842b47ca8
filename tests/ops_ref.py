"""Plain 64-bit implementations of the transformer operators, their error bounds,
and device arrays of any type and layout for their tests (numpy only)."""
import numpy as np

# half a step relative to the value (a rounding's largest error)
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# the smallest step (below the normal range errors are absolute)
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def to_bits(x, dtype):
    """f64/f32 values as the type's bits, rounded to nearest even."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x.view(np.uint32)
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype):
    if dtype == "f32":
        return b.view(np.float32).astype(np.float64)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def round_to(x, dtype):
    return from_bits(to_bits(x, dtype), dtype)


def e4m3_values():
    """The 256 codes' values (OCP e4m3fn)."""
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = np.nan if (c & 127) == 127 else (-x if c & 128 else x)
    return v


class Dev:
    """`values` (any shape, f64) as a device array of `dtype`, laid out with
    `order` (the dimensions from the outermost to the innermost in memory), `gap`
    elements between neighbours of the second innermost dimension, and `lead`
    elements ahead of the first. What lies between is `fill`."""

    def __init__(self, pkg, values, dtype, order=None, gap=0, lead=0, fill=0.0, whole=False):
        values = np.asarray(values)
        self.dtype, self.shape = dtype, values.shape
        order = list(order or range(values.ndim))
        strides, n = [0] * values.ndim, 1
        for k, d in enumerate(reversed(order)):
            strides[d] = n
            n *= max(values.shape[d], 1)
            if k == 0:
                n += gap
        self.strides, self.lead, self.n = tuple(strides), lead, n + lead
        if whole:
            bits = values.astype(np.int32).view(np.uint32)
            flat = np.zeros(self.n, np.uint32)
        elif dtype == "e4m3":
            bits = values.astype(np.uint8)
            flat = np.full(self.n, 0x55, np.uint8)
        else:
            bits = to_bits(values, dtype)
            flat = np.full(self.n, to_bits(np.float32(fill), dtype))
        self.kind = "i32" if whole else dtype
        self.np_type = flat.dtype
        flat = np.ascontiguousarray(flat)
        view = self.view(flat)
        view[...] = bits
        raw = flat.tobytes()
        raw += b"\0" * (-len(raw) % 4)
        self.buf = pkg.hip.DeviceBuffer.from_array(np.frombuffer(raw, np.float32))
        self.before = flat
        self.array = pkg.ops.Array(self.buf.ptr + lead * flat.dtype.itemsize, self.shape, self.kind, self.strides)

    def view(self, flat):
        size = flat.dtype.itemsize
        return np.lib.stride_tricks.as_strided(flat[self.lead:], self.shape, [s * size for s in self.strides])

    def bits(self):
        raw = self.buf.download().tobytes()[:self.n * np.dtype(self.np_type).itemsize]
        return np.frombuffer(raw, self.np_type).copy()

    def get(self):
        b = self.view(self.bits())
        if self.kind == "i32":
            return np.ascontiguousarray(b).view(np.int32)
        if self.kind == "e4m3":
            return np.ascontiguousarray(b)
        return from_bits(np.ascontiguousarray(b), self.dtype)

    def gaps_kept(self):
        """Whether what lies between the array's elements is as it was."""
        now, was = self.bits(), self.before.copy()
        self.view(now)[...] = 0
        self.view(was)[...] = 0
        return np.array_equal(now, was)


def attention(dtype, q, k, v, scale, cap=0.0, causal=False, q_lens=None, k_lens=None, prefix=None, q_docs=None,
              k_docs=None, q_pos=None, k_pos=None, slopes=None, table=None, window=0, sinks=0,
              least=0.0):
    """(out, bound, written): the result in 64 bits for inputs that are values of
    `dtype`, the error a 32-bit evaluation may have, and which rows are written.

    The bound, with u = 2^-24 and P the weights (sum 1), first order: a score is a
    sum of D products (D u of their magnitudes), then scaled, capped, biased and
    turned into an exponent with the row's maximum taken off (4 u of each of their
    magnitudes; cap tanh by a formula good to 8 u of the cap), so with delta the
    largest such error of the row's scores every P is off by 2 delta relative,
    and by 4 u for exp and the sums' own roundings sqrt-free n u. A weight is
    rounded to the type before it multiplies v (HALF), the f16 one also by half
    its smallest step, 2^-25 at weights that have 2^0 or more for the row's
    largest. The result is rounded once (HALF of it, or half the smallest step).
    `least`: keys of smaller weights, for the row's largest, are left out.
    """
    B, Lq, H, D = q.shape
    Lk, G = k.shape[1], H // k.shape[2]
    u = 2.0 ** -24
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    written = np.zeros((B, Lq), bool)
    at2 = lambda x, b: x[b] if x.ndim == 2 else x  # noqa: E731
    for b in range(B):
        n = Lk if k_lens is None else min(max(int(k_lens[b]), 0), Lk)
        m = Lq if q_lens is None else min(max(int(q_lens[b]), 0), Lq)
        written[b, :m] = True
        i, j = np.arange(m)[:, None], np.arange(n)[None, :]
        ok = np.ones((m, n), bool)
        if causal:
            ok = j <= n - m + i
            if prefix is not None:
                ok |= j < int(prefix[b])
        if window:
            place = n - m + i
            ok = ok & ((j > place - window) | (j < sinks))
            if not causal:
                ok = ok & (j < place + window)
        if q_docs is not None:
            dq, dk = at2(q_docs, b)[:m, None], at2(k_docs, b)[None, :n]
            ok = ok & (dq == dk) & (dq >= 0)
        dist = (at2(q_pos, b)[:m, None].astype(np.int64) - at2(k_pos, b)[None, :n]) if q_pos is not None else n - m + i - j
        for h in range(H):
            kk, vv = k[b, :n, h // G], v[b, :n, h // G]
            use = ok.copy()
            with np.errstate(invalid="ignore", over="ignore"):
                kz = np.where(use.any(0)[:, None], kk, 0.0)
                s = np.where(use, q[b, :m, h] @ kz.T if m and n else 0.0, 0.0)
                # rows whose own keys are finite must not see others' NaN
                for r, c in np.argwhere(use & ~np.isfinite(s)):
                    s[r, c] = q[b, r, h] @ kk[c]
                if not np.isfinite(kz).all() or not np.isfinite(q[b, :m, h]).all():
                    for r in range(m):
                        for c in range(n):
                            if use[r, c]:
                                s[r, c] = q[b, r, h] @ kk[c]
                s = s * scale
                err = np.where(use, np.abs(np.nan_to_num(q[b, :m, h])) @ np.abs(np.nan_to_num(kz)).T if m and n else 0.0, 0)
                err = (D + 4) * u * abs(scale) * err
                if cap:
                    s = cap * np.tanh(s / cap)
                    err = err + 8 * u * cap
                mag = np.abs(s)
                if slopes is not None:
                    s = s - slopes[h] * np.abs(dist)
                    mag = mag + np.abs(slopes[h] * dist)
                if table is not None:
                    T = table.shape[1]
                    bias = table[h][np.clip(dist, -(T // 2), T // 2) + T // 2]
                    use = use & ~np.isneginf(bias)
                    bias = np.where(np.isneginf(bias), 0, bias)
                    s = s + bias
                    mag = mag + np.abs(bias)
                err = np.where(use, err + 8 * u * mag, 0)
                s = np.where(use, s, -np.inf)
                top = s.max(1, initial=-np.inf, keepdims=True)
                p = np.where(use, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                p = np.where(np.isnan(s) & use, np.nan, p)
                total = p.sum(1, keepdims=True)
                w = p / np.where(total == 0, 1, total)
                va = np.abs(vv)
                for r in range(m):
                    live = use[r] & ~(p[r] < least)
                    if not live.any():
                        continue
                    out[b, r, h] = w[r, live] @ vv[live]
                    # keys whose weight is nothing do not widen the bound
                    heavy = live & (w[r] > 1e-12)
                    delta = err[r, heavy].max(initial=0.0)
                    e = 2 * delta + (4 + live.sum()) * u
                    if dtype != "f32":
                        e = e + HALF[dtype]
                    bound[b, r, h] = e * (w[r, live] @ va[live])
                    if dtype == "f16":
                        bound[b, r, h] += 2.0 ** -25 * va[live].sum(0) / max(total[r, 0], 1.0)
                    bound[b, r, h] += np.maximum(HALF[dtype] * np.abs(out[b, r, h]), TINY[dtype] / 2)
    return out, bound, written


def rotary(x, angle, pairs, adjacent, inverse):
    """x [B][L][H][D] turned by angle [B][L][pairs]."""
    y = np.array(x)
    c, s = np.cos(angle)[:, :, None], np.sin(angle)[:, :, None] * (-1 if inverse else 1)
    i, j = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def norm_rotary(dtype, x, weight, offset, eps, angle, pairs, adjacent, inverse):
    """(out, bound): heads x [B][L][H][D] (values of `dtype`) normed, times weight [D] or [H][D] plus
    offset, and turned by angle [B][L][pairs], in 64 bits, and what a 32-bit evaluation may be off.

    The bound, with u = 2^-24: the squares' sum is a chain of at most max(16, D / 64) additions in
    a lane and 6 across lanes, halved by the root; the mean and eps (2 u, halved), root, reciprocal
    and three roundings of the product with the weight (whose own sum is one): max(16, D / 64) / 2
    + 9 u of the normed channel. Sin and cos are off by 3 u, two products and a sum: 6 u of the pair's
    magnitudes. The result is rounded once."""
    u, D = 2.0 ** -24, x.shape[-1]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (np.asarray(weight, np.float64) + offset)
        out = rotary(y, angle, pairs, adjacent, inverse)
        mag = np.abs(y)
        i, j = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
        both = mag[..., i] + mag[..., j]
        mag[..., i], mag[..., j] = both, both
        return out, (max(16, D / 64) / 2 + 15) * u * mag + np.maximum(HALF[dtype] * np.abs(out), TINY[dtype] / 2)
