"""The transformer operators of include/swin2sr_hip.h on arrays in HBM: attention
(capped scores, distance biases, document, causal and prefix masks, padded
batches, grouped heads), rotary positions with several axes, and the
root-mean-square norm with the residual's addition and an 8-bit output.

Arrays are anything with `data_ptr()`, `shape`, `stride()` and `dtype` as torch
tensors have them (torch itself is not imported here; a process that uses it
imports it before this library is loaded, so that both share one HIP runtime),
or an `Array` over a device address. Calls enqueue on `stream` (a hipStream_t as
an int; 0 is the current device's default stream) and do not wait; the arrays
have to live until the work is done. Errors surface as `S2SError` with the
library's message; shapes and types that do not fit raise it too.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

from .abi import Attention_, RmsNorm_, Rotary_, S2SError, Tokens_, check, load_library

F32, F16, BF16, E4M3 = 0, 1, 2, 3
_NAMES = {"f32": F32, "float32": F32, "f16": F16, "float16": F16, "bf16": BF16, "bfloat16": BF16,
          "e4m3": E4M3, "float8_e4m3fn": E4M3}
_codes = {}


class Array:
    """`shape` elements of `dtype` ("f32", "f16", "bf16", "e4m3", "i32", "u8") at a
    device address; `strides` in elements, contiguous by default."""

    def __init__(self, ptr: int, shape: Sequence[int], dtype: str, strides: Optional[Sequence[int]] = None):
        self.ptr, self.shape, self.dtype = int(ptr), tuple(int(n) for n in shape), dtype
        if strides is None:
            strides, n = [], 1
            for d in reversed(self.shape):
                strides.insert(0, n)
                n *= d
        self._strides = tuple(int(n) for n in strides)
        if len(self._strides) != len(self.shape):
            raise S2SError(f"Array: {len(self.shape)} dimensions, {len(self._strides)} strides")

    def data_ptr(self) -> int:
        return self.ptr

    def stride(self):
        return self._strides


def _type(dtype) -> int:
    """The s2s_dtype of a type's name, or of a torch type; -1 for another."""
    try:
        return _codes[dtype]
    except KeyError:
        code = _codes[dtype] = _NAMES.get(str(dtype).replace("torch.", ""), -1)
        return code


def _is_int32(dtype) -> bool:
    return str(dtype) in ("torch.int32", "int32", "i32")


def _is_f32(dtype) -> bool:
    return _type(dtype) == F32


def _need(ok, what: str):
    if not ok:
        raise S2SError(what)


def _contiguous(a) -> bool:
    n = 1
    for d, s in zip(reversed(tuple(a.shape)), reversed(tuple(a.stride()))):
        if d != 1 and s != n:
            return False
        n *= d
    return True


def _tokens(where: Tokens_, a, shape, dtype: int, op: str, name: str):
    """An array [batch][tokens][heads][width] into its C struct."""
    if tuple(a.shape) != shape or _type(a.dtype) != dtype:
        raise S2SError(f"{op}: {name} is {tuple(a.shape)} of {a.dtype}, wanted {shape} of the call's type")
    s = a.stride()
    if s[3] != 1 and shape[3] > 1:
        raise S2SError(f"{op}: the channels of {name} are not adjacent")
    where.data, where.batch, where.token, where.head = a.data_ptr(), s[0], s[1], s[2]


def _vector(a, n: int, op: str, name: str):
    """A contiguous int32 vector of n."""
    if a is None:
        return None
    _need(tuple(a.shape) == (n,) and _is_int32(a.dtype) and _contiguous(a), f"{op}: {name} is no int32 vector of {n}")
    return a.data_ptr()


def _per_token(a, batch: int, tokens: int, op: str, name: str):
    """int32 [batch][tokens], or [tokens] shared by the batch: address and batch stride."""
    if a is None:
        return None, 0
    shape, s = tuple(a.shape), tuple(a.stride())
    _need(_is_int32(a.dtype) and shape in ((tokens,), (batch, tokens)) and (s[-1] == 1 or tokens <= 1),
          f"{op}: {name} is not int32 [{batch}][{tokens}] or [{tokens}] with adjacent tokens")
    return a.data_ptr(), (s[0] if len(shape) == 2 else 0)


class Attention:
    """A plan of `s2s_attention` for one set of sizes.

    `dtype` ("f32", "f16", "bf16") is the type of q, k, v and out; `scale` is
    1 / sqrt(width) by default, `cap` 0 for none. `workspace_bytes` of device
    memory go with every call: one buffer serves all calls of a stream, calls
    that may overlap on the device (other streams, replays of captured graphs)
    need one each.

        plan = ops.Attention("bf16", batch, q_tokens, k_tokens, q_heads, k_heads, width, causal=True)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
        plan(q, k, v, out, workspace=ws, stream=stream, k_lens=lens, cap=...)
    """

    def __init__(self, dtype, batch: int, q_tokens: int, k_tokens: int, q_heads: int, k_heads: int, width: int,
                 scale: Optional[float] = None, cap: float = 0.0, causal: bool = False):
        sizes = (batch, q_tokens, k_tokens, q_heads, k_heads, width)
        _need(all(-2 ** 31 <= n < 2 ** 31 for n in sizes), "attention: a size that is no 32-bit int")
        self.lib = load_library()
        a = self.args = Attention_()
        a.dtype = self.dtype = _type(dtype)
        a.batch, a.q_tokens, a.k_tokens = batch, q_tokens, k_tokens
        a.q_heads, a.k_heads, a.width = q_heads, k_heads, width
        a.scale = float(scale) if scale is not None else max(width, 1) ** -0.5
        a.cap, a.causal = float(cap), int(bool(causal))
        self.q_shape, self.k_shape = (batch, q_tokens, q_heads, width), (batch, k_tokens, k_heads, width)
        n = C.c_uint64()
        check(self.lib.s2s_attention_workspace(C.byref(a), C.byref(n)), "attention")
        self.workspace_bytes = n.value

    def __call__(self, q, k, v, out, workspace=None, stream: int = 0, q_lens=None, k_lens=None, prefix=None,
                 q_docs=None, k_docs=None, q_pos=None, k_pos=None, slopes=None, table=None):
        """out [batch][q_tokens][q_heads][width] from q (the same shape), k and v
        [batch][k_tokens][k_heads][width]; lengths and prefix int32 [batch];
        documents and positions int32 [batch][tokens] or [tokens]; slopes f32
        [q_heads]; table f32 [q_heads][odd]."""
        a = Attention_.from_buffer_copy(self.args)
        op = "attention"
        _tokens(a.q, q, self.q_shape, self.dtype, op, "q")
        _tokens(a.k, k, self.k_shape, self.dtype, op, "k")
        _tokens(a.v, v, self.k_shape, self.dtype, op, "v")
        _tokens(a.out, out, self.q_shape, self.dtype, op, "out")
        if q_lens is not None:
            a.q_lens = _vector(q_lens, a.batch, op, "q_lens")
        if k_lens is not None:
            a.k_lens = _vector(k_lens, a.batch, op, "k_lens")
        if prefix is not None:
            a.prefix = _vector(prefix, a.batch, op, "prefix")
        if q_docs is not None or k_docs is not None:
            a.q_docs, a.q_docs_batch = _per_token(q_docs, a.batch, a.q_tokens, op, "q_docs")
            a.k_docs, a.k_docs_batch = _per_token(k_docs, a.batch, a.k_tokens, op, "k_docs")
        if q_pos is not None or k_pos is not None:
            a.q_pos, a.q_pos_batch = _per_token(q_pos, a.batch, a.q_tokens, op, "q_pos")
            a.k_pos, a.k_pos_batch = _per_token(k_pos, a.batch, a.k_tokens, op, "k_pos")
        if slopes is not None:
            _need(tuple(slopes.shape) == (a.q_heads,) and _is_f32(slopes.dtype) and _contiguous(slopes),
                  f"{op}: slopes is no f32 vector of {a.q_heads}")
            a.slopes = slopes.data_ptr()
        if table is not None:
            _need(len(table.shape) == 2 and table.shape[0] == a.q_heads and _is_f32(table.dtype) and _contiguous(table),
                  f"{op}: table is no contiguous f32 [{a.q_heads}][entries]")
            a.table, a.table_size = table.data_ptr(), table.shape[1]
        ws, n = (None, 0) if workspace is None else (workspace.data_ptr(), _bytes(workspace))
        check(self.lib.s2s_attention(C.byref(a), ws, n, stream), op)
        return out


def _bytes(a) -> int:
    n = 1
    for d in a.shape:
        n *= d
    _need(_contiguous(a), "workspace: not contiguous")
    size = {"u8": 1, "uint8": 1, "i32": 4, "int32": 4, "f32": 4, "float32": 4}.get(str(a.dtype).replace("torch.", ""))
    _need(size is not None, f"workspace: of {a.dtype}, wanted u8, i32 or f32")
    return n * size


class Rotary:
    """Rotary positions: pair p of every head is turned by
    pos[b][token][pair_axis[p]] * inv_freq[p].

    `Rotary.of(sections, theta)` makes the common frequencies: sections[a] pairs
    for axis a, one behind the other, pair i of a section at theta ** (-i /
    sections[a]). `adjacent` pairs channels (2p, 2p + 1) instead of (p, p +
    pairs); `inverse` turns back."""

    def __init__(self, inv_freq: Sequence[float], pair_axis: Sequence[int], adjacent: bool = False,
                 inverse: bool = False):
        _need(len(inv_freq) == len(pair_axis) and len(inv_freq) >= 1, "rotary: a frequency and an axis for each pair")
        _need(all(0 <= int(x) <= 255 for x in pair_axis), "rotary: an axis that is none")
        self.lib = load_library()
        self.inv_freq = (C.c_double * len(inv_freq))(*[float(f) for f in inv_freq])
        self.pair_axis = (C.c_uint8 * len(pair_axis))(*[int(x) for x in pair_axis])
        a = self.args = Rotary_()
        a.pairs, a.adjacent, a.inverse = len(inv_freq), int(bool(adjacent)), int(bool(inverse))
        a.inv_freq = C.cast(self.inv_freq, C.POINTER(C.c_double))
        a.pair_axis = C.cast(self.pair_axis, C.POINTER(C.c_uint8))

    @classmethod
    def of(cls, sections: Sequence[int], theta: float = 10000.0, adjacent: bool = False, inverse: bool = False):
        return cls([theta ** (-i / n) for n in sections for i in range(n)],
                   [a for a, n in enumerate(sections) for _ in range(n)], adjacent=adjacent, inverse=inverse)

    def __call__(self, q, pos, q_out=None, k=None, k_out=None, lens=None, stream: int = 0):
        """q (and k) [batch][tokens][heads][width] into q_out (and k_out), in place
        without them; pos int32 [batch][tokens][axes] or [tokens][axes]; tokens
        from lens[b] on are not written."""
        op = "rotary"
        a = Rotary_.from_buffer_copy(self.args)
        shape = tuple(q.shape)
        _need(len(shape) == 4 and max(shape) < 2 ** 31, f"{op}: q is {shape}, wanted [batch][tokens][heads][width]")
        a.dtype = dt = _type(q.dtype)
        a.batch, a.tokens, a.q_heads, a.width = shape
        _tokens(a.q, q, shape, dt, op, "q")
        _tokens(a.q_out, q if q_out is None else q_out, shape, dt, op, "q_out")
        if k is not None:
            ks = tuple(k.shape)
            _need(len(ks) == 4 and ks[2] >= 1, f"{op}: k is {ks}, wanted [batch][tokens][heads][width]")
            ks = (shape[0], shape[1], ks[2], shape[3])
            a.k_heads = ks[2]
            _tokens(a.k, k, ks, dt, op, "k")
            _tokens(a.k_out, k if k_out is None else k_out, ks, dt, op, "k_out")
        else:
            _need(k_out is None, f"{op}: k_out without k")
        ps, pstr = tuple(pos.shape), tuple(pos.stride())
        a.axes = ps[-1] if ps else 0
        _need(_is_int32(pos.dtype) and ps in (shape[1:2] + ps[-1:], shape[:2] + ps[-1:]),
              f"{op}: pos is {ps} of {pos.dtype}, wanted int32 [batch][tokens][axes] or [tokens][axes]")
        _need((pstr[-1] == 1 or ps[-1] == 1) and (pstr[-2] == ps[-1] or ps[-2] <= 1),
              f"{op}: the tokens and axes of pos are not adjacent")
        a.pos, a.pos_batch = pos.data_ptr(), (pstr[0] if len(ps) == 3 else 0)
        if lens is not None:
            a.lens = _vector(lens, a.batch, op, "lens")
        check(self.lib.s2s_rotary(C.byref(a), stream), op)
        return (q if q_out is None else q_out) if k is None else (q if q_out is None else q_out, k if k_out is None else k_out)


def _rows(a, rows: int, cols: int, dtype: int, op: str, name: str):
    s = a.stride()
    if tuple(a.shape) != (rows, cols) or _type(a.dtype) != dtype or (s[1] != 1 and cols > 1):
        raise S2SError(f"{op}: {name} is {tuple(a.shape)} of {a.dtype}, wanted [{rows}][{cols}] with adjacent columns "
                       "and the call's type")
    return a.data_ptr(), s[0]


def rms_norm(x, weight, out, eps: float = 1e-6, res=None, sum=None, scales=None, group: int = 0,
             weight_offset: float = 0.0, stream: int = 0):
    """out = h / sqrt(mean(h^2) + eps) * (weight + weight_offset) of the rows of h =
    x + res, with h in `sum`. x, res, sum [rows][cols] of one type, out of that type
    or e4m3 (then with `scales` f32 [rows][ceil(cols / group)], group 0 being the
    row); weight f32 [cols]."""
    op = "rms_norm"
    a = RmsNorm_()
    _need(len(x.shape) == 2, f"{op}: x is {tuple(x.shape)}, wanted [rows][cols]")
    rows, cols = x.shape
    _need(cols < 2 ** 31 and abs(group) < 2 ** 31, f"{op}: columns or a group that are no 32-bit int")
    a.rows, a.cols, a.eps, a.weight_offset, a.group = rows, cols, eps, weight_offset, group
    a.dtype = dt = _type(x.dtype)
    a.out_dtype = E4M3 if _type(out.dtype) == E4M3 else dt
    a.x, a.x_stride = _rows(x, rows, cols, dt, op, "x")
    if res is not None:
        a.res, a.res_stride = _rows(res, rows, cols, dt, op, "res")
    if sum is not None:
        a.sum, a.sum_stride = _rows(sum, rows, cols, dt, op, "sum")
    a.out, a.out_stride = _rows(out, rows, cols, a.out_dtype, op, "out")
    _need(tuple(weight.shape) == (cols,) and _is_f32(weight.dtype) and _contiguous(weight),
          f"{op}: weight is no f32 vector of {cols}")
    a.weight = weight.data_ptr()
    if scales is not None:
        _need(group >= 0, f"{op}: a negative group")
        n = -(-cols // group) if group else 1
        _need(tuple(scales.shape) == (rows, n) and _is_f32(scales.dtype) and _contiguous(scales),
              f"{op}: scales is no contiguous f32 [{rows}][{n}]")
        a.scales = scales.data_ptr()
    check(load_library().s2s_rms_norm(C.byref(a), stream), op)
    return out
