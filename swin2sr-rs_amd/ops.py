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
import struct
from typing import Optional, Sequence

from .abi import Attention_, S2SError, check, last_error, load_library

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


_int32 = {}


def _is_int32(dtype) -> bool:
    try:
        return _int32[dtype]
    except KeyError:
        _int32[dtype] = str(dtype) in ("torch.int32", "int32", "i32")
        return _int32[dtype]


def _is_f32(dtype) -> bool:
    return _type(dtype) == F32


def _need(ok, what: str):
    if not ok:
        raise S2SError(what)


def _f32(x) -> float:
    """As a C float takes it: an infinity (which the library refuses) past its range."""
    return C.c_float(x).value


def _contiguous(a) -> bool:
    n = 1
    for d, s in zip(reversed(tuple(a.shape)), reversed(tuple(a.stride()))):
        if d != 1 and s != n:
            return False
        n *= d
    return True


def _tokens(a, shape, dtype: int, op: str, name: str):
    """An array [batch][tokens][heads][width] as its C struct's fields."""
    if a.shape != shape or _type(a.dtype) != dtype:
        raise S2SError(f"{op}: {name} is {tuple(a.shape)} of {a.dtype}, wanted {shape} of the call's type")
    b, t, h, d = a.stride()
    if d != 1 and shape[3] > 1:
        raise S2SError(f"{op}: the channels of {name} are not adjacent")
    return a.data_ptr(), b, t, h


# The argument structs as one pack each (a call's fields set one by one through
# ctypes take as long as the call): the C structs' layout, null pointers as 0.
_ATTENTION = struct.Struct("@8i2f 4q4q4q4q 3P 2P2q 2P2q 2Pi0q")
_ROTARY = struct.Struct("@10i 4q4q4q4q Pq3P")
_RMS = struct.Struct("@2iqi4P4qP2fPi0q")


def _vector(a, n: int, op: str, name: str):
    """A contiguous int32 vector of n: its address, 0 for none."""
    if a is None:
        return 0
    _need(tuple(a.shape) == (n,) and _is_int32(a.dtype) and _contiguous(a), f"{op}: {name} is no int32 vector of {n}")
    return a.data_ptr()


def _per_token(a, batch: int, tokens: int, op: str, name: str):
    """int32 [batch][tokens], or [tokens] shared by the batch: address and batch stride."""
    if a is None:
        return 0, 0
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
        self.dtype = _type(dtype)
        self.head = (self.dtype, batch, q_tokens, k_tokens, q_heads, k_heads, width, int(bool(causal)),
                     _f32(scale) if scale is not None else max(width, 1) ** -0.5, _f32(cap))
        self.batch, self.q_tokens, self.k_tokens, self.q_heads = batch, q_tokens, k_tokens, q_heads
        self.q_shape, self.k_shape = (batch, q_tokens, q_heads, width), (batch, k_tokens, k_heads, width)
        a = Attention_(*self.head)
        n = C.c_uint64()
        check(self.lib.s2s_attention_workspace(C.byref(a), C.byref(n)), "attention")
        self.workspace_bytes = n.value

    def __call__(self, q, k, v, out, workspace=None, stream: int = 0, q_lens=None, k_lens=None, prefix=None,
                 q_docs=None, k_docs=None, q_pos=None, k_pos=None, slopes=None, table=None):
        """out [batch][q_tokens][q_heads][width] from q (the same shape), k and v
        [batch][k_tokens][k_heads][width]; lengths and prefix int32 [batch];
        documents and positions int32 [batch][tokens] or [tokens]; slopes f32
        [q_heads]; table f32 [q_heads][odd]."""
        op, dt, batch, nq, nk = "attention", self.dtype, self.batch, self.q_tokens, self.k_tokens
        arrays = (*_tokens(q, self.q_shape, dt, op, "q"), *_tokens(k, self.k_shape, dt, op, "k"),
                  *_tokens(v, self.k_shape, dt, op, "v"), *_tokens(out, self.q_shape, dt, op, "out"))
        lens = (_vector(q_lens, batch, op, "q_lens"), _vector(k_lens, batch, op, "k_lens"), _vector(prefix, batch, op, "prefix"))
        docs = pos = (0, 0, 0, 0)
        if q_docs is not None or k_docs is not None:
            (a, sa), (b, sb) = _per_token(q_docs, batch, nq, op, "q_docs"), _per_token(k_docs, batch, nk, op, "k_docs")
            docs = (a, b, sa, sb)
        if q_pos is not None or k_pos is not None:
            (a, sa), (b, sb) = _per_token(q_pos, batch, nq, op, "q_pos"), _per_token(k_pos, batch, nk, op, "k_pos")
            pos = (a, b, sa, sb)
        slope_ptr = table_ptr = entries = 0
        if slopes is not None:
            _need(slopes.shape == (self.q_heads,) and _is_f32(slopes.dtype) and _contiguous(slopes),
                  f"{op}: slopes is no f32 vector of {self.q_heads}")
            slope_ptr = slopes.data_ptr()
        if table is not None:
            _need(len(table.shape) == 2 and table.shape[0] == self.q_heads and _is_f32(table.dtype) and _contiguous(table),
                  f"{op}: table is no contiguous f32 [{self.q_heads}][entries]")
            table_ptr, entries = table.data_ptr(), table.shape[1]
            _need(entries < 2 ** 31, f"{op}: a table of {entries} entries")
        args = _ATTENTION.pack(*self.head, *arrays, *lens, *docs, *pos, slope_ptr, table_ptr, entries)
        ws, n = (None, 0) if workspace is None else (workspace.data_ptr(), _bytes(workspace))
        if self.lib.s2s_attention(args, ws, n, stream):
            raise S2SError(f"{op}: {last_error()}")
        return out


_SIZES = {}


def _bytes(a) -> int:
    n = 1
    for d in a.shape:
        n *= d
    size = _SIZES.get(a.dtype)
    if size is None:
        size = {"u8": 1, "uint8": 1, "i32": 4, "int32": 4, "f32": 4, "float32": 4}.get(str(a.dtype).replace("torch.", ""))
        _need(size is not None, f"workspace: of {a.dtype}, wanted u8, i32 or f32")
        _SIZES[a.dtype] = size
    _need(len(a.shape) == 1 and a.stride()[0] == 1 or _contiguous(a), "workspace: not contiguous")
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
        self.flags = (len(inv_freq), int(bool(adjacent)), int(bool(inverse)))
        self.host = (C.addressof(self.inv_freq), C.addressof(self.pair_axis))

    @classmethod
    def of(cls, sections: Sequence[int], theta: float = 10000.0, adjacent: bool = False, inverse: bool = False):
        return cls([theta ** (-i / n) for n in sections for i in range(n)],
                   [a for a, n in enumerate(sections) for _ in range(n)], adjacent=adjacent, inverse=inverse)

    def __call__(self, q, pos, q_out=None, k=None, k_out=None, lens=None, stream: int = 0):
        """q (and k) [batch][tokens][heads][width] into q_out (and k_out), in place
        without them; pos int32 [batch][tokens][axes] or [tokens][axes]; tokens
        from lens[b] on are not written."""
        op = "rotary"
        shape = q.shape
        _need(len(shape) == 4 and max(shape) < 2 ** 31, f"{op}: q is {tuple(shape)}, wanted [batch][tokens][heads][width]")
        dt = _type(q.dtype)
        if q_out is None:
            q_out = q
        arrays = _tokens(q, shape, dt, op, "q"), _tokens(q_out, shape, dt, op, "q_out")
        k_arrays, k_heads = ((0, 0, 0, 0), (0, 0, 0, 0)), 0
        if k is not None:
            ks = k.shape
            _need(len(ks) == 4 and 1 <= ks[2] < 2 ** 31, f"{op}: k is {tuple(ks)}, wanted [batch][tokens][heads][width]")
            k_heads = ks[2]
            ks = (shape[0], shape[1], k_heads, shape[3])
            if k_out is None:
                k_out = k
            k_arrays = _tokens(k, ks, dt, op, "k"), _tokens(k_out, ks, dt, op, "k_out")
        else:
            _need(k_out is None, f"{op}: k_out without k")
        ps, pstr = tuple(pos.shape), pos.stride()
        _need(_is_int32(pos.dtype) and ps in ((shape[1],) + ps[-1:], (shape[0], shape[1]) + ps[-1:]),
              f"{op}: pos is {ps} of {pos.dtype}, wanted int32 [batch][tokens][axes] or [tokens][axes]")
        _need((pstr[-1] == 1 or ps[-1] == 1) and (pstr[-2] == ps[-1] or ps[-2] <= 1),
              f"{op}: the tokens and axes of pos are not adjacent")
        args = _ROTARY.pack(dt, shape[0], shape[1], shape[2], k_heads, shape[3], min(ps[-1], 2 ** 31 - 1), *self.flags, *arrays[0],
                            *k_arrays[0], *arrays[1], *k_arrays[1], pos.data_ptr(), pstr[0] if len(ps) == 3 else 0,
                            _vector(lens, shape[0], op, "lens"), *self.host)
        if self.lib.s2s_rotary(args, stream):
            raise S2SError(f"{op}: {last_error()}")
        return q_out if k is None else (q_out, k_out)


def _rows(a, shape, dtype: int, op: str, name: str):
    """An array [rows][cols]: address and row stride; zeros for none."""
    if a is None:
        return 0, 0
    if a.shape != shape or _type(a.dtype) != dtype or (a.stride()[1] != 1 and shape[1] > 1):
        raise S2SError(f"{op}: {name} is {tuple(a.shape)} of {a.dtype}, wanted {tuple(shape)} with adjacent columns "
                       "and the call's type")
    return a.data_ptr(), a.stride()[0]


def rms_norm(x, weight, out, eps: float = 1e-6, res=None, sum=None, scales=None, group: int = 0,
             weight_offset: float = 0.0, stream: int = 0):
    """out = h / sqrt(mean(h^2) + eps) * (weight + weight_offset) of the rows of h =
    x + res, with h in `sum`. x, res, sum [rows][cols] of one type, out of that type
    or e4m3 (then with `scales` f32 [rows][ceil(cols / group)], group 0 being the
    row); weight f32 [cols]."""
    op, shape = "rms_norm", x.shape
    _need(len(shape) == 2, f"{op}: x is {tuple(shape)}, wanted [rows][cols]")
    rows, cols = shape
    _need(cols < 2 ** 31 and 0 <= group < 2 ** 31, f"{op}: columns or a group that are negative or no 32-bit int")
    dt = _type(x.dtype)
    odt = E4M3 if _type(out.dtype) == E4M3 else dt
    xp, xs = _rows(x, shape, dt, op, "x")
    rp, rs = _rows(res, shape, dt, op, "res")
    sp, ss = _rows(sum, shape, dt, op, "sum")
    op_, os_ = _rows(out, shape, odt, op, "out")
    _need(weight.shape == (cols,) and _is_f32(weight.dtype) and (weight.stride()[0] == 1 or cols <= 1),
          f"{op}: weight is no f32 vector of {cols}")
    scale_ptr = 0
    if scales is not None:
        n = -(-cols // group) if group else 1
        _need(scales.shape == (rows, n) and _is_f32(scales.dtype) and _contiguous(scales),
              f"{op}: scales is no contiguous f32 [{rows}][{n}]")
        scale_ptr = scales.data_ptr()
    args = _RMS.pack(dt, odt, rows, cols, xp, rp, sp, op_, xs, rs, ss, os_, weight.data_ptr(), _f32(weight_offset), _f32(eps), scale_ptr,
                     group)
    if load_library().s2s_rms_norm(args, stream):
        raise S2SError(f"{op}: {last_error()}")
    return out
