"""Heads' norms with the rotation, attention with a sliding window and attention of a batch that
shares a prefix, without a GPU: every refusal that needs no device, and the plain implementations."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import ops_ref as R
from test_ops import arr, plan, tensors

# ---- heads' norms with the rotation ------------------------------------------------


def turn(pkg, q=(2, 5, 4, 64), k=None, qw=(64,), kw=None, sections=(16, 16), plan=None, **more):
    p = plan or pkg.ops.NormRotary.of(sections)
    p(arr(pkg, q), arr(pkg, (q[0], q[1], len(sections)), "i32"), arr(pkg, qw, "f32"), k=arr(pkg, k, ptr=8192) if k else None,
      k_weight=arr(pkg, kw, "f32") if kw else None, **more)


@pytest.mark.parametrize("call,word", [
    (dict(qw=(63,)), "q_weight"), (dict(qw=(3, 64)), "q_weight"), (dict(qw=(2, 5, 64)), "q_weight"),
    (dict(k=(2, 5, 2, 64)), "k without k_weight"), (dict(kw=(64,)), "k_weight without k"),
    (dict(k=(2, 5, 2, 64), kw=(4, 64)), "k_weight"), (dict(k=(2, 4, 2, 64), kw=(64,)), "k is"),
    (dict(sections=(16, 17)), "pairs"), (dict(sections=(8,) * 5), "axes"), (dict(q=(5, 4, 64)), "wanted"),
])
def test_norm_rotary_refused(pkg, call, word):
    with pytest.raises(pkg.S2SError, match=word):
        turn(pkg, **call)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_norm_rotary_weight_type_refused(pkg, dtype):
    p = pkg.ops.NormRotary.of((16, 16))
    with pytest.raises(pkg.S2SError, match="q_weight"):
        p(arr(pkg, (2, 5, 4, 64)), arr(pkg, (2, 5, 2), "i32"), arr(pkg, (64,), dtype))
    with pytest.raises(pkg.S2SError, match="q_weight"):
        p(arr(pkg, (2, 5, 4, 64)), arr(pkg, (2, 5, 2), "i32"), arr(pkg, (4, 64), "f32", strides=(128, 2)))


@pytest.mark.parametrize("number", [-1.0, float("nan"), float("inf"), 1e39])
def test_norm_rotary_eps_refused(pkg, number):
    with pytest.raises(pkg.S2SError, match="eps"):
        turn(pkg, plan=pkg.ops.NormRotary.of((16, 16), eps=number))
    if number != -1.0:
        with pytest.raises(pkg.S2SError, match="weight_offset"):
            turn(pkg, plan=pkg.ops.NormRotary.of((16, 16), weight_offset=number))


def test_norm_rotary_nothing_to_do(pkg):
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        pkg.ops.NormRotary.of((16, 16))(arr(pkg, shape, ptr=0), arr(pkg, shape[:2] + (2,), "i32", ptr=0), arr(pkg, (64,), "f32", ptr=0))


def test_norm_rotary_across_refused(pkg):
    q, k, o = (arr(pkg, (1, 4, 2, 64), ptr=4096 * (1 + i)) for i in range(3))
    w = arr(pkg, (64,), "f32")
    with pytest.raises(pkg.S2SError, match="q's output is k"):
        pkg.ops.NormRotary.of((16, 16))(q, arr(pkg, (1, 4, 2), "i32"), w, q_out=k, k=k, k_weight=w, k_out=o)


# ---- attention with a sliding window ---------------------------------------------------


@pytest.mark.parametrize("more,word", [
    (dict(window=-1), "a window of -1"), (dict(window=2 ** 30 + 1), "window"), (dict(window=8, sinks=-1), "sinks"),
    (dict(window=8, sinks=2 ** 30 + 1), "sinks"), (dict(sinks=4), "sinks without"), (dict(window=2 ** 31), "int"),
    (dict(window=8, width=129), "width"), (dict(window=8, q_heads=3), "multiple"),
])
def test_window_sizes_refused(pkg, more, word):
    with pytest.raises(pkg.S2SError, match=word):
        plan(pkg, **more)


def test_window_calls_refused(pkg):
    """Sinks with documents: the entry's first keys are not each document's."""
    with pytest.raises(pkg.S2SError, match="sinks with documents"):
        plan(pkg, window=3, sinks=1)(**tensors(pkg), q_docs=arr(pkg, (2, 5), "i32"), k_docs=arr(pkg, (2, 7), "i32"))
    with pytest.raises(pkg.S2SError, match="scale"):
        plan(pkg, window=3, scale=float("nan"))(**tensors(pkg))
    with pytest.raises(pkg.S2SError, match="prefix without"):
        plan(pkg, window=3)(**tensors(pkg), prefix=arr(pkg, (2,), "i32"))


def test_window_nothing_to_do(pkg):
    for more in (dict(batch=0), dict(q_tokens=0)):
        b, n = more.get("batch", 2), more.get("q_tokens", 5)
        plan(pkg, window=4, **more)(arr(pkg, (b, n, 4, 64)), arr(pkg, (b, 7, 2, 64)), arr(pkg, (b, 7, 2, 64)), arr(pkg, (b, n, 4, 64)))


def test_window_workspace_goes_by_the_window(pkg):
    """A step over a long cache needs ranges for its whole length, one over a short window few or none."""
    sizes = dict(batch=1, q_tokens=1, k_tokens=100000, q_heads=4, k_heads=1)
    assert plan(pkg, window=64, **sizes).workspace_bytes < plan(pkg, window=4096, **sizes).workspace_bytes < plan(pkg, **sizes).workspace_bytes
    assert plan(pkg, window=2 ** 30, **sizes).workspace_bytes == plan(pkg, **sizes).workspace_bytes


# ---- attention of a batch that shares its first keys ------------------------------------


def shared(pkg, **more):
    a = dict(dtype="bf16", batch=2, q_tokens=5, shared_tokens=9, k_tokens=7, q_heads=4, k_heads=2, width=64)
    a.update(more)
    return pkg.ops.SharedAttention(**a)


def shared_tensors(pkg):
    return dict(tensors(pkg), shared_k=arr(pkg, (9, 2, 64)), shared_v=arr(pkg, (9, 2, 64)))


@pytest.mark.parametrize("more,word", [
    (dict(dtype="f64"), "dtype"), (dict(batch=-1), "negative"), (dict(shared_tokens=-1), "negative shared"), (dict(k_tokens=-1), "negative"),
    (dict(q_heads=3), "multiple"), (dict(width=129), "width"), (dict(shared_tokens=2 ** 30), "2.30 shared"),
    (dict(shared_tokens=2 ** 31), "int"), (dict(batch=2 ** 12, q_tokens=2 ** 12 + 1, q_heads=4), "2.26"),
])
def test_shared_sizes_refused(pkg, more, word):
    with pytest.raises(pkg.S2SError, match=word):
        shared(pkg, **more)


@pytest.mark.parametrize("name,bad", [
    ("q", dict(shape=(2, 5, 4, 63))), ("k", dict(shape=(2, 9, 2, 64))), ("shared_k", dict(shape=(2, 9, 2, 64))),
    ("shared_k", dict(shape=(8, 2, 64))), ("shared_v", dict(shape=(9, 4, 64))), ("shared_v", dict(shape=(9, 2, 64), dtype="f16")),
    ("shared_k", dict(shape=(9, 2, 64), strides=(128, 1, 2))), ("out", dict(shape=(2, 5, 4, 64), dtype="f32")),
])
def test_shared_arrays_refused(pkg, name, bad):
    t = shared_tensors(pkg)
    t[name] = arr(pkg, **bad)
    with pytest.raises(pkg.S2SError, match=name):
        shared(pkg)(**t)


@pytest.mark.parametrize("extra,word", [
    (dict(shared_lens=((3,), "i32")), "shared_lens"), (dict(shared_lens=((2,), "f32")), "shared_lens"), (dict(k_lens=((3,), "i32")), "k_lens"),
    (dict(q_lens=((2, 1), "i32")), "q_lens"), (dict(slopes=((2,), "f32")), "slopes"),
])
def test_shared_extras_refused(pkg, extra, word):
    with pytest.raises(pkg.S2SError, match=word):
        shared(pkg)(**shared_tensors(pkg), **{n: arr(pkg, *x) for n, x in extra.items()})


@pytest.mark.parametrize("more,word", [(dict(scale=float("nan")), "scale"), (dict(scale=2e30), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=1e-9), "cap")])
def test_shared_numbers_refused(pkg, more, word):
    with pytest.raises(pkg.S2SError, match=word):
        shared(pkg, **more)(**shared_tensors(pkg))


@pytest.mark.parametrize("name", ["prefix", "q_docs", "k_docs", "q_pos", "k_pos", "table"])
def test_shared_other_masks_refused(pkg, name):
    a = pkg.abi.SharedAttention_(pkg.abi.Attention_(2, 2, 5, 7, 4, 2, 64, 1, 1.0, 0.0), 9)
    setattr(a.own, name, 4096)
    lib = pkg.load_library()
    assert lib.s2s_shared_attention(C.addressof(a), None, 0, None) != 0 and b"not taken" in lib.s2s_last_error()


def test_shared_nothing_to_do(pkg):
    for more in (dict(batch=0), dict(q_tokens=0)):
        b, n = more.get("batch", 2), more.get("q_tokens", 5)
        s = arr(pkg, (9, 2, 64))
        shared(pkg, **more)(arr(pkg, (b, n, 4, 64)), s, s, arr(pkg, (b, 7, 2, 64)), arr(pkg, (b, 7, 2, 64)), arr(pkg, (b, n, 4, 64)))


def test_shared_workspace_goes_by_the_way(pkg):
    """Whole keys over enough column tiles need no sums, a step over long keys does."""
    assert shared(pkg, batch=64, q_tokens=500, shared_tokens=8000, k_tokens=500, q_heads=32, k_heads=8, width=128).workspace_bytes == 0
    step = dict(q_tokens=1, k_tokens=64, q_heads=32, k_heads=8, width=128)
    assert shared(pkg, batch=4, shared_tokens=300, **step).workspace_bytes == 0
    assert 0 < shared(pkg, batch=4, shared_tokens=3000, **step).workspace_bytes < shared(pkg, batch=40, shared_tokens=3000, **step).workspace_bytes


# ---- the C interface ------------------------------------------------------------------

STRUCTS = [("S2sSharedAttentionArgs", "s2s_shared_attention_args", "SharedAttention_", "_SHARED"),
           ("S2sNormRotaryArgs", "s2s_norm_rotary_args", "NormRotary_", "_NORM_ROTARY")]
RUST = {"s2s_rotary_args": "S2sRotaryArgs", "s2s_attention_args": "S2sAttentionArgs", "s2s_tokens": "S2sTokens", "int": "c_int",
        "float": "f32", "int64_t": "i64"}


@pytest.mark.parametrize("rust,c,py,pack", STRUCTS)
def test_structs_are_the_headers(pkg, rust, c, py, pack):
    """The Rust and Python structs have the header's fields, in its order and of its types, and the pack that a call sends is
    the struct: distinct values packed come back under the fields, nested ones flattened."""
    root = Path(__file__).resolve().parent.parent
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (c, c), (root / "include" / "swin2sr_hip.h").read_text(), re.S).group(1)
    fields = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        m = re.match(r"\s*((?:const )?\w+)\s+(.*)", decl.strip(), re.S)
        if m:
            for name in m.group(2).split(","):
                fields.append((name.strip().lstrip("*"), "pointer" if name.strip().startswith("*") else m.group(1)))
    rs = re.search(r"pub struct %s \{(.*?)\n\}" % rust, (root / "swin2sr-rs_amd" / "rust" / "src" / "hip.rs").read_text(), re.S).group(1)
    rs = re.findall(r"pub (\w+): ([^,\n]+),", rs)
    struct = getattr(pkg.abi, py)
    assert [n for n, _ in rs] == [n for n, _ in fields] == [n for n, _ in struct._fields_]
    for (name, kind), (_, rt), (_, pt) in zip(fields, rs, struct._fields_):
        if kind == "pointer":
            assert rt.startswith("*") and C.sizeof(pt) == 8, name
        else:
            assert rt == RUST[kind], name
            assert pt in {"int": [C.c_int], "float": [C.c_float], "int64_t": [C.c_int64], "s2s_tokens": [pkg.abi.Tokens_],
                          "s2s_rotary_args": [pkg.abi.Rotary_], "s2s_attention_args": [pkg.abi.Attention_]}[kind], name
    packer = getattr(pkg.ops, pack)
    assert packer.size == C.sizeof(struct)

    def leaves(s):
        for f, t in s._fields_:
            v = getattr(s, f)
            if isinstance(v, C.Structure):
                yield from leaves(v)
            elif isinstance(v, C._Pointer):
                yield C.cast(v, C.c_void_p).value
            else:
                yield v
    n = len(list(leaves(struct())))
    assert list(leaves(struct.from_buffer_copy(packer.pack(*range(1, n + 1))))) == list(range(1, n + 1))


def test_null_arguments_refused(pkg):
    lib = pkg.load_library()
    assert lib.s2s_norm_rotary(None, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_shared_attention_workspace(None, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_shared_attention(None, None, 0, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_window_attention_workspace(None, 1, 0, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_window_attention(None, 1, 0, None, 0, None) != 0 and b"null" in lib.s2s_last_error()


# ---- the plain implementations ----------------------------------------------------------


def test_plain_norm_rotary():
    """A head of equal channels has the weights, turned, whatever its size."""
    x = np.full((1, 2, 1, 6), 7.0)
    w = np.arange(1.0, 7.0)
    for adjacent in (False, True):
        y, bound = R.norm_rotary("f32", x, w, 0.0, 0.0, np.full((1, 2, 2), np.pi / 2), 2, adjacent, False)
        i, j = ([0, 2], [1, 3]) if adjacent else ([0, 1], [2, 3])
        assert np.allclose(y[..., i], -w[j]) and np.allclose(y[..., j], w[i]) and np.allclose(y[..., 4:], w[4:])
        assert (bound > 0).all() and (bound < 1e-4).all()


def test_plain_window():
    """Uniform weights average the window and the sinks; not causal, what lies less than the window away."""
    g = np.random.default_rng(1)
    k, v = g.standard_normal((1, 9, 1, 4)), g.standard_normal((1, 9, 1, 4))
    q = np.zeros((1, 9, 2, 4))
    out, _, _ = R.attention("f32", q, k, v, 1.0, causal=True, window=3, sinks=2)
    for i in range(9):
        seen = sorted(set(range(max(0, i - 2), i + 1)) | set(range(min(2, i + 1))))
        assert np.allclose(out[0, i, 1], v[0, seen, 0].mean(0))
    out, _, _ = R.attention("f32", q, k, v, 1.0, window=3, sinks=2)
    for i in range(9):
        seen = sorted(set(range(max(0, i - 2), min(9, i + 3))) | {0, 1})
        assert np.allclose(out[0, i, 1], v[0, seen, 0].mean(0))
    # more queries than keys: the first ones have no key
    out, _, _ = R.attention("f32", q, k[:, :4], v[:, :4], 1.0, causal=True, window=2, sinks=1)
    assert not out[0, :5].any() and np.allclose(out[0, 5, 0], v[0, 0, 0])
