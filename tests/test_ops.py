"""The transformer operators without a GPU: every refusal that needs no device, and
the plain implementations that the GPU tests use."""
import numpy as np
import pytest

import ops_ref as R


def arr(pkg, shape, dtype="bf16", ptr=4096, strides=None):
    return pkg.ops.Array(ptr, shape, dtype, strides)


def plan(pkg, **more):
    a = dict(dtype="bf16", batch=2, q_tokens=5, k_tokens=7, q_heads=4, k_heads=2, width=64)
    a.update(more)
    return pkg.ops.Attention(**a)


@pytest.mark.parametrize("more,word", [
    (dict(dtype="f64"), "dtype"), (dict(dtype="e4m3"), "dtype"), (dict(batch=-1), "negative"), (dict(q_tokens=-1), "negative"),
    (dict(k_tokens=-2), "negative"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"), (dict(k_heads=0), "multiple"),
    (dict(width=0), "width"), (dict(width=129), "width"), (dict(k_tokens=2 ** 31 - 1), "2^30"),
    (dict(q_tokens=2 ** 30, q_heads=4), "2^30"), (dict(batch=2 ** 20), "2^20"), (dict(batch=2 ** 32 + 1), "int"),
])
def test_attention_sizes_refused(pkg, more, word):
    with pytest.raises(pkg.S2SError, match=word.replace("^", r"\^")):
        plan(pkg, **more)


def tensors(pkg):
    return dict(q=arr(pkg, (2, 5, 4, 64)), k=arr(pkg, (2, 7, 2, 64)), v=arr(pkg, (2, 7, 2, 64)), out=arr(pkg, (2, 5, 4, 64)))


@pytest.mark.parametrize("name,bad", [
    ("q", dict(shape=(2, 5, 4, 63))), ("q", dict(shape=(2, 5, 64))), ("k", dict(shape=(2, 7, 4, 64))), ("v", dict(shape=(2, 5, 2, 64))),
    ("out", dict(shape=(2, 5, 4, 64), dtype="f16")), ("k", dict(shape=(2, 7, 2, 64), strides=(896, 128, 1, 2))),
])
def test_attention_arrays_refused(pkg, name, bad):
    t = tensors(pkg)
    t[name] = arr(pkg, **bad)
    with pytest.raises(pkg.S2SError, match=name):
        plan(pkg)(**t)


@pytest.mark.parametrize("extra,word", [
    (dict(k_lens=((3,), "i32")), "k_lens"), (dict(q_lens=((2,), "f32")), "q_lens"), (dict(prefix=((2,), "i32")), "prefix"),
    (dict(q_docs=((2, 5), "i32")), "together"), (dict(q_docs=((2, 5), "i32"), k_docs=((3, 7), "i32")), "k_docs"),
    (dict(slopes=((2,), "f32")), "slopes"), (dict(slopes=((4,), "bf16")), "slopes"), (dict(table=((4, 6), "f32")), "odd"),
    (dict(table=((2, 5), "f32")), "table"), (dict(q_pos=((5,), "i32"), k_pos=((7,), "i32")), "without slopes"),
])
def test_attention_extras_refused(pkg, extra, word):
    e = {n: arr(pkg, *x) for n, x in extra.items()}
    with pytest.raises(pkg.S2SError, match=word):
        plan(pkg)(**tensors(pkg), **e)


def test_attention_one_of_a_pair_refused(pkg):
    with pytest.raises(pkg.S2SError):
        plan(pkg)(**tensors(pkg), k_docs=arr(pkg, (2, 7), "i32"))
    with pytest.raises(pkg.S2SError):
        plan(pkg)(**tensors(pkg), slopes=arr(pkg, (4,), "f32"), k_pos=arr(pkg, (2, 7), "i32"))


@pytest.mark.parametrize("more,word", [
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(cap=-1.0), "cap"),
    (dict(cap=float("inf")), "cap"), (dict(cap=1e-9), "cap"),
])
def test_attention_numbers_refused(pkg, more, word):
    with pytest.raises(pkg.S2SError, match=word):
        plan(pkg, **more)(**tensors(pkg))


def test_attention_nothing_to_do(pkg):
    """No batch entry or no query: done without a device."""
    for more in (dict(batch=0), dict(q_tokens=0)):
        b, n = more.get("batch", 2), more.get("q_tokens", 5)
        p = plan(pkg, **more)
        p(arr(pkg, (b, n, 4, 64)), arr(pkg, (b, 7, 2, 64)), arr(pkg, (b, 7, 2, 64)), arr(pkg, (b, n, 4, 64)))


@pytest.mark.parametrize("freq,axis,word", [
    ([1.0, float("nan")], [0, 0], "inv_freq"), ([2.0 ** 20], [0], "inv_freq"), ([1.0], [2], "axis"), ([1.0, 1.0], [0], "axis"),
    ([], [], "axis"), ([1.0] * 129, [0] * 129, "pairs"), ([1.0] * 33, [0] * 33, "pairs"), ([1.0], [256], "axis"), ([1.0], [-1], "axis"),
])
def test_rotary_frequencies_refused(pkg, freq, axis, word):
    with pytest.raises(pkg.S2SError, match=word):
        r = pkg.ops.Rotary(freq, axis)
        r(arr(pkg, (1, 4, 2, 64)), arr(pkg, (1, 4, 2), "i32"))


@pytest.mark.parametrize("q,pos,more,word", [
    (((4, 2, 64),), ((1, 4, 2), "i32"), {}, "wanted"), (((1, 4, 2, 64), "e4m3"), ((1, 4, 2), "i32"), {}, "dtype"),
    (((1, 4, 2, 64),), ((1, 4, 2), "f32"), {}, "pos"), (((1, 4, 2, 64),), ((1, 5, 2), "i32"), {}, "pos"),
    (((1, 4, 2, 64),), ((1, 4, 5), "i32"), {}, "axes"), (((1, 4, 2, 64),), ((1, 4, 2), "i32", 4096, (8, 4, 1)), {}, "pos"),
    (((1, 4, 2, 64),), ((1, 4, 2), "i32"), dict(k=((1, 5, 2, 64),)), "k"),
    (((1, 4, 2, 64),), ((1, 4, 2), "i32"), dict(k_out=((1, 4, 2, 64),)), "k_out"),
    (((1, 4, 2, 64),), ((1, 4, 2), "i32"), dict(lens=((2,), "i32")), "lens"),
])
def test_rotary_arrays_refused(pkg, q, pos, more, word):
    r = pkg.ops.Rotary.of((16, 16))
    with pytest.raises(pkg.S2SError, match=word):
        r(arr(pkg, *q), arr(pkg, *pos), **{n: arr(pkg, *x) for n, x in more.items()})


@pytest.mark.parametrize("x,out,more,word", [
    (((4, 8, 2), "f32"), ((4, 8), "f32"), {}, "rows"), (((4, 8), "e4m3"), ((4, 8), "e4m3"), {}, "dtype"),
    (((4, 8), "f32"), ((4, 9), "f32"), {}, "out"), (((4, 8), "f32"), ((4, 8), "f16"), {}, "out"),
    (((4, 8), "f32", 4096, (16, 2)), ((4, 8), "f32"), {}, "x"),
    (((4, 8), "f32"), ((4, 8), "f32"), dict(group=8), "group"), (((4, 8), "f32"), ((4, 8), "e4m3"), {}, "scales"),
    (((4, 8), "f32"), ((4, 8), "e4m3"), dict(scales=((4, 2), "f32")), "scales"),
    (((4, 24), "f32"), ((4, 24), "e4m3"), dict(scales=((4, 2), "f32"), group=12), "multiple of 8"),
    (((4, 24), "f32"), ((4, 24), "e4m3"), dict(scales=((4, 2), "f32"), group=-8), "negative"),
    (((4, 8), "f32"), ((4, 8), "f32"), dict(eps=-1.0), "eps"), (((4, 8), "f32"), ((4, 8), "f32"), dict(eps=float("nan")), "eps"),
    (((4, 8), "f32"), ((4, 8), "f32"), dict(res=((4, 8), "f16")), "res"), (((4, 8), "f32"), ((4, 8), "f32"), dict(sum=((3, 8), "f32")), "sum"),
])
def test_rms_norm_refused(pkg, x, out, more, word):
    more = {n: arr(pkg, *v) if isinstance(v, tuple) else v for n, v in more.items()}
    with pytest.raises(pkg.S2SError, match=word):
        pkg.ops.rms_norm(arr(pkg, *x), arr(pkg, (x[0][1],), "f32"), arr(pkg, *out, ptr=8192), **more)


@pytest.mark.parametrize("more,fewer", [
    (dict(batch=2 ** 10, q_tokens=2 ** 21, q_heads=1, k_heads=1), 2 ** 20 - 64),
    (dict(batch=2 ** 19, q_tokens=2 ** 11 - 63, q_heads=2, k_heads=2), 2 ** 10 - 64),
    (dict(batch=1, q_tokens=2 ** 30 - 63, q_heads=1, k_heads=1), 2 ** 30 - 64),
])
def test_attention_more_than_a_launch_refused(pkg, more, fewer):
    """Query tokens times heads of the whole batch: a launch holds less than 2^24 tiles of 64."""
    with pytest.raises(pkg.S2SError, match="of the batch"):
        plan(pkg, **more)
    assert plan(pkg, **{**more, "q_tokens": fewer}).workspace_bytes > 0


def test_attention_more_documents_than_a_launch_refused(pkg):
    b, nk = 2 ** 13, 2 ** 18
    p = plan(pkg, batch=b, k_tokens=nk, q_heads=2, k_heads=2, q_tokens=1)
    a = [arr(pkg, (b, n, 2, 64)) for n in (1, nk, nk, 1)]
    with pytest.raises(pkg.S2SError, match="documents"):
        p(*a, q_docs=arr(pkg, (1,), "i32"), k_docs=arr(pkg, (nk,), "i32"))


@pytest.mark.parametrize("big", [1e39, -1e39, 1e300])
def test_numbers_past_a_float_refused(pkg, big):
    for more in (dict(scale=big), dict(cap=big)):
        with pytest.raises(pkg.S2SError, match="scale|cap"):
            plan(pkg, **more)(**tensors(pkg))
    for more in (dict(eps=big), dict(weight_offset=big)):
        with pytest.raises(pkg.S2SError, match="eps"):
            pkg.ops.rms_norm(arr(pkg, (4, 8), "f32"), arr(pkg, (8,), "f32"), arr(pkg, (4, 8), "f32"), **more)


@pytest.mark.parametrize("name", ["q_out", "k_out"])
def test_rotary_across_refused(pkg, name):
    """q's output where k lies, or k's where q lies: read by other workgroups still."""
    q, k, o = (arr(pkg, (1, 4, 2, 64), ptr=4096 * (1 + i)) for i in range(3))
    out = dict(q_out=k, k_out=o) if name == "q_out" else dict(q_out=o, k_out=q)
    with pytest.raises(pkg.S2SError, match="q's output is k"):
        pkg.ops.Rotary.of((16, 16))(q, arr(pkg, (1, 4, 2), "i32"), k=k, **out)


def test_nothing_to_do(pkg):
    """No row, no token: done without a device or an address."""
    none = arr(pkg, (0, 8), "f32", ptr=0)
    pkg.ops.rms_norm(none, arr(pkg, (8,), "f32"), none)
    pkg.ops.rms_norm(none, arr(pkg, (8,), "f32"), arr(pkg, (0, 8), "e4m3", ptr=0), scales=arr(pkg, (0, 1), "f32", ptr=0))
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        pkg.ops.Rotary.of((16, 16))(arr(pkg, shape, ptr=0), arr(pkg, shape[:2] + (2,), "i32", ptr=0))


def test_rms_norm_weight_refused(pkg):
    with pytest.raises(pkg.S2SError, match="weight"):
        pkg.ops.rms_norm(arr(pkg, (4, 8), "f32"), arr(pkg, (9,), "f32"), arr(pkg, (4, 8), "f32", ptr=8192))


@pytest.mark.parametrize("pack,name", [("_ATTENTION", "Attention_"), ("_ROTARY", "Rotary_"), ("_RMS", "RmsNorm_")])
def test_argument_packs_are_the_c_structs(pkg, pack, name):
    """The packs that the calls send are the C structs, field by field: distinct values packed
    come back under the structs' names in order, nested ones flattened."""
    import ctypes as C
    packer, struct = getattr(pkg.ops, pack), getattr(pkg.abi, name)
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
    data = packer.pack(*range(1, n + 1))
    assert list(leaves(struct.from_buffer_copy(data))) == list(range(1, n + 1))


@pytest.mark.parametrize("rust,c,py", [("S2sAttentionArgs", "s2s_attention_args", "Attention_"), ("S2sRotaryArgs", "s2s_rotary_args", "Rotary_"),
                                       ("S2sRmsNormArgs", "s2s_rms_norm_args", "RmsNorm_"), ("S2sTokens", "s2s_tokens", "Tokens_")])
def test_structs_are_the_headers(pkg, rust, c, py):
    """The Rust and Python structs have the header's fields, in its order and of its sizes."""
    import ctypes as C
    import re
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (c, c), (root / "include" / "swin2sr_hip.h").read_text(), re.S).group(1)
    fields = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        m = re.match(r"\s*((?:const )?\w+)\s+(.*)", decl.strip(), re.S)
        if m:
            for name in m.group(2).split(","):
                name = name.strip()
                fields.append((name.lstrip("*"), "pointer" if name.startswith("*") else m.group(1)))
    rs = re.search(r"pub struct %s \{(.*?)\n\}" % rust, (root / "swin2sr-rs_amd" / "rust" / "src" / "hip.rs").read_text(), re.S).group(1)
    rs = re.findall(r"pub (\w+): ([^,\n]+),", rs)
    kinds = {"int": ("c_int", C.c_int), "float": ("f32", C.c_float), "int64_t": ("i64", C.c_int64), "s2s_tokens": ("S2sTokens", pkg.abi.Tokens_)}
    assert [n for n, _ in rs] == [n for n, _ in fields] == [n for n, _ in getattr(pkg.abi, py)._fields_]
    for (name, kind), (_, rt), (_, pt) in zip(fields, rs, getattr(pkg.abi, py)._fields_):
        if kind == "pointer":
            assert rt.startswith("*"), name
            assert C.sizeof(pt) == 8, name
        else:
            assert (rt, pt) == kinds[kind], name


def test_null_arguments_refused(pkg):
    lib = pkg.load_library()
    assert lib.s2s_attention_workspace(None, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_attention(None, None, 0, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_rotary(None, None) != 0 and b"null" in lib.s2s_last_error()
    assert lib.s2s_rms_norm(None, None) != 0 and b"null" in lib.s2s_last_error()


# ---- the oracle ------------------------------------------------------------------


def test_roundings():
    g = np.random.default_rng(0)
    x = g.standard_normal(1000) * 10.0 ** g.integers(-3, 4, 1000)
    for t in ("f16", "bf16"):
        y = R.round_to(x, t)
        # below its normal range (f16: 2^-14) a type's steps are all the smallest one
        assert (np.abs(y - x.astype(np.float32)) <= np.maximum(R.HALF[t] * np.abs(x), R.TINY[t] / 2)).all()
        assert np.array_equal(R.round_to(y, t), y)
    v = R.e4m3_values()
    assert v[0x7E] == 448 and v[1] == 2.0 ** -9 and v[0x38] == 1 and np.isnan(v[0x7F]) and v[0xB8] == -1


def test_plain_attention():
    """Uniform weights average what the masks leave; a row with nothing gives zeros; what is
    masked may hold anything."""
    g = np.random.default_rng(1)
    k, v = g.standard_normal((1, 6, 1, 4)), g.standard_normal((1, 6, 1, 4))
    q = np.zeros((1, 3, 2, 4))
    out, bound, _ = R.attention("f32", q, k, v, 1.0, causal=True)
    for i in range(3):
        assert np.allclose(out[0, i, 1], v[0, :4 + i, 0].mean(0), atol=1e-14)
    v[0, 5] = np.nan
    docs = np.array([0, 0, 1, 1, -1, -1])
    out, _, _ = R.attention("f32", q, k, v, 1.0, q_docs=np.array([1, -1, 2]), k_docs=docs)
    assert np.allclose(out[0, 0, 0], v[0, 2:4, 0].mean(0)) and not out[0, 1:].any()
    out, _, w = R.attention("f32", q, k, v, 1.0, k_lens=np.array([2]), q_lens=np.array([1]))
    assert np.allclose(out[0, 0, 0], v[0, :2, 0].mean(0)) and w.sum() == 1


def test_plain_rotary():
    x = np.random.default_rng(2).standard_normal((1, 1, 1, 6))
    for adjacent in (False, True):
        y = R.rotary(x, np.full((1, 1, 2), np.pi / 2), 2, adjacent, False)
        i, j = ([0, 2], [1, 3]) if adjacent else ([0, 1], [2, 3])
        assert np.allclose(y[..., i], -x[..., j]) and np.allclose(y[..., j], x[..., i]) and np.array_equal(y[..., 4:], x[..., 4:])
        assert np.allclose(R.rotary(y, np.full((1, 1, 2), np.pi / 2), 2, adjacent, True), x)
