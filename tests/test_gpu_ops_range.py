"""The attention operator over the range of its values, on the GPU: values far from one, and
keys that a mask hides, in every kernel that large calls take."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_ops as T

pytestmark = pytest.mark.gpu


# ---- values far from one ----------------------------------------------------------


def saturated(scale):
    """Scores at minus the cap in the first half of the heads and at the cap in the second; values of
    size `scale`."""
    def change(q, k, v, more):
        h = q.shape[2] // 2
        q[...], k[...] = 5.0, 5.0
        k[:, :, :h] = -5.0
        v *= scale
        v[...] = T.R.round_to(v, "bf16")  # (values of f32 too)
    return change


@pytest.mark.parametrize("dtype,scale", [(t, x) for t in ("f32", "bf16") for x in (1e-4, 1e-6, 1e-12, 1e-30, 1e30, 1e36)] + [("f16", 1e-4)])
def test_attention_values_under_a_cap(pkg, dtype, scale):
    """Scores of a cap's size either way leave the values' precision alone, however small or large they
    are: a row whose keys all score -50 has the same result as one whose keys all score 50."""
    T.check_attention(pkg, T.case(dtype, D=64, causal=True, cap=50.0, **T.WIDE), saturated(scale))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [dict(Lq=1, Lk=130, H=2), dict(Lq=80, Lk=130, H=2), T.WIDE])
def test_attention_values_near_the_largest(pkg, dtype, shape):
    """Values of 2e37 whose weighted mean is no larger: one key scores 5 above the others, in a tile behind
    theirs."""
    def change(q, k, v, more):
        q[...], k[...] = 1.0, 0.0
        k[:, 70] = 0.625  # times 64 / 8
        v *= 2e37 / 8
        v[...] = T.R.round_to(v, "bf16")
    T.check_attention(pkg, T.case(dtype, D=64, **shape), change)


# ---- slopes past what a product with a distance holds -----------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [dict(Lq=1, Lk=200, H=8), dict(Lq=90, Lk=200, H=8, KV=2), dict(T.WIDE, H=12)])
@pytest.mark.parametrize("mask", ["causal", "all", "positions", "cap"])
def test_attention_steep_slopes(pkg, dtype, shape, mask):
    """However steep the slopes, infinite ones too, the key in the query's own place scores without a bias: it is
    all that the row sees."""
    c = T.case(dtype, D=64, causal=mask in ("causal", "cap"), cap=30.0 if mask == "cap" else 0.0, slopes=True,
               pos=(lambda g, c: (np.arange(c["Lq"]) + 1000, np.arange(c["Lk"]) + 1000)) if mask == "positions" else None, **shape)
    q, k, v, more = T.inputs(c)
    steep = np.array([1e21, 1e30, 5e36, 1e37, 1e38, 3e38, np.inf, 2.0], np.float32)
    more["slopes"] = steep[np.arange(c["H"]) % 8]
    plan, ws, _ = T.make_plan(pkg, c)
    d, m = T.upload(pkg, c, q, k, v, more)
    T.call(plan, ws, d, m)
    got = d["out"].get()
    first = 0 if mask == "positions" else c["Lk"] - c["Lq"]
    for h in np.flatnonzero(more["slopes"] > 1e20):
        want = v[:, first:first + c["Lq"], h // (c["H"] // c["KV"])]
        # one weight, which the sum divides away: a product and a division in f32, and the type's rounding
        assert (np.abs(got[:, :, h] - want) <= (T.R.HALF[dtype] + 4 * 2.0 ** -24) * np.abs(want)).all(), h


# ---- calls that the documentation allows ------------------------------------------------


def test_operators_after_an_error_of_the_callers(pkg):
    """A failed call of the caller's own to the runtime, whose error nobody has taken, is no error of the operators."""
    h = pkg.hip.rt()
    c = T.case("bf16", Lq=3, Lk=70, H=2, KV=1)
    q, k, v, more = T.inputs(c)
    plan, ws, scale = T.make_plan(pkg, c)
    want, bound, _ = T.R.attention("bf16", q, k, v, scale)
    d, m = T.upload(pkg, c, q, k, v, more)
    pos = T.R.Dev(pkg, np.zeros((1, 3, 1), np.int32), "f32", whole=True)
    x, w, out = (T.R.Dev(pkg, a, "f32") for a in (np.ones((4, 32)), np.ones(32), np.zeros((4, 32))))
    rot = pkg.ops.Rotary.of((8,))
    assert h.hipSetDevice(9999) != 0
    T.call(plan, ws, d, m)
    assert h.hipSetDevice(9999) != 0
    rot(d["q"].array, pos.array)
    assert h.hipSetDevice(9999) != 0
    pkg.ops.rms_norm(x.array, w.array, out.array)
    h.hipGetLastError()
    pkg.hip.synchronize()
    assert (np.abs(d["out"].get() - want) <= bound).all()
    assert (np.abs(out.get() - 1) <= 1e-6).all()


def test_rotary_in_place_strides_of_one(pkg):
    """In place the strides have to be the same, but that of a dimension of one counts for nothing."""
    x = np.random.default_rng(0).standard_normal((1, 1, 1, 16))
    d, one = T.R.Dev(pkg, x, "f32"), T.R.Dev(pkg, x, "f32")
    pos = T.R.Dev(pkg, np.full((1, 1, 1), 3, np.int32), "f32", whole=True)
    rot, A = pkg.ops.Rotary.of((8,)), pkg.ops.Array
    rot(one.array, pos.array)
    rot(A(d.array.ptr, (1, 1, 1, 16), "f32", (5, 7, 9, 1)), pos.array, A(d.array.ptr, (1, 1, 1, 16), "f32", (64, 16, 16, 1)))
    assert np.array_equal(d.get(), one.get())


@pytest.mark.parametrize("Lq", [2, 100])
def test_attention_no_keys_with_documents_and_positions(pkg, Lq):
    """No key: the keys' documents and positions are arrays of nothing, whose address may be zero."""
    plan = pkg.ops.Attention("bf16", 2, Lq, 0, 4, 2, 64)
    q, out = (T.R.Dev(pkg, np.full((2, Lq, 4, 64), 3.0), "bf16") for _ in range(2))
    empty, none = pkg.ops.Array(0, (2, 0, 2, 64), "bf16"), pkg.ops.Array(0, (2, 0), "i32")
    ids = T.R.Dev(pkg, np.zeros((2, Lq), np.int32), "f32", whole=True)
    slopes = T.R.Dev(pkg, np.ones(4), "f32")
    ws = T.R.Dev(pkg, np.zeros(max(plan.workspace_bytes // 4, 1)), "f32")
    plan(q.array, empty, empty, out.array, workspace=ws.array, q_docs=ids.array, k_docs=none)
    assert not out.get().any()
    out.buf.upload(np.ones(out.buf.n, np.float32))
    plan(q.array, empty, empty, out.array, workspace=ws.array, q_pos=ids.array, k_pos=none, slopes=slopes.array)
    assert not out.get().any()
    # nor does the address of nothing say anything: here the output's, and one past every array
    out.buf.upload(np.ones(out.buf.n, np.float32))
    at_out, past = pkg.ops.Array(out.array.ptr, (2, 0, 2, 64), "bf16"), pkg.ops.Array(8, (2, 0), "i32")
    plan(q.array, at_out, at_out, out.array, workspace=ws.array, q_docs=ids.array, k_docs=past, q_pos=ids.array, k_pos=past, slopes=slopes.array)
    assert not out.get().any()


@pytest.mark.parametrize("cols", [100, 4096])
def test_rms_norm_largest_group(pkg, cols):
    """A group far past the row is the row."""
    T.rms_case(pkg, "bf16", 5, cols, e4m3=True, group=2 ** 31 - 8)


@pytest.mark.parametrize("mode", [0, 1])
def test_operators_captured_in_every_mode(pkg, mode):
    """Capture in the global and the thread's own mode, which refuse calls that a capture cannot hold: a call makes none.
    Replays, with eager work between them, are the eager run."""
    h, vp = pkg.hip.rt(), C.c_void_p
    for name, args in {"hipStreamBeginCapture": [vp, C.c_int], "hipStreamEndCapture": [vp, C.POINTER(vp)],
                       "hipGraphInstantiate": [C.POINTER(vp), vp, vp, vp, C.c_size_t], "hipGraphLaunch": [vp, vp],
                       "hipGraphExecDestroy": [vp], "hipGraphDestroy": [vp]}.items():
        getattr(h, name).argtypes = args
    b, other, st = T.Block(pkg, 7), T.Block(pkg, 8), T.new_stream(pkg)
    b.run()
    pkg.hip.synchronize()
    want = b.bits()
    g, e = vp(), vp()
    assert h.hipStreamBeginCapture(st, mode) == 0
    b.run(stream=st.value)
    assert h.hipStreamEndCapture(st, C.byref(g)) == 0
    assert h.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
    for _ in range(4):
        for dev in (b.h, b.turned, b.out, b.last):
            dev.buf.upload(np.zeros(dev.buf.n, np.float32))
        other.run()
        pkg.hip.synchronize()
        assert h.hipGraphLaunch(e, st) == 0
        pkg.hip.stream_synchronize(st.value)
        assert b.bits() == want
    h.hipGraphExecDestroy(e)
    h.hipGraphDestroy(g)
    h.hipStreamDestroy(st)


# ---- hidden keys in the kernels of large calls --------------------------------------------

HIDDEN = {
    "f16": dict(dtype="f16", D=128),
    "bf16": dict(dtype="bf16", D=64),
    "f32": dict(dtype="f32", D=64),
    "cap_bf16": dict(dtype="bf16", D=128, cap=50.0, spread=4.0),
    "cap_f32": dict(dtype="f32", D=32, cap=50.0, spread=4.0),
    "slopes_bf16": dict(dtype="bf16", D=64, slopes=True),
    "slopes_f32": dict(dtype="f32", D=128, slopes=True),
    "cap_slopes_f16": dict(dtype="f16", D=96, slopes=True, cap=30.0),
    "documents_bf16": dict(dtype="bf16", D=128, docs=T.scattered, cap=50.0),
    "documents_f32": dict(dtype="f32", D=96, docs=T.scattered, slopes=True),
}


@pytest.mark.parametrize("where,name", [(w, n) for w in ("future", "past_the_length", "documents") for n in HIDDEN
                                        if w != "documents" or "docs" in HIDDEN[n]])
def test_attention_hidden_keys_of_large_calls(pkg, name, where):
    """NaN and infinities in keys that some or all of the queries do not see, by the causal mask, the
    lengths or the documents: as they are not there for those, and are for the others."""
    more = dict(causal=True) if where == "future" else dict(k_lens=[90 - i for i in range(43)]) if where == "past_the_length" else {}

    def change(q, k, v, extra):
        if where == "future":
            v[:, 89, 0, 5], v[:, 88, 3, 2], k[:, 89, 4, 0], v[:, 60, 5, 7] = np.nan, np.inf, np.nan, -np.inf
        elif where == "past_the_length":
            for b in range(43):
                k[b, 90 - b:], v[b, 90 - b:] = np.nan, (np.inf, -np.inf, np.nan)[b % 3]
        else:
            k[:, 80:], v[:, 70:75], v[:, 75:] = np.inf, np.nan, -np.inf
            extra["k_docs"][:, 70:] = np.where(np.arange(20) % 2, -1, 7)
    T.check_attention(pkg, T.case(**HIDDEN[name], **more, **T.WIDE), change)


# ---- rows whose squares pass an f32 --------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [60, 180, 177, 4096, 16400])
@pytest.mark.parametrize("e4m3", [False, True])
def test_rms_norm_rows_far_from_one(pkg, dtype, cols, e4m3):
    """Rows of 1e19 to 1e37 and, without eps, of 1e-19 to 1e-30: their squares' mean is past what an f32 holds, or below
    its precision, and the norm is not."""
    def change(x, r):
        for n, s in enumerate((1e19, 1e25, 1e37, 1.0, 1e-19, 1e-25, 1e-30)):
            x[n] *= s
            r[n] *= s
    for group in (0, 64) if e4m3 else (0,):
        T.rms_case(pkg, dtype, 8, cols, e4m3=e4m3, group=group, change=change, eps=0.0)

    def large(x, r):
        x[1:4], r[1:4] = x[1:4] * 1e30, r[1:4] * 1e30
    T.rms_case(pkg, dtype, 8, cols, e4m3=e4m3, change=large, alias=("sum",))
