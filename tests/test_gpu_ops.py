"""The transformer operators on the GPU against their definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import ops_ref as R

pytestmark = pytest.mark.gpu

ORDERS = {"packed": (0, 1, 2, 3), "cache": (0, 2, 1, 3)}


def case(dtype="bf16", B=1, Lq=64, Lk=64, H=2, KV=1, D=64, order="packed", gap=0, lead=0, cap=0.0, causal=False,
         q_lens=None, k_lens=None, prefix=None, docs=None, pos=None, slopes=False, table=0, seed=0, scale=None, spread=1.0):
    return dict(locals())


def inputs(c):
    g = np.random.default_rng(c["seed"])
    B, Lq, Lk, H, KV, D, t = (c[x] for x in ("B", "Lq", "Lk", "H", "KV", "D", "dtype"))
    q = R.round_to(c["spread"] * g.standard_normal((B, Lq, H, D)), t)
    k = R.round_to(g.standard_normal((B, Lk, KV, D)), t)
    v = R.round_to(g.standard_normal((B, Lk, KV, D)), t)
    more = {}
    for name in ("q_lens", "k_lens", "prefix"):
        if c[name] is not None:
            more[name] = np.array(c[name], np.int32)
    if c["docs"] is not None:
        q_docs, k_docs = c["docs"](g, c) if callable(c["docs"]) else c["docs"]
        more["q_docs"], more["k_docs"] = np.asarray(q_docs, np.int32), np.asarray(k_docs, np.int32)
    if c["pos"] is not None:
        more["q_pos"], more["k_pos"] = (np.asarray(x, np.int32) for x in c["pos"](g, c))
    if c["slopes"]:
        more["slopes"] = (2.0 ** -(np.arange(H) % 8 + 1)).astype(np.float32)
    if c["table"]:
        more["table"] = (2 * g.standard_normal((H, c["table"]))).astype(np.float32)
    return q, k, v, more


def upload(pkg, c, q, k, v, more):
    o = ORDERS[c["order"]]
    d = {n: R.Dev(pkg, x, c["dtype"], o, c["gap"], c["lead"], np.nan) for n, x in (("q", q), ("k", k), ("v", v))}
    d["out"] = R.Dev(pkg, np.full(q.shape, 7.5), c["dtype"], ORDERS["packed"], c["gap"], c["lead"], 3.25)
    m = {n: R.Dev(pkg, x, "f32", whole=x.dtype == np.int32) for n, x in more.items()}
    return d, m


def make_plan(pkg, c):
    scale = c["D"] ** -0.5 if c["scale"] is None else c["scale"]
    plan = pkg.ops.Attention(c["dtype"], c["B"], c["Lq"], c["Lk"], c["H"], c["KV"], c["D"], scale=scale, cap=c["cap"],
                             causal=c["causal"])
    # stale contents of a workspace must not matter: NaN everywhere
    ws = R.Dev(pkg, np.full(max(plan.workspace_bytes // 4, 1), np.nan), "f32")
    return plan, ws, np.float64(np.float32(scale))


def call(plan, ws, d, m, stream=0):
    plan(d["q"].array, d["k"].array, d["v"].array, d["out"].array, workspace=ws.array, stream=stream,
         **{n: x.array for n, x in m.items()})


def check_attention(pkg, c, change=None):
    q, k, v, more = inputs(c)
    if change:
        change(q, k, v, more)
    plan, ws, scale = make_plan(pkg, c)
    want, bound, written = R.attention(c["dtype"], q, k, v, scale, np.float64(np.float32(c["cap"])), c["causal"],
                                       **{n: x.astype(np.float64) if x.dtype == np.float32 else x for n, x in more.items()})
    d, m = upload(pkg, c, q, k, v, more)
    call(plan, ws, d, m)
    pkg.hip.synchronize()
    got = d["out"].get()
    assert d["out"].gaps_kept()
    w = written[:, :, None, None] & np.ones(got.shape, bool)
    assert np.all(got[~w] == 7.5), "rows past the sequence were written"
    got, want, bound = got[w], want[w], bound[w]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    off = np.abs(got[fine] - want[fine])
    worst = (off / np.maximum(bound[fine], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, (worst, off.max())
    return d, m, plan, ws


def segments(*sizes):
    """Consecutive documents of these sizes over queries and keys alike, the rest padding."""
    def make(g, c):
        ids = np.full(c["Lk"], -1)
        at = 0
        for n, s in enumerate(sizes):
            ids[at:at + s] = n
            at += s
        return ids[:c["Lq"]], ids
    return make


def scattered(g, c):
    return g.integers(-1, 4, (c["B"], c["Lq"])), g.integers(-1, 4, (c["B"], c["Lk"]))


def scattered_blocks(g, c):
    ids = np.repeat(g.integers(-1, 5, (c["B"], c["Lk"] // 50 + 1)), 50, 1)[:, :c["Lk"]]
    return ids[:, :c["Lq"]], ids


def far_apart(g, c):
    return np.full(c["Lq"], 3), np.full((c["B"], c["Lk"]), 5)


def grid(g, c):
    w = 8
    return (np.arange(c["Lq"]) // w * (2 * w - 1) + np.arange(c["Lq"]) % w,
            np.arange(c["Lk"]) // w * (2 * w - 1) + np.arange(c["Lk"]) % w)


CASES = {
    "one": case(Lq=1, Lk=1, H=1),
    "one_key_f32": case("f32", Lq=3, Lk=1, H=3, KV=3, D=30),
    "width_1": case("f16", Lq=5, Lk=9, D=1),
    "width_10": case("f32", B=2, Lq=64, Lk=64, H=6, KV=6, D=10, docs=scattered),
    "width_30_f32": case("f32", B=3, Lq=64, Lk=64, H=6, KV=6, D=30, table=225, pos=grid),
    "width_30_bf16": case("bf16", B=2, Lq=70, Lk=70, H=6, KV=3, D=30, slopes=True),
    "width_80": case("f16", Lq=33, Lk=190, H=4, KV=2, D=80, cap=30.0),
    "width_96": case("bf16", Lq=200, Lk=200, H=4, KV=1, D=96, causal=True),
    "width_127": case("bf16", Lq=17, Lk=131, H=3, KV=3, D=127, lead=1),
    "width_128": case("f16", B=2, Lq=257, Lk=257, H=8, KV=2, D=128, causal=True, cap=50.0),
    "width_128_f32": case("f32", Lq=130, Lk=201, H=4, KV=2, D=128, causal=True, slopes=True),
    "cache": case("bf16", B=3, Lq=20, Lk=301, H=8, KV=4, order="cache", causal=True, q_lens=[20, 3, 11], k_lens=[301, 64, 128]),
    "odd_address": case("f16", B=2, Lq=40, Lk=77, H=4, KV=2, D=64, gap=3, lead=1, causal=True),
    "gap_8": case("bf16", B=2, Lq=40, Lk=77, H=4, KV=2, D=64, gap=8, lead=8),
    "prefix": case("bf16", B=3, Lq=150, Lk=150, H=4, KV=2, causal=True, prefix=[0, 37, 1000]),
    "prefix_behind": case("f16", B=2, Lq=30, Lk=200, H=4, KV=2, causal=True, prefix=[190, 5]),
    "more_queries_than_keys": case("bf16", Lq=90, Lk=30, H=2, causal=True),
    "lengths": case("f16", B=5, Lq=33, Lk=70, H=2, q_lens=[0, 1, 33, 5, 40], k_lens=[70, 0, 1, -3, 64], causal=True),
    "documents": case("bf16", Lq=500, Lk=500, H=4, KV=2, docs=segments(130, 1, 64, 200)),
    "documents_packed": case("bf16", Lq=2600, Lk=2600, H=2, KV=1, D=32, docs=segments(300, 900, 64, 1100, 200)),
    "documents_backwards": case("f16", B=2, Lq=700, Lk=700, H=2, KV=1, D=64, docs=lambda g, c: (9 - np.arange(700) // 71, 9 - np.arange(700) // 71)),
    "documents_lengths": case("f32", B=3, Lq=700, Lk=700, H=2, KV=2, D=32, docs=scattered_blocks, q_lens=[700, 1, 333], k_lens=[650, 700, 333]),
    "rows_of_4_bytes": case("f16", B=2, Lq=40, Lk=150, H=2, KV=2, D=62, causal=True),
    "rows_of_4_bytes_f32": case("f32", B=2, Lq=40, Lk=150, H=2, KV=1, D=97, causal=True, cap=20.0),
    "documents_causal": case("f16", Lq=300, Lk=300, H=2, KV=2, docs=segments(7, 100, 150), causal=True, slopes=True),
    "documents_scattered": case("f32", B=2, Lq=65, Lk=190, H=2, docs=scattered),
    "documents_empty": case("bf16", B=2, Lq=65, Lk=190, H=2, docs=far_apart),
    "step": case("bf16", B=4, Lq=1, Lk=900, H=8, KV=2, D=128, order="cache", causal=True, cap=50.0, k_lens=[900, 1, 333, 0]),
    "step_f16_slopes": case("f16", B=1, Lq=1, Lk=5003, H=16, KV=2, order="cache", causal=True, slopes=True),
    "step_f32": case("f32", B=2, Lq=1, Lk=1500, H=4, KV=4, D=64, order="cache", causal=True, table=63),
    "step_f32_128": case("f32", B=2, Lq=1, Lk=700, H=4, KV=2, D=128, order="cache", causal=True),
    "step_4": case("bf16", B=2, Lq=4, Lk=2100, H=8, KV=2, D=128, order="cache", causal=True, prefix=[0, 2099]),
    "step_documents": case("f16", B=2, Lq=2, Lk=1100, H=4, KV=2, D=96, order="cache", docs=scattered),
    "group_33": case("f16", B=1, Lq=2, Lk=700, H=33, KV=1, D=32),
    "large_scores": case("bf16", Lq=64, Lk=300, H=2, D=64, spread=30.0),
    "large_scores_capped": case("f16", Lq=64, Lk=300, H=2, D=64, spread=30.0, cap=30.0),
    "large_cap": case("f32", Lq=64, Lk=100, H=2, D=32, cap=30000.0, spread=3.0),
    "huge_cap": case("bf16", Lq=3, Lk=100, H=2, D=32, cap=1e9, spread=3.0),
    "mixed_cap": case("f32", Lq=64, Lk=300, H=2, D=64, spread=4.0, cap=8.0),
    "small_cap": case("f32", Lq=64, Lk=100, H=2, D=32, cap=0.5),
    "negative_scale": case("f32", Lq=20, Lk=100, H=2, D=32, scale=-0.3),
    "long_f16": case("f16", Lq=130, Lk=2000, H=2, KV=1, D=64, causal=True),
}


# enough (batch entry, key head) pairs for the waves of 32 columns, in every kernel of theirs
WIDE = dict(B=43, H=12, KV=12, Lq=70, Lk=90)
CASES.update({
    "wide_bf16": case("bf16", D=128, **WIDE),
    "wide_causal_f16": case("f16", D=64, causal=True, **WIDE),
    "wide_f32": case("f32", D=64, causal=True, **WIDE),
    "wide_cap_bf16": case("bf16", D=128, causal=True, cap=50.0, spread=4.0, **WIDE),
    "wide_cap_saturated_bf16": case("bf16", D=32, cap=50.0, spread=40.0, **WIDE),
    "wide_cap_f32": case("f32", D=96, causal=True, cap=30.0, spread=8.0, **WIDE),
    "wide_cap_running_bf16": case("bf16", D=64, causal=True, cap=80.0, spread=20.0, **WIDE),
    "wide_cap_f16": case("f16", D=128, causal=True, cap=50.0, spread=10.0, **WIDE),
    "wide_slopes_bf16": case("bf16", D=96, slopes=True, **WIDE),
    "wide_slopes_causal_f16": case("f16", D=128, slopes=True, causal=True, **WIDE),
    "wide_slopes_f32": case("f32", D=128, slopes=True, causal=True, **WIDE),
    "wide_cap_slopes_bf16": case("bf16", D=64, slopes=True, causal=True, cap=50.0, **WIDE),
    "wide_docs_bf16": case("bf16", D=128, docs=scattered, causal=True, cap=50.0, slopes=True, **WIDE),
    "wide_docs_f32": case("f32", D=96, docs=scattered, **WIDE),
    "wide_lengths_bf16": case("bf16", D=128, causal=True, cap=50.0, k_lens=[(7 * i) % 91 for i in range(43)],
                              q_lens=[(5 * i) % 71 for i in range(43)], **WIDE),
})


@pytest.mark.parametrize("name", CASES)
def test_attention(pkg, name):
    check_attention(pkg, CASES[name])


def test_attention_shared_rows(pkg):
    """Strides of zero: one key and value row for all tokens, one batch entry for all."""
    for dtype, Lk in (("bf16", 100), ("f32", 1), ("f16", 65)):
        c = case(dtype, B=2, Lq=20, Lk=Lk, H=2, KV=2, D=64, causal=False)
        q, k, v, more = inputs(c)
        k[:], v[:] = k[:1, :1], v[:1, :1]
        plan, ws, scale = make_plan(pkg, c)
        want, bound, _ = R.attention(dtype, q, k, v, scale)
        d, m = upload(pkg, c, q, k, v, more)
        one = {n: pkg.ops.Array(d[n].array.ptr, (2, Lk, 2, 64), dtype, (0, 0, 64, 1)) for n in "kv"}
        plan(d["q"].array, one["k"], one["v"], d["out"].array, workspace=ws.array)
        assert (np.abs(d["out"].get() - want) <= bound).all()


def masked_nan(c):
    """NaN and infinities wherever no query of the case may look."""
    def change(q, k, v, more):
        n = c["Lk"]
        for x, bad in ((k, np.nan), (v, np.inf)):
            x[:, n - 7:n - 4] = bad
            x[:, n - 4:] = np.nan
        for b in range(c["B"]):
            more["k_docs"][b, n - 7:] = -1
    return change


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Lq", [1, 90])
def test_attention_nan_in_masked_documents(pkg, dtype, Lq):
    c = case(dtype, B=2, Lq=Lq, Lk=200, H=4, KV=2, docs=scattered)
    check_attention(pkg, c, masked_nan(c))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Lq", [3, 150])
def test_attention_nan_past_the_length(pkg, dtype, Lq):
    c = case(dtype, B=2, Lq=Lq, Lk=200, H=4, KV=2, k_lens=[150, 61])

    def change(q, k, v, more):
        k[0, 150:], v[0, 150:], k[1, 61:], v[1, 61:] = np.nan, np.inf, -np.inf, np.nan
    check_attention(pkg, c, change)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Lq,Lk", [(150, 150), (3, 150), (2, 2000)])
def test_attention_nan_in_the_future(pkg, dtype, Lq, Lk):
    """A causal query before a key that holds NaN or an infinity does not see it; one behind does."""
    c = case(dtype, Lq=Lq, Lk=Lk, H=4, KV=2, causal=True, order="cache")

    def change(q, k, v, more):
        v[0, Lk - 1, 0, 5] = np.nan
        v[0, Lk - 2, 1, 3] = np.inf
        k[0, Lk - 1, 1, 0] = np.nan
    check_attention(pkg, c, change)


def test_attention_infinity_seen(pkg):
    c = case("bf16", Lq=40, Lk=100, H=2, KV=1)
    q, k, v, more = inputs(c)
    v[0, 10, 0, 3], v[0, 70, 0, 9] = np.inf, -np.inf
    plan, ws, scale = make_plan(pkg, c)
    d, m = upload(pkg, c, q, k, v, more)
    call(plan, ws, d, m)
    got = d["out"].get()
    assert np.all(np.isposinf(got[..., 3])) and np.all(np.isneginf(got[..., 9]))
    assert np.isfinite(np.delete(got, (3, 9), -1)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Lq", [2, 80])
def test_attention_table_takes_keys_out(pkg, dtype, Lq):
    """A bias of minus infinity is a mask; one of the type's lowest value leaves a row of
    nothing but such keys its even weights."""
    c = case(dtype, Lq=Lq, Lk=80, H=2, KV=1, table=41, causal=False)

    def change(q, k, v, more):
        more["table"][0, :15] = -np.inf
        more["table"][0, 30:] = -np.inf
        more["table"][1, :] = -np.inf
    check_attention(pkg, c, change)

    def lowest(q, k, v, more):
        more["table"][0, :] = np.finfo(np.float32).min
        q[...] = 0
    check_attention(pkg, c, lowest)


@pytest.mark.parametrize("shift", [0, 4])
@pytest.mark.parametrize("heads,hd", [(6, 30), (6, 10), (2, 16)])
def test_attention_is_the_window_attention(pkg, heads, hd, shift):
    """The framework's own window attention as a case of the operator: windows as the batch,
    shift bands as documents, the (dy, dx) table by positions y * 15 + x, unit q and k."""
    lib = pkg.load_library()
    g = np.random.default_rng(3)
    hp, wp, c = 16, 24, heads * hd
    qkv = g.standard_normal((hp * wp, 3 * c)).astype(np.float32)
    ls = np.full(heads, np.log(10), np.float32)
    rel = g.standard_normal((15, 15, heads))
    y, x = np.divmod(np.arange(64), 8)
    cpb = rel[y[:, None] - y[None, :] + 7, x[:, None] - x[None, :] + 7].astype(np.float32)
    want = np.empty((hp * wp, c), np.float32)
    rc = lib.s2s_test_attention(hp, wp, 8, heads, hd, shift, pkg.abi.fptr(qkv), pkg.abi.fptr(ls),
                                pkg.abi.fptr(np.ascontiguousarray(cpb.reshape(4096, heads))), pkg.abi.fptr(want))
    assert rc == 0, pkg.abi.last_error()
    n = hp * wp // 64
    yx, reg = np.empty((n, 64, 2), np.int32), np.empty((n, 64, 2), np.uint8)
    assert lib.s2s_test_window_map(hp, wp, 8, shift, yx.ctypes.data_as(C.POINTER(C.c_int32)),
                                   reg.ctypes.data_as(C.POINTER(C.c_uint8))) == 0
    at = yx[..., 0] * wp + yx[..., 1]
    win = qkv[at].reshape(n, 64, 3, heads, hd).astype(np.float64)
    q, k = (win[:, :, i] / np.linalg.norm(win[:, :, i], axis=-1, keepdims=True) for i in (0, 1))
    table = np.zeros((heads, 225), np.float32)
    dy, dx = np.meshgrid(np.arange(-7, 8), np.arange(-7, 8), indexing="ij")
    table[:, (dy * 15 + dx + 112).ravel()] = rel.reshape(225, heads).T
    dev = {k_: R.Dev(pkg, x_, "f32") for k_, x_ in (("q", q), ("k", k), ("v", win[:, :, 2]))}
    dev["out"] = R.Dev(pkg, np.zeros((n, 64, heads, hd)), "f32")
    pos = R.Dev(pkg, (y * 15 + x).astype(np.int32), "f32", whole=True)
    docs = R.Dev(pkg, (reg[..., 0].astype(np.int32) * 3 + reg[..., 1]), "f32", whole=True)
    plan = pkg.ops.Attention("f32", n, 64, 64, heads, heads, hd, scale=10.0)
    ws = R.Dev(pkg, np.zeros(max(plan.workspace_bytes // 4, 1)), "f32")
    call(plan, ws, dev, dict(q_pos=pos, k_pos=pos, q_docs=docs, k_docs=docs, table=R.Dev(pkg, table, "f32")))
    got = dev["out"].get().reshape(n * 64, c)
    # two f32 evaluations of scores up to 10 + |bias|: 2 (hd + 12) 2^-24 of each other relative
    # in the weights, twice, and -100 against no weight (e^-80 at most)
    assert np.abs(got - want[at.ravel()]).max() <= 8 * (hd + 12) * 14 * 2.0 ** -24


def test_attention_table_sizes(pkg):
    """A table of the group's heads in LDS and one that is too large for it."""
    for entries, heads in ((2047, 1), (4097, 2), (681, 6)):
        check_attention(pkg, case("f16", B=2, Lq=70, Lk=190, H=heads, KV=1, D=32, table=entries))
        check_attention(pkg, case("bf16", B=1, Lq=2, Lk=1300, H=heads, KV=1, D=64, table=entries, causal=True, order="cache"))


def test_attention_lowest_bias_is_even(pkg):
    """Every score at the type's lowest value: the weights are equal."""
    for dtype, Lq in (("f32", 2), ("f32", 70), ("bf16", 70)):
        c = case(dtype, Lq=Lq, Lk=80, H=2, KV=1, D=32, table=3)
        q, k, v, more = inputs(c)
        more["table"][:] = np.finfo(np.float32).min
        plan, ws, _ = make_plan(pkg, c)
        d, m = upload(pkg, c, q, k, v, more)
        call(plan, ws, d, m)
        want = v[:, :, 0].mean(1)[:, None, None, :]
        tol = (80 + 8) * 2.0 ** -24 * np.abs(v).mean() * 2 + 2 * R.HALF[dtype] * (np.abs(want) + np.abs(v).mean())
        assert (np.abs(d["out"].get() - want) <= tol).all()


def test_attention_no_keys(pkg):
    """No key at all gives zeros and reads nothing."""
    for Lq in (1, 100):
        plan = pkg.ops.Attention("bf16", 2, Lq, 0, 4, 2, 64, causal=True)
        q, out = (R.Dev(pkg, np.full((2, Lq, 4, 64), 3.0), "bf16") for _ in range(2))
        empty = pkg.ops.Array(0, (2, 0, 2, 64), "bf16")
        ws = R.Dev(pkg, np.zeros(max(plan.workspace_bytes // 4, 1)), "f32")
        plan(q.array, empty, empty, out.array, workspace=ws.array)
        assert not out.get().any()


def test_attention_is_deterministic(pkg):
    """The same call gives the same bits, whatever order its workgroups come in."""
    for c in (case("bf16", B=2, Lq=1500, Lk=1500, H=4, KV=2, D=64, docs=segments(400, 90, 700)),
              case("f16", B=1, Lq=1, Lk=20000, H=8, KV=1, D=64, order="cache", causal=True),
              case("f32", B=2, Lq=300, Lk=300, H=2, KV=2, D=30, docs=scattered)):
        q, k, v, more = inputs(c)
        plan, ws, _ = make_plan(pkg, c)
        d, m = upload(pkg, c, q, k, v, more)
        seen = set()
        for _ in range(6):
            call(plan, ws, d, m)
            seen.add(d["out"].bits().tobytes())
        assert len(seen) == 1


@pytest.mark.parametrize("Lq", [1, 40])
def test_attention_offsets_past_32_bits(pkg, Lq):
    """A cache whose tokens lie 4 MiB apart: 8.8 GB from the first to the last, of which only the
    tokens' own bytes are written."""
    Lk, D, stride = 2100, 64, 1 << 21
    g = np.random.default_rng(1)
    q, k, v = (R.round_to(g.standard_normal(s), "bf16") for s in ((1, Lq, 2, D), (1, Lk, 1, D), (1, Lk, 1, D)))
    buf = pkg.hip.DeviceBuffer((stride * (Lk - 1) + 2 * D + 1) // 2)
    rows = np.concatenate([R.to_bits(k[0, :, 0], "bf16"), R.to_bits(v[0, :, 0], "bf16")], 1)
    copy, vp = pkg.hip.rt().hipMemcpy, C.c_void_p
    for j in range(Lk):
        row = np.ascontiguousarray(rows[j])
        assert copy(vp(buf.ptr + j * stride * 2), row.ctypes.data_as(vp), row.nbytes, 1) == 0
    kd, vd = (pkg.ops.Array(buf.ptr + off, (1, Lk, 1, D), "bf16", (0, stride, 0, 1)) for off in (0, 2 * D))
    qd, out = R.Dev(pkg, q, "bf16"), R.Dev(pkg, np.zeros(q.shape), "bf16")
    plan = pkg.ops.Attention("bf16", 1, Lq, Lk, 2, 1, D, causal=True)
    ws = R.Dev(pkg, np.zeros(max(plan.workspace_bytes // 4, 1)), "f32")
    plan(qd.array, kd, vd, out.array, workspace=ws.array)
    want, bound, _ = R.attention("bf16", q, k, v, np.float64(np.float32(D ** -0.5)), causal=True)
    got = out.get()
    buf.free()
    assert (np.abs(got - want) <= bound).all()


# ---- what a call refuses with a device at hand ---------------------------------------


def refused(pkg, word, f):
    with pytest.raises(pkg.S2SError, match=word):
        f()


def test_attention_refuses(pkg):
    c = case("bf16", B=1, Lq=1, Lk=5000, H=8, KV=2, D=64)
    q, k, v, more = inputs(c)
    plan, ws, _ = make_plan(pkg, c)
    d, m = upload(pkg, c, q, k, v, more)
    A = pkg.ops.Array
    a = {n: x.array for n, x in d.items()}
    assert plan.workspace_bytes > 0
    refused(pkg, "workspace", lambda: plan(**a))
    refused(pkg, "workspace", lambda: plan(**a, workspace=A(ws.buf.ptr, (plan.workspace_bytes - 1,), "u8")))
    refused(pkg, "workspace is not aligned", lambda: plan(**a, workspace=A(ws.buf.ptr + 4, (plan.workspace_bytes,), "u8")))
    host = np.zeros(64, np.float32)
    refused(pkg, "workspace is not device memory",
            lambda: plan(**a, workspace=A(host.ctypes.data // 16 * 16, (plan.workspace_bytes,), "u8")))
    w = dict(workspace=ws.array)
    refused(pkg, "q is not device memory", lambda: plan(**{**a, "q": A(host.ctypes.data, (1, 1, 8, 64), "bf16")}, **w))
    refused(pkg, "k_lens is not device memory", lambda: plan(**a, **w, k_lens=A(host.ctypes.data, (1,), "i32")))
    refused(pkg, "k is null", lambda: plan(**{**a, "k": A(0, (1, 5000, 2, 64), "bf16")}, **w))
    refused(pkg, "v is not aligned", lambda: plan(**{**a, "v": A(d["v"].array.ptr + 1, (1, 5000, 2, 64), "bf16")}, **w))
    refused(pkg, "overlap", lambda: plan(**{**a, "out": A(d["out"].array.ptr, (1, 1, 8, 64), "bf16", (512, 512, 63, 1))}, **w))
    refused(pkg, "out is an input", lambda: plan(**{**a, "out": a["q"]}, **w))
    refused(pkg, "stride", lambda: plan(**{**a, "k": A(d["k"].array.ptr, (1, 5000, 2, 64), "bf16", (0, 1 << 23, 64, 1))}, **w))
    refused(pkg, "stride", lambda: plan(**{**a, "k": A(d["k"].array.ptr, (1, 5000, 2, 64), "bf16", (0, -64, 64, 1))}, **w))
    refused(pkg, "prefix without", lambda: plan(**a, **w, prefix=R.Dev(pkg, np.zeros(1, np.int32), "f32", whole=True).array))
    # and nothing of these was run
    assert np.all(d["out"].get() == 7.5)


def test_rotary_and_norm_refuse(pkg):
    A = pkg.ops.Array
    x = R.Dev(pkg, np.ones((2, 4, 3, 16)), "bf16")
    pos = R.Dev(pkg, np.zeros((2, 4, 1), np.int32), "f32", whole=True)
    rot = pkg.ops.Rotary.of((8,))
    p = x.array.ptr
    refused(pkg, "in place", lambda: rot(x.array, pos.array, A(p, (2, 4, 3, 16), "bf16", (400, 48, 16, 1))))
    refused(pkg, "overlap", lambda: rot(x.array, pos.array, A(p, (2, 4, 3, 16), "bf16", (0, 48, 16, 1))))
    refused(pkg, "same array", lambda: rot(x.array, pos.array, x.array, x.array, x.array))
    host = np.zeros(64, np.int32)
    refused(pkg, "pos is not device memory", lambda: rot(x.array, A(host.ctypes.data, (2, 4, 1), "i32")))
    y, w = R.Dev(pkg, np.ones((4, 32)), "f32"), R.Dev(pkg, np.ones(32), "f32")
    out = R.Dev(pkg, np.zeros((4, 32)), "f32")
    norm = pkg.ops.rms_norm
    refused(pkg, "overlap", lambda: norm(y.array, w.array, A(out.array.ptr, (4, 32), "f32", (16, 1))))
    refused(pkg, "not in its rows", lambda: norm(y.array, w.array, A(y.array.ptr, (4, 32), "f32", (64, 1))))
    refused(pkg, "not in its rows", lambda: norm(y.array, w.array, A(y.array.ptr, (4, 32), "e4m3"), scales=A(out.array.ptr, (4, 1), "f32")))
    refused(pkg, "same array", lambda: norm(y.array, w.array, out.array, sum=out.array))
    refused(pkg, "weight is not device memory", lambda: norm(y.array, A(host.ctypes.data, (32,), "f32"), out.array))
    assert not out.get().any()


# ---- streams, graphs, the operators one after another --------------------------------------


class Block:
    """The front half of a transformer block on `tokens` image tokens: norm with the residual's
    addition, a projection (made on the host beforehand: q, k, v are read from the norm's output
    by strides), rotary positions, attention over documents and over a cache."""

    def __init__(self, pkg, seed, tokens=700, heads=4, kv=2, D=32):
        self.pkg, self.D = pkg, D
        g = np.random.default_rng(seed)
        cols = (heads + 2 * kv) * D
        self.x, self.res = (R.round_to(g.standard_normal((tokens, cols)), "bf16") for _ in range(2))
        self.weight = (1 + 0.1 * g.standard_normal(cols)).astype(np.float32)
        self.pos = np.stack([np.arange(tokens) // 25, np.arange(tokens) % 25], 1)[None].astype(np.int32)
        self.docs = np.where(np.arange(tokens) < 333, 0, np.where(np.arange(tokens) < 680, 1, -1)).astype(np.int32)
        up = lambda v, t="bf16": R.Dev(pkg, v, t, whole=v.dtype == np.int32)  # noqa: E731
        self.dx, self.dres, self.dw, self.dpos, self.ddocs = up(self.x), up(self.res), up(self.weight, "f32"), up(self.pos), up(self.docs)
        self.h = up(np.zeros((tokens, cols)))
        self.turned = up(np.zeros((1, tokens, heads + kv, D)))
        self.out, self.last = up(np.zeros((1, tokens, heads, D))), up(np.zeros((1, 1, heads, D)))
        self.rot = pkg.ops.Rotary.of((8, 8))
        self.plan = pkg.ops.Attention("bf16", 1, tokens, tokens, heads, kv, D, cap=30.0)
        self.step = pkg.ops.Attention("bf16", 1, 1, tokens, heads, kv, D, causal=True)
        n = max(self.plan.workspace_bytes, self.step.workspace_bytes)
        self.ws = R.Dev(pkg, np.zeros(n // 4 + 1), "f32")
        self.tokens, self.heads, self.kv = tokens, heads, kv

    def view(self, dev, first, n, width_heads):
        ptr = dev.array.ptr + first * self.D * 2
        return self.pkg.ops.Array(ptr, (1, self.tokens, n, self.D), "bf16", (0, width_heads * self.D, self.D, 1))

    def run(self, stream=0):
        H, KV = self.heads, self.kv
        all_ = H + 2 * KV
        self.pkg.ops.rms_norm(self.dx.array, self.dw.array, self.h.array, res=self.dres.array, stream=stream)
        q, k, v = self.view(self.h, 0, H, all_), self.view(self.h, H, KV, all_), self.view(self.h, H + KV, KV, all_)
        tq, tk = self.view(self.turned, 0, H, H + KV), self.view(self.turned, H, KV, H + KV)
        self.rot(q, self.dpos.array, tq, k, tk, stream=stream)
        self.plan(tq, tk, v, self.out.array, workspace=self.ws.array, stream=stream, q_docs=self.ddocs.array, k_docs=self.ddocs.array)
        last = self.pkg.ops.Array(tq.ptr + (self.tokens - 1) * (H + KV) * self.D * 2, (1, 1, H, self.D), "bf16")
        self.step(last, tk, v, self.last.array, workspace=self.ws.array, stream=stream)

    def bits(self):
        return self.h.bits().tobytes() + self.turned.bits().tobytes() + self.out.bits().tobytes() + self.last.bits().tobytes()


def test_norm_rotary_attention(pkg):
    """The three operators as they follow one another, each stage against 64 bits from what the
    stage before left in memory."""
    b = Block(pkg, 0)
    b.run()
    pkg.hip.synchronize()
    H, KV, D, n = b.heads, b.kv, b.D, b.tokens
    sum_ = b.x + b.res
    y = sum_ / np.sqrt((sum_ * sum_).mean(1, keepdims=True) + 1e-6) * b.weight
    h = b.h.get()
    assert (np.abs(h - y) <= (40 * 2.0 ** -24 + R.HALF["bf16"]) * np.abs(y) + 1e-30).all()
    qkv = h.reshape(1, n, H + 2 * KV, D)
    axis, freq = np.array(b.rot.pair_axis[:]), np.array(b.rot.inv_freq[:])
    turned = R.rotary(qkv[:, :, :H + KV], b.pos[..., axis] * freq, 16, False, False)
    got = b.turned.get()
    both = np.tile(np.abs(qkv[:, :, :H + KV, :16]) + np.abs(qkv[:, :, :H + KV, 16:]), 2)
    assert (np.abs(got - turned) <= 6 * 2.0 ** -24 * both + R.HALF["bf16"] * np.abs(turned) + 1e-30).all()
    scale = np.float64(np.float32(D ** -0.5))
    want, bound, _ = R.attention("bf16", got[:, :, :H], got[:, :, H:], qkv[:, :, H + KV:], scale, 30.0, q_docs=b.docs, k_docs=b.docs)
    assert (np.abs(b.out.get() - want) <= bound).all()
    want, bound, _ = R.attention("bf16", got[:, -1:, :H], got[:, :, H:], qkv[:, :, H + KV:], scale, causal=True)
    assert (np.abs(b.last.get() - want) <= bound).all()


def new_stream(pkg):
    h, st = pkg.hip.rt(), C.c_void_p()
    h.hipStreamCreateWithFlags.argtypes = [C.POINTER(C.c_void_p), C.c_uint]
    h.hipStreamDestroy.argtypes = [C.c_void_p]
    assert h.hipStreamCreateWithFlags(C.byref(st), 1) == 0
    return st


def test_operators_on_streams(pkg):
    """Two runs on streams of their own, at once, are each the run on the default stream."""
    blocks = [Block(pkg, s) for s in (1, 2)]
    want = []
    for b in blocks:
        b.run()
        pkg.hip.synchronize()
        want.append(b.bits())
    streams = [new_stream(pkg) for _ in blocks]
    for b in blocks:
        for dev in (b.h, b.turned, b.out, b.last):
            dev.buf.upload(np.zeros(dev.buf.n, np.float32))
    pkg.hip.synchronize()
    for _ in range(3):
        for b, st in zip(blocks, streams):
            b.run(stream=st.value)
    for st in streams:
        pkg.hip.stream_synchronize(st.value)
    assert [b.bits() for b in blocks] == want
    for st in streams:
        pkg.hip.rt().hipStreamDestroy(st)


def test_operators_captured(pkg):
    """The run captured into a graph: every replay, with eager work between, is the eager run on
    the inputs of the moment; a second graph has a workspace of its own."""
    h, vp = pkg.hip.rt(), C.c_void_p
    for name, args in {"hipStreamBeginCapture": [vp, C.c_int], "hipStreamEndCapture": [vp, C.POINTER(vp)],
                       "hipGraphInstantiate": [C.POINTER(vp), vp, vp, vp, C.c_size_t], "hipGraphLaunch": [vp, vp],
                       "hipGraphExecDestroy": [vp], "hipGraphDestroy": [vp]}.items():
        getattr(h, name).argtypes = args
    blocks, st = [Block(pkg, s) for s in (3, 4)], new_stream(pkg)
    graphs, execs = [], []
    for b in blocks:
        assert h.hipStreamBeginCapture(st, 2) == 0
        b.run(stream=st.value)
        g, e = vp(), vp()
        assert h.hipStreamEndCapture(st, C.byref(g)) == 0
        assert h.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
        graphs.append(g)
        execs.append(e)
    other = Block(pkg, 5)
    for turn in range(4):
        for b in blocks:
            b.x = R.round_to(np.random.default_rng(10 + turn).standard_normal(b.x.shape), "bf16")
            raw = R.to_bits(b.x, "bf16").tobytes()
            b.dx.buf.upload(np.frombuffer(raw, np.float32))
            b.run()
            pkg.hip.synchronize()
            want = b.bits()
            for dev in (b.h, b.turned, b.out, b.last):
                dev.buf.upload(np.zeros(dev.buf.n, np.float32))
            pkg.hip.synchronize()
            assert h.hipGraphLaunch(execs[blocks.index(b)], st) == 0
            other.run()
            pkg.hip.stream_synchronize(st.value)
            pkg.hip.synchronize()
            assert b.bits() == want, turn
        for e in execs:  # both at once: nothing shared
            assert h.hipGraphLaunch(e, st) == 0
        pkg.hip.stream_synchronize(st.value)
        assert blocks[-1].bits() == want
    for e, g in zip(execs, graphs):
        h.hipGraphExecDestroy(e)
        h.hipGraphDestroy(g)
    h.hipStreamDestroy(st)


# ---- rotary ---------------------------------------------------------------------


def rotary_case(pkg, dtype, B, L, H, KV, D, sections, adjacent, inverse=False, order="packed", gap=0, lead=0, in_place=False,
                lens=None, far=False, seed=0, shared=False):
    g = np.random.default_rng(seed)
    x = {n: R.round_to(g.standard_normal((B, L, h, D)), dtype) for n, h in (("q", H), ("k", KV)) if h}
    top = 2 ** 31 - 1 if far else 4096
    pos = g.integers(-top if far else 0, top, (L, len(sections)) if shared else (B, L, len(sections))).astype(np.int32)
    rot = pkg.ops.Rotary.of(sections, adjacent=adjacent, inverse=inverse)
    P = sum(sections)
    axis, freq = np.array(rot.pair_axis[:]), np.array(rot.inv_freq[:])
    angle = (pos[..., axis].astype(np.longdouble) * freq.astype(np.longdouble))
    angle = np.asarray(np.fmod(angle, 2 * np.longdouble("3.14159265358979323846264338327950288")), np.float64)
    if shared:
        angle = np.broadcast_to(angle, (B,) + angle.shape)
    dev = {n: R.Dev(pkg, v, dtype, ORDERS[order], gap, lead, 2.5) for n, v in x.items()}
    out = dev if in_place else {n: R.Dev(pkg, np.full(v.shape, 9.0), dtype, ORDERS["packed"], gap, lead, 2.5) for n, v in x.items()}
    args = dict(k=dev["k"].array, k_out=out["k"].array) if KV else {}
    if lens is not None:
        args["lens"] = R.Dev(pkg, np.array(lens, np.int32), "f32", whole=True).array
    keep = R.Dev(pkg, pos, "f32", whole=True)
    lens_dev = None
    if lens is not None:
        lens_dev = R.Dev(pkg, np.array(lens, np.int32), "f32", whole=True)
        args["lens"] = lens_dev.array
    rot(dev["q"].array, keep.array, out["q"].array, **args)
    pkg.hip.synchronize()
    for n, v in x.items():
        want = R.rotary(v, angle, P, adjacent, inverse)
        got = out[n].get()
        assert out[n].gaps_kept()
        # sin and cos to 3 u (their angle's rounding, the polynomial, its sum), two products
        # and a sum, then the type's rounding; channels past the pairs are copied
        mag = R.rotary(np.abs(v), np.zeros_like(angle), P, adjacent, False)
        i, j = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if adjacent else (slice(0, P), slice(P, 2 * P))
        both = np.abs(v[..., i]) + np.abs(v[..., j])
        mag[..., i], mag[..., j] = both, both
        tol = 6 * 2.0 ** -24 * mag + np.maximum(R.HALF[dtype] * np.abs(want), R.TINY[dtype] / 2)
        tol[..., 2 * P:] = 0
        rows = np.ones(v.shape[:2], bool) if lens is None else np.arange(L)[None, :] < np.array(lens)[:, None]
        off = np.abs(got - want)[rows] - tol[rows]
        assert off.max(initial=-1.0) <= 0, off.max()
        untouched = v if in_place else np.full(v.shape, 9.0)
        assert np.array_equal(got[~rows], untouched[~rows])


ROTARY = {
    "one": dict(dtype="bf16", B=1, L=1, H=1, KV=0, D=2, sections=(1,), adjacent=False),
    "step": dict(dtype="bf16", B=5, L=1, H=32, KV=8, D=128, sections=(22, 21, 21), adjacent=False),
    "halves_f32": dict(dtype="f32", B=2, L=77, H=6, KV=6, D=64, sections=(8, 12, 12), adjacent=False),
    "adjacent_f16": dict(dtype="f16", B=2, L=77, H=6, KV=2, D=64, sections=(8, 12, 12), adjacent=True),
    "adjacent_30_f32": dict(dtype="f32", B=2, L=90, H=6, KV=6, D=30, sections=(5, 5, 5), adjacent=True),
    "halves_30_bf16": dict(dtype="bf16", B=2, L=90, H=6, KV=6, D=30, sections=(7, 8), adjacent=False),
    "part": dict(dtype="f16", B=1, L=300, H=3, KV=1, D=96, sections=(8, 8, 4, 4), adjacent=False),
    "part_odd": dict(dtype="bf16", B=1, L=33, H=3, KV=1, D=31, sections=(5, 4), adjacent=True),
    "odd_address": dict(dtype="f16", B=2, L=40, H=4, KV=2, D=64, sections=(32,), adjacent=True, gap=3, lead=1),
    "odd_address_halves": dict(dtype="bf16", B=2, L=40, H=4, KV=2, D=64, sections=(32,), adjacent=False, gap=1, lead=3),
    "cache_order": dict(dtype="bf16", B=2, L=40, H=4, KV=2, D=128, sections=(32, 32), adjacent=False, order="cache"),
    "in_place": dict(dtype="bf16", B=2, L=50, H=4, KV=2, D=128, sections=(32, 32), adjacent=False, in_place=True),
    "in_place_padded": dict(dtype="f32", B=3, L=50, H=4, KV=2, D=32, sections=(8, 8), adjacent=True, in_place=True, lens=[50, 0, 7]),
    "padded": dict(dtype="f16", B=3, L=50, H=4, KV=2, D=32, sections=(16,), adjacent=False, lens=[0, 49, 13]),
    "inverse": dict(dtype="f32", B=1, L=60, H=2, KV=2, D=64, sections=(16, 16), adjacent=False, inverse=True),
    "far": dict(dtype="f32", B=1, L=500, H=2, KV=1, D=64, sections=(10, 11, 11), adjacent=False, far=True),
    "far_inverse": dict(dtype="f32", B=1, L=500, H=2, KV=1, D=64, sections=(10, 11, 11), adjacent=True, far=True, inverse=True),
    "shared": dict(dtype="bf16", B=4, L=30, H=2, KV=1, D=64, sections=(16, 16), adjacent=False, shared=True),
    "pairs_128": dict(dtype="bf16", B=1, L=30, H=2, KV=1, D=256, sections=(64, 64), adjacent=False),
}


@pytest.mark.parametrize("name", ROTARY)
def test_rotary(pkg, name):
    rotary_case(pkg, **ROTARY[name])


def test_rotary_quarter_turns(pkg):
    """Angles of whole quarter turns, where sin and cos change places: the signs and zeros."""
    n = 64
    pos = np.arange(-n // 2, n // 2, dtype=np.int32)[None, :, None]
    rot = pkg.ops.Rotary([np.pi / 2], [0], adjacent=True)
    x = np.tile(np.array([3.0, 5.0]), (1, n, 1, 1))
    d, p = R.Dev(pkg, x, "f32"), R.Dev(pkg, pos, "f32", whole=True)
    rot(d.array, p.array)
    want = R.rotary(x, pos.astype(np.float64) * np.pi / 2, 1, True, False)
    assert np.abs(d.get() - want).max() <= 8 * 6 * 2.0 ** -24


def test_rotary_inverse_is_the_gradient(pkg):
    """The gradient of sum(g * rotary(x)) by x is the inverse rotation of g: against central
    differences (exact for a linear map but for the roundings of f32, 1e-5 at steps of 1)."""
    g = np.random.default_rng(5)
    L, D = 6, 8
    x, up = (R.round_to(g.standard_normal((1, L, 1, D)), "f32") for _ in range(2))
    pos = R.Dev(pkg, g.integers(0, 1000, (1, L, 2)).astype(np.int32), "f32", whole=True)
    fwd, inv = (pkg.ops.Rotary.of((2, 2), inverse=i) for i in (False, True))

    def run(rot, v):
        d, o = R.Dev(pkg, v, "f32"), R.Dev(pkg, np.zeros(v.shape), "f32")
        rot(d.array, pos.array, o.array)
        return o.get()
    grad = run(inv, up)
    for at in range(L * D):
        step = np.zeros(L * D)
        step[at] = 1.0
        step = step.reshape(x.shape)
        diff = ((run(fwd, x + step) - run(fwd, x - step)) * up).sum() / 2
        assert abs(diff - grad.reshape(-1)[at]) <= 1e-5


# ---- root-mean-square norm ----------------------------------------------------------


def rms_case(pkg, dtype, rows, cols, res=True, sum_=True, e4m3=False, group=0, gap=0, lead=0, offset=0.0, alias=None,
             seed=0, change=None, eps=1e-6):
    g = np.random.default_rng(seed)
    x, r = (R.round_to(s * g.standard_normal((rows, cols)), dtype) for s in (1.0, 3.0))
    if change:
        change(x, r)
        x, r = R.round_to(x, dtype), R.round_to(r, dtype)
    wt = (1 + 0.3 * g.standard_normal(cols)).astype(np.float32)
    n_groups = -(-cols // group) if group else 1
    dx, dr = (R.Dev(pkg, v, dtype, gap=gap, lead=lead, fill=np.nan) for v in (x, r))
    dw = R.Dev(pkg, wt, "f32")
    out = R.Dev(pkg, np.zeros((rows, cols)), "e4m3" if e4m3 else dtype, gap=gap, lead=lead, fill=1.0)
    dsum = R.Dev(pkg, np.zeros((rows, cols)), dtype, gap=gap, lead=lead, fill=1.0)
    if alias:
        dsum = dr if "sum" in alias else dsum
        out = dx if "out" in alias else out
    sc = R.Dev(pkg, np.zeros((rows, n_groups)), "f32")
    pkg.ops.rms_norm(dx.array, dw.array, out.array, eps=eps, res=dr.array if res else None, sum=dsum.array if sum_ else None,
                     scales=sc.array if e4m3 else None, group=group, weight_offset=offset)
    pkg.hip.synchronize()
    u = 2.0 ** -24
    h = x + r if res else x
    with np.errstate(invalid="ignore", over="ignore"):
        ms = (h * h).mean(1, keepdims=True) + np.float64(np.float32(eps))
        y = h / np.sqrt(ms) * (wt.astype(np.float64) + offset)
    # the sum in f32, a chain of at most cols / 64 + 8 additions of squares under the root,
    # root and reciprocal, two products and the weight's sum
    rel = (cols / 64 + 8 + 8) * u
    if sum_:
        got = dsum.get()
        tol = np.maximum(R.HALF[dtype] * np.abs(h), R.TINY[dtype] / 2) + u * np.abs(h)
        ok = np.isfinite(h)
        assert (np.abs(got - h)[ok] <= tol[ok]).all()
        assert dsum.gaps_kept()
    got = out.get()
    assert out.gaps_kept()
    if not e4m3:
        tol = rel * np.abs(y) + np.maximum(R.HALF[dtype] * np.abs(y), R.TINY[dtype] / 2)
        assert np.array_equal(np.isnan(got), np.isnan(y))
        ok = np.isfinite(y)
        assert (np.abs(got - y)[ok] <= tol[ok]).all()
        return
    gs = group or cols
    scale = sc.get()
    vals = R.e4m3_values()[got]
    for k in range(n_groups):
        part = y[:, k * gs:(k + 1) * gs]
        want = np.maximum(np.abs(part).max(1) / 448, 2.0 ** -126)
        fine = np.isfinite(want)
        assert (np.abs(scale[:, k] - want)[fine] <= (rel + u) * want[fine]).all()
        assert np.array_equal(np.isnan(scale[:, k]), np.isnan(want))
        back = vals[:, k * gs:(k + 1) * gs][fine] * want[fine][:, None]
        # half a step of e4m3 (2^-4 of the value, at least half of 2^-9), one more part in 2^20
        # for a value so near a border that f32 puts it on the other side
        tol = np.maximum(2.0 ** -4 * np.abs(part[fine]), 2.0 ** -10 * want[fine][:, None]) * (1 + 2.0 ** -10)
        assert (np.abs(back - part[fine]) <= tol + 2 * rel * np.abs(part[fine])).all()
        assert np.isnan(vals[:, k * gs:(k + 1) * gs][~fine]).any(1).all()


RMS = {
    "one": dict(dtype="f32", rows=1, cols=1),
    "plane": dict(dtype="f32", rows=300, cols=180),
    "plane_f16": dict(dtype="f16", rows=300, cols=180),
    "plane_e4m3": dict(dtype="bf16", rows=300, cols=180, e4m3=True, group=128),
    "plane_e4m3_row": dict(dtype="f16", rows=77, cols=60, e4m3=True),
    "plane_720": dict(dtype="bf16", rows=77, cols=716, e4m3=True, group=32, alias=("sum",)),
    "narrow": dict(dtype="bf16", rows=70, cols=60, res=False, sum_=False),
    "odd": dict(dtype="f16", rows=9, cols=1023, gap=1, lead=1),
    "offset": dict(dtype="bf16", rows=5, cols=4096, offset=1.0),
    "no_sum": dict(dtype="bf16", rows=5, cols=2048, sum_=False),
    "no_res_but_sum": dict(dtype="bf16", rows=5, cols=2048, res=False),
    "wide": dict(dtype="f32", rows=3, cols=20000),
    "wide_bf16": dict(dtype="bf16", rows=3, cols=40008),
    "in_place_sum": dict(dtype="bf16", rows=30, cols=1024, alias=("sum",)),
    "in_place_both": dict(dtype="f32", rows=30, cols=1000, alias=("sum", "out")),
    "in_place_wide": dict(dtype="f16", rows=3, cols=30001, alias=("sum", "out")),
    "e4m3_row": dict(dtype="bf16", rows=4, cols=4096, e4m3=True),
    "e4m3_128": dict(dtype="bf16", rows=33, cols=5120, e4m3=True, group=128),
    "e4m3_128_alias": dict(dtype="bf16", rows=33, cols=5120, e4m3=True, group=128, alias=("sum",)),
    "e4m3_ragged": dict(dtype="f16", rows=33, cols=1000, e4m3=True, group=64),
    "e4m3_odd": dict(dtype="f32", rows=33, cols=77, e4m3=True, group=32, gap=3, lead=1),
    "e4m3_group_8": dict(dtype="f16", rows=33, cols=333, e4m3=True, group=8),
    "e4m3_group_past_row": dict(dtype="f16", rows=33, cols=333, e4m3=True, group=4096),
    "e4m3_group_48": dict(dtype="bf16", rows=7, cols=960, e4m3=True, group=48),
    "e4m3_wide": dict(dtype="f32", rows=2, cols=33333, e4m3=True, group=128),
    "e4m3_wide_row": dict(dtype="bf16", rows=2, cols=33333, e4m3=True, alias=("sum",)),
}


@pytest.mark.parametrize("name", RMS)
def test_rms_norm(pkg, name):
    rms_case(pkg, **RMS[name])


@pytest.mark.parametrize("cols", [180, 4096, 20001])
@pytest.mark.parametrize("e4m3", [False, True])
def test_rms_norm_rows_apart(pkg, cols, e4m3):
    """Rows of zeros, of NaN, of the largest and of tiny values: each its own."""
    def change(x, r):
        x[0], r[0] = 0, 0
        x[1, 3] = np.nan
        x[2], r[2] = x[2] * 1e15, r[2] * 1e15
        x[3], r[3] = x[3] * 1e-12, r[3] * 1e-12
    rms_case(pkg, "f32", 6, cols, e4m3=e4m3, group=0, change=change)
    rms_case(pkg, "f32", 6, cols, e4m3=e4m3, group=64 if e4m3 else 0, change=change)


# ---- more rows than one launch holds, dimensions of one -------------------------------------


@pytest.mark.parametrize("e4m3", [False, True])
def test_rms_norm_more_rows_than_workgroups(pkg, e4m3):
    """2^24 + 5 rows of 3: every row the same (its stride is 0), so that each is the first one."""
    rows, cols = 2 ** 24 + 5, 3
    x, w = R.Dev(pkg, R.round_to(np.array([[1.5, -2.25, 0.125]]), "f16"), "f16"), R.Dev(pkg, np.array([1.0, 0.5, 2.0]), "f32")
    out = pkg.hip.DeviceBuffer((rows * cols * (1 if e4m3 else 2) + 3) // 4)
    out.upload(np.full(out.n, np.nan, np.float32))
    scales = pkg.hip.DeviceBuffer(rows)
    A = pkg.ops.Array
    pkg.ops.rms_norm(A(x.array.ptr, (rows, cols), "f16", (0, 1)), w.array, A(out.ptr, (rows, cols), "e4m3" if e4m3 else "f16"),
                     scales=A(scales.ptr, (rows, 1), "f32") if e4m3 else None)
    pkg.hip.synchronize()
    got = out.download().view(np.uint8 if e4m3 else np.float16)[:rows * cols].reshape(rows, cols)
    h = np.array([1.5, -2.25, 0.125])
    want = h / np.sqrt((h * h).mean() + np.float64(np.float32(1e-6))) * np.array([1.0, 0.5, 2.0])
    # one rounding to f16 (one of e4m3 after the scale), and a dozen f32 ones before it
    first = R.e4m3_values()[got[0]] * (np.abs(want).max() / 448) if e4m3 else got[0].astype(np.float64)
    assert (np.abs(first - want) <= (2.0 ** -4 if e4m3 else 2.0 ** -11) * np.abs(want) + 24 * 2.0 ** -24 * np.abs(want)).all()
    assert (got == got[0]).all()
    if e4m3:
        s = scales.download()
        assert (s == s[0]).all() and abs(s[0] / (np.abs(want).max() / 448) - 1) <= 24 * 2.0 ** -24
    out.free()
    scales.free()


def test_rotary_more_tokens_than_workgroups(pkg):
    """2^28 + 2^14 tokens of one pair, the batch's entries all the same: each is the first one."""
    batch, tokens = 2 ** 14 + 1, 2 ** 14
    g = np.random.default_rng(3)
    q = R.Dev(pkg, R.round_to(g.standard_normal((1, tokens, 1, 2)), "f16"), "f16")
    pos = R.Dev(pkg, g.integers(0, 2 ** 31 - 1, (1, tokens, 1)).astype(np.int32), "f32", whole=True)
    out, one = pkg.hip.DeviceBuffer(batch * tokens), R.Dev(pkg, np.zeros((1, tokens, 1, 2)), "f16")
    rot, A = pkg.ops.Rotary([0.7], [0]), pkg.ops.Array
    rot(q.array, pos.array, one.array)
    rot(A(q.array.ptr, (batch, tokens, 1, 2), "f16", (0, 2, 2, 1)), A(pos.array.ptr, (tokens, 1), "i32"),
        A(out.ptr, (batch, tokens, 1, 2), "f16"))
    pkg.hip.synchronize()
    want = one.bits().view(np.uint32).reshape(-1)[:tokens]
    got = out.download().view(np.uint32).reshape(batch, tokens)
    out.free()
    assert (got == want).all()


@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 70), (5, 1)])
def test_attention_strides_of_one(pkg, Lq, Lk):
    """The stride of a dimension of one counts for nothing: odd, zero, or far past any array."""
    c = case("bf16", Lq=Lq, Lk=Lk, H=2, KV=1, D=64)
    q, k, v, more = inputs(c)
    plan, ws, scale = make_plan(pkg, c)
    d, m = upload(pkg, c, q, k, v, more)
    want, bound, _ = R.attention("bf16", q, k, v, scale)
    for odd in (0, 1, (1 << 23) + 1):
        def moved(a, n):
            b, t, h, w = a.stride()
            return pkg.ops.Array(a.ptr, a.shape, a.dtype, (odd, odd if n == 1 else t, odd if a.shape[2] == 1 else h, w))
        d["out"].buf.upload(np.zeros(d["out"].buf.n, np.float32))
        plan(moved(d["q"].array, Lq), moved(d["k"].array, Lk), moved(d["v"].array, Lk), moved(d["out"].array, Lq), workspace=ws.array)
        assert (np.abs(d["out"].get() - want) <= bound).all()


# ---- key ranges joined column by column -----------------------------------------------------

JOIN = {
    "bf16_128": case("bf16", Lq=140, Lk=1500, H=8, KV=8, D=128, causal=True),
    "f16_96": case("f16", Lq=140, Lk=1500, H=8, KV=4, D=96, cap=20.0),
    "f32_64": case("f32", Lq=140, Lk=900, H=8, KV=8, D=64, slopes=True, causal=True),
    "f32_32": case("f32", Lq=260, Lk=800, H=6, KV=6, D=30, order="cache", gap=2),
    "odd": case("bf16", Lq=140, Lk=1100, H=8, KV=2, D=17, gap=1, lead=1, causal=True),
    "two": case("f16", Lq=140, Lk=1300, H=8, KV=8, D=34, gap=2),
    "lengths": case("bf16", B=4, Lq=70, Lk=1024, H=8, KV=4, D=80, causal=True, q_lens=[70, 0, 33, 70], k_lens=[1024, 900, 20, 0]),
    "prefix": case("bf16", B=2, Lq=90, Lk=1024, H=8, KV=8, D=64, causal=True, prefix=[1000, 0], cap=50.0),
    "step": case("bf16", B=40, Lq=1, Lk=512, H=32, KV=8, D=128, order="cache", causal=True, k_lens=[1 + 13 * i for i in range(40)]),
}


@pytest.mark.parametrize("name", JOIN)
def test_attention_few_ranges(pkg, name):
    check_attention(pkg, JOIN[name])


# ---- rows of odd widths and addresses ------------------------------------------------

ODD = {
    "wave": dict(dtype="f16", rows=2001, cols=177, gap=1, lead=1),
    "wave_row": dict(dtype="bf16", rows=1501, cols=177, e4m3=True, lead=1),
    "wave_groups": dict(dtype="f16", rows=1030, cols=1023, e4m3=True, group=128, gap=1),
    "wave_group_8": dict(dtype="f32", rows=1027, cols=333, e4m3=True, group=8, alias=("sum",)),
    "wave_group_24": dict(dtype="bf16", rows=1025, cols=1024, e4m3=True, group=24),
    "wave_group_past_row": dict(dtype="bf16", rows=1025, cols=77, e4m3=True, group=80),
    "in_place": dict(dtype="f32", rows=1100, cols=61, alias=("sum", "out")),
    "widest": dict(dtype="bf16", rows=5, cols=8191, lead=1),
    "widest_groups": dict(dtype="bf16", rows=5, cols=8191, lead=1, e4m3=True, group=8),
    "group_1000": dict(dtype="f32", rows=9, cols=8192, e4m3=True, group=1000),
    "past": dict(dtype="f16", rows=5, cols=8193, e4m3=True, group=200),
}


@pytest.mark.parametrize("name", ODD)
def test_rms_norm_odd_rows(pkg, name):
    rms_case(pkg, **ODD[name])


@pytest.mark.parametrize("cols,rows", [(179, 1030), (4095, 6)])
@pytest.mark.parametrize("group", [0, 64])
def test_rms_norm_odd_rows_apart(pkg, cols, rows, group):
    """Rows of zeros, of NaN, of the largest and of tiny values: each its own."""
    def change(x, r):
        x[0], r[0] = 0, 0
        x[1, 3] = np.nan
        x[2], r[2] = x[2] * 1e15, r[2] * 1e15
        x[3], r[3] = x[3] * 1e-12, r[3] * 1e-12
    rms_case(pkg, "f32", rows, cols, e4m3=True, group=group, change=change)
    rms_case(pkg, "f32", rows, cols, change=change)


# ---- documents' summaries: in one launch up to 64 tiles of keys and of columns, in three past them


def doc_lengths(g, c):
    ids = np.sort(g.integers(0, 9, (c["B"], c["Lk"])), 1)
    ids[:, -c["Lk"] // 20:] = -1
    return ids[:, :c["Lq"]], ids


DOCS = {
    "five_tiles": case("bf16", B=3, Lq=300, Lk=300, H=2, KV=2, D=32, docs=doc_lengths, q_lens=[300, 0, 123], k_lens=[300, 300, 123]),
    "64_tiles": case("f16", Lq=4096, Lk=4096, H=1, KV=1, D=16, docs=doc_lengths),
    "65_tiles": case("f16", Lq=4097, Lk=4097, H=1, KV=1, D=16, docs=doc_lengths),
    "65_columns": case("bf16", B=2, Lq=1100, Lk=1100, H=4, KV=1, D=40, docs=doc_lengths, causal=True),
    "few_columns": case("bf16", B=2, Lq=2, Lk=4000, H=4, KV=1, D=64, docs=scattered, order="cache"),
    "half_tiles": case("f32", B=2, Lq=1500, Lk=1500, H=1, KV=1, D=100, docs=doc_lengths),
    "none": case("f32", B=2, Lq=500, Lk=500, H=1, KV=1, D=24, docs=lambda g, c: (np.full(500, -1), np.full(500, -1))),
}


@pytest.mark.parametrize("name", DOCS)
def test_attention_document_summaries(pkg, name):
    check_attention(pkg, DOCS[name])
