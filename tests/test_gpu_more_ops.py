"""Heads' norms with the rotation, attention with a sliding window and attention of a batch that
shares a prefix, on the GPU against their definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import ops_ref as R
import test_gpu_ops as T

pytestmark = pytest.mark.gpu


# ---- heads' norms with the rotation ------------------------------------------------------


def turned(pkg, dtype, B, L, H, KV, D, sections, adjacent=False, inverse=False, order="packed", gap=0, lead=0, in_place=False,
           lens=None, each=False, offset=0.0, eps=1e-6, far=False, seed=0, change=None, weight_gap=0):
    g = np.random.default_rng(seed)
    x = {n: g.standard_normal((B, L, h, D)) * np.exp(g.standard_normal((B, L, h, 1))) for n, h in (("q", H), ("k", KV)) if h}
    if change:
        change(x)
    x = {n: R.round_to(v, dtype) for n, v in x.items()}
    w = {n: (1 + 0.3 * g.standard_normal((h, D) if each else D)).astype(np.float32) for n, h in (("q", H), ("k", KV)) if h}
    top = 2 ** 31 - 1 if far else 4096
    pos = g.integers(-top if far else 0, top, (B, L, len(sections))).astype(np.int32)
    rot = pkg.ops.NormRotary.of(sections, eps=eps, weight_offset=offset, adjacent=adjacent, inverse=inverse)
    axis, freq = np.array(rot.pair_axis[:]), np.array(rot.inv_freq[:])
    angle = pos[..., axis].astype(np.longdouble) * freq.astype(np.longdouble)
    angle = np.asarray(np.fmod(angle, 2 * np.longdouble("3.14159265358979323846264338327950288")), np.float64)
    dev = {n: R.Dev(pkg, v, dtype, T.ORDERS[order], gap, lead, 2.5) for n, v in x.items()}
    out = dev if in_place else {n: R.Dev(pkg, np.full(v.shape, 9.0), dtype, T.ORDERS["packed"], gap, lead, 2.5) for n, v in x.items()}
    dw = {n: R.Dev(pkg, v, "f32", gap=weight_gap, lead=weight_gap) for n, v in w.items()}
    args = dict(k=dev["k"].array, k_out=out["k"].array, k_weight=dw["k"].array) if KV else {}
    lens_dev = None
    if lens is not None:
        lens_dev = R.Dev(pkg, np.array(lens, np.int32), "f32", whole=True)
        args["lens"] = lens_dev.array
    dpos = R.Dev(pkg, pos, "f32", whole=True)
    rot(dev["q"].array, dpos.array, dw["q"].array, out["q"].array, **args)
    pkg.hip.synchronize()
    for n, v in x.items():
        want, bound = R.norm_rotary(dtype, v, w[n], np.float64(np.float32(offset)), np.float64(np.float32(eps)), angle, sum(sections), adjacent, inverse)
        got = out[n].get()
        assert out[n].gaps_kept()
        rows = np.ones(v.shape[:2], bool) if lens is None else np.arange(L)[None, :] < np.array(lens)[:, None]
        untouched = v if in_place else np.full(v.shape, 9.0)
        assert np.array_equal(got[~rows], untouched[~rows])
        got, want, bound = got[rows], want[rows], bound[rows]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        worst = (np.abs(got - want)[fine] / np.maximum(bound[fine], 1e-300)).max(initial=0.0)
        assert worst <= 1.0, (n, worst)


TURNED = {
    "one": dict(dtype="bf16", B=1, L=1, H=1, KV=0, D=2, sections=(1,)),
    "step": dict(dtype="bf16", B=5, L=1, H=32, KV=8, D=128, sections=(22, 21, 21)),
    "halves_f32": dict(dtype="f32", B=2, L=77, H=6, KV=6, D=64, sections=(8, 12, 12)),
    "halves_f16": dict(dtype="f16", B=1, L=300, H=16, KV=2, D=128, sections=(64,)),
    "adjacent_f16": dict(dtype="f16", B=2, L=77, H=6, KV=2, D=64, sections=(8, 12, 12), adjacent=True),
    "adjacent_bf16": dict(dtype="bf16", B=2, L=77, H=6, KV=2, D=128, sections=(32, 32), adjacent=True, each=True),
    "adjacent_30_f32": dict(dtype="f32", B=2, L=90, H=6, KV=6, D=30, sections=(5, 5, 5), adjacent=True, each=True),
    "halves_30_bf16": dict(dtype="bf16", B=2, L=90, H=6, KV=6, D=30, sections=(7, 8)),
    "halves_10_f32": dict(dtype="f32", B=2, L=90, H=6, KV=6, D=10, sections=(3, 2)),
    "part": dict(dtype="f16", B=1, L=300, H=3, KV=1, D=96, sections=(8, 8, 4, 4)),
    "part_80": dict(dtype="f16", B=1, L=301, H=16, KV=16, D=80, sections=(10, 10)),
    "part_odd": dict(dtype="bf16", B=1, L=33, H=3, KV=1, D=31, sections=(5, 4), adjacent=True),
    "part_one": dict(dtype="f32", B=1, L=33, H=3, KV=1, D=97, sections=(1,), each=True),
    "odd_address": dict(dtype="f16", B=2, L=40, H=4, KV=2, D=64, sections=(32,), adjacent=True, gap=3, lead=1),
    "odd_address_halves": dict(dtype="bf16", B=2, L=40, H=4, KV=2, D=64, sections=(32,), gap=1, lead=3, weight_gap=1, each=True),
    "gap_8": dict(dtype="bf16", B=2, L=40, H=4, KV=2, D=64, sections=(32,), gap=8, lead=8, weight_gap=3),
    "cache_order": dict(dtype="bf16", B=2, L=40, H=4, KV=2, D=128, sections=(32, 32), order="cache"),
    "in_place": dict(dtype="bf16", B=2, L=50, H=4, KV=2, D=128, sections=(32, 32), in_place=True),
    "in_place_30": dict(dtype="f16", B=2, L=50, H=4, KV=2, D=30, sections=(4, 3), in_place=True, each=True),
    "in_place_padded": dict(dtype="f32", B=3, L=50, H=4, KV=2, D=32, sections=(8, 8), adjacent=True, in_place=True, lens=[50, 0, 7]),
    "padded": dict(dtype="f16", B=3, L=50, H=4, KV=2, D=32, sections=(16,), lens=[0, 49, 13]),
    "inverse": dict(dtype="f32", B=1, L=60, H=2, KV=2, D=64, sections=(16, 16), inverse=True),
    "far": dict(dtype="f32", B=1, L=500, H=2, KV=1, D=64, sections=(10, 11, 11), far=True),
    "offset": dict(dtype="bf16", B=1, L=60, H=2, KV=2, D=64, sections=(16, 16), offset=1.0),
    "wide": dict(dtype="bf16", B=1, L=30, H=2, KV=1, D=256, sections=(64, 64)),
    "wide_f32": dict(dtype="f32", B=1, L=30, H=2, KV=1, D=512, sections=(64, 64), each=True),
    "wide_part": dict(dtype="bf16", B=1, L=30, H=2, KV=1, D=2000, sections=(64, 64), adjacent=True),
    "wide_odd": dict(dtype="f16", B=1, L=7, H=2, KV=1, D=777, sections=(100,)),
    "heads_65": dict(dtype="f32", B=1, L=3, H=65, KV=3, D=64, sections=(32,)),
    "tokens": dict(dtype="bf16", B=1, L=5003, H=4, KV=1, D=128, sections=(32, 32)),
}


@pytest.mark.parametrize("name", TURNED)
def test_norm_rotary(pkg, name):
    turned(pkg, **TURNED[name])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,adjacent", [(64, False), (30, True), (97, False), (1030, True)])
def test_norm_rotary_heads_apart(pkg, dtype, D, adjacent):
    """Heads of zeros, of NaN, and from 1e-30 to 1e37 beside one another: each its own, without an eps too."""
    def change(x):
        for v in x.values():
            for n, s in enumerate((1e19, 1e25, 1e37, 1.0, 1e-19, 1e-25, 1e-30)):
                v[:, n] *= s / np.abs(v[:, n]).max()
            v[:, 7, 0] = np.nan
    turned(pkg, dtype, 2, 9, 3, 2, D, (5,), adjacent=adjacent, eps=0.0, change=change)

    def zeros(x):
        x["q"][0, 3, 1] = 0
        x["k"][1, 4] = 0
    turned(pkg, dtype, 2, 9, 3, 2, D, (5,), adjacent=adjacent, change=zeros)


def test_norm_rotary_is_the_norm_and_the_rotation(pkg):
    """f32 heads through rms_norm and rotary one after the other, and through the one call."""
    g = np.random.default_rng(4)
    B, L, H, D = 2, 40, 6, 60
    x, w = R.round_to(g.standard_normal((B, L, H, D)), "f32"), (1 + 0.3 * g.standard_normal(D)).astype(np.float32)
    pos = R.Dev(pkg, g.integers(0, 500, (B, L, 2)).astype(np.int32), "f32", whole=True)
    d, dw, y, z, one = (R.Dev(pkg, v, "f32") for v in (x, w, 0 * x, 0 * x, 0 * x))
    A = pkg.ops.Array
    pkg.ops.rms_norm(A(d.array.ptr, (B * L * H, D), "f32"), dw.array, A(y.array.ptr, (B * L * H, D), "f32"))
    pkg.ops.Rotary.of((15, 15))(y.array, pos.array, z.array)
    pkg.ops.NormRotary.of((15, 15))(d.array, pos.array, dw.array, one.array)
    # twice the error that one evaluation may have (23 u of the pair's magnitudes)
    both = np.tile(np.abs(y.get()[..., :30]) + np.abs(y.get()[..., 30:]), 2)
    assert (np.abs(z.get() - one.get()) <= 2 * 24 * 2.0 ** -24 * both).all()


def test_norm_rotary_refuses(pkg):
    A = pkg.ops.Array
    x, w = R.Dev(pkg, np.ones((2, 4, 3, 16)), "bf16"), R.Dev(pkg, np.ones(16), "f32")
    pos = R.Dev(pkg, np.zeros((2, 4, 1), np.int32), "f32", whole=True)
    rot, p, host = pkg.ops.NormRotary.of((8,)), x.array.ptr, np.zeros(64, np.float32)
    T.refused(pkg, "in place", lambda: rot(x.array, pos.array, w.array, A(p, (2, 4, 3, 16), "bf16", (400, 48, 16, 1))))
    T.refused(pkg, "overlap", lambda: rot(x.array, pos.array, w.array, A(p, (2, 4, 3, 16), "bf16", (0, 48, 16, 1))))
    T.refused(pkg, "q_weight is not device memory", lambda: rot(x.array, pos.array, A(host.ctypes.data, (16,), "f32")))
    T.refused(pkg, "q_weight or k_weight is null", lambda: rot(x.array, pos.array, A(0, (16,), "f32")))
    k, out = R.Dev(pkg, np.ones((2, 4, 1, 16)), "bf16"), R.Dev(pkg, np.ones((2, 4, 3, 16)), "bf16")
    T.refused(pkg, "k_weight is not aligned", lambda: rot(x.array, pos.array, w.array, out.array, k=k.array, k_weight=A(w.array.ptr + 2, (16,), "f32")))
    T.refused(pkg, "stride", lambda: rot(x.array, pos.array, A(w.array.ptr, (3, 16), "f32", (-16, 1))))
    assert (x.get() == 1).all()


# ---- attention with a sliding window ------------------------------------------------------


def wcase(dtype="bf16", window=16, sinks=0, **more):
    return dict(T.case(dtype, **more), window=window, sinks=sinks)


def window_plan(pkg, c):
    scale = c["D"] ** -0.5 if c["scale"] is None else c["scale"]
    p = pkg.ops.Attention(c["dtype"], c["B"], c["Lq"], c["Lk"], c["H"], c["KV"], c["D"], scale=scale, cap=c["cap"],
                          causal=c["causal"], window=c["window"], sinks=c["sinks"])
    ws = R.Dev(pkg, np.full(max(p.workspace_bytes // 4, 1), np.nan), "f32")
    return p, ws, np.float64(np.float32(scale))


def check_window(pkg, c, change=None):
    q, k, v, more = T.inputs(c)
    if change:
        change(q, k, v, more)
    p, ws, scale = window_plan(pkg, c)
    want, bound, written = R.attention(c["dtype"], q, k, v, scale, np.float64(np.float32(c["cap"])), c["causal"], window=c["window"],
                                       sinks=c["sinks"], **{n: x.astype(np.float64) if x.dtype == np.float32 else x for n, x in more.items()})
    d, m = T.upload(pkg, c, q, k, v, more)
    T.call(p, ws, d, m)
    pkg.hip.synchronize()
    got = d["out"].get()
    assert d["out"].gaps_kept()
    w = written[:, :, None, None] & np.ones(got.shape, bool)
    assert np.all(got[~w] == 7.5), "rows past the sequence were written"
    got, want, bound = got[w], want[w], bound[w]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    worst = (np.abs(got[fine] - want[fine]) / np.maximum(bound[fine], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, worst
    # (infinities of the same sign too)
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


WINDOWS = {
    "one": wcase(Lq=1, Lk=1, H=1, window=1),
    "one_key": wcase("f32", Lq=9, Lk=200, H=2, causal=True, window=1),
    "one_key_both_ways": wcase("f16", Lq=90, Lk=200, H=2, window=1),
    "sinks_alone": wcase("f32", Lq=9, Lk=200, H=2, causal=True, window=1, sinks=1),
    "step": wcase("bf16", B=4, Lq=1, Lk=3000, H=8, KV=2, D=128, order="cache", causal=True, window=500, sinks=4, k_lens=[3000, 1, 333, 0]),
    "step_f16_slopes": wcase("f16", Lq=1, Lk=5003, H=16, KV=2, order="cache", causal=True, slopes=True, window=1000, sinks=130),
    "step_f32": wcase("f32", B=2, Lq=1, Lk=1500, H=4, KV=4, D=64, order="cache", causal=True, table=63, window=300, sinks=3),
    "step_f32_128": wcase("f32", B=2, Lq=1, Lk=1700, H=4, KV=2, D=128, order="cache", causal=True, window=900),
    "step_4": wcase("bf16", B=2, Lq=4, Lk=2100, H=8, KV=2, D=128, order="cache", causal=True, window=777, sinks=1, cap=30.0),
    "step_short": wcase("f16", B=2, Lq=1, Lk=900, H=4, KV=1, order="cache", causal=True, window=5, sinks=2),
    "step_window_past_all": wcase("f16", B=2, Lq=1, Lk=900, H=4, KV=1, order="cache", causal=True, window=2 ** 30, sinks=2 ** 30),
    "sinks_past_all": wcase("bf16", Lq=100, Lk=300, H=2, causal=True, window=7, sinks=1000),
    "sinks_meet_window": wcase("bf16", Lq=300, Lk=300, H=2, causal=True, window=64, sinks=65),
    "prompt": wcase("bf16", Lq=700, Lk=700, H=4, KV=2, D=128, causal=True, window=100, sinks=4),
    "prompt_f16": wcase("f16", Lq=513, Lk=513, H=4, KV=1, D=64, causal=True, window=64, sinks=64),
    "prompt_f32": wcase("f32", Lq=400, Lk=400, H=2, KV=2, D=128, causal=True, window=33, sinks=1, slopes=True),
    "both_ways": wcase("f32", Lq=500, Lk=500, H=6, KV=6, D=30, window=50),
    "both_ways_sinks": wcase("bf16", Lq=500, Lk=500, H=2, KV=1, D=96, window=70, sinks=9, cap=20.0),
    "table": wcase("f32", B=2, Lq=256, Lk=256, H=6, KV=6, D=30, table=225, pos=T.grid, window=40),
    "documents": wcase("bf16", Lq=1200, Lk=1200, H=4, KV=2, docs=T.segments(130, 1, 64, 700, 200), causal=True, window=90),
    "documents_both_ways": wcase("f16", Lq=1200, Lk=1200, H=2, KV=2, docs=T.segments(130, 1, 64, 700, 200), window=90),
    "documents_scattered": wcase("f32", B=2, Lq=65, Lk=790, H=2, docs=T.scattered, window=30),
    "documents_blocks": wcase("f32", B=3, Lq=700, Lk=700, H=2, KV=2, D=32, docs=T.scattered_blocks, window=200, causal=True, q_lens=[700, 1, 333], k_lens=[650, 700, 333]),
    "documents_step": wcase("f16", B=2, Lq=2, Lk=9100, H=4, KV=2, D=96, order="cache", docs=T.scattered_blocks, window=3000, causal=True),
    "prefix": wcase("bf16", B=3, Lq=150, Lk=150, H=4, KV=2, causal=True, prefix=[0, 37, 1000], window=20, sinks=2),
    "lengths": wcase("f16", B=5, Lq=33, Lk=70, H=2, q_lens=[0, 1, 33, 5, 40], k_lens=[70, 0, 1, -3, 64], causal=True, window=3, sinks=1),
    "lengths_both_ways": wcase("f16", B=5, Lq=33, Lk=170, H=2, q_lens=[0, 1, 33, 5, 40], k_lens=[170, 0, 1, -3, 64], window=3),
    "more_queries_than_keys": wcase("bf16", Lq=190, Lk=30, H=2, causal=True, window=10, sinks=2),
    "more_queries_than_keys_both_ways": wcase("bf16", Lq=190, Lk=30, H=2, window=10, sinks=2),
    "odd_address": wcase("f16", B=2, Lq=40, Lk=277, H=4, KV=2, D=64, gap=3, lead=1, causal=True, window=50, sinks=5),
    "rows_of_4_bytes": wcase("f16", B=2, Lq=40, Lk=350, H=2, KV=2, D=62, causal=True, window=50, sinks=5),
    "odd_step": wcase("bf16", B=2, Lq=1, Lk=2277, H=4, KV=2, D=63, gap=3, lead=1, causal=True, window=1050, sinks=5),
    "group_33": wcase("f16", Lq=2, Lk=700, H=33, KV=1, D=32, causal=True, window=80, sinks=3),
    "ranges": wcase("bf16", Lq=140, Lk=3500, H=8, KV=8, D=128, causal=True, window=1500, sinks=4),
    "ranges_f32": wcase("f32", Lq=260, Lk=1800, H=6, KV=6, D=30, order="cache", gap=2, window=700, sinks=70),
    "negative_scale": wcase("f32", Lq=20, Lk=100, H=2, D=32, scale=-0.3, window=20, causal=True),
    "large_scores": wcase("bf16", Lq=64, Lk=300, H=2, D=64, spread=30.0, window=100, sinks=3, causal=True),
}
WIDE = dict(B=23, H=12, KV=12, Lq=170, Lk=190)
WINDOWS.update({
    "wide_bf16": wcase("bf16", D=128, window=30, sinks=3, causal=True, **WIDE),
    "wide_f16": wcase("f16", D=64, window=70, **WIDE),
    "wide_f32": wcase("f32", D=64, window=33, sinks=1, causal=True, **WIDE),
    "wide_f32_128": wcase("f32", D=128, window=65, sinks=1, causal=True, **WIDE),
    "wide_cap_bf16": wcase("bf16", D=96, window=64, sinks=64, cap=50.0, spread=4.0, causal=True, **WIDE),
    "wide_slopes_bf16": wcase("bf16", D=64, window=100, slopes=True, **WIDE),
    "wide_cap_slopes_f16": wcase("f16", D=32, window=100, slopes=True, cap=30.0, causal=True, **WIDE),
    "wide_docs_bf16": wcase("bf16", D=128, window=20, docs=T.scattered, causal=True, cap=50.0, slopes=True, **WIDE),
    "wide_lengths_bf16": wcase("bf16", D=128, window=20, sinks=2, causal=True, k_lens=[(17 * i) % 191 for i in range(23)],
                               q_lens=[(13 * i) % 171 for i in range(23)], **WIDE),
})


@pytest.mark.parametrize("name", WINDOWS)
def test_window(pkg, name):
    check_window(pkg, WINDOWS[name])


HIDDEN = {
    "step": wcase("bf16", Lq=1, Lk=900, H=4, KV=2, D=128, causal=True, window=300, sinks=4),
    "steps_f32": wcase("f32", Lq=3, Lk=900, H=4, KV=2, causal=True, window=300, sinks=4),
    "prompt_f16": wcase("f16", Lq=300, Lk=900, H=4, KV=2, causal=True, window=300, sinks=4),
    "prompt_f32": wcase("f32", Lq=300, Lk=900, H=2, D=100, causal=True, window=300, sinks=4),
    "table": wcase("bf16", Lq=300, Lk=900, H=4, KV=2, causal=True, window=300, sinks=4, table=63),
    "wide": wcase("bf16", causal=True, window=20, sinks=4, **WIDE),
    "wide_f32": wcase("f32", causal=True, window=20, sinks=4, D=96, **WIDE),
}


@pytest.mark.parametrize("name", HIDDEN)
def test_window_hides_what_keys_hold(pkg, name):
    """NaN and infinities in keys that have left some or all of the windows: as if they were not there for the queries
    that do not see them, and there for those that do; the same in a sink."""
    c = HIDDEN[name]
    first = c["Lk"] - c["Lq"] - c["window"] + 1  # the first key of the first query's window

    def gone(q, k, v, more):
        k[:, 4:max(first, 4)], v[:, 4:max(first, 4)] = np.nan, np.inf
        if c["Lq"] > 20:
            v[:, first + 5 if first > 0 else 7, 0, 3] = np.inf  # seen by the first few queries
            k[:, first + 9 if first > 0 else 9, -1, 2] = np.nan
    check_window(pkg, c, gone)

    def sink(q, k, v, more):
        v[:, 2, 0, 3] = -np.inf
        v[:, 3, -1, 1] = np.nan
    check_window(pkg, c, sink)


def test_window_past_all_is_no_window(pkg):
    """A window of all keys gives the attention without one."""
    for c in (wcase("bf16", Lq=300, Lk=300, H=4, KV=2, D=128, causal=True, window=300),
              wcase("f32", Lq=1, Lk=1300, H=4, KV=2, causal=True, window=1300), wcase("f16", **dict(WIDE, B=30), D=64, window=2 ** 30)):
        q, k, v, more = T.inputs(c)
        d, m = T.upload(pkg, c, q, k, v, more)
        p, ws, scale = window_plan(pkg, c)
        T.call(p, ws, d, m)
        got = d["out"].get()
        p, ws, scale = T.make_plan(pkg, c)
        T.call(p, ws, d, m)
        want, bound, _ = R.attention(c["dtype"], q, k, v, scale, causal=c["causal"])
        assert (np.abs(got - d["out"].get()) <= 2 * bound).all()


def test_window_refuses(pkg):
    c = wcase("bf16", Lq=1, Lk=9000, H=8, KV=2, causal=True, window=5000, sinks=4)
    q, k, v, more = T.inputs(c)
    p, ws, _ = window_plan(pkg, c)
    d, m = T.upload(pkg, c, q, k, v, more)
    a = {n: x.array for n, x in d.items()}
    assert p.workspace_bytes > 0
    T.refused(pkg, "workspace", lambda: p(**a))
    T.refused(pkg, "workspace", lambda: p(**a, workspace=pkg.ops.Array(ws.buf.ptr, (p.workspace_bytes - 1,), "u8")))
    T.refused(pkg, "out is an input", lambda: p(**{**a, "out": a["q"]}, workspace=ws.array))
    assert np.all(d["out"].get() == 7.5)


# ---- attention of a batch that shares its first keys ---------------------------------------


def scase(dtype="bf16", S=100, shared_lens=None, shared_order="cache", **more):
    return dict(T.case(dtype, **more), S=S, shared_lens=shared_lens, shared_order=shared_order)


def shared_inputs(c):
    q, k, v, more = T.inputs(c)
    g = np.random.default_rng(c["seed"] + 1000)
    sk, sv = (R.round_to(g.standard_normal((c["S"], c["KV"], c["D"])), c["dtype"]) for _ in range(2))
    if c["shared_lens"] is not None:
        more["shared_lens"] = np.array(c["shared_lens"], np.int32)
    return q, k, v, sk, sv, more


def shared_want(c, q, k, v, sk, sv, more, scale, least=0.0):
    """Entry by entry, the entry's shared keys ahead of its own."""
    outs = []
    for b in range(c["B"]):
        n = int(np.clip(more["shared_lens"][b], 0, c["S"])) if "shared_lens" in more else c["S"]
        own = int(np.clip(more["k_lens"][b], 0, c["Lk"])) if "k_lens" in more else c["Lk"]
        kk, vv = (np.concatenate((x[:n], y[b, :own]))[None] for x, y in ((sk, k), (sv, v)))
        extra = {"q_lens": more["q_lens"][b:b + 1], "least": least} if "q_lens" in more else {"least": least}
        if "slopes" in more:
            extra["slopes"] = more["slopes"].astype(np.float64)
        outs.append(R.attention(c["dtype"], q[b:b + 1], kk, vv, scale, np.float64(np.float32(c["cap"])), c["causal"], **extra))
    return [np.concatenate(x) for x in zip(*outs)]


def shared_setup(pkg, c, arrays):
    q, k, v, sk, sv, more = arrays
    scale = c["D"] ** -0.5 if c["scale"] is None else c["scale"]
    p = pkg.ops.SharedAttention(c["dtype"], c["B"], c["Lq"], c["S"], c["Lk"], c["H"], c["KV"], c["D"], scale=scale, cap=c["cap"], causal=c["causal"])
    ws = R.Dev(pkg, np.full(max(p.workspace_bytes // 4, 1), np.nan), "f32")
    d, m = T.upload(pkg, c, q, k, v, more)
    order = (1, 0, 2) if c["shared_order"] == "cache" else (0, 1, 2)
    d["shared_k"], d["shared_v"] = (R.Dev(pkg, x, c["dtype"], order, c["gap"], c["lead"], np.nan) for x in (sk, sv))
    return p, ws, d, m, np.float64(np.float32(scale))


def shared_call(p, ws, d, m, stream=0):
    p(*(d[n].array for n in ("q", "shared_k", "shared_v", "k", "v", "out")), workspace=ws.array, stream=stream, **{n: x.array for n, x in m.items()})


def check_shared(pkg, c, change=None):
    arrays = shared_inputs(c)
    if change:
        change(*arrays)
    p, ws, d, m, scale = shared_setup(pkg, c, arrays)
    want, bound, written = shared_want(c, *arrays, scale)
    # the ranges' weights and their sum: a rescaling and an addition each, f32
    bound = bound + 8 * 2.0 ** -24 * np.abs(want)
    shared_call(p, ws, d, m)
    pkg.hip.synchronize()
    got = d["out"].get()
    assert d["out"].gaps_kept()
    w = written[:, :, None, None] & np.ones(got.shape, bool)
    assert np.all(got[~w] == 7.5), "rows past the sequence were written"
    got, want, bound = got[w], want[w], bound[w]
    if not np.isfinite(want).all():
        # a key whose weight is below 2^-126 of its row's largest has none in 32 bits (e^(s - max) is no normal number), so
        # that an infinity it holds may count or not: such rows are not compared
        held = np.isfinite(shared_want(c, *arrays, scale, least=2.0 ** -126)[0][w]) == np.isfinite(want)
        assert held.mean() > 0.5
        got, want, bound = got[held], want[held], bound[held]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    worst = (np.abs(got[fine] - want[fine]) / np.maximum(bound[fine], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, worst
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


SHARED = {
    "one": scase(S=1, Lq=1, Lk=1, H=1),
    "step": scase("bf16", S=900, B=5, Lq=1, Lk=70, H=8, KV=2, D=128, causal=True, k_lens=[70, 1, 33, 64, 0]),
    "step_many": scase("bf16", S=2000, B=40, Lq=1, Lk=130, H=16, KV=4, D=128, causal=True, k_lens=[1 + 3 * i for i in range(40)]),
    "step_f16": scase("f16", S=1501, B=16, Lq=1, Lk=20, H=8, KV=8, D=64, causal=True, cap=20.0),
    "step_f32": scase("f32", S=700, B=16, Lq=1, Lk=20, H=8, KV=2, D=64, causal=True, slopes=True),
    "step_f32_128": scase("f32", S=300, B=30, Lq=1, Lk=20, H=8, KV=2, D=128, causal=True),
    "step_few": scase("f16", S=2700, B=2, Lq=1, Lk=500, H=4, KV=2, D=96, causal=True, slopes=True, order="cache"),
    "step_long_own": scase("bf16", S=64, B=3, Lq=1, Lk=3000, H=8, KV=2, D=128, causal=True, order="cache"),
    "steps_of_4": scase("bf16", S=800, B=7, Lq=4, Lk=100, H=8, KV=2, D=64, causal=True, k_lens=[100, 4, 50, 2, 0, 99, 7], q_lens=[4, 4, 3, 2, 0, 1, 4]),
    "parts": scase("bf16", S=500, B=6, Lq=1, Lk=40, H=8, KV=2, D=64, causal=True, shared_lens=[0, 1, 64, 333, 500, 1000]),
    "parts_none": scase("f16", S=500, B=6, Lq=2, Lk=40, H=2, KV=2, D=64, causal=True, shared_lens=[0, -5, 0, 0, 0, 0]),
    "parts_f32_slopes": scase("f32", S=500, B=6, Lq=3, Lk=40, H=4, KV=2, D=32, causal=True, slopes=True, shared_lens=[0, 1, 64, 333, 500, 499], k_lens=[40, 3, 2, 0, 1, 30], q_lens=[3, 3, 2, 0, 3, 3]),
    "nothing": scase("bf16", S=50, B=3, Lq=2, Lk=40, H=2, D=64, causal=True, shared_lens=[0, 0, 50], k_lens=[0, 40, 0]),
    "more_queries_than_keys": scase("f32", S=20, B=3, Lq=90, Lk=30, H=2, D=32, causal=True, shared_lens=[20, 0, 7], slopes=True),
    "tail": scase("bf16", S=700, B=4, Lq=130, Lk=130, H=8, KV=2, D=128, causal=True),
    "tail_f16": scase("f16", S=333, B=3, Lq=257, Lk=257, H=4, KV=4, D=64, causal=True, cap=30.0, k_lens=[257, 100, 31], q_lens=[257, 100, 31]),
    "tail_f32": scase("f32", S=333, B=3, Lq=100, Lk=150, H=4, KV=2, D=128, causal=True, slopes=True),
    "all": scase("f32", S=289, B=9, Lq=64, Lk=64, H=6, KV=6, D=30),
    "all_bf16": scase("bf16", S=400, B=4, Lq=33, Lk=70, H=4, KV=2, D=80, shared_lens=[400, 17, 0, 399]),
    "no_own": scase("bf16", S=400, B=4, Lq=3, Lk=0, H=4, KV=2, D=64),
    "no_shared": scase("bf16", S=0, B=4, Lq=3, Lk=90, H=4, KV=2, D=64, causal=True),
    "odd_address": scase("f16", S=277, B=3, Lq=5, Lk=40, H=4, KV=2, D=64, gap=3, lead=1, causal=True),
    "rows_of_4_bytes": scase("f16", S=350, B=3, Lq=5, Lk=40, H=2, KV=2, D=62, causal=True),
    "odd_width": scase("bf16", S=350, B=20, Lq=5, Lk=40, H=2, KV=1, D=17, causal=True, shared_order="packed"),
    "packed": scase("bf16", S=350, B=20, Lq=2, Lk=40, H=4, KV=2, D=64, causal=True, shared_order="packed", order="cache"),
    "negative_scale": scase("f32", S=90, B=3, Lq=20, Lk=30, H=2, D=32, scale=-0.3, causal=True),
    "large_scores": scase("bf16", S=300, B=3, Lq=40, Lk=100, H=2, D=64, spread=30.0, causal=True),
    "group_33": scase("f16", S=500, B=2, Lq=2, Lk=70, H=33, KV=1, D=32, causal=True),
    "batch_of_one": scase("bf16", S=500, B=1, Lq=1, Lk=70, H=8, KV=2, D=128, causal=True),
    "wide": scase("bf16", S=190, B=40, Lq=40, Lk=50, H=12, KV=12, D=128, causal=True),
    "wide_f32": scase("f32", S=190, B=40, Lq=40, Lk=50, H=12, KV=12, D=64, slopes=True, causal=True),
    "wide_cap_f16": scase("f16", S=190, B=40, Lq=40, Lk=50, H=12, KV=12, D=96, cap=50.0, spread=4.0),
}


@pytest.mark.parametrize("name", SHARED)
def test_shared(pkg, name):
    check_shared(pkg, SHARED[name])


SHARED_HIDDEN = {
    "step": scase("bf16", S=300, B=5, Lq=1, Lk=40, H=8, KV=2, D=128, causal=True, shared_lens=[0, 200, 100, 1, 250]),
    "steps_f32": scase("f32", S=300, B=5, Lq=3, Lk=40, H=4, KV=2, D=64, causal=True, shared_lens=[0, 200, 100, 1, 250]),
    "few_f16": scase("f16", S=300, B=2, Lq=1, Lk=40, H=4, KV=2, D=64, causal=True, shared_lens=[0, 200]),
    "tail": scase("bf16", S=300, B=4, Lq=100, Lk=100, H=4, KV=2, D=64, causal=True, shared_lens=[0, 200, 100, 250]),
    "all_f32": scase("f32", S=300, B=4, Lq=100, Lk=100, H=4, KV=2, D=100, shared_lens=[0, 200, 100, 250]),
    "wide_f16": scase("f16", S=300, B=40, Lq=40, Lk=50, H=12, KV=12, D=64, causal=True, shared_lens=[(7 * i) % 260 for i in range(40)]),
}


@pytest.mark.parametrize("name", SHARED_HIDDEN)
def test_shared_hides_what_keys_hold(pkg, name):
    """NaN and infinities in shared keys that no entry, or only some, have a part of."""
    def past(q, k, v, sk, sv, more):
        sk[260:], sv[260:] = np.nan, np.inf
        sv[150, 0, 3], sv[151, 1, 5], sk[180, 1, 0] = np.inf, np.nan, np.nan  # seen where the part is longer
    check_shared(pkg, SHARED_HIDDEN[name], past)


def test_shared_is_the_attention_of_whole_keys(pkg):
    """The same batch with every entry's keys laid out whole, through the attention without sharing."""
    c = scase("bf16", S=600, B=6, Lq=3, Lk=50, H=8, KV=2, D=64, causal=True)
    arrays = shared_inputs(c)
    p, ws, d, m, scale = shared_setup(pkg, c, arrays)
    shared_call(p, ws, d, m)
    got = d["out"].get()
    q, k, v, sk, sv, _ = arrays
    whole = {n: np.concatenate((np.broadcast_to(s, (6,) + s.shape), x), 1) for n, s, x in (("k", sk, k), ("v", sv, v))}
    big = T.case("bf16", B=6, Lq=3, Lk=650, H=8, KV=2, D=64, causal=True)
    plan, ws2, _ = T.make_plan(pkg, big)
    d2, m2 = T.upload(pkg, big, q, whole["k"], whole["v"], {})
    T.call(plan, ws2, d2, m2)
    _, bound, _ = R.attention("bf16", q, whole["k"], whole["v"], scale, causal=True)
    assert (np.abs(got - d2["out"].get()) <= 2.01 * bound).all()


def test_shared_refuses(pkg):
    c = scase("bf16", S=900, B=5, Lq=1, Lk=70, H=8, KV=2, D=128, causal=True)
    p, ws, d, m, _ = shared_setup(pkg, c, shared_inputs(c))
    a = {n: x.array for n, x in d.items()}
    A = pkg.ops.Array
    host = np.zeros(64, np.float32)
    T.refused(pkg, "workspace", lambda: p(**a))
    T.refused(pkg, "workspace", lambda: p(**a, workspace=A(ws.buf.ptr, (p.workspace_bytes - 1,), "u8")))
    w = dict(workspace=ws.array)
    T.refused(pkg, "out is an input", lambda: p(**{**a, "q": a["out"]}, **w))
    T.refused(pkg, "out is an input", lambda: p(**{**a, "shared_v": A(a["out"].ptr, (900, 2, 128), "bf16")}, **w))
    T.refused(pkg, "shared_k is null", lambda: p(**{**a, "shared_k": A(0, (900, 2, 128), "bf16")}, **w))
    T.refused(pkg, "shared_v is not device memory", lambda: p(**{**a, "shared_v": A(host.ctypes.data, (900, 2, 128), "bf16")}, **w))
    T.refused(pkg, "shared_lens is not device memory", lambda: p(**a, **w, shared_lens=A(host.ctypes.data, (5,), "i32")))
    T.refused(pkg, "2.22", lambda: p(**{**a, "shared_k": A(a["shared_k"].ptr, (900, 2, 128), "bf16", (1 << 23, 128, 1))}, **w))
    T.refused(pkg, "stride", lambda: p(**{**a, "shared_k": A(a["shared_k"].ptr, (900, 2, 128), "bf16", (-128, 128, 1))}, **w))
    assert np.all(d["out"].get() == 7.5)


# ---- infinities that a step sees -----------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("op", ["attention", "window", "shared"])
@pytest.mark.parametrize("keys", [120, 2000])
def test_steps_see_infinities(pkg, dtype, op, keys):
    """An infinity of v in the middle of what a step reads is infinite in its channel and nowhere else; one of either
    sign is NaN."""
    H, KV, D = 4, 2, 64
    sizes = dict(B=2, Lq=1, Lk=keys, H=H, KV=KV, D=D, causal=True, order="cache")

    def put(v):
        v[..., keys // 2, 0, 3], v[..., keys // 2 + 1, 1, 9], v[..., 70, 1, 5], v[..., keys - 60, 1, 5] = np.inf, -np.inf, np.inf, -np.inf
    if op == "shared":
        check_shared(pkg, scase(dtype, S=keys, **dict(sizes, Lk=50)), lambda q, k, v, sk, sv, more: put(sv))
        check_shared(pkg, scase(dtype, S=50, **sizes), lambda q, k, v, sk, sv, more: put(v))
    elif op == "window":
        check_window(pkg, wcase(dtype, window=keys - 3, sinks=1, **sizes), lambda q, k, v, more: put(v))
    else:
        T.check_attention(pkg, T.case(dtype, **sizes), lambda q, k, v, more: put(v))


# ---- every way over shared keys ---------------------------------------------------------------

WAYS = {
    # 17 to 32 columns an entry beside the shared keys' ranges: f32 always, 16-bit types from many keys times entries on
    "f32_24": scase("f32", S=500, B=7, Lq=24, Lk=50, H=6, KV=6, D=30, causal=True, slopes=True),
    "f32_20_128": scase("f32", S=300, B=5, Lq=5, Lk=70, H=8, KV=2, D=128, causal=True, q_lens=[5, 0, 3, 5, 1], k_lens=[70, 9, 64, 65, 0]),
    "f32_32_part": scase("f32", S=400, B=6, Lq=16, Lk=40, H=4, KV=2, D=64, shared_lens=[0, 400, 64, 1, 333, 65], cap=20.0),
    "bf16_32_many": scase("bf16", S=3100, B=64, Lq=8, Lk=20, H=16, KV=4, D=64, causal=True),
    "f16_17_many": scase("f16", S=3100, B=64, Lq=17, Lk=20, H=4, KV=4, D=32, causal=True, shared_lens=[(97 * i) % 3200 for i in range(64)]),
    # ranges of whole keys
    "whole_ranges": scase("bf16", S=1500, B=3, Lq=20, Lk=200, H=8, KV=4, D=64, causal=True),
    "whole_ranges_part": scase("f16", S=900, B=4, Lq=40, Lk=300, H=4, KV=2, D=96, causal=True, shared_lens=[0, 900, 100, 449], k_lens=[300, 20, 0, 100], q_lens=[40, 20, 0, 33]),
    "whole_ranges_own": scase("f32", S=10, B=2, Lq=40, Lk=1900, H=4, KV=2, D=64, causal=True, order="cache"),
    "whole_general": scase("bf16", S=1500, B=3, Lq=1, Lk=200, H=8, KV=4, D=64, causal=True, scale=-0.1, slopes=True),
    "whole_odd": scase("bf16", S=1500, B=3, Lq=1, Lk=200, H=8, KV=4, D=63, causal=True, gap=3, lead=1, slopes=True),
    # steps in ranges, rows of 4-byte multiples, waves of 16 and of 32 columns over the shared keys
    "step_30_f32": scase("f32", S=1500, B=9, Lq=1, Lk=200, H=6, KV=6, D=30, causal=True),
    "step_30_f32_many": scase("f32", S=1100, B=270, Lq=1, Lk=20, H=2, KV=2, D=30, causal=True),
    "step_62_f16": scase("f16", S=1100, B=70, Lq=1, Lk=80, H=8, KV=2, D=62, causal=True, cap=30.0),
    "step_300_columns": scase("bf16", S=1100, B=75, Lq=1, Lk=80, H=8, KV=2, D=128, causal=True, k_lens=[i % 81 for i in range(75)]),
    "no_shared_long": scase("bf16", S=0, B=4, Lq=1, Lk=900, H=8, KV=2, D=64, causal=True),
    "no_own_step": scase("f16", S=1500, B=4, Lq=1, Lk=0, H=8, KV=2, D=64, causal=True),
    "step_nine_tiles": scase("bf16", S=505, B=3, Lq=1, Lk=10, H=8, KV=2, D=64, causal=True),
}


@pytest.mark.parametrize("name", WAYS)
def test_shared_ways(pkg, name):
    check_shared(pkg, WAYS[name])


@pytest.mark.parametrize("name", ["f32_24", "bf16_32_many", "whole_ranges", "step_30_f32_many", "step_300_columns"])
def test_shared_ways_hide_what_keys_hold(pkg, name):
    c = dict(WAYS[name])
    S, B = c["S"], c["B"]
    c["shared_lens"] = [(S - 90) * i // (B - 1) for i in range(B)]

    def past(q, k, v, sk, sv, more):
        sk[S - 80:], sv[S - 70:] = np.nan, -np.inf
        sv[S // 2, 0, 3], sv[S // 2 + 1, -1, 5], sk[S // 2 + 70, -1, 0] = np.inf, np.nan, np.nan
    check_shared(pkg, c, past)


# ---- calls at the edges ------------------------------------------------------------------------


@pytest.mark.parametrize("L", [1, 3, 50])
def test_norm_rotary_lengths_of_any_size(pkg, L):
    """Lengths past the tokens write them all, negative ones none, at an int's ends too."""
    lens = [2 ** 31 - 1, -2 ** 31, 2, 0, 2 ** 31 - 1, -1, L]
    turned(pkg, "bf16", 7, L, 3, 2, 64, (16, 16), lens=lens)
    turned(pkg, "f32", 7, L, 3, 2, 31, (5,), lens=lens, adjacent=True)


def test_norm_rotary_strides_past_32_bits(pkg):
    """Tokens, heads and batch entries 3 GB apart."""
    D, g = 16, np.random.default_rng(2)
    x, w = R.round_to(g.standard_normal((2, 2, 2, D)), "f16"), np.ones(D, np.float32)
    pos = R.Dev(pkg, g.integers(0, 100, (2, 2, 1)).astype(np.int32), "f32", whole=True)
    dw, plain, rot, A = R.Dev(pkg, w, "f32"), R.Dev(pkg, x, "f16"), pkg.ops.NormRotary.of((8,)), pkg.ops.Array
    rot(plain.array, pos.array, dw.array)
    want, far, vp = plain.get(), (3 << 30) // 2, C.c_void_p
    for strides in ((far, D, 2 * D, 1), (2 * D, far, D, 1), (4 * D, 2 * D, far, 1)):
        buf = pkg.hip.DeviceBuffer((far + 8 * D) // 2)
        places = [(b, t, h, (b * strides[0] + t * strides[1] + h * strides[2]) * 2) for b in (0, 1) for t in (0, 1) for h in (0, 1)]
        for b, t, h, at in places:
            row = np.ascontiguousarray(R.to_bits(x[b, t, h], "f16"))
            assert pkg.hip.rt().hipMemcpy(vp(buf.ptr + at), row.ctypes.data_as(vp), row.nbytes, 1) == 0
        rot(A(buf.ptr, (2, 2, 2, D), "f16", strides), pos.array, dw.array)
        for b, t, h, at in places:
            row = np.empty(D, np.uint16)
            assert pkg.hip.rt().hipMemcpy(row.ctypes.data_as(vp), vp(buf.ptr + at), row.nbytes, 2) == 0
            # (another kernel where strides pass 32 bits: two evaluations of at most the bound each, and a step of f16)
            assert np.abs(R.from_bits(row, "f16") - want[b, t, h]).max() <= 2.0 ** -10 * np.abs(want[b, t, h]).max()
        buf.free()


def test_norm_rotary_more_tokens_than_workgroups(pkg):
    """2^28 + 2^14 tokens of one pair, the batch's entries all the same: each is the first one."""
    batch, tokens = 2 ** 14 + 1, 2 ** 14
    g = np.random.default_rng(3)
    q, w = R.Dev(pkg, R.round_to(g.standard_normal((1, tokens, 1, 2)), "f16"), "f16"), R.Dev(pkg, np.array([1.0, 0.5]), "f32")
    pos = R.Dev(pkg, g.integers(0, 2 ** 31 - 1, (1, tokens, 1)).astype(np.int32), "f32", whole=True)
    out, one = pkg.hip.DeviceBuffer(batch * tokens), R.Dev(pkg, np.zeros((1, tokens, 1, 2)), "f16")
    rot, A = pkg.ops.NormRotary([0.7], [0]), pkg.ops.Array
    rot(q.array, pos.array, w.array, one.array)
    rot(A(q.array.ptr, (batch, tokens, 1, 2), "f16", (0, 2, 2, 1)), A(pos.array.ptr, (tokens, 1), "i32"), w.array,
        A(out.ptr, (batch, tokens, 1, 2), "f16"))
    pkg.hip.synchronize()
    want, got = one.bits().view(np.uint32).reshape(-1)[:tokens], out.download().view(np.uint32).reshape(batch, tokens)
    out.free()
    assert (got == want).all()


@pytest.mark.parametrize("order", [(1, 0, 2, 3), (2, 1, 0, 3), (1, 2, 0, 3), (2, 0, 1, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rotary_entries_side_by_side(pkg, order, in_place):
    """A token's entries, or a head's, next to each other: the next entry's first token lies ahead of this one's last."""
    for dtype, adjacent, D in (("bf16", False, 64), ("f32", True, 30)):
        T.ORDERS["other"] = order
        try:
            turned(pkg, dtype, 9, 7, 3, 2, D, (5, 4), adjacent=adjacent, order="other", in_place=in_place)
            turned(pkg, dtype, 3, 500, 3, 2, D, (5, 4), adjacent=adjacent, order="other", in_place=in_place, lens=[500, 13, 499])
        finally:
            del T.ORDERS["other"]


@pytest.mark.parametrize("op", ["window", "shared"])
@pytest.mark.parametrize("Lq", [1, 40])
def test_offsets_past_32_bits(pkg, op, Lq):
    """Keys 4 MiB apart: 8.8 GB from the first to the last."""
    Lk, D, stride, vp = 2100, 64, 1 << 21, C.c_void_p
    g = np.random.default_rng(1)
    q, k, v = (R.round_to(g.standard_normal(s), "bf16") for s in ((1, Lq, 2, D), (1, Lk, 1, D), (1, Lk, 1, D)))
    buf = pkg.hip.DeviceBuffer((stride * (Lk - 1) + 2 * D + 1) // 2)
    rows = np.concatenate([R.to_bits(k[0, :, 0], "bf16"), R.to_bits(v[0, :, 0], "bf16")], 1)
    for j in range(Lk):
        row = np.ascontiguousarray(rows[j])
        assert pkg.hip.rt().hipMemcpy(vp(buf.ptr + j * stride * 2), row.ctypes.data_as(vp), row.nbytes, 1) == 0
    qd, out, A = R.Dev(pkg, q, "bf16"), R.Dev(pkg, np.zeros(q.shape), "bf16"), pkg.ops.Array
    scale = np.float64(np.float32(D ** -0.5))
    if op == "window":
        kd, vd = (A(buf.ptr + off, (1, Lk, 1, D), "bf16", (0, stride, 0, 1)) for off in (0, 2 * D))
        p = pkg.ops.Attention("bf16", 1, Lq, Lk, 2, 1, D, causal=True, window=700, sinks=70)
        ws = R.Dev(pkg, np.zeros(max(p.workspace_bytes // 4, 1)), "f32")
        p(qd.array, kd, vd, out.array, workspace=ws.array)
        want, bound, _ = R.attention("bf16", q, k, v, scale, causal=True, window=700, sinks=70)
    else:
        n = Lk - 60
        sk, sv = (A(buf.ptr + off, (n, 1, D), "bf16", (stride, 0, 1)) for off in (0, 2 * D))
        kd, vd = (A(buf.ptr + off + n * stride * 2, (1, 60, 1, D), "bf16", (0, stride, 0, 1)) for off in (0, 2 * D))
        p = pkg.ops.SharedAttention("bf16", 1, Lq, n, 60, 2, 1, D, causal=True)
        ws = R.Dev(pkg, np.zeros(max(p.workspace_bytes // 4, 1)), "f32")
        p(qd.array, sk, sv, kd, vd, out.array, workspace=ws.array)
        want, bound, _ = R.attention("bf16", q, k, v, scale, causal=True)
    got = out.get()
    buf.free()
    assert (np.abs(got - want) <= bound + 8 * 2.0 ** -24 * np.abs(want)).all()


def test_strides_of_one(pkg):
    """The stride of a dimension of one counts for nothing, the shared keys' batch stride neither."""
    c = scase("bf16", S=1, B=1, Lq=1, Lk=1, H=2, KV=1, D=64)
    arrays = shared_inputs(c)
    p, ws, d, m, scale = shared_setup(pkg, c, arrays)
    want, bound, _ = shared_want(c, *arrays, scale)
    A = pkg.ops.Array
    for odd in (0, 1, (1 << 23) + 1):
        d["out"].buf.upload(np.zeros(d["out"].buf.n, np.float32))
        a = {n: A(d[n].array.ptr, d[n].array.shape, "bf16", (odd, odd, 64 if n in ("q", "out") else odd, 1)) for n in ("q", "k", "v", "out")}
        s = {n: A(d[n].array.ptr, (1, 1, 64), "bf16", (odd, odd, 1)) for n in ("shared_k", "shared_v")}
        p(a["q"], s["shared_k"], s["shared_v"], a["k"], a["v"], a["out"], workspace=ws.array)
        assert (np.abs(d["out"].get() - want) <= bound + 8 * 2.0 ** -24 * np.abs(want)).all()


def test_keys_of_all_tokens_one_row(pkg):
    """Strides of zero: one shared row and one own row for all tokens."""
    for dtype, Lq in (("bf16", 1), ("f32", 1), ("f16", 40)):
        c = scase(dtype, S=700, B=3, Lq=Lq, Lk=70, H=2, KV=2, D=64)
        q, k, v, sk, sv, more = shared_inputs(c)
        k[:], v[:], sk[:], sv[:] = k[:1, :1], v[:1, :1], sk[:1], sv[:1]
        p, ws, d, m, scale = shared_setup(pkg, c, (q, k, v, sk, sv, more))
        want, bound, _ = shared_want(c, q, k, v, sk, sv, more, scale)
        A = pkg.ops.Array
        one = [A(d[n].array.ptr, (700, 2, 64), dtype, (0, 700 * 64, 1)) for n in ("shared_k", "shared_v")]
        one += [A(d[n].array.ptr, (3, 70, 2, 64), dtype, (0, 0, 64, 1)) for n in "kv"]
        p(d["q"].array, *one, d["out"].array, workspace=ws.array)
        assert (np.abs(d["out"].get() - want) <= bound + 8 * 2.0 ** -24 * np.abs(want)).all()


def test_operators_are_deterministic(pkg):
    """The same call gives the same bits, whatever order its workgroups come in."""
    for c in (wcase("bf16", B=2, Lq=700, Lk=700, H=4, KV=2, D=64, causal=True, window=99, sinks=3),
              wcase("f16", Lq=1, Lk=20000, H=8, KV=1, D=64, order="cache", causal=True, window=9000, sinks=3)):
        d, m = T.upload(pkg, c, *T.inputs(c))
        p, ws, _ = window_plan(pkg, c)
        seen = set()
        for _ in range(6):
            T.call(p, ws, d, m)
            seen.add(d["out"].bits().tobytes())
        assert len(seen) == 1
    for c in (SHARED["step_many"], SHARED["tail"], WAYS["bf16_32_many"], WAYS["whole_ranges"]):
        p, ws, d, m, _ = shared_setup(pkg, c, shared_inputs(c))
        seen = set()
        for _ in range(6):
            shared_call(p, ws, d, m)
            seen.add(d["out"].bits().tobytes())
        assert len(seen) == 1


# ---- the operators one after another, on streams and in graphs ------------------------------------


class Tail:
    """What several views of one image do with it, in one batch: the image's tokens are normed, turned and
    attended to in a window once; then every view's tokens, normed and turned, attend to the image's keys (shared) and
    their own, and one step of one token each follows, over the views' windows."""

    def __init__(self, pkg, seed, tokens=600, views=5, own=40, heads=4, kv=2, D=64, dtype="bf16"):
        self.pkg, self.D, self.heads, self.kv, self.dtype = pkg, D, heads, kv, dtype
        self.tokens, self.views, self.own = tokens, views, own
        g = np.random.default_rng(seed)
        up = lambda v, t=dtype: R.Dev(pkg, v, t, whole=np.asarray(v).dtype == np.int32)  # noqa: E731
        rows = heads + 2 * kv
        self.x, self.y = (R.round_to(g.standard_normal((b, n, rows, D)), dtype) for b, n in ((1, tokens), (views, own)))
        self.w = [(1 + 0.2 * g.standard_normal(s)).astype(np.float32) for s in ((heads, D), (D,))]
        self.pos = [np.stack([np.arange(n) // 25, np.arange(n) % 25], 1)[None].repeat(b, 0).astype(np.int32) for b, n in ((1, tokens), (views, own))]
        self.lens = np.array([own - 7 * i for i in range(views)], np.int32)
        self.dx, self.dy, self.dw, self.dpos, self.dlens = up(self.x), up(self.y), [up(v, "f32") for v in self.w], [up(p) for p in self.pos], up(self.lens)
        zeros = lambda *s: up(np.zeros(s))  # noqa: E731
        self.tx, self.ty = zeros(1, tokens, heads + kv, D), zeros(views, own, heads + kv, D)
        self.ox, self.oy, self.last = zeros(1, tokens, heads, D), zeros(views, own, heads, D), zeros(views, 1, heads, D)
        self.turn = pkg.ops.NormRotary.of((16, 16), eps=1e-5)
        self.windows = pkg.ops.Attention(dtype, 1, tokens, tokens, heads, kv, D, causal=True, window=100, sinks=4)
        self.shared = pkg.ops.SharedAttention(dtype, views, own, tokens, own, heads, kv, D, causal=True)
        self.step = pkg.ops.Attention(dtype, views, 1, own, heads, kv, D, causal=True, window=16, sinks=2)
        self.steps = pkg.ops.SharedAttention(dtype, views, 1, tokens, own, heads, kv, D, causal=True)
        self.last2 = zeros(views, 1, heads, D)
        n = max(p.workspace_bytes for p in (self.windows, self.shared, self.step, self.steps))
        self.ws = up(np.full(n // 4 + 1, np.nan), "f32")
        self.outputs = (self.tx, self.ty, self.ox, self.oy, self.last, self.last2)

    def part(self, dev, first, n):
        """Heads first to first + n of an array, as an array."""
        size = 4 if self.dtype == "f32" else 2
        return self.pkg.ops.Array(dev.array.ptr + first * self.D * size, dev.shape[:2] + (n, self.D), self.dtype, dev.array.stride())

    def run(self, stream=0):
        H, KV, A = self.heads, self.kv, self.pkg.ops.Array
        for x, t, pos, lens in ((self.dx, self.tx, self.dpos[0], None), (self.dy, self.ty, self.dpos[1], self.dlens)):
            self.turn(self.part(x, 0, H), pos.array, self.dw[0].array, self.part(t, 0, H), k=self.part(x, H, KV), k_weight=self.dw[1].array,
                      k_out=self.part(t, H, KV), lens=lens.array if lens else None, stream=stream)
        k, v = self.part(self.tx, H, KV), self.part(self.dx, H + KV, KV)
        self.windows(self.part(self.tx, 0, H), k, v, self.ox.array, workspace=self.ws.array, stream=stream)
        sk, sv = (A(a.ptr, a.shape[1:], self.dtype, a.stride()[1:]) for a in (k, v))
        yk, yv = self.part(self.ty, H, KV), self.part(self.dy, H + KV, KV)
        self.shared(self.part(self.ty, 0, H), sk, sv, yk, yv, self.oy.array, workspace=self.ws.array, stream=stream, q_lens=self.dlens.array,
                    k_lens=self.dlens.array)
        one = self.part(self.ty, 0, H)
        q = A(one.ptr, (self.views, 1, H, self.D), self.dtype, one.stride())
        self.step(q, yk, yv, self.last.array, workspace=self.ws.array, stream=stream, k_lens=self.dlens.array)
        self.steps(q, sk, sv, yk, yv, self.last2.array, workspace=self.ws.array, stream=stream, k_lens=self.dlens.array)

    def bits(self):
        return b"".join(d.bits().tobytes() for d in self.outputs)

    def clear(self):
        for d in self.outputs:
            d.buf.upload(np.zeros(d.buf.n, np.float32))
        self.pkg.hip.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_operators_together(pkg, dtype):
    """Each stage against 64 bits from what the stage before left in memory."""
    b = Tail(pkg, 0, dtype=dtype)
    b.run()
    pkg.hip.synchronize()
    H, KV, D = b.heads, b.kv, b.D
    axis, freq = np.array(b.turn.pair_axis[:]), np.array(b.turn.inv_freq[:])
    for x, t, pos, lens in ((b.x, b.tx.get(), b.pos[0], [b.tokens]), (b.y, b.ty.get(), b.pos[1], b.lens)):
        angle = pos[..., axis] * freq
        for first, n, w in ((0, H, b.w[0]), (H, KV, b.w[1])):
            want, bound = R.norm_rotary(dtype, x[:, :, first:first + n], w, 0.0, np.float64(np.float32(1e-5)), angle, 32, False, False)
            for i, m in enumerate(lens):
                assert (np.abs(t[i, :m, first:first + n] - want[i, :m]) <= bound[i, :m]).all()
                assert not t[i, m:].any()
    tx, ty, scale = b.tx.get(), b.ty.get(), np.float64(np.float32(D ** -0.5))
    k, v = tx[:, :, H:], b.x[:, :, H + KV:]
    want, bound, _ = R.attention(dtype, tx[:, :, :H], k, v, scale, causal=True, window=100, sinks=4)
    assert (np.abs(b.ox.get() - want) <= bound).all()
    oy, last, last2 = b.oy.get(), b.last.get(), b.last2.get()
    for i, m in enumerate(b.lens):
        q, yk, yv = ty[i:i + 1, :m, :H], ty[i:i + 1, :m, H:], b.y[i:i + 1, :m, H + KV:]
        kk, vv = np.concatenate((k, yk), 1), np.concatenate((v, yv), 1)
        want, bound, _ = R.attention(dtype, q, kk, vv, scale, causal=True)
        assert (np.abs(oy[i, :m] - want[0]) <= bound[0] + 8 * 2.0 ** -24 * np.abs(want[0])).all() and not oy[i, m:].any()
        want, bound, _ = R.attention(dtype, ty[i:i + 1, :1, :H], yk, yv, scale, causal=True, window=16, sinks=2)
        assert (np.abs(last[i] - want[0]) <= bound[0]).all()
        want, bound, _ = R.attention(dtype, ty[i:i + 1, :1, :H], kk, vv, scale, causal=True)
        assert (np.abs(last2[i] - want[0]) <= bound[0] + 8 * 2.0 ** -24 * np.abs(want[0])).all()


def test_operators_together_on_streams(pkg):
    """Two runs on streams of their own, at once, are each the run on the default stream."""
    runs, want = [Tail(pkg, s) for s in (1, 2)], []
    for b in runs:
        b.run()
        pkg.hip.synchronize()
        want.append(b.bits())
        b.clear()
    streams = [T.new_stream(pkg) for _ in runs]
    for _ in range(3):
        for b, st in zip(runs, streams):
            b.run(stream=st.value)
    for st in streams:
        pkg.hip.stream_synchronize(st.value)
    assert [b.bits() for b in runs] == want
    for st in streams:
        pkg.hip.rt().hipStreamDestroy(st)


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_operators_together_captured(pkg, mode):
    """Captured in each mode: every replay, with eager work of another run between, is the eager run on the inputs of the
    moment; two graphs with workspaces of their own run at once."""
    h, vp = pkg.hip.rt(), C.c_void_p
    for name, args in {"hipStreamBeginCapture": [vp, C.c_int], "hipStreamEndCapture": [vp, C.POINTER(vp)],
                       "hipGraphInstantiate": [C.POINTER(vp), vp, vp, vp, C.c_size_t], "hipGraphLaunch": [vp, vp],
                       "hipGraphExecDestroy": [vp], "hipGraphDestroy": [vp]}.items():
        getattr(h, name).argtypes = args
    runs, other, st, two = [Tail(pkg, s) for s in (3, 4)], Tail(pkg, 5), T.new_stream(pkg), T.new_stream(pkg)
    graphs, execs = [], []
    for b in runs:
        b.run()
        pkg.hip.synchronize()
        assert h.hipStreamBeginCapture(st, mode) == 0
        b.run(stream=st.value)
        g, e = vp(), vp()
        assert h.hipStreamEndCapture(st, C.byref(g)) == 0
        assert h.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
        graphs.append(g)
        execs.append(e)
    for turn in range(4):
        want = []
        for b, e in zip(runs, execs):
            b.x = R.round_to(np.random.default_rng(10 + turn).standard_normal(b.x.shape), b.dtype)
            b.dx.buf.upload(np.frombuffer(R.to_bits(b.x, b.dtype).tobytes(), np.float32))
            b.run()
            pkg.hip.synchronize()
            want.append(b.bits())
            b.clear()
            assert h.hipGraphLaunch(e, st) == 0
            other.run()
            pkg.hip.stream_synchronize(st.value)
            pkg.hip.synchronize()
            assert b.bits() == want[-1], turn
            b.clear()
        for e, s in zip(execs, (st, two)):
            assert h.hipGraphLaunch(e, s) == 0
        for s in (st, two):
            pkg.hip.stream_synchronize(s.value)
        assert [b.bits() for b in runs] == want
    for e, g in zip(execs, graphs):
        h.hipGraphExecDestroy(e)
        h.hipGraphDestroy(g)
    for s in (st, two):
        h.hipStreamDestroy(s)


# ---- hidden keys in the kernels of large calls -------------------------------------------------

LARGE = {
    "f16": dict(dtype="f16", D=128),
    "cap_bf16": dict(dtype="bf16", D=128, cap=50.0, spread=4.0),
    "cap_f32": dict(dtype="f32", D=32, cap=50.0, spread=4.0),
    "slopes_bf16": dict(dtype="bf16", D=64, slopes=True),
    "slopes_f32": dict(dtype="f32", D=128, slopes=True),
    "cap_slopes_f16": dict(dtype="f16", D=96, slopes=True, cap=30.0),
    "rows_of_4_bytes_f32": dict(dtype="f32", D=30, slopes=True),
    "rows_of_4_bytes_f16": dict(dtype="f16", D=62, cap=30.0),
    "odd_bf16": dict(dtype="bf16", D=63, gap=1),
}


@pytest.mark.parametrize("name", LARGE)
@pytest.mark.parametrize("causal", [True, False])
def test_window_large_calls_hide_what_keys_hold(pkg, name, causal):
    def change(q, k, v, more):
        # left behind by all but the first queries, ahead of all but the last ones, and a sink
        v[:, 25, 0, 5], v[:, 30, 1, 2], k[:, 27, 2, 0] = np.nan, np.inf, np.nan
        v[:, 180, 3, 7], v[:, 1, 5, 3] = -np.inf, np.inf
    check_window(pkg, wcase(**LARGE[name], window=20, sinks=3, causal=causal, **WIDE), change)


@pytest.mark.parametrize("name", LARGE)
def test_shared_large_calls_hide_what_keys_hold(pkg, name):
    """Whole keys by waves of 32 columns: keys past an entry's part, past its own, and in the future."""
    c = dict(LARGE[name])
    cap = c.pop("slopes", False)  # (slopes leave far keys without a weight in 32 bits: gentle ones)
    c = scase(**c, B=23, S=130, Lq=70, Lk=80, H=12, KV=12, causal=True, slopes=cap, shared_lens=[5 * i for i in range(23)],
              k_lens=[80 - i for i in range(23)], q_lens=[70 - i for i in range(23)])

    def change(q, k, v, sk, sv, more):
        if "slopes" in more:
            more["slopes"] /= 64
        sk[111:], sv[115:] = np.nan, -np.inf
        sv[60, 0, 3], sv[61, 1, 5], sk[62, 2, 0] = np.inf, np.nan, np.nan
        for b in range(23):
            k[b, 80 - b:], v[b, 80 - b:] = np.nan, (np.inf, np.nan)[b % 2]
            v[b, 79 - b, 4, 1] = np.inf
    check_shared(pkg, c, change)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,pairs", [(136, 66), (144, 72), (160, 80), (200, 65), (192, 96), (256, 128), (258, 65), (300, 128)])
def test_norm_rotary_many_pairs(pkg, dtype, D, pairs):
    """More than 64 pairs, in lanes of one to eight."""
    for adjacent in (False, True):
        turned(pkg, dtype, 2, 21, 3, 1, D, (pairs - 30, 30), adjacent=adjacent, each=D % 16 == 0)
