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
