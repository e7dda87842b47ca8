"""Heads' norms with the rotation of one long sequence, on the GPU: past 2^29 bytes of an array."""
import numpy as np
import pytest

import ops_ref as R

pytestmark = pytest.mark.gpu

BLOCK, H, KV, D = 256, 6, 2, 128


@pytest.mark.parametrize("blocks", [511, 512, 515])
def test_norm_rotary_one_long_sequence(pkg, blocks):
    """256 f32 tokens again and again, q's 131072 of them 2^29 bytes (each 8 heads of 128, k behind q): as one
    sequence they are what they are as two and as steps, to the bit, and the first ones right against 64 bits."""
    tokens, width = blocks * BLOCK, (H + KV) * D
    g = np.random.default_rng(5)
    x = R.round_to(g.standard_normal((BLOCK, H + KV, D)), "f32").astype(np.float32)
    w = (1 + 0.3 * g.standard_normal(D)).astype(np.float32)
    place = g.integers(0, 4096, (BLOCK, 2)).astype(np.int32)
    A = pkg.ops.Array
    src, dst = pkg.hip.DeviceBuffer(tokens * width), pkg.hip.DeviceBuffer(tokens * width)
    src.upload(np.tile(x.reshape(-1), blocks))
    dw, dpos = R.Dev(pkg, w, "f32"), R.Dev(pkg, np.tile(place, (blocks, 1)), "f32", whole=True)
    rot = pkg.ops.NormRotary.of((32, 32))

    def run(batch, n):
        dst.upload(np.full(tokens * width, np.nan, np.float32))
        strides = (n * width, width, D, 1)
        q, k, qo, ko = (A(b.ptr + 4 * at * D, (batch, n, h, D), "f32", strides)
                        for b in (src, dst) for at, h in ((0, H), (H, KV)))
        rot(q, A(dpos.array.ptr, (batch, n, 2), "i32"), dw.array, qo, k=k, k_weight=dw.array, k_out=ko)
        pkg.hip.synchronize()
        return dst.download().view(np.uint32).reshape(blocks, BLOCK, H + KV, D)

    whole = run(1, tokens)
    assert (whole == whole[0]).all()
    angle = place[:, np.array(rot.pair_axis[:])].astype(np.float64) * np.array(rot.inv_freq[:])
    want, bound = R.norm_rotary("f32", x[None].astype(np.float64), w, 0.0, np.float64(np.float32(1e-6)), angle[None], 64, False, False)
    assert (np.abs(whole[0].view(np.float32) - want[0]) <= bound[0]).all()
    assert np.array_equal(whole, run(tokens, 1))
    if blocks % 2 == 0:
        assert np.array_equal(whole, run(2, tokens // 2))
    else:
        assert np.array_equal(whole[0], run(blocks, BLOCK)[0])
    src.free()
    dst.free()
