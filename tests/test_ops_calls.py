"""Calls of the transformer operators at the edges of their sizes, without a GPU."""
import pytest

from test_ops import arr, plan, tensors


def test_attention_of_no_batch_entry_with_documents(pkg):
    """No batch entry: done without a device, also where documents that the batch shares stand beside an array of none."""
    p = plan(pkg, batch=0)
    p(arr(pkg, (0, 5, 4, 64)), arr(pkg, (0, 7, 2, 64)), arr(pkg, (0, 7, 2, 64)), arr(pkg, (0, 5, 4, 64)),
      q_docs=arr(pkg, (5,), "i32"), k_docs=arr(pkg, (0, 7), "i32", ptr=0))


@pytest.mark.parametrize("name", ["res", "sum", "out", "x"])
@pytest.mark.parametrize("shape", [(4,), (1, 4, 8), ()])
def test_rms_norm_dimensions_refused(pkg, name, shape):
    """Arrays that are no rows and columns raise the library's error, as other wrong shapes do."""
    a = dict(x=arr(pkg, (4, 8), "f32"), out=arr(pkg, (4, 8), "f32", ptr=8192))
    a[name] = arr(pkg, shape, "f32", ptr=16384)
    with pytest.raises(pkg.S2SError, match=name):
        pkg.ops.rms_norm(weight=arr(pkg, (8,), "f32"), **a)


@pytest.mark.parametrize("big", [1.1e30, 3e38, -3e38])
def test_attention_numbers_past_their_products_refused(pkg, big):
    """A scale or cap whose product with log2(e) or with a score of one overflows would give NaN."""
    for more, word in ((dict(scale=big), "the scale"), (dict(cap=abs(big)), "the cap")):
        with pytest.raises(pkg.S2SError, match=word):
            plan(pkg, **more)(**tensors(pkg))


def test_attention_document_tiles_past_a_launch_refused(pkg):
    """The last counts of key tiles below 2^26, whose last workgroup would be the launch's 2^24th."""
    b, nk = 24573, 32 * 2731
    assert b * (nk // 32) == 2 ** 26 - 1
    p = plan(pkg, dtype="f32", batch=b, q_tokens=17, k_tokens=nk, q_heads=1, k_heads=1, width=100)
    a = [arr(pkg, (b, n, 1, 100), "f32", strides=(0, 100, 100, 1)) for n in (17, nk, nk, 17)]
    with pytest.raises(pkg.S2SError, match="documents"):
        p(*a, q_docs=arr(pkg, (17,), "i32"), k_docs=arr(pkg, (nk,), "i32"))
