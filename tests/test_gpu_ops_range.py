"""The attention operator over the range of its values, on the GPU: values far from one, and
keys that a mask hides, in every kernel that large calls take."""
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
