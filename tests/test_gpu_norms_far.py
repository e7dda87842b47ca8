"""The operators' norms at the ends of the types' range, on the GPU: heads and rows of subnormal values
and of nearly the largest, whose squares and whose root's reciprocal are no normal f32."""
import numpy as np
import pytest

import test_gpu_more_ops as M
import test_gpu_ops as T

pytestmark = pytest.mark.gpu

# (the smallest is one step of f32; bf16, whose steps are 2^-133, takes the others)
FAR = (3.3e38, 1.5e38, 2.0 ** -126, 2.0 ** -128.5, 1e-39, 1e-40, 2.0 ** -149)


def far(x, dtype):
    """Tokens or rows of `x` scaled to the sizes of FAR, by their largest magnitude."""
    for n, s in enumerate(FAR):
        x[n] *= max(s, 2.0 ** -133 if dtype == "bf16" else 0.0) / np.abs(x[n]).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,adjacent", [(64, False), (30, True), (97, False), (1030, True)])
@pytest.mark.parametrize("each", [False, True])
def test_norm_rotary_heads_at_the_ends_of_the_range(pkg, dtype, D, adjacent, each):
    """Every head's norm is about one, also without an eps and where the head's own is 2^-149."""
    def change(x):
        for v in x.values():
            for b in range(2):
                far(v[b], dtype)
    M.turned(pkg, dtype, 2, 9, 3, 2, D, (5,), adjacent=adjacent, eps=0.0, change=change, each=each)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [60, 180, 177, 4096, 16400])
@pytest.mark.parametrize("e4m3", [False, True])
def test_rms_norm_rows_at_the_ends_of_the_range(pkg, dtype, cols, e4m3):
    def change(x, r):
        far(x, dtype)
        r[:len(FAR)] = 0.0
    for group in (0, 64) if e4m3 else (0,):
        T.rms_case(pkg, dtype, 8, cols, e4m3=e4m3, group=group, change=change, eps=0.0)
