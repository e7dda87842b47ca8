"""What the built library holds of the attention's kernels: those that a call can reach."""
import re
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent.parent / "swin2sr-rs_amd" / "libswin2sr_hip.so"


def attention_kernels():
    """(width, column blocks a wave, few columns, alignment, mode) of every k_attn that the library names."""
    if not LIB.exists():
        pytest.skip("the library is not built")
    name = rb"6k_attnI(?:f|DF16_|DF16b|Dh|u6__bf16)Li(\d+)ELi(\d)ELb([01])ELi(\d+)ELi(\d+)E"
    return {tuple(int(x) for x in m) for m in re.findall(name, LIB.read_bytes())}


def test_wide_waves_are_of_known_masks():
    """Waves of 32 columns take arrays of 16-byte multiples with the cap and slopes compiled in (modes 0 to 3) or
    documents of heads over 64 wide (24); those that ask in every tile (8) are the windows' and the shared prefix's, of
    4-byte multiples."""
    wide = {k for k in attention_kernels() if k[1] == 2}
    assert {k[4] for k in wide} >= {0, 1, 2, 3, 24}
    for dp, _, few, align, mode in wide:
        kind, of = mode & 63, mode & ~63
        assert not few
        if align == 16:
            assert kind in (0, 1, 2, 3) or (kind == 24 and of in (0, 64) and dp > 64), (dp, align, mode)
        else:
            assert align == 4 and kind == 8 and of in (64, 256), (dp, align, mode)
