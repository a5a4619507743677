"""How many tokens cache4_move moves in one launch, without a workspace: 4096 blocks of 32
elements of a head (no GPU)."""
import ctypes

import pytest

from test_decode4_host import cache, lib  # noqa: F401


@pytest.mark.parametrize("dh", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads", [1, 8])
def test_the_border_of_one_launch(lib, dh, heads):  # noqa: F811
    c, n = ctypes.byref(cache(dh=dh, heads=heads)), ctypes.c_size_t(1)
    most = 4096 * 32 // dh
    assert lib.qph_cache4_move_workspace(c, most, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.qph_cache4_move_workspace(c, most + 1, ctypes.byref(n)) == 0
    assert n.value == (most + 1) * 2 * heads * (dh // 32) * 17
