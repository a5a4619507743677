"""cache4_move at the most tokens that one launch takes, one before and one past them."""
import numpy as np
import pytest

from test_gpu_decode4 import HEAD_DIMS, make_cache
from test_gpu_step4 import check_move

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("past", [-1, 0, 1])
def test_the_border_of_one_launch(gpu, dh, past):
    rng = np.random.default_rng(dh)
    tokens = 4096 * 32 // dh + past
    pages = tokens // 64 + 2
    c = make_cache(gpu, rng, pages, 64, 2, dh)
    slots = rng.permutation(pages * 64)[:tokens]
    print("move", dh, tokens, flush=True)
    check_move(gpu, c, slots.tolist(), np.roll(slots, 1).tolist(), "a cycle")
    check_move(gpu, c, list(range(1, tokens)), list(range(tokens - 1)), "one place down")
