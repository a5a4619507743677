"""Attention over the 4-bit cache with sinks and drafted trees where keys or values that
were written held a NaN or an infinity: cache4_write marks such a block with its scale and
leaves its codes zero, and every row that sees it reads NaN there, in each form of the
kernel.  Against the definition in 64 bits, at the tolerances of test_gpu_mask4."""
import math

import numpy as np
import pytest

from test_gpu_decode4 import DTYPES, HEAD_DIMS, tables
from test_gpu_mask4 import check, drafted, paths, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("part", ["k", "v"])
@pytest.mark.parametrize("group,news,bound", [
    (1, [3, 2], None),                      # few rows
    (8, [70, 40], None),                    # many
    (8, [16, 9], 1 << 20)])                 # even shares
def test_written_nan_and_infinity(gpu, dtype, dh, part, group, news, bound):
    from qppocr_amd import ops
    rng = np.random.default_rng(dh + group)
    t = getattr(gpu, dtype)
    page, lens = 16, [300, 130]
    pages = 30
    c = ops.cache4(pages, page, 1, dh)
    table = tables(rng, pages, page, lens)
    context = [n - m for n, m in zip(lens, news)]
    trees = [paths(drafted(rng, n, 5)) for n in news]
    # a token that the window hides, one that it shows, one of the first, and a drafted one
    marks = [(0, 100, 0, math.nan), (0, 4, dh - 1, math.inf), (1, context[1] + 1, dh // 2, -math.inf)]
    for b, n in enumerate(lens):
        pos = np.arange(n)
        slots = np.array(table[b])[pos // page] * page + pos % page
        kv = rng.standard_normal((2, n, 1, dh))
        for at, j, d, x in marks:
            if at == b:
                kv["kv".index(part), j, 0, d] = x
        kv = gpu.from_numpy(kv.astype(np.float32)).cuda().to(t)
        ops.cache4_write(c, kv[0], kv[1], gpu.from_numpy(slots.astype(np.int64)).cuda())
    s = (c.k_scales if part == "k" else c.v_scales).cpu().numpy()
    assert (s == 255).sum() == len(marks)
    q = queries(gpu, rng, sum(news), group, dh, dtype)
    print("written NaN", dtype, dh, part, group, news, flush=True)
    # (a window of 40 behind 3 first tokens sees neither of sequence 0's two)
    for tr, window, sinks, whole in ((trees, 0, 0, True), (trees, 40, 3, False), (None, 40, 3, False),
                                     (None, 40, 5, True)):
        y, lse = check(gpu, c, q, table, lens, news, window, sinks, tr, max_len=bound)
        bad = np.isnan(y).any(axis=(1, 2))
        assert bad[:news[0]].all() if whole else not bad[:news[0]].any()
        want = [see[1] for see in trees[1]] if tr is not None else [i >= 1 for i in range(news[1])]
        assert (bad[news[0]:] == want).all()
        assert (np.isnan(lse).any(axis=1) == (bad if part == "k" else False)).all()
