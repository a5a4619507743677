"""Attention over the 4-bit cache with sinks and drafted trees at the borders of what one
launch takes, against the definition in 64 bits (tolerances: test_gpu_mask4)."""
import numpy as np
import pytest

from test_gpu_decode4 import DTYPES, close, half_step, host, make_cache, numbers
from test_gpu_mask4 import attend, drafted, paths, queries, visible, words_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tree", [False, True])
def test_more_sequences_than_eight_waves_each_can_be_launched_for(gpu, dtype, tree):
    """1100000 sequences of 8 heads with up to 240 rows a head: 8.8 million workgroups, which
    eight waves each would make 4.5 10^9 threads, past the 2^32 of a launch.  All sequences
    but three are empty; those are computed whole."""
    from qppocr_amd import ops
    rng = np.random.default_rng(3)
    batch, heads, group, dh, page = 1100000, 8, 4, 32, 16
    c = make_cache(gpu, rng, 6, page, heads, dh)
    at, news, lens = (0, 555555, batch - 1), (50, 7, 33), (90, 50, 40)
    table = np.full((batch, 6), -1, dtype=np.int32)
    ln, n = np.zeros(batch, dtype=np.int32), np.zeros(batch, dtype=np.int32)
    for b, m, l in zip(at, news, lens):
        table[b], ln[b], n[b] = rng.permutation(6), l, m
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    q = queries(gpu, rng, sum(news), heads * group, dh, dtype)
    trees = [paths(drafted(rng, m, 4)) for m in news]
    def dev(x):
        return gpu.from_numpy(x).cuda()
    kw = dict(starts=dev(starts), max_new=60, lse=True)
    window, sinks = (0, 0) if tree else (15, 5)
    print("launch", dtype, tree, flush=True)
    if tree:
        bits = np.concatenate([words_of(t, 1) for t in trees])
        y, s = ops.attention_tree4(q, c, dev(table), dev(ln), dh ** -0.5, dev(bits), **kw)
    else:
        y, s = ops.attention_cache4(q, c, dev(table), dev(ln), dh ** -0.5, window=window, sinks=sinks, **kw)
    y, s, qd = host(y), host(s), host(q)
    k, v = numbers(c)
    terms = {"float32": 3, "float16": 2, "bfloat16": 1}[dtype]
    row = 0
    for b, m, l, t in zip(at, news, lens, trees):
        pos = np.arange(l)
        pg = table[b].astype(np.int64)[pos // page]
        for i in range(m):
            see = visible(l, m, i, True, window, sinks, t if tree else None)
            want, tol, (lse, ltol) = attend(qd[row], k[pg[see], pos[see] % page], v[pg[see], pos[see] % page],
                                            dh ** -0.5, terms, group)
            close(y[row], want, tol + half_step(gpu, q.dtype, want) * 1.001, f"row {b} {i}")
            close(s[row], lse, ltol, f"lse {b} {i}")
            row += 1
