"""Attention over the 4-bit cache with sinks and drafted trees where a head has more
rows than a few workgroups' own: the form in which waves share a tile's operands.
Against the definition in 64 bits, at the tolerances of test_gpu_mask4."""
import math

import numpy as np
import pytest

from test_gpu_decode4 import DTYPES, HEAD_DIMS, close, half_step, host, make_cache, numbers
from test_gpu_mask4 import attend, check, drafted, paths, queries, setup, visible, words_of

pytestmark = pytest.mark.gpu


def some(news, each=9):
    """Pairs (sequence, new token): the ends of a sequence's tokens and some between."""
    return [(b, i) for b, n in enumerate(news) for i in sorted({*range(0, n, max(1, n // each)), n - 1} if n else ())]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("heads,group,news,context,window,sinks,tree", [
    (1, 8, [33, 1, 0, 12], [100, 0, 40, 31], 0, 0, True),     # 264 rows; idle waves; no context
    (2, 3, [100, 87], [333, 1], 0, 0, True),                  # heads and tokens end inside a tile
    (1, 1, [300, 257], [31, 700], 0, 0, True),                # several words, several row tiles
    (1, 5, [64, 60], [64, 200], 17, 3, True),
    (1, 4, [129, 65], [500, 3], 40, 35, False),
    (1, 2, [140, 150], [0, 90], 1, 1, False),
    (1, 7, [40, 38], [260, 9], 100, 1000, False)])
def test_shapes(gpu, dtype, dh, heads, group, news, context, window, sinks, tree):
    print("many rows", dtype, dh, heads, group, news, context, window, sinks, tree, flush=True)
    rng = np.random.default_rng(dh + sum(news) + group)
    lens = [a + b for a, b in zip(context, news)]
    c, table = setup(gpu, rng, lens, heads, dh, 16)
    trees = [paths(drafted(rng, n, 5)) for n in news] if tree else None
    check(gpu, c, queries(gpu, rng, sum(news), heads * group, dh, dtype), table, lens, news, window, sinks, trees,
          rows=some(news, 20), causal=group != 7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [64, 128, 192])
@pytest.mark.parametrize("heads,lens,news,group", [
    (1, [9000, 300], [40, 41], 8),                            # many splits, several rows a wave join them
    (1, [20000], [34], 8),                                    # many splits, few rows
    (2, [3000, 0, 2111], [90, 3, 77], 4)])
def test_splits(gpu, dtype, dh, heads, lens, news, group):
    """Keys that workgroups share, bounds too small and too large; the same bits again."""
    rng = np.random.default_rng(dh + sum(lens))
    c, table = setup(gpu, rng, lens, heads, dh, 64)
    q = queries(gpu, rng, sum(news), heads * group, dh, dtype)
    trees = [paths(drafted(rng, n, 4)) for n in news]
    rows, got = some(news, 4), []
    for bound, tr, window, sinks in ((max(lens), trees, 0, 0), (500, trees, 0, 0), (1 << 20, trees, 0, 0),
                                     (max(lens), None, 2500, 600), (max(lens), trees, 1030, 5),
                                     (max(lens), trees, 0, 0)):
        print("splits", dtype, dh, lens, bound, window, sinks, flush=True)
        got.append(check(gpu, c, q, table, lens, news, window, sinks, tr, max_len=bound, rows=rows))
    assert (got[0][0] == got[-1][0]).all() and (got[0][1] == got[-1][1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 96, 128, 192])
@pytest.mark.parametrize("low,high", [(96, 106), (138, 143), (27, 30)])
def test_scales_past_float16(gpu, dtype, dh, low, high):
    """Values, then keys, with scales that float16 does not hold in a few rows, blocks of
    zeros with the smallest scale among ordinary ones, and both in places that no row
    sees."""
    rng = np.random.default_rng(dh + low)
    lens, news, group = [230, 400], [70, 40], 8
    for part in ("v_scales", "k_scales"):
        c, table = setup(gpu, rng, lens, 1, dh, 32)
        s = getattr(c, part)
        for b, keys in ((0, (3, 100, 228)), (1, (40, 399))):
            for j in keys:
                s[table[b][j // 32], :, j % 32] = gpu.from_numpy(
                    rng.integers(low, high, (1, dh // 32)).astype(np.uint8)).cuda()
        codes = getattr(c, part.replace("scales", "codes"))
        for b, j in ((0, 17), (1, 111), (1, 112)):
            codes[table[b][j // 32], :, j % 32], s[table[b][j // 32], :, j % 32] = 0, 27
        s[table[0][7], :, 6:] = 255                            # behind the last token
        q = queries(gpu, rng, sum(news), group, dh, dtype)
        trees = [paths(drafted(rng, n, 5)) for n in news]
        print("scales", dtype, dh, low, part, flush=True)
        check(gpu, c, q, table, lens, news, trees=trees, rows=some(news))
        check(gpu, c, q, table, lens, news, 60, 50, rows=some(news))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 96, 128, 192])
def test_nan_stays_with_its_rows(gpu, dtype, dh):
    rng = np.random.default_rng(6 + dh)
    page, news, lens, group = 16, [66, 5], [150, 40], 8
    c, table = setup(gpu, rng, lens, 1, dh, page)
    for s in (c.k_scales, c.v_scales):
        s[table[0][9], :, 6:], s[table[1][2], :, 8:] = 255, 255
    for s, b, j, block in ((c.k_scales, 0, 104, 0), (c.v_scales, 0, 117, dh // 32 - 1), (c.v_scales, 1, 37, 0)):
        s[table[b][j // page], 0, j % page, block] = 255
    trees = [paths(drafted(rng, n, 6)) for n in news]
    q = queries(gpu, rng, sum(news), group, dh, dtype)
    print("NaN", dtype, dh, flush=True)
    y, _ = check(gpu, c, q, table, lens, news, trees=trees)
    bad = np.isnan(y).any(axis=(1, 2))
    assert (bad == [*(t[20] | t[33] for t in trees[0]), *(t[2] for t in trees[1])]).all()
    check(gpu, c, q, table, lens, news, 3, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 60])
def test_scores_of_any_size(gpu, dtype, size):
    """(as in test_gpu_mask4: rows whose best key is far ahead are that key's value)"""
    from qppocr_amd import ops
    scale, big = (size, 1.0) if dtype == "float16" and size > 2.0 ** 12 else (1.0, size)
    rng = np.random.default_rng(2)
    dh, group, n, length = 64, 4, 70, 150
    c, table = setup(gpu, rng, [length], 1, dh, 32)
    q = queries(gpu, rng, n, group, dh, dtype) * big
    tree = paths(drafted(rng, n, 3))
    y = host(ops.attention_tree4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                 gpu.tensor([length], dtype=gpu.int32, device="cuda"), scale,
                                 gpu.from_numpy(words_of(tree, 2)).cuda()))
    k, v = numbers(c)
    pos = np.arange(length)
    pg = np.array(table[0])[pos // 32]
    k, v, qd = k[pg, pos % 32, 0], v[pg, pos % 32, 0], host(q)
    seen = 0
    for i in range(n):
        see = visible(length, n, i, True, 0, 0, tree)
        for g in range(group):
            s = np.where(see, k @ qd[i, g] * scale, -np.inf)
            first, second = np.sort(s)[::-1][:2]
            if first - second > 30 + 2.0 ** -16 * (np.abs(k) @ np.abs(qd[i, g])).max() * scale:
                want = v[s.argmax()]
                tol = half_step(gpu, q.dtype, want) + 2.0 ** -22 * np.abs(want) + np.exp(-20.0) * 6
                close(y[i, g], want, tol, f"row {i} {g}")
                seen += 1
    assert seen > n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,bound", [(1, 1), (4, 3), (8, 34), (1, 260)])
def test_more_new_tokens_than_the_bound(gpu, dtype, group, bound):
    """max_new only shapes the launch: sequences with more are computed whole."""
    from qppocr_amd import ops
    rng = np.random.default_rng(bound)
    news, lens, dh = [300, 2], [340, 90], 64
    c, table = setup(gpu, rng, lens, 1, dh, 32)
    q = queries(gpu, rng, sum(news), group, dh, dtype)
    tab = gpu.tensor(table, dtype=gpu.int32, device="cuda")
    ln = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    st = gpu.tensor([0, 300, 302], dtype=gpu.int32, device="cuda")
    trees = [paths(drafted(rng, n, 4)) for n in news]
    bits = np.zeros((sum(news), 5), dtype=np.int64)
    bits[:300], bits[300:] = words_of(trees[0], 5), words_of(trees[1], 5)
    print("past max_new", dtype, group, bound, flush=True)
    k, v = numbers(c)
    terms = {"float32": 3, "float16": 2, "bfloat16": 1}[dtype]
    for tr, window, sinks in ((trees, 0, 0), (None, 50, 20)):
        kw = dict(starts=st, max_new=bound, window=window, sinks=sinks, lse=True)
        y, s = (ops.attention_cache4(q, c, tab, ln, 0.125, **kw) if tr is None else
                ops.attention_tree4(q, c, tab, ln, 0.125, gpu.from_numpy(bits).cuda(), **kw))
        y, s, qd = host(y), host(s), host(q)
        for b, i in some(news, 12):
            pos = np.arange(lens[b])
            pg = np.array(table[b])[pos // 32]
            see = visible(lens[b], news[b], i, True, window, sinks, tr and tr[b])
            want, tol, (lse, ltol) = attend(qd[300 * b + i], k[pg[see], pos[see] % 32], v[pg[see], pos[see] % 32],
                                            0.125, terms, group)
            close(y[300 * b + i], want, tol + half_step(gpu, q.dtype, want) * 1.001, f"row {b} {i}")
            close(s[300 * b + i], lse, ltol, f"lse {b} {i}")


def test_bits_bad_pages_and_lengths(gpu):
    """Rows of no bits, of all and of later tokens; page numbers outside the pool; lengths
    past the table; more new tokens than cached ones."""
    rng = np.random.default_rng(5)
    page, pages = 16, 12
    c = make_cache(gpu, rng, pages, page, 2, 64)
    table = [[3, -1, 5, 7, 1, 0, 2, 6], [pages, 1, 2, 1 << 30, 4, 4, -5, 9], [8, 9, 10, 11, 0, 4, 6, -5],
             [-(1 << 31)] * 8]
    lens, news = [128, 1 << 20, 10, 80], [70, 68, 40, 66]
    for dtype in DTYPES:
        print("bad pages", dtype, flush=True)
        q = queries(gpu, rng, sum(news), 8, 64, dtype)
        trees = [rng.random((n, n)) < 0.4 for n in news]
        trees[0][2] = trees[1][:] = False
        trees[2][39] = True
        rows = some(news, 8) + [(0, 2)]
        check(gpu, c, q, table, lens, news, trees=trees, rows=rows)
        check(gpu, c, q, table, lens, news, 30, 18, trees, rows=rows)
        check(gpu, c, q, table, lens, news, 20, 18, rows=rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_and_rows_left_alone(gpu, dtype):
    from qppocr_amd import ops
    rng = np.random.default_rng(8)
    lens, news, dh, group = [300, 133], [70, 66], 64, 4
    c, table = setup(gpu, rng, lens, 2, dh, 32)
    n = sum(news)
    trees = [paths(drafted(rng, m, 3)) for m in news]
    packed = queries(gpu, rng, n + 5, 12, dh, dtype)
    q, big = packed[:, 1:9], gpu.full((n + 5, 9, dh), 7.0, device="cuda", dtype=packed.dtype)
    starts = [2, 2 + news[0], 2 + n]
    y, _ = check(gpu, c, q, table, lens, news, out=big[:, :8], trees=trees, starts=starts, rows=some(news, 4))
    for left in (big[:2], big[2 + n:], big[:, 8]):
        assert (host(left) == 7).all()
    was = host(packed.clone())
    words = gpu.zeros((n + 5, 2), dtype=gpu.int64, device="cuda")
    for b in range(2):
        words[starts[b]:starts[b + 1]] = gpu.from_numpy(words_of(trees[b], 2)).cuda()
    ops.attention_tree4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                        gpu.tensor(lens, dtype=gpu.int32, device="cuda"), dh ** -0.5, words,
                        starts=gpu.tensor(starts, dtype=gpu.int32, device="cuda"), max_new=max(news), out=q)
    got = host(packed)
    assert (got[2:2 + n, 1:9] == y[2:2 + n]).all()
    got[2:2 + n, 1:9] = was[2:2 + n, 1:9]
    assert (got == was).all()


def test_past_32_bits(gpu):
    """A pool whose bytes pass 2^32: the last pages' keys."""
    from qppocr_amd import ops
    rng = np.random.default_rng(12)
    page, heads, dh, news = 1024, 8, 256, 80
    pages = (1 << 32) // (page * heads * dh // 2) + 3
    c = ops.cache4(pages, page, heads, dh)
    last = [pages - 1, pages - 2]
    for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)):
        for p in last:
            codes[p] = gpu.from_numpy(rng.integers(0, 256, codes[p].shape, dtype=np.uint8)).cuda()
            scales[p] = gpu.from_numpy(rng.integers(121, 128, scales[p].shape).astype(np.uint8)).cuda()
    small = ops.Cache4(*(x[last].contiguous() for x in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)))
    i32 = dict(dtype=gpu.int32, device="cuda")
    for dtype in DTYPES:
        q = queries(gpu, rng, news, 32, dh, dtype)
        bits = gpu.from_numpy(words_of(paths(drafted(rng, news, 3)), 2)).cuda()
        y = [host(ops.attention_tree4(q, x, gpu.tensor([t], **i32), gpu.tensor([1500], **i32), 0.1, bits,
                                      max_len=2048)) for x, t in ((c, last), (small, [0, 1]))]
        assert (y[0] == y[1]).all() and np.isfinite(y[0]).all()


@pytest.mark.parametrize("length", [300, 30000])
def test_captured(gpu, length):
    """Two captured calls, replayed in turn and in flight together on two streams."""
    from qppocr_amd import ops
    rng = np.random.default_rng(15)
    news, pages = 80, length // 64 + 2
    c = make_cache(gpu, rng, pages, 64, 2, 128)
    table = gpu.from_numpy(rng.permutation(pages)[None].astype(np.int32)).cuda()
    lens = gpu.tensor([length], dtype=gpu.int32, device="cuda")
    qs = [gpu.zeros((news, 8, 128), device="cuda", dtype=gpu.bfloat16) for _ in range(2)]
    bits = [gpu.zeros((news, 2), dtype=gpu.int64, device="cuda") for _ in range(2)]
    graphs, outs = [], []
    for q, t in zip(qs, bits):
        ops.attention_tree4(q, c, table, lens, 0.1, t)
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(ops.attention_tree4(q, c, table, lens, 0.1, t, lse=True))
        graphs.append(g)
    side = gpu.cuda.Stream()
    for i in range(4):
        for q, t in zip(qs, bits):
            q.copy_(queries(gpu, rng, news, 8, 128, "bfloat16"))
            t.copy_(gpu.from_numpy(words_of(paths(drafted(rng, news, 3)), 2)).cuda())
        lens.fill_(length - 51 * i)
        gpu.cuda.synchronize()
        graphs[0].replay()
        with gpu.cuda.stream(side):
            graphs[1].replay()
        gpu.cuda.synchronize()
        for q, t, (y, s) in zip(qs, bits, outs):
            y2, s2 = ops.attention_tree4(q, c, table, lens, 0.1, t, lse=True)
            assert (host(y) == host(y2)).all() and (host(s) == host(s2)).all()
            assert np.isfinite(host(y)).all() and not (host(s) == -math.inf).any()


# ------------------------------------- several sequences of a row tile, even shares of their keys

EVEN = 1 << 20            # a bound for which keys are split however short the sequences are


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("heads,group,news,context,window,sinks,tree", [
    (2, 4, [31, 0, 1, 17, 9], [4000, 50, 0, 700, 2100], 0, 0, True),
    (1, 8, [16, 15, 2], [33, 2900, 0], 0, 0, True),
    (1, 3, [20, 33, 7, 1, 40], [64, 1000, 0, 31, 1900], 500, 70, True),
    (3, 1, [60, 90], [1500, 1700], 1030, 5, False),
    (1, 2, [50, 13, 64], [900, 0, 2500], 0, 0, False)])
def test_even_shares(gpu, dtype, dh, heads, group, news, context, window, sinks, tree):
    print("even", dtype, dh, heads, group, news, context, window, sinks, tree, flush=True)
    rng = np.random.default_rng(dh + sum(news) + group)
    lens = [a + b for a, b in zip(context, news)]
    c, table = setup(gpu, rng, lens, heads, dh, 32)
    trees = [paths(drafted(rng, n, 5)) for n in news] if tree else None
    q = queries(gpu, rng, sum(news), heads * group, dh, dtype)
    got = [check(gpu, c, q, table, lens, news, window, sinks, trees, rows=some(news, 5), max_len=bound,
                 causal=group != 2) for bound in (EVEN, max(lens), EVEN)]
    assert (got[0][0] == got[2][0]).all() and (got[0][1] == got[2][1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [2, 30, 64, 65])
def test_even_shares_of_short_sequences(gpu, dtype, batch):
    """Many parts to a workgroup; one long sequence among short ones; as many sequences as
    a wave has lanes, and one more."""
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0, 200, batch)]
    lens[batch // 2] = 3000
    news = [int(x) for x in rng.integers(0, 9, batch)]
    news[-1], news[batch // 2] = 20, 20
    c, table = setup(gpu, rng, lens, 1, 64, 16)
    q = queries(gpu, rng, sum(news), 8, 64, dtype)
    trees = [paths(drafted(rng, n, 5)) for n in news]
    print("short", dtype, batch, flush=True)
    check(gpu, c, q, table, lens, news, trees=trees, rows=some(news, 2), max_len=EVEN)
    check(gpu, c, q, table, lens, news, 50, 33, rows=some(news, 2), max_len=EVEN)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [64, 192])
def test_even_shares_walked_again(gpu, dtype, dh):
    """Values that float16 does not hold, NaN, and scores far from zero in some parts of a
    sequence; lengths past the table and below zero; pages outside the pool."""
    rng = np.random.default_rng(dh)
    lens, news, group = [1900, 700, 1 << 20, -5, 64], [16, 9, 12, 3, 16], 8
    c, table = setup(gpu, rng, [1900, 700, 90, 0, 64], 1, dh, 32)
    wide = max(len(t) for t in table)
    table = [t + [-1] * (wide - len(t)) for t in table]
    table[1][3] = c.pages
    for b, j, scale in ((0, 30, 145), (0, 1700, 100), (1, 400, 142), (4, 5, 103)):
        c.v_scales[table[b][j // 32], :, j % 32] = scale
    for b, j, scale in ((0, 900, 142), (1, 5, 255), (4, 50, 150)):
        c.k_scales[table[b][j // 32], :, j % 32] = scale
    c.v_scales[table[0][1890 // 32], :, 1890 % 32] = 255         # a drafted token
    q = queries(gpu, rng, sum(news), group, dh, dtype)
    trees = [paths(drafted(rng, n, 4)) for n in news]
    print("again", dtype, dh, flush=True)
    check(gpu, c, q, table, lens, news, trees=trees, max_len=EVEN)
    check(gpu, c, q, table, lens, news, 700, 31, max_len=EVEN)


@pytest.mark.parametrize("dtype", DTYPES)
def test_even_shares_past_the_bound(gpu, dtype):
    """Sequences with more new tokens than max_new, their further rows in the same parts;
    captured and replayed with other lengths."""
    from qppocr_amd import ops
    rng = np.random.default_rng(4)
    news, dh, group = [130, 20], 64, 8
    c = make_cache(gpu, rng, 80, 32, 1, dh)
    table = gpu.from_numpy(rng.permutation(80).reshape(2, 40).astype(np.int32)).cuda()
    q = queries(gpu, rng, 150, group, dh, dtype)
    trees = [paths(drafted(rng, n, 4)) for n in news]
    bits = np.zeros((150, 3), dtype=np.int64)
    bits[:130], bits[130:] = words_of(trees[0], 3), words_of(trees[1], 3)
    words = gpu.from_numpy(bits).cuda()
    st = gpu.tensor([0, 130, 150], dtype=gpu.int32, device="cuda")
    ln = gpu.tensor([1200, 900], dtype=gpu.int32, device="cuda")

    def call(bound, most=EVEN):
        return ops.attention_tree4(q, c, table, ln, 0.125, words, starts=st, max_new=bound, max_len=most, lse=True)
    call(20)
    g = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(g):
        y, s = call(20)
    terms = {"float32": 3, "float16": 2, "bfloat16": 1}[dtype]
    k, v = numbers(c)
    for lens in ([1200, 900], [131, 1280], [1280, 20]):
        ln.copy_(gpu.tensor(lens, dtype=gpu.int32))
        gpu.cuda.synchronize()
        g.replay()
        gpu.cuda.synchronize()
        y2, s2 = call(20)
        assert (host(y) == host(y2)).all() and (host(s) == host(s2)).all()
        for b, i in some(news, 8):
            pos = np.arange(lens[b])
            pg = host(table)[b].astype(np.int64)[pos // 32]
            see = visible(lens[b], news[b], i, True, 0, 0, trees[b])
            want, tol, (lse, ltol) = attend(host(q)[130 * b + i], k[pg[see], pos[see] % 32],
                                            v[pg[see], pos[see] % 32], 0.125, terms, group)
            close(host(y)[130 * b + i], want, tol + half_step(gpu, q.dtype, want) * 1.001, f"row {b} {i}")
            close(host(s)[130 * b + i], lse, ltol, f"lse {b} {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("part", ["v", "k"])
def test_numbers_below_the_smallest_normal_float16(gpu, dtype, part):
    """All values, then all keys, so small that float16 holds them below its normal
    numbers: nothing of them is lost."""
    rng = np.random.default_rng(44)
    lens, news, group, dh = [300], [70], 4, 64
    c, table = setup(gpu, rng, lens, 1, dh, 32)
    s = getattr(c, part + "_scales")
    s.copy_(gpu.from_numpy(rng.integers(104, 109, s.shape).astype(np.uint8)))
    q = queries(gpu, rng, 70, group, dh, dtype)
    trees = [paths(drafted(rng, 70, 5))]
    scale = dh ** -0.5 if part == "v" else 2.0 ** 17
    print("small", dtype, part, flush=True)
    if part == "v" and dtype == "float16":       # (the result has its own smallest number)
        q = q.float().bfloat16()
    y, _ = check(gpu, c, q, table, lens, news, trees=trees, rows=some(news, 30), scale=scale)
    assert (y != 0).any(axis=-1).all()
