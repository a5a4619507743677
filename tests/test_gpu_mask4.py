"""Attention over the 4-bit cache with first tokens that stay visible and with
drafted trees, against the definition in 64 bits (tolerances: attend_row of
test_gpu_decode4, derived at its top): lengths, windows, sinks and trees at the
borders of tiles, pages, words and splits; rows that see nothing; NaN and garbage
in places that a row does not see; bad pages; strides; graphs and streams."""
import math

import numpy as np
import pytest

from test_gpu_decode4 import (DTYPES, HEAD_DIMS, attend_row, close, half_step, host, make_cache,
                              numbers, tables)

pytestmark = pytest.mark.gpu

TERMS = {"float32": 3, "float16": 2, "bfloat16": 1}


def drafted(rng, n, spread):
    """Parents of a tree, each among the `spread` tokens before."""
    return [int(rng.integers(max(-1, i - spread), i)) for i in range(n)]


def paths(parents):
    """[n, n] truth values: token i's own path."""
    a = np.zeros((len(parents), len(parents)), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def words_of(see, words):
    """Masks of rows of truth values, int64 [rows, words]; bits past a row's tokens set
    at random would count for nothing."""
    wide = np.zeros((see.shape[0], 64 * words), dtype=bool)
    wide[:, :min(see.shape[1], 64 * words)] = see[:, :64 * words]
    return np.packbits(wide, axis=1, bitorder="little").view(np.int64)


def visible(n, news, i, causal, window, sinks, see):
    """Truth values over the keys 0 .. n - 1 of the i-th of `news` new tokens."""
    j, c = np.arange(n), n - news
    if see is None:
        p = c + i
        v = j <= p if causal else np.ones(n, dtype=bool)
    else:
        p = c - 1 + int(see[i].sum())
        v = j < c
    if window:
        v = v & ((j > p - window) | (j < sinks))
    if see is not None:
        for k in range(news):
            if 0 <= c + k < n:
                v[c + k] = see[i, k]
    return v


def check(torch, c, q, table, lens, news, window=0, sinks=0, trees=None, causal=True, max_len=None,
          starts=None, words=None, rows=None, name="mask", out=None, scale=None):
    """Runs and checks a call; table, lens, news are host lists, trees [news, news] of
    truth values a sequence.  rows: pairs (sequence, new token) to check (default: all)."""
    from qppocr_amd import ops
    scale = c.dh ** -0.5 if scale is None else scale
    terms = TERMS[str(q.dtype)[6:]]
    group = q.shape[1] // c.heads
    starts = [0] + list(np.cumsum(news)) if starts is None else starts
    kw = dict(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_new=max(news),
              max_len=max_len, window=window, sinks=sinks, lse=True, out=out)
    tab = torch.tensor(table, dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if trees is None:
        y, sums = ops.attention_cache4(q, c, tab, ln, scale, causal=causal, **kw)
    else:
        words = words or (max(news) + 63) // 64
        bits = np.zeros((q.shape[0], words), dtype=np.int64)
        for b, see in enumerate(trees):
            bits[starts[b]:starts[b] + news[b]] = words_of(see, words)
        y, sums = ops.attention_tree4(q, c, tab, ln, scale, torch.from_numpy(bits).cuda(), **kw)
    y, sums, qd = host(y), host(sums), host(q)
    k, v = numbers(c)
    page = c.page_size
    for b, n in enumerate(lens):
        n = max(0, min(n, len(table[b]) * page))
        pos = np.arange(n)
        pg = np.array(table[b] + [-1], dtype=np.int64)[pos // page] if n else np.zeros(0, np.int64)
        there = (pg >= 0) & (pg < c.pages)
        for i in range(news[b]):
            if rows is not None and (b, i) not in rows:
                continue
            see = there & visible(n, news[b], i, causal, window, sinks, None if trees is None else trees[b])
            row = starts[b] + i
            want, tol, (lse, ltol) = attend(qd[row], k[pg[see], pos[see] % page],
                                            v[pg[see], pos[see] % page], scale, terms, group)
            close(y[row], want, tol + half_step(torch, q.dtype, want) * 1.001, f"{name}: row {row} ({b}, {i})")
            close(sums[row], lse, ltol, f"{name}: lse of row {row}")
    return y, sums


def attend(q, k, v, scale, terms, group):
    """attend_row; a bfloat16 row's probabilities may be held as float16, each off by half a
    step of it, 2^-11 of itself, which the values pass on."""
    out, tol, sums = attend_row(q, k, v, scale, terms, group)
    for h in range(q.shape[0] if terms == 1 and k.shape[0] else 0):
        s = k[:, h // group] @ q[h] * scale
        p = np.exp(s - s.max())
        with np.errstate(invalid="ignore"):
            tol[h] += 2.0 ** -11 * (p / p.sum() @ np.abs(v[:, h // group]))
    return out, tol, sums


def queries(torch, rng, tokens, heads, dh, dtype):
    x = torch.from_numpy(rng.standard_normal((tokens, heads, dh)).astype(np.float32)).cuda()
    return x.to(getattr(torch, dtype))


def setup(torch, rng, lens, heads, dh, page, extra=2):
    pages = sum((max(n, 0) + page - 1) // page for n in lens) + extra
    return make_cache(torch, rng, pages, page, heads, dh), tables(rng, pages, page, lens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
def test_sinks_steps(gpu, dtype, dh):
    """One token of each sequence: windows that reach the sinks, end beside them or far
    behind, sinks at a tile's border and past the sequence."""
    rng = np.random.default_rng(dh)
    lens = [1, 0, 5, 32, 33, 64, 100, 131, 400, 900]
    for page, heads, group, window, sinks in ((16, 2, 1, 40, 4), (32, 1, 4, 1, 32), (64, 1, 7, 130, 33),
                                              (16, 1, 2, 64, 1000)):
        print("sinks step", dtype, dh, page, heads, group, window, sinks, flush=True)
        c, table = setup(gpu, rng, lens, heads, dh, page)
        check(gpu, c, queries(gpu, rng, len(lens), heads * group, dh, dtype), table, lens,
              [1] * len(lens), window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("heads,group,news,lens,causal,window,sinks", [
    (2, 4, [5, 1, 8], [90, 1, 8], True, 13, 3),             # 32 rows: two column tiles a wave
    (1, 1, [3, 7, 2], [2, 7, 0], True, 2, 1),               # more new tokens than cached ones
    (1, 16, [2, 2], [200, 31], False, 20, 5),
    (1, 2, [70, 0, 33], [300, 9, 33], True, 40, 35),        # rows of their own, gaps, odd ends
    (1, 3, [45, 60], [60, 400], False, 100, 70),
    (1, 1, [130], [500], True, 1, 1)])
def test_sinks_chunks(gpu, dtype, dh, heads, group, news, lens, causal, window, sinks):
    print("sinks chunk", dtype, dh, heads, group, news, lens, causal, window, sinks, flush=True)
    rng = np.random.default_rng(dh + sum(news))
    c, table = setup(gpu, rng, lens, heads, dh, 16)
    check(gpu, c, queries(gpu, rng, sum(news), heads * group, dh, dtype), table, lens, news, window,
          sinks, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("heads,group,news,context,window,sinks", [
    (2, 1, [8, 1, 5], [20, 0, 31], 0, 0),                   # few rows; a tree without a context
    (1, 4, [8, 3, 7], [300, 64, 33], 0, 0),                 # 32 rows
    (1, 2, [40, 17, 64, 2], [100, 1, 31, 500], 0, 0),       # rows of their own
    (1, 1, [65, 130, 64], [90, 3, 200], 0, 0),              # more than a word, more than two
    (1, 2, [33, 12], [400, 90], 50, 0),
    (2, 3, [20, 6, 50], [300, 0, 45], 7, 40)])
def test_trees(gpu, dtype, dh, heads, group, news, context, window, sinks):
    print("trees", dtype, dh, heads, group, news, context, window, sinks, flush=True)
    rng = np.random.default_rng(dh + sum(news) + window)
    lens = [a + b for a, b in zip(context, news)]
    c, table = setup(gpu, rng, lens, heads, dh, 16)
    trees = [paths(drafted(rng, n, s)) for n, s in zip(news, (4, 1, 9, 2))]
    check(gpu, c, queries(gpu, rng, sum(news), heads * group, dh, dtype), table, lens, news, window,
          sinks, trees)


@pytest.mark.parametrize("dtype", DTYPES)
def test_trees_of_any_bits(gpu, dtype):
    """Masks that are no paths: rows without a bit (with and without a context), with
    all, with those of later tokens; bits past the sequence's tokens; more words than
    the tokens need; drafted tokens that are not cached (a length below their number)."""
    rng = np.random.default_rng(9)
    news, lens, heads, dh = [6, 40, 5, 3, 70], [6, 160, 2, 0, 71], 2, 64
    c, table = setup(gpu, rng, lens, heads, dh, 32)
    trees = [rng.random((n, n)) < 0.4 for n in news]
    trees[0][2] = trees[1][7] = trees[4][69] = False
    trees[1][8] = trees[0][0] = True
    for group in (1, 4):
        for window, sinks in ((0, 0), (9, 0), (60, 20)):
            print("any bits", dtype, group, window, sinks, flush=True)
            q = queries(gpu, rng, sum(news), heads * group, dh, dtype)
            y, s = check(gpu, c, q, table, lens, news, window, sinks, trees, words=3)
            assert (y[2] == 0).all() and (s[2] == -math.inf).all()
            assert (y[51:54] == 0).all() and (s[51:54] == -math.inf).all()
    # the bits from a sequence's tokens on
    from qppocr_amd import ops
    q = queries(gpu, rng, 9, heads, dh, dtype)
    tab = gpu.tensor(table[:2], dtype=gpu.int32, device="cuda")
    ln = gpu.tensor([20, 100], dtype=gpu.int32, device="cuda")
    st = gpu.tensor([0, 4, 9], dtype=gpu.int32, device="cuda")
    bits = np.concatenate([words_of(paths([-1, 0, 0, 2]), 1), words_of(paths([-1, 0, 1, 1, 3]), 1)])
    got = []
    for high in (0, -32):                    # ~31: the bits from the sixth on
        t = gpu.from_numpy(bits | high).cuda()
        got.append(ops.attention_tree4(q, c, tab, ln, 0.125, t, starts=st, max_new=5, window=9, sinks=3))
    assert (host(got[0]) == host(got[1])).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,news", [(1, [9, 3, 16]), (4, [8, 8, 7]), (8, [30, 9, 12])])
def test_trees_long(gpu, dtype, group, news):
    """Contexts that many workgroups share, in all three forms, bounds that are too small
    or too large for them; the same call gives the same bits."""
    rng = np.random.default_rng(77)
    context, dh = [9000, 100, 4097 - news[2]], 128
    lens = [a + b for a, b in zip(context, news)]
    c, table = setup(gpu, rng, lens, 1, dh, 64)
    q = queries(gpu, rng, sum(news), group, dh, dtype)
    trees = [paths(drafted(rng, n, 4)) for n in news]
    rows = [(b, i) for b in range(3) for i in (0, 1, news[b] // 2, news[b] - 1)]
    got = []
    for bound in (9100, 300, 5000, 1 << 20, 9100):
        print("trees long", dtype, group, bound, flush=True)
        got.append(check(gpu, c, q, table, lens, news, trees=trees, max_len=bound, rows=rows))
    assert (got[0][0] == got[-1][0]).all() and (got[0][1] == got[-1][1]).all()
    for window, sinks in ((2500, 600), (4000, 3000), (1030, 5), (3, 2100)):
        print("trees long", dtype, group, window, sinks, flush=True)
        check(gpu, c, q, table, lens, news, window, sinks, trees, rows=rows)
        check(gpu, c, q, table, lens, news, window, sinks, rows=rows)
        check(gpu, c, q, table, lens, news, window, sinks, rows=rows, causal=False)
    check(gpu, c, q, table, lens, news, trees=trees, rows=rows, scale=-(dh ** -0.5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_a_gap_it_is_the_plain_attention(gpu, dtype):
    """A chain is a causal chunk, and sinks that reach the window are no window: within
    the tolerance of both, the plain call's result."""
    from qppocr_amd import ops
    rng = np.random.default_rng(3)
    news, lens, dh = [7, 60], [200, 90], 64
    c, table = setup(gpu, rng, lens, 2, dh, 32)
    q = queries(gpu, rng, sum(news), 4, dh, dtype)
    chain = [np.tril(np.ones((n, n), dtype=bool)) for n in news]
    y, s = check(gpu, c, q, table, lens, news, trees=chain)
    z, r = check(gpu, c, q, table, lens, news, window=40, sinks=1 << 40)
    st = gpu.tensor([0, 7, 67], dtype=gpu.int32, device="cuda")
    p, u = ops.attention_cache4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                gpu.tensor(lens, dtype=gpu.int32, device="cuda"), dh ** -0.5, starts=st,
                                max_new=60, lse=True)
    eps = gpu.finfo(q.dtype).eps + 2.0 ** -14
    for a, b in ((y, s), (z, r)):
        close(a, host(p), eps * np.abs(host(p)) + 2.0 ** -12, "rows")
        close(b, host(u), 2.0 ** -16 * (1 + np.abs(host(u))), "sums")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 96, 128, 192])
@pytest.mark.parametrize("group", [1, 4, 12])
def test_nan_stays_with_its_rows(gpu, dtype, dh, group):
    """Blocks of NaN behind the last token, between the sinks and the window, on other
    branches of the tree: only the rows that see them, all of a row for a key's, the
    block's elements for a value's."""
    rng = np.random.default_rng(6 + dh)
    page, news, lens = 16, [9, 5], [110, 40]
    c = make_cache(gpu, rng, 14, page, 1, dh)
    table = [[1, 4, 2, 6, 8, 9, 10], [0, 3, 12, -1, -1, -1, -1]]
    for s in (c.k_scales, c.v_scales):
        s[10, :, 14:], s[12, :, 8:], s[5], s[7], s[11], s[13] = 255, 255, 255, 255, 255, 255
        s[4, :, 2:12] = 255                      # keys 18 to 27 of sequence 0
    c.k_scales[10, 0, 8, 0] = 255                # key 104: drafted token 3
    c.v_scales[10, 0, 10, (dh // 32) - 1] = 255  # value 106: drafted token 5, its last block
    c.v_scales[12, 0, 4, 0] = 255                # value 36: drafted token 1 of sequence 1
    q = queries(gpu, rng, 14, group, dh, dtype)
    trees = [paths([-1, 0, 0, 1, 2, 2, 5, 4, -1]), paths([-1, 0, 0, 2, 1])]
    print("NaN", dtype, dh, group, flush=True)
    y, s = check(gpu, c, q, table, lens, news, 60, 17, trees)
    bad = np.isnan(y).any(axis=(1, 2))
    assert (bad == [False, False, False, True, False, True, True, False, False,
                    False, True, False, False, True]).all()
    y, _ = check(gpu, c, q, table, lens, news, 60, 17)
    assert (np.isnan(y).any(axis=(1, 2)) == [False] * 3 + [True] * 6 + [False] + [True] * 4).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_over_memory_never_written(gpu, dtype):
    """A pool whose unwritten tokens hold any bytes at all (scales that overflow among
    them): only the written ones that a row sees count."""
    from qppocr_amd import ops
    rng = np.random.default_rng(31)
    t = getattr(gpu, dtype)
    for dh, heads, group, news, lens, window, sinks in (
            (64, 2, 3, [1, 1, 1], [17, 64, 31], 12, 3), (128, 1, 4, [5, 2], [1500, 1239], 700, 40),
            (96, 1, 1, [60], [170], 0, 0), (32, 1, 16, [66, 65], [166, 90], 20, 5)):
        print("never written", dtype, dh, lens, flush=True)
        page = 64
        pages = sum((n + page - 1) // page for n in lens) + 2
        c = ops.cache4(pages, page, heads, dh)
        for x in (c.k_codes, c.k_scales, c.v_codes, c.v_scales):
            x.copy_(gpu.from_numpy(rng.integers(0, 256, x.shape, dtype=np.uint8)))
        for x in (c.k_scales, c.v_scales):
            x[:, :, 1::2] = gpu.from_numpy(rng.integers(250, 256, x[:, :, 1::2].shape, dtype=np.uint8)).cuda()
        table = tables(rng, pages, page, lens)
        for b, n in enumerate(lens):
            pos = np.arange(n)
            slots = np.array(table[b])[pos // page] * page + pos % page
            kv = gpu.from_numpy(rng.standard_normal((2, n, heads, dh)).astype(np.float32)).cuda().to(t)
            ops.cache4_write(c, kv[0], kv[1], gpu.from_numpy(slots.astype(np.int64)).cuda())
        q = queries(gpu, rng, sum(news), heads * group, dh, dtype)
        trees = [paths(drafted(rng, n, 3)) for n in news]
        rows = [(b, i) for b in range(len(news)) for i in (0, news[b] // 2, news[b] - 1)]
        for tr in (None, trees):
            y, s = check(gpu, c, q, table, lens, news, window, sinks, tr, rows=rows)
            assert np.isfinite(y).all() and np.isfinite(s).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 21, 2.0 ** 60])
def test_scores_of_any_size(gpu, dtype, size):
    """Scores far from zero, where a product with log2 e has no fraction left: each form
    gives the softmax of the scores as they are (they differ by far more than one, so a
    row's result is a value of the cache)."""
    from qppocr_amd import ops
    if dtype == "float16" and size > 2.0 ** 12:
        scale, big = size, 1.0
    else:
        scale, big = 1.0, size
    rng = np.random.default_rng(2)
    dh, lens = 64, [90]
    for group, n in ((1, 5), (4, 8), (4, 40)):
        c, table = setup(gpu, rng, lens, 1, dh, 32)
        q = queries(gpu, rng, n, group, dh, dtype) * big
        trees = [paths(drafted(rng, n, 3))]
        bits = gpu.from_numpy(words_of(trees[0], 1)).cuda()
        y = host(ops.attention_tree4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                     gpu.tensor(lens, dtype=gpu.int32, device="cuda"), scale, bits))
        k, v = numbers(c)
        pos = np.arange(90)
        pg = np.array(table[0])[pos // 32]
        k, v, qd = k[pg, pos % 32, 0], v[pg, pos % 32, 0], host(q)
        for i in range(n):
            see = visible(90, n, i, True, 0, 0, trees[0])
            for g in range(group):
                s = np.where(see, k @ qd[i, g] * scale, -np.inf)
                first, second = np.sort(s)[::-1][:2]
                # (a float32 sum of 64 exact products is off by 2^-17 of their size at most)
                if first - second > 30 + 2.0 ** -16 * (np.abs(k) @ np.abs(qd[i, g])).max() * scale:
                    # (the one term's product, its sum's reciprocal and their product are rounded)
                    want = v[s.argmax()]
                    tol = half_step(gpu, q.dtype, want) + 2.0 ** -22 * np.abs(want) + np.exp(-20.0) * 6
                    close(y[i, g], want, tol, f"row {i} {g}")


def test_bad_pages_and_lengths(gpu):
    """Page numbers outside the pool hold no keys; lengths past the table are cut at it;
    a negative length is none; starts past the rows are cut at them."""
    from qppocr_amd import ops
    rng = np.random.default_rng(5)
    page, pages = 16, 12
    c = make_cache(gpu, rng, pages, page, 2, 64)
    table = [[3, -1, 5, 7], [pages, 1, 2, 1 << 30], [-1, -1, -1, -1], [8, 9, 10, 11], [0, 4, 6, -5],
             [-(1 << 31), 0, 2, 2]]
    lens, news = [60, 64, 50, 1 << 20, 49, 33], [3, 9, 2, 30, 1, 4]
    for dtype in DTYPES:
        for heads in (2, 8):
            q = queries(gpu, rng, sum(news), heads, 64, dtype)
            trees = [paths(drafted(rng, n, 3)) for n in news]
            check(gpu, c, q, table, lens, news, trees=trees)
            check(gpu, c, q, table, lens, news, 20, 18, trees)
            check(gpu, c, q, table, lens, news, 20, 18)
    tab = gpu.tensor(table, dtype=gpu.int32, device="cuda")
    y, s = ops.attention_cache4(q[:6], c, tab, gpu.full((6,), -7, dtype=gpu.int32, device="cuda"), 0.125,
                                window=5, sinks=2, lse=True)
    assert (host(y) == 0).all() and (host(s) == -math.inf).all()
    st = gpu.tensor([-4, 2, 1, 60, 70, 1 << 30, 6], dtype=gpu.int32, device="cuda")
    y = ops.attention_cache4(q, c, tab, gpu.tensor(lens, dtype=gpu.int32, device="cuda"), 0.125, starts=st,
                             max_new=9, window=5, sinks=2)
    assert np.isfinite(host(y[:2])).all()


def test_strides_and_rows_left_alone(gpu):
    """Queries out of a packed projection, results into another, in place too; rows of no
    sequence keep what out holds."""
    from qppocr_amd import ops
    rng = np.random.default_rng(8)
    lens, dh, page = [70, 33], 64, 32
    for news in ([4, 3], [30, 21]):
        for dtype in DTYPES:
            c, table = setup(gpu, rng, lens, 2, dh, page)
            n = sum(news)
            trees = [paths(drafted(rng, m, 3)) for m in news]
            packed = queries(gpu, rng, n + 5, 12, dh, dtype)
            q = packed[:, 1:9]
            big = gpu.full((n + 5, 9, dh), 7.0, device="cuda", dtype=q.dtype)
            out = big[:, :8]
            starts = [2, 2 + news[0], 2 + n]
            args = dict(trees=trees, starts=starts)
            y, _ = check(gpu, c, q, table, lens, news, out=out, **args)
            for left in (big[:2], big[2 + n:], big[:, 8]):
                assert (host(left) == 7).all()
            was = packed.clone()
            z, _ = check(gpu, c, q.clone(), table, lens, news, **args)
            assert (z[2:2 + n] == y[2:2 + n]).all()
            words = gpu.zeros((n + 5, 1), dtype=gpu.int64, device="cuda")
            for b in range(2):
                words[starts[b]:starts[b + 1]] = gpu.from_numpy(words_of(trees[b], 1)).cuda()
            ops.attention_tree4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                gpu.tensor(lens, dtype=gpu.int32, device="cuda"), dh ** -0.5, words,
                                starts=gpu.tensor(starts, dtype=gpu.int32, device="cuda"),
                                max_new=max(news), out=q)
            got = host(packed)
            assert (got[2:2 + n, 1:9] == y[2:2 + n]).all()
            got[2:2 + n, 1:9] = host(was)[2:2 + n, 1:9]
            assert (got == host(was)).all()


def test_nothing_to_do(gpu):
    from qppocr_amd import ops
    c = ops.cache4(2, 16, 2, 64)
    i32 = dict(dtype=gpu.int32, device="cuda")
    q = gpu.zeros((0, 4, 64), device="cuda")
    y = ops.attention_cache4(q, c, gpu.zeros((3, 2), **i32), gpu.zeros(3, **i32), 0.1, window=3, sinks=1)
    assert tuple(y.shape) == (0, 4, 64)
    t = gpu.zeros((0, 1), dtype=gpu.int64, device="cuda")
    y = ops.attention_tree4(q, c, gpu.zeros((0, 2), **i32), gpu.zeros(0, **i32), 0.1, t)
    assert tuple(y.shape) == (0, 4, 64)
    # a table without pages holds no keys
    q = gpu.ones((2, 4, 64), device="cuda")
    y, s = ops.attention_cache4(q, c, gpu.zeros((2, 0), **i32), gpu.full((2,), 9, **i32), 0.1, window=3,
                                sinks=1, lse=True)
    assert (host(y) == 0).all() and (host(s) == -math.inf).all()


def test_past_32_bits(gpu):
    """A pool whose bytes pass 2^32: the last pages' keys, read by every form."""
    rng = np.random.default_rng(12)
    from qppocr_amd import ops
    page, heads, dh = 1024, 8, 256
    pages = (1 << 32) // (page * heads * dh // 2) + 3
    c = ops.cache4(pages, page, heads, dh)
    last = [pages - 1, pages - 2]
    for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)):
        for p in last:
            codes[p] = gpu.from_numpy(rng.integers(0, 256, codes[p].shape, dtype=np.uint8)).cuda()
            scales[p] = gpu.from_numpy(rng.integers(121, 128, scales[p].shape).astype(np.uint8)).cuda()
    small = ops.Cache4(*(x[last].contiguous() for x in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)))
    i32 = dict(dtype=gpu.int32, device="cuda")
    for news in (1, 4, 40):
        q = queries(gpu, rng, news, 32, dh, "bfloat16")
        bits = gpu.from_numpy(words_of(paths(drafted(rng, news, 3)), 1)).cuda()
        y = [ops.attention_tree4(q, x, gpu.tensor([t], **i32), gpu.tensor([1500], **i32), 0.1, bits,
                                 max_len=2048) for x, t in ((c, last), (small, [0, 1]))]
        assert (host(y[0]) == host(y[1])).all() and np.isfinite(host(y[0])).all()


@pytest.mark.parametrize("news", [3, 40])
def test_captured(gpu, news):
    """Two captured calls whose keys many workgroups share, replayed in turn and in flight
    together on two streams: a workspace each; masks and lengths change between."""
    from qppocr_amd import ops
    rng = np.random.default_rng(15)
    c = make_cache(gpu, rng, 130, 64, 2, 128)
    table = gpu.from_numpy(rng.permutation(128)[None].astype(np.int32)).cuda()
    lens = gpu.tensor([8000], dtype=gpu.int32, device="cuda")
    qs = [gpu.zeros((news, 8, 128), device="cuda", dtype=gpu.float16) for _ in range(2)]
    bits = [gpu.zeros((news, 1), dtype=gpu.int64, device="cuda") for _ in range(2)]
    graphs, outs = [], []
    for q, t in zip(qs, bits):
        ops.attention_tree4(q, c, table, lens, 0.1, t, window=5000, sinks=40)
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(ops.attention_tree4(q, c, table, lens, 0.1, t, window=5000, sinks=40, lse=True))
        graphs.append(g)
    side = gpu.cuda.Stream()
    for i in range(5):
        new = [queries(gpu, rng, news, 8, 128, "float16") for _ in qs]
        masks = [gpu.from_numpy(words_of(paths(drafted(rng, news, 3)), 1)).cuda() for _ in qs]
        for q, v, t, w in zip(qs, new, bits, masks):
            q.copy_(v)
            t.copy_(w)
        lens.fill_(8000 - 1111 * i)
        gpu.cuda.synchronize()
        graphs[0].replay()
        with gpu.cuda.stream(side):
            graphs[1].replay()
        gpu.cuda.synchronize()
        for v, w, (y, s) in zip(new, masks, outs):
            y2, s2 = ops.attention_tree4(v, c, table, lens, 0.1, w, window=5000, sinks=40, max_len=8192, lse=True)
            assert (host(y) == host(y2)).all() and (host(s) == host(s2)).all()


def test_refusals(gpu):
    from qppocr_amd import ops
    c = ops.cache4(4, 16, 2, 64)
    i32 = dict(dtype=gpu.int32, device="cuda")
    q, tab, ln = gpu.zeros((3, 4, 64), device="cuda"), gpu.zeros((3, 4), **i32), gpu.ones(3, **i32)
    t = gpu.ones((3, 1), dtype=gpu.int64, device="cuda")
    def tree(q=q, tree=t, **kw):
        return ops.attention_tree4(q, c, tab, ln, 0.1, tree, **kw)
    tree()
    for bad, text in ((dict(tree=t[:2]), "tree int64"), (dict(tree=t[:, :0]), "tree int64"),
                      (dict(tree=t[:, 0]), "tree int64"), (dict(tree=t.int()), "contiguous torch.int64"),
                      (dict(tree=t.cpu()), "is on cpu"), (dict(tree=t.expand(3, 2)), "contiguous"),
                      (dict(starts=gpu.zeros(4, **i32)), "max_new"),
                      (dict(starts=gpu.zeros(4, **i32), max_new=65), "words"),
                      (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
                      (dict(q=q.double()), "float64"), (dict(out=q[:, :, :32]), "must be"),
                      (dict(q=q.clone().requires_grad_()), "gradient")):
        with pytest.raises(ValueError, match=text):
            tree(**bad)
    with pytest.raises(ValueError, match="negative"):
        ops.attention_cache4(q, c, tab, ln, 0.1, window=4, sinks=-1)
