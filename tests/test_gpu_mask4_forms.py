"""Attention over the 4-bit cache with sinks and drafted trees in the forms that only
particular batches take: twelve waves that share a few rows, and even shares of the keys of
sequences with a window and first tokens.  Against the definition in 64 bits, at the
tolerances of test_gpu_mask4; few rows at those of test_gpu_decode4, which leave a bfloat16
row's probabilities 16 bits."""
import math

import numpy as np
import pytest

import test_gpu_mask4
from test_gpu_decode4 import DTYPES, HEAD_DIMS, attend_row, host, tables
from test_gpu_mask4 import check, drafted, paths, queries, setup

pytestmark = pytest.mark.gpu

LONG = 1 << 20            # a bound of lengths for which keys are split however short they are


@pytest.fixture
def sixteen_bits(monkeypatch):
    """The few-row form's tolerance, without the many-row form's 11-bit probabilities."""
    monkeypatch.setattr(test_gpu_mask4, "attend", attend_row)


def picked(news, sequences, each=3):
    return [(b, i) for b in sequences for i in sorted({0, news[b] // 2, news[b] - 1} if news[b] else ())][:each * len(sequences)]


# -------------------------------------- a workgroup of twelve waves for a head's few rows

# 25 sequences of 8 heads are 200 workgroups: three splits fit the chip, which these are in place of
LENS25 = [0, 1, 31, 32, 33, 64, 95, 352, 384, 385, 416, 767, 768, 769, 1500, 2, 700, 40, 90, 200, 383, 5, 3, 17, 1030]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("group,most,window,sinks,tree", [
    (2, 1, 1000, 70, False),                # single tokens, sinks and window in one run or two
    (1, 9, 0, 0, True),
    (4, 4, 1040, 5, True),
    (1, 16, 1000, 1, False)])
def test_twelve_waves(gpu, sixteen_bits, dtype, dh, group, most, window, sinks, tree):
    """Sequences with fewer tiles of keys than waves, as many, one more, and none; ragged
    numbers of new tokens."""
    rng = np.random.default_rng(dh + most)
    news = [1] * 25 if most == 1 else [int(x) for x in rng.integers(0, most + 1, 25)]
    news[14] = news[24] = most
    c, table = setup(gpu, rng, LENS25, 8, dh, 16)
    trees = [paths(drafted(rng, n, 4)) for n in news] if tree else None
    q = queries(gpu, rng, sum(news), 8 * group, dh, dtype)
    print("twelve waves", dtype, dh, group, most, window, sinks, tree, flush=True)
    got = [check(gpu, c, q, table, LENS25, news, window, sinks, trees, max_len=LONG, rows=picked(news, range(25)))
           for _ in range(2)]
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,lens", [(1, [700]), (1, [513]), (2, [768, 520]), (16, [530, 760, 3, 641, 0, 99, 600, 700])])
def test_twelve_waves_for_short_sequences(gpu, sixteen_bits, dtype, dh, heads, lens):
    """Three splits' worth of keys, in few workgroups and in many."""
    rng = np.random.default_rng(dh + sum(lens))
    news = [min(3, 1 + b) for b in range(len(lens))]
    c, table = setup(gpu, rng, lens, heads, dh, 32)
    q = queries(gpu, rng, sum(news), heads * 4, dh, dtype)
    trees = [paths(drafted(rng, n, 3)) for n in news]
    print("twelve waves, short", dtype, dh, heads, lens, flush=True)
    check(gpu, c, q, table, lens, news, trees=trees, max_len=max(lens))
    check(gpu, c, q, table, lens, news, 500, 40, max_len=max(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 96, 128])
@pytest.mark.parametrize("scale", [None, 2.0 ** 21])
def test_twelve_waves_walked_again(gpu, sixteen_bits, dtype, dh, scale):
    """NaN in some waves' keys and values, seen and not; with the large scale, scores far
    from zero, of which a row's result is the best key's value: both go through the second
    walk, whose tiles are twelve apart too.  Lengths past the table and below zero, pages
    outside the pool."""
    from qppocr_amd import ops
    rng = np.random.default_rng(dh)
    lens = list(LENS25)
    c, table = setup(gpu, rng, lens, 8, dh, 32)
    wide = max(len(t) for t in table)
    table = [list(t) + [-1] * (wide - len(t)) for t in table]
    q = queries(gpu, rng, 25, 8, dh, dtype)
    print("twelve waves again", dtype, dh, scale, flush=True)
    if scale is None:
        table[12][3] = c.pages
        lens[16], lens[20] = 1 << 20, -5
        for b, j, part in ((14, 700, "v_scales"), (14, 1499, "k_scales"), (13, 8, "v_scales"), (11, 400, "k_scales")):
            getattr(c, part)[table[b][j // 32], 0, j % 32, dh // 32 - 1] = 255
        y, s = check(gpu, c, q, table, lens, [1] * 25, 1000, 70, max_len=LONG)
        bad = np.isnan(y).any(axis=(1, 2))
        assert bad[[11, 13, 14]].all() and bad.sum() == 3
        assert (y[20] == 0).all() and (s[20] == -math.inf).all()
        return
    from test_gpu_decode4 import close, half_step, numbers
    from test_gpu_mask4 import visible
    i32 = dict(dtype=gpu.int32, device="cuda")
    y = host(ops.attention_cache4(q, c, gpu.tensor(table, **i32), gpu.tensor(lens, **i32), scale, window=1000,
                                  sinks=70, max_len=LONG))
    k, v = numbers(c)
    qd, seen = host(q), 0
    for b, n in enumerate(lens):
        pos = np.flatnonzero(visible(n, 1, 0, True, 1000, 70, None)) if n else np.zeros(0, int)
        pg = np.array(table[b], dtype=np.int64)[pos // 32]
        for h in range(8 if n else 0):
            kh, vh = k[pg, pos % 32, h], v[pg, pos % 32, h]
            score = kh @ qd[b, h] * scale
            first, second = np.sort(np.append(score, -np.inf))[::-1][:2]
            # (a float32 sum of dh exact products is off by 2^-16 of their size at most)
            if first - second > 30 + 2.0 ** -15 * (np.abs(kh) @ np.abs(qd[b, h])).max() * scale:
                want = vh[score.argmax()]
                tol = half_step(gpu, q.dtype, want) + 2.0 ** -22 * np.abs(want) + np.exp(-20.0) * 6
                close(y[b, h], want, tol, f"row {b} {h}")
                seen += 1
    assert seen > 100


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_twelve_waves_captured(gpu, dtype):
    """Captured and replayed with other lengths and masks, two in flight together."""
    from qppocr_amd import ops
    rng = np.random.default_rng(5)
    c, table = setup(gpu, rng, [1600] * 4 + [300] * 21, 8, 64, 64)
    i32 = dict(dtype=gpu.int32, device="cuda")
    wide = max(len(t) for t in table)
    tab = gpu.tensor([list(t) + [-1] * (wide - len(t)) for t in table], **i32)
    ln = gpu.zeros(25, **i32)
    qs = [gpu.zeros((25, 32, 64), device="cuda", dtype=getattr(gpu, dtype)) for _ in range(2)]
    graphs, outs = [], []

    def call(q):
        return ops.attention_cache4(q, c, tab, ln, 0.125, window=1100, sinks=9, lse=True)
    for q in qs:
        call(q)
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(call(q))
        graphs.append(g)
    side = gpu.cuda.Stream()
    for i in range(4):
        for q in qs:
            q.copy_(queries(gpu, rng, 25, 32, 64, dtype))
        ln.copy_(gpu.tensor([1600 - 333 * i] * 4 + rng.integers(0, 300, 21).tolist(), dtype=gpu.int32))
        gpu.cuda.synchronize()
        graphs[0].replay()
        with gpu.cuda.stream(side):
            graphs[1].replay()
        gpu.cuda.synchronize()
        for q, (y, s) in zip(qs, outs):
            y2, s2 = call(q)
            assert (host(y) == host(y2)).all() and (host(s) == host(s2)).all()


# ------------------------------------- even shares of the keys that a window and sinks leave

def most_new(dtype, dh, one, two):
    """New tokens for which a workgroup has a sequence's rows: waves of 16 rows (one) or 32."""
    return two if dh <= (64 if dtype == "float32" else 128) else one


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("window,sinks,tree", [(1000, 70, False), (1000, 70, True), (1100, 1, False), (40, 1100, True)])
def test_even_shares_of_windows(gpu, dtype, dh, window, sinks, tree):
    """64 sequences of 5 heads: parts that begin in the first tokens, in the window and end
    in either; windows that reach the first tokens; sequences without keys or new tokens."""
    rng = np.random.default_rng(dh + window + sinks)
    most = most_new(dtype, dh, 16, 24)
    lens = [int(x) for x in rng.integers(0, 120, 64)]
    for b, n in ((0, 1700), (5, 1095), (6, 2500), (31, 1060), (32, 1070), (40, 71), (41, 64), (63, 1333)):
        lens[b] = n
    news = [int(x) for x in rng.integers(0, most // 2, 64)]
    for b, n in ((0, most), (5, 1), (6, most), (10, 0), (31, most - 1), (32, 7), (40, 5), (41, most), (63, 3)):
        news[b] = n
    lens[11], news[11] = 0, 4
    c, table = setup(gpu, rng, lens, 5, dh, 32)
    trees = [paths(drafted(rng, n, 5)) for n in news] if tree else None
    q = queries(gpu, rng, sum(news), 20, dh, dtype)
    print("even windows", dtype, dh, window, sinks, tree, flush=True)
    got = [check(gpu, c, q, table, lens, news, window, sinks, trees, max_len=LONG,
                 rows=picked(news, (0, 5, 6, 10, 11, 17, 31, 32, 40, 41, 63))) for _ in range(2)]
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh,most", [(32, 24), (64, 50), (128, 16), (192, 16)])
def test_even_shares_of_a_long_window(gpu, dtype, dh, most):
    """A window of 60000 keys of one sequence of 66000 in many workgroups' shares, short
    sequences beside it; four waves a workgroup and more."""
    rng = np.random.default_rng(dh)
    most = max(most, most_new(dtype, dh, 16, 24))
    lens, news = [300, 66000, 0, 61000, 90, 2000], [most, 5, 0, most, 2, 9]
    c, table = setup(gpu, rng, lens, 1, dh, 128)
    trees = [paths(drafted(rng, n, 5)) for n in news]
    q = queries(gpu, rng, sum(news), 4, dh, dtype)
    rows = [(0, 0), (0, most - 1), (1, 0), (1, 4), (3, most // 2), (4, 1), (5, 8)]
    for tr, window, sinks in ((None, 60000, 333), (trees, 60000, 1)):
        print("even, a long window", dtype, dh, window, sinks, flush=True)
        check(gpu, c, q, table, lens, news, window, sinks, tr, max_len=LONG, rows=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [64, 192])
def test_even_shares_of_windows_walked_again(gpu, dtype, dh):
    """Values and keys that float16 does not hold and NaN: among the first tokens, between
    them and the window, in the window, at its borders; lengths past the table and below
    zero; pages outside the pool."""
    rng = np.random.default_rng(dh)
    window, sinks = 1000, 70
    most = most_new(dtype, dh, 16, 24)
    lens = [int(x) for x in rng.integers(0, 100, 64)]
    for b, n in ((0, 1700), (6, 2500), (31, 1200), (63, 1333)):
        lens[b] = n
    news = [int(x) for x in rng.integers(0, most // 2, 64)]
    news[0], news[6], news[31], news[63] = most, 3, 5, most
    c, table = setup(gpu, rng, lens, 5, dh, 32)
    wide = max(len(t) for t in table)
    table = [list(t) + [-1] * (wide - len(t)) for t in table]
    lens[9], lens[17] = 1 << 20, -5
    news[9], news[17] = 4, 6
    table[31][9] = c.pages
    # 1676 is sequence 0's first position and 1700 its last: window and sinks hide 70 to 676 from all rows
    for b, j, scale in ((0, 69, 145), (0, 300, 255), (0, 1690, 100), (6, 69, 142), (6, 70, 255), (63, 400, 103)):
        c.v_scales[table[b][j // 32], :, j % 32] = scale
    for b, j, scale in ((0, 5, 142), (0, 310, 255), (31, 250, 150), (63, 1332, 255)):
        c.k_scales[table[b][j // 32], :, j % 32] = scale
    q = queries(gpu, rng, sum(news), 20, dh, dtype)
    trees = [paths(drafted(rng, n, 4)) for n in news]
    rows = picked(news, (0, 6, 9, 17, 31, 40, 63), 4) + [(0, i) for i in range(0, most, 5)]
    print("even windows again", dtype, dh, flush=True)
    for tr in (None, trees):
        y, _ = check(gpu, c, q, table, lens, news, window, sinks, tr, max_len=LONG, rows=rows)
        at = sum(news[:6])
        assert np.isfinite(y[:news[0]]).all() and np.isfinite(y[at:at + 3]).all()
        assert np.isnan(y[-1]).any(axis=-1).any() if tr is None else True
