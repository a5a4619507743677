"""A step's pages, slots, positions and masks, rotation by positions and moves inside
the cache, against plain loops and 64-bit arithmetic; and a decoder's steps that draft,
check and accept trees with all of them together."""
import math

import numpy as np
import pytest

from test_gpu_decode4 import DTYPES, HEAD_DIMS, close, half_step, host, make_cache, numbers
from test_gpu_mask4 import attend, drafted, paths, words_of

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ extend

def extend(table, lens, news, page, ring, ends, tokens, parents=None, max_new=0):
    """The definition, sequence by sequence; writes table and ring."""
    head, tail = ends
    free, limit, out_of_pages = head, tail, False
    cap, wide = len(ring), table.shape[1]
    room = min(wide * page, (1 << 31) - 256)
    was = ring.copy()
    starts, after = [0], []
    slots = np.full(tokens, -1, dtype=np.int64)
    positions = np.zeros(tokens, dtype=np.int64)
    words = (max_new + 63) // 64
    tree = np.zeros((tokens, words), dtype=np.int64)
    at = 0
    for b, (n0, m) in enumerate(zip(lens, news)):
        n0 = min(max(n0, 0), room)
        r0, r1 = at, at + max(m, 0)
        at = r1
        starts.append(min(r1, tokens))
        held = -(-n0 // page)
        rows = np.arange(min(r0, tokens), min(r1, tokens))
        depth = rows - r0 + 1
        if parents is not None and len(rows):
            p = parents[rows[0]:rows[-1] + 1]
            see = paths([int(x) if 0 <= x < i else -1 for i, x in enumerate(p)])
            depth = see.sum(1)
            tree[rows] = words_of(see, words)
        positions[rows] = np.minimum(n0 + depth - 1, (1 << 31) - 1)
        if m < 0:
            n1 = max(n0 + m, 0)
            for col in range(-(-n1 // page), held):
                if tail - ends[1] < cap - min(max(limit - head, 0), cap):      # (else dropped)
                    ring[tail % cap] = table[b, col]
                    tail += 1
            after.append(n1)
            continue
        need = -(-(n0 + m) // page) - held
        if n0 + m > room or r1 > tokens:
            after.append(n0)
            continue
        if need and (out_of_pages or free + need > max(limit, free)):
            out_of_pages = True
            after.append(n0)
            continue
        for col in range(held, held + need):
            table[b, col] = was[free % cap]
            free += 1
        pos = n0 + np.arange(m)
        pg = table[b, pos // page].astype(np.int64)
        slots[rows] = np.where(pg >= 0, pg * page + pos % page, -1)
        after.append(n0 + m)
    return starts, after, slots, positions, (free, tail), tree


def check_extend(torch, table, lens, news, page, ring, ends, tokens, parents=None, max_new=None, name=""):
    from qppocr_amd import ops
    def dev(x, t=np.int32):
        return torch.from_numpy(np.ascontiguousarray(x, dtype=t)).cuda()
    tb, rg = dev(table), dev(ring)
    step = ops.cache4_extend(tb, dev(lens), dev(news), page, rg, dev(ends, np.int64), tokens,
                             None if parents is None else dev(parents), max_new)
    table, ring = table.copy(), ring.copy()
    starts, after, slots, positions, left, tree = extend(table, lens, news, page, ring, ends, tokens,
                                                         parents, max_new or 0)
    for what, got, want in (("starts", step.starts, starts), ("lens", step.lens, after),
                            ("slots", step.slots, slots), ("positions", step.positions, positions),
                            ("ends", step.ends, left), ("table", tb, table), ("ring", rg, ring)):
        got, want = got.cpu().numpy(), np.asarray(want)
        assert got.shape == want.shape and (got == want).all(), \
            (name, what, np.argwhere(got != want)[:3].tolist(), got[got != want][:5], want[got != want][:5])
    if parents is not None:
        assert (step.tree.cpu().numpy() == tree).all(), name
    else:
        assert step.tree is None
    return step


def pool(rng, lens, news, page, wide, spare=3, head=0):
    """A table of distinct pages, and a ring whose free ones start at `head`."""
    batch = len(lens)
    held = [-(-n // page) for n in lens]
    need = [max(0, -(-(n + m) // page) - h) for n, m, h in zip(lens, news, held)]
    pages = sum(held) + sum(need) + spare
    order = rng.permutation(pages)
    table = np.full((batch, wide), -1, dtype=np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    ring = np.full(pages, -1, dtype=np.int32)
    free = order[at:]
    ring[(head + np.arange(len(free))) % pages] = free
    return table, ring, (head, head + len(free))


@pytest.mark.parametrize("page", [16, 64, 32768])
@pytest.mark.parametrize("batch,context,most", [
    (1, 0, 1), (1, 100, 300), (3, 40, 17), (64, 500, 1), (65, 50, 40), (700, 300, 9), (2048, 40, 3),
    (2049, 40, 3), (9000, 20, 2)])
def test_extend(gpu, page, batch, context, most):
    rng = np.random.default_rng(batch + page)
    lens = rng.integers(0, context + 1, batch).tolist()
    news = rng.integers(0, most + 1, batch).tolist()
    for b in range(0, batch, 5):
        news[b] = -int(rng.integers(0, lens[b] + 3))
    wide = -(-(context + most) // page) + 1
    rows = sum(n for n in news if n > 0)
    print("extend", page, batch, context, most, flush=True)
    for head, more in ((0, 0), (12345678901, 9)):
        table, ring, ends = pool(rng, lens, news, page, wide, head=head)
        check_extend(gpu, table, lens, news, page, ring, ends, rows + more)


@pytest.mark.parametrize("batch", [5, 300, 3000])
def test_extend_that_is_not_granted(gpu, batch):
    """Pages run out in the middle; a table that is too narrow; rows past `tokens`;
    lengths outside the table; an empty or overfull ring; numbers at their types' ends."""
    rng = np.random.default_rng(batch)
    page, wide = 16, 6
    lens = rng.integers(0, 96, batch).tolist()
    news = rng.integers(0, 30, batch).tolist()
    rows = sum(news)
    table, ring, ends = pool(rng, lens, news, page, wide + 4)
    table = np.ascontiguousarray(table[:, :wide])
    cap = len(ring)
    for tokens in (rows, rows // 2, 0):
        for free in (cap, cap // 2, 3, 0, -5):
            check_extend(gpu, table, lens, news, page, ring, (ends[0], ends[0] + free), tokens,
                         name=f"{tokens} {free}")
    odd = list(lens)
    odd[0], odd[1], odd[2] = -3, 1 << 30, (1 << 31) - 1
    hard = list(news)
    hard[3], hard[4] = (1 << 31) - 1, -(1 << 31)
    check_extend(gpu, table, odd, hard, page, ring, (7, 7 + cap), rows, name="odd")
    hard[0] = hard[1] = hard[2] = (1 << 31) - 1
    check_extend(gpu, table, odd, hard, page, ring, (7, 7 + cap), rows, name="sums past 32 bits")
    check_extend(gpu, table, odd, [-(1 << 31)] * batch, page, ring[:5], (-3, -1), 4, name="more given than held")


@pytest.mark.parametrize("batch,most,spread", [(1, 1, 1), (4, 63, 3), (3, 64, 1), (5, 65, 70), (40, 33, 8),
                                               (2, 200, 5), (2100, 5, 2), (3, 700, 1)])
def test_extend_trees(gpu, batch, most, spread):
    """Paths and depths, over more than a word; parents that are none."""
    rng = np.random.default_rng(batch + most)
    lens = rng.integers(0, 300, batch).tolist()
    news = rng.integers(0, most + 1, batch).tolist()
    news[0] = most
    if batch > 2:
        news[2] = -lens[2]
    page, wide = 32, (300 + most) // 32 + 1
    parents = [p for n in news for p in drafted(rng, max(n, 0), spread)]
    print("extend trees", batch, most, spread, flush=True)
    table, ring, ends = pool(rng, lens, news, page, wide)
    check_extend(gpu, table, lens, news, page, ring, ends, len(parents) + 3,
                 np.array(parents + [0, 5, -1]), most)
    wild = rng.integers(-(1 << 31), 1 << 31, len(parents))
    keep = rng.random(len(parents)) < 0.7
    wild = np.where(keep, parents, wild)
    check_extend(gpu, table, lens, news, page, ring, ends, len(parents), wild, most)
    # fewer words than a sequence's tokens need, fewer rows than there are
    check_extend(gpu, table, lens, news, page, ring, ends, len(parents), wild, max(1, most - 70))
    check_extend(gpu, table, lens, news, page, ring, ends, max(0, len(parents) - 2),
                 wild[:max(0, len(parents) - 2)], most)


def test_extend_nothing_to_do(gpu):
    table, ring = np.zeros((0, 3), np.int32), np.arange(4, dtype=np.int32)
    check_extend(gpu, table, [], [], 16, ring, (1, 4), 0)
    check_extend(gpu, table, [], [], 16, ring, (1, 4), 5)
    check_extend(gpu, np.zeros((2, 0), np.int32), [0, 3], [1, 0], 16, ring, (1, 4), 1)
    check_extend(gpu, np.zeros((2, 3), np.int32), [4, 5], [0, 0], 16, ring, (0, 0), 0, np.zeros(0, np.int32), 1)


def test_extend_table_of_other_strides(gpu):
    from qppocr_amd import ops
    big = gpu.full((3, 10), 99, dtype=gpu.int32, device="cuda")
    ring = gpu.arange(8, dtype=gpu.int32, device="cuda")
    i32 = dict(dtype=gpu.int32, device="cuda")
    s = ops.cache4_extend(big[:, 2:6], gpu.tensor([0, 16, 5], **i32), gpu.tensor([20, 1, 2], **i32), 16, ring,
                          gpu.tensor([2, 8], device="cuda"), 23)
    want = np.full((3, 10), 99)
    want[0, 2:4], want[1, 3] = [2, 3], 4
    assert (big.cpu().numpy() == want).all()
    assert s.ends.tolist() == [5, 8] and s.lens.tolist() == [20, 17, 7]


def test_extend_captured(gpu):
    """A step captured once: lengths and ends go round by copies inside the graph; every
    replay is the definition's next step."""
    from qppocr_amd import ops
    rng = np.random.default_rng(1)
    batch, page, wide = 30, 16, 20
    lens, news = [0] * batch, [3] * batch
    table, ring, ends = pool(rng, [wide * page] * batch, [0] * batch, page, wide, spare=1)
    ring[:] = rng.permutation(len(ring))
    ends = (0, len(ring))
    table[:] = -1
    i32 = dict(dtype=gpu.int32, device="cuda")
    tb, rg = gpu.from_numpy(table).cuda(), gpu.from_numpy(ring).cuda()
    ln, nw = gpu.tensor(lens, **i32), gpu.tensor(news, **i32)
    en = gpu.tensor(ends, device="cuda")
    ops.cache4_extend(tb.clone(), ln, nw, page, rg.clone(), en, 200)
    gpu.cuda.synchronize()
    g = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(g):
        s = ops.cache4_extend(tb, ln, nw, page, rg, en, 200)
        ln.copy_(s.lens)
        en.copy_(s.ends)
    for i in range(9):
        g.replay()
        gpu.cuda.synchronize()
        starts, lens, slots, positions, ends, _ = extend(table, lens, news, page, ring, ends, 200)
        assert s.lens.tolist() == lens and s.ends.tolist() == list(ends), i
        assert (s.slots.cpu().numpy() == slots).all() and (s.positions.cpu().numpy() == positions).all(), i
        assert (rg.cpu().numpy() == ring).all() and (tb.cpu().numpy() == table).all(), i
        news = rng.integers(-9, 14, batch).tolist()
        nw.copy_(gpu.tensor(news, **i32))


# ------------------------------------------------------------------ rotary

def rotate(x, pos, freqs, axes, neighbours, inverse):
    """In 64 bits: x [tokens, heads, dh], pos [axes, tokens] (whole numbers)."""
    y, r = x.copy(), len(freqs)
    for i in range(r):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + r)
        # angles of far positions: whole turns taken off in long numbers
        t = np.array([math.remainder(float(int(p) * f_exact(freqs[i]) % TWO_PI), 2 * math.pi)
                      for p in pos[axes[i]]])[:, None]
        s, c = np.sin(t) * (-1 if inverse else 1), np.cos(t)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def f_exact(f):
    import fractions
    return fractions.Fraction(f)


TWO_PI = f_exact(628318530717958647692528676655900576839433879875021) / 10 ** 50


def check_rotary(torch, x, pos, freqs, axes=None, neighbours=False, inverse=False, out=None, name=""):
    from qppocr_amd import ops
    plan = ops.rotary_plan(x.shape[2], freqs, axes, neighbours)
    xd = host(x)
    p = pos.cpu().numpy()
    axes = [0] * len(freqs) if axes is None else axes
    if p.ndim == 1:
        p = np.stack([p] * (max(axes) + 1))
    y = ops.rotary(x, pos, plan, inverse=inverse, out=out)
    want = rotate(xd, p, freqs, axes, neighbours, inverse)
    # cosine and sine: the angle's float32 (2^-24 of pi / 4 at most, two roundings), the
    # series' (four roundings of at most half a unit of 1) and its first term left out:
    # 2^-22 altogether; then two products and their sum
    r = len(freqs)
    size = np.abs(xd).copy()
    for i in range(r):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + r)
        size[..., a] = size[..., b] = size[..., a] + size[..., b]
    tol = size * (2.0 ** -22 + 2.0 ** -23)
    tol[..., 2 * r:] = 0
    close(host(y), want, tol + half_step(torch, x.dtype, want) * 1.001 * (tol > 0), name)
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("tokens,heads,dh,pairs,axes", [
    (1, 1, 2, 1, 1), (1, 40, 128, 64, 1), (7, 3, 64, 32, 3), (5, 2, 96, 24, 2), (3, 5, 80, 37, 4),
    (33, 1, 32, 5, 2), (200, 2, 256, 128, 3), (2, 2, 7, 3, 1), (3, 1, 130, 8, 1)])
def test_rotary(gpu, dtype, neighbours, tokens, heads, dh, pairs, axes):
    rng = np.random.default_rng(dh + tokens)
    t = getattr(gpu, dtype)
    freqs = [10000.0 ** (-i / pairs) for i in range(pairs)]
    ax = [i % axes for i in range(pairs)]
    print("rotary", dtype, neighbours, tokens, heads, dh, pairs, axes, flush=True)
    for index in (gpu.int32, gpu.int64):
        x = gpu.from_numpy(rng.standard_normal((tokens, heads, dh)).astype(np.float32)).cuda().to(t)
        pos = gpu.from_numpy(rng.integers(-300, 5000, (axes, tokens))).cuda().to(index)
        y = check_rotary(gpu, x, pos, freqs, ax, neighbours, False, name="forward")
        z = check_rotary(gpu, y, pos, freqs, ax, neighbours, True, name="back")
        # there and back: two roundings of each element of a pair
        u = 4 * gpu.finfo(t).eps / 2 + 2.0 ** -20
        close(host(z), host(x), u * 2 * (np.abs(host(x)).max() + 1), "there and back")
        one = pos[0].contiguous()
        check_rotary(gpu, x, one, freqs, ax, neighbours, False, name="one position for all axes")


def test_rotary_far_positions(gpu):
    """Positions up to the types' ends, whose angles float32 or float64 products lose;
    fast and slow pairs; frequencies past a turn a position and below zero."""
    rng = np.random.default_rng(2)
    freqs = [1.0, 0.75, 1e-3, 10000.0 ** (-63 / 64), 1e-7, 2.0 ** -40, -0.3, 100.0, math.pi, 0.0]
    for index, values in ((gpu.int32, [0, 1, -1, 131071, 1 << 20, (1 << 31) - 1, -(1 << 31)]),
                          (gpu.int64, [(1 << 31), 1 << 38, -(1 << 38) + 7])):
        pos = gpu.tensor(values, dtype=index, device="cuda")
        x = gpu.from_numpy(rng.standard_normal((len(values), 2, 20)).astype(np.float32)).cuda()
        # (2^38 positions of 2^-65 turns: 2^-27 turns, a fifth of the tolerance)
        check_rotary(gpu, x, pos, freqs, name=str(index))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_strides(gpu, dtype):
    """Out of a packed projection, in place, into another; positions of any strides."""
    from qppocr_amd import ops
    rng = np.random.default_rng(3)
    t = getattr(gpu, dtype)
    freqs = [100.0 ** (-i / 13) for i in range(13)]
    ax = [0] * 5 + [1] * 8
    packed = gpu.from_numpy(rng.standard_normal((9, 6, 31)).astype(np.float32)).cuda().to(t)
    x = packed[:, 1:4, 2:31]
    pos = gpu.from_numpy(rng.integers(0, 3000, (9, 2))).cuda().t()
    y = check_rotary(gpu, x, pos, freqs, ax)
    big = gpu.full((3, 9, 31), 5.0, device="cuda", dtype=t)
    z = check_rotary(gpu, x, pos, freqs, ax, out=big[:, :, 1:30].transpose(0, 1))
    assert (host(z) == host(y)).all() and (host(big[:, :, 0]) == 5).all() and (host(big[:, :, 30]) == 5).all()
    was = host(packed)
    ops.rotary(x, pos, ops.rotary_plan(29, freqs, ax), out=x)
    want = was.copy()
    want[:, 1:4, 2:31] = host(y)
    assert (host(packed) == want).all()


def test_rotary_keeps_numbers_that_are_none(gpu):
    """An infinity or NaN reaches its own pair alone; elements that are not turned are
    copied bit for bit; positions of zero change nothing."""
    from qppocr_amd import ops
    x = gpu.ones((3, 2, 16), device="cuda", dtype=gpu.float16)
    x[1, 0, 2], x[1, 1, 5], x[2, 0, 15] = math.inf, math.nan, math.nan
    plan = ops.rotary_plan(16, [1.0] * 6)
    y = host(ops.rotary(x, gpu.tensor([0, 1, 2], dtype=gpu.int32, device="cuda"), plan))
    assert (y[0] == 1).all()
    bad = ~np.isfinite(y)
    assert bad[1, 0, [2, 8]].all() and bad[1, 1, [5, 11]].all() and bad[2, 0, 15] and bad.sum() == 5


def test_rotary_nothing_to_do(gpu):
    from qppocr_amd import ops
    plan = ops.rotary_plan(32, [1.0, 0.5])
    i32 = dict(dtype=gpu.int32, device="cuda")
    assert ops.rotary(gpu.zeros((0, 3, 32), device="cuda"), gpu.zeros(0, **i32), plan).shape == (0, 3, 32)
    assert ops.rotary(gpu.zeros((4, 0, 32), device="cuda"), gpu.zeros(4, **i32), plan).shape == (4, 0, 32)


# -------------------------------------------------------------------- move

def pools(c):
    return [x.cpu().numpy().copy() for x in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]


def check_move(torch, c, src, dst, name=""):
    from qppocr_amd import ops
    before, page = pools(c), c.page_size
    ops.cache4_move(c, torch.tensor(src, dtype=torch.int64, device="cuda"),
                    torch.tensor(dst, dtype=torch.int64, device="cuda"))
    want = [x.copy() for x in before]
    total = c.pages * page
    for s, d in zip(src, dst):
        if 0 <= s < total and 0 <= d < total:
            for w, x in zip(want, before):
                w[d // page, :, d % page] = x[s // page, :, s % page]
    for got, w in zip(pools(c), want):
        assert (got == w).all(), (name, np.argwhere(got != w)[:4].tolist())


@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("heads,page,tokens", [(1, 16, 1), (8, 16, 70), (3, 64, 600), (2, 32, 1100), (1, 16, 5000),
                                               (16, 128, 1030)])
def test_move(gpu, dh, heads, page, tokens):
    """Any slots to any others, left and taken in one call: permutations, shifts, slots
    outside the pool."""
    rng = np.random.default_rng(dh + tokens)
    pages = tokens // page + 3
    c = make_cache(gpu, rng, pages, page, heads, dh)
    total = pages * page
    print("move", dh, heads, page, tokens, flush=True)
    check_move(gpu, c, rng.integers(0, total, tokens).tolist(), rng.permutation(total)[:tokens].tolist(), "any")
    cycle = rng.permutation(total)[:tokens]
    check_move(gpu, c, cycle.tolist(), np.roll(cycle, 1).tolist(), "a cycle")
    check_move(gpu, c, list(range(1, tokens)), list(range(tokens - 1)), "one place down")
    src, dst = rng.integers(0, total, tokens), rng.permutation(total)[:tokens]
    src[::3], dst[1::4] = -1, total + rng.integers(0, 1 << 40, len(dst[1::4]))
    src[2::5] = -(1 << 62)
    check_move(gpu, c, src.tolist(), dst.tolist(), "outside the pool")


def test_move_nothing_to_do(gpu):
    rng = np.random.default_rng(0)
    c = make_cache(gpu, rng, 3, 16, 2, 64)
    check_move(gpu, c, [], [])
    check_move(gpu, c, [5], [5])
    check_move(gpu, c, [-1], [3])
    check_move(gpu, c, [3], [48])


def test_move_past_32_bits(gpu):
    from qppocr_amd import ops
    page, heads, dh = 1024, 8, 256
    pages = (1 << 32) // (page * heads * dh // 2) + 3
    c = ops.cache4(pages, page, heads, dh)
    rng = np.random.default_rng(0)
    last = pages * page - 700
    kv = gpu.from_numpy(rng.standard_normal((2, 700, heads, dh)).astype(np.float32)).cuda()
    at = gpu.arange(last, last + 700, device="cuda")
    ops.cache4_write(c, kv[0], kv[1], at)
    want = ops.cache4_read(c, at)
    for n in (40, 700):
        ops.cache4_move(c, at[:n], gpu.arange(5, 5 + n, device="cuda"))
        got = ops.cache4_read(c, gpu.arange(5, 5 + n, device="cuda"))
        assert all((host(a) == host(b[:n])).all() for a, b in zip(got, want))
        ops.cache4_move(c, gpu.arange(5, 5 + n, device="cuda"), at[:n])
        assert all((host(a) == host(b)).all() for a, b in zip(ops.cache4_read(c, at), want))


def test_move_captured(gpu):
    """Two captured moves of many tokens, in flight together: a workspace each."""
    from qppocr_amd import ops
    rng = np.random.default_rng(4)
    cs = [make_cache(gpu, rng, 60, 64, 8, 128) for _ in range(2)]
    n = 1800
    src = [gpu.zeros(n, dtype=gpu.int64, device="cuda") for _ in cs]
    dst = [gpu.arange(n, device="cuda") for _ in cs]
    graphs = []
    for c, s, d in zip(cs, src, dst):
        ops.cache4_move(c, s, s)
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            ops.cache4_move(c, s, d)
        graphs.append(g)
    side = gpu.cuda.Stream()
    for i in range(4):
        order = [rng.permutation(60 * 64) for _ in cs]
        for o, s, d in zip(order, src, dst):
            s.copy_(gpu.from_numpy(o[:n]))
            d.copy_(gpu.from_numpy(np.roll(o[:n], 3)))
        before = [pools(c) for c in cs]
        gpu.cuda.synchronize()
        graphs[0].replay()
        with gpu.cuda.stream(side):
            graphs[1].replay()
        gpu.cuda.synchronize()
        for c, o, was in zip(cs, order, before):
            s, d = o[:n], np.roll(o[:n], 3)
            for got, w in zip(pools(c), was):
                want = w.copy()
                want[d // 64, :, d % 64] = w[s // 64, :, s % 64]
                assert (got == want).all(), i


# ------------------------------------------------------- all of them together

@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_that_check_drafted_trees(gpu, dtype):
    """Prompts, then steps of a batch that draft a tree a sequence, turn its queries and
    keys by sheet, row and column, check it in one attention and keep one path: pages
    taken and given back, accepted tokens moved, a sequence that ends.  Every attention
    against 64 bits over the keys that the cache holds, and after each acceptance the
    cache against one that was written without drafts."""
    from qppocr_amd import ops
    rng = np.random.default_rng(7)
    t = getattr(gpu, dtype)
    batch, heads, group, dh, page, wide = 4, 2, 2, 64, 16, 12
    pages = batch * wide
    c, kept = ops.cache4(pages, page, heads, dh), ops.cache4(pages, page, heads, dh)
    i32 = dict(dtype=gpu.int32, device="cuda")
    table = gpu.full((batch, wide), -1, **i32)
    ring = gpu.from_numpy(rng.permutation(pages).astype(np.int32)).cuda()
    ends = gpu.tensor([0, pages], device="cuda")
    lens = gpu.zeros(batch, **i32)
    plan = ops.rotary_plan(dh, [1000.0 ** (-i / 32) for i in range(32)], [0] * 8 + [1] * 12 + [2] * 12)
    terms = {"float32": 3, "float16": 2, "bfloat16": 1}[dtype]
    host_lens = [0] * batch
    for step, news in enumerate(([20, 3, 17, 40], [5, 6, 7, 3], [6, 1, 9, 6], [8, 8, 2, 8], [7, 5, 3, 4])):
        print("drafted step", dtype, step, news, flush=True)
        if step == 3:
            gone = gpu.tensor([0, -host_lens[1], 0, 0], **i32)         # a sequence ends, another begins
            s = ops.cache4_extend(table, lens, gone, page, ring, ends, 0)
            lens, ends = s.lens, s.ends
            host_lens[1] = 0
        n = sum(news)
        parents = [p for m in news for p in ([-1] + list(range(m - 1)) if step == 0 else drafted(rng, m, 4))]
        s = ops.cache4_extend(table, lens, gpu.tensor(news, **i32), page, ring, ends, n,
                              gpu.tensor(parents, **i32), max(news))
        qkv = gpu.from_numpy(rng.standard_normal((n, heads * (group + 2), dh)).astype(np.float32)).cuda().to(t)
        sheet = gpu.stack([s.positions, s.positions // 10, s.positions % 10])
        qk = qkv[:, :heads * (group + 1)]
        ops.rotary(qk, sheet, plan, out=qk)
        q, k, v = qkv.split([heads * group, heads, heads], 1)
        ops.cache4_write(c, k, v, s.slots)
        y, sums = ops.attention_tree4(q, c, table, s.lens, dh ** -0.5, s.tree, starts=s.starts,
                                      max_new=max(news), lse=True)
        # the rows against 64 bits
        kd, vd = numbers(c)
        st, ln, tab = s.starts.tolist(), s.lens.tolist(), table.cpu().numpy()
        path, count, left = [], [], []
        for b in range(batch):
            assert ln[b] == host_lens[b] + news[b]
            see = paths(parents[st[b]:st[b + 1]])
            pos = np.arange(ln[b])
            pg = tab[b, pos // page]
            for i in range(news[b]):
                vis = (pos < host_lens[b]) | np.concatenate([np.zeros(host_lens[b], bool), see[i]])
                want, tol, (lse, ltol) = attend(host(q[st[b] + i]), kd[pg[vis], pos[vis] % page],
                                                    vd[pg[vis], pos[vis] % page], dh ** -0.5, terms, group)
                close(host(y[st[b] + i]), want, tol + half_step(gpu, t, want) * 1.001, f"step {step} row {b} {i}")
                close(host(sums[st[b] + i]), lse, ltol, f"step {step} sum {b} {i}")
            # one path is accepted: the deepest token's
            end = int(see.sum(1).argmax())
            path.append(np.flatnonzero(see[end]))
            count.append(len(path[-1]))
            left.append(news[b] - count[-1])
        src = gpu.cat([s.slots[st[b]:st[b + 1]][gpu.from_numpy(path[b]).cuda()] for b in range(batch)])
        dst = gpu.cat([s.slots[st[b]:st[b] + count[b]] for b in range(batch)])
        rows = gpu.cat([st[b] + gpu.from_numpy(path[b]).cuda() for b in range(batch)])
        ops.cache4_move(c, src, dst)
        ops.cache4_write(kept, k[rows], v[rows], dst)
        s2 = ops.cache4_extend(table, s.lens, gpu.tensor([-m for m in left], **i32), page, ring, s.ends, 0)
        lens, ends = s2.lens, s2.ends
        host_lens = [a + b for a, b in zip(host_lens, count)]
        assert lens.tolist() == host_lens
        tab = table.cpu().numpy()
        slots = np.concatenate([tab[b, np.arange(host_lens[b]) // page] * page + np.arange(host_lens[b]) % page
                                for b in range(batch)])
        at = gpu.from_numpy(slots.astype(np.int64)).cuda()
        for a, b in zip(ops.cache4_read(c, at), ops.cache4_read(kept, at)):
            assert (host(a) == host(b)).all(), f"step {step}: accepted tokens"
        # no page is held twice or lost
        held = [int(p) for b in range(batch) for p in tab[b, :-(-host_lens[b] // page)]]
        e = ends.tolist()
        free = [int(ring[i % pages]) for i in range(*e)]
        assert sorted(held + free) == list(range(pages)), f"step {step}: pages"


def test_other_streams(gpu):
    """Calls from several threads, each on a stream of its own, in its order."""
    import threading
    from qppocr_amd import ops
    rng = np.random.default_rng(16)
    plan = ops.rotary_plan(64, [50.0 ** (-i / 32) for i in range(32)])
    x0 = [gpu.from_numpy(rng.standard_normal((50, 3, 64)).astype(np.float32)).cuda() for _ in range(4)]
    pos = gpu.arange(50, dtype=gpu.int32, device="cuda")
    def chain(x):
        for i in range(40):
            x = ops.rotary(x, pos, plan, inverse=i % 3 == 0)
        return x
    want = [host(chain(x)) for x in x0]
    gpu.cuda.synchronize()
    got = [None] * 4
    def work(i):
        s = gpu.cuda.Stream()
        with gpu.cuda.stream(s):
            y = chain(x0[i])
            s.synchronize()
            got[i] = host(y)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for a, b in zip(got, want):
        assert (a == b).all()


def test_refusals(gpu):
    from qppocr_amd import ops
    i32 = dict(dtype=gpu.int32, device="cuda")
    table, lens, news = gpu.zeros((3, 4), **i32), gpu.zeros(3, **i32), gpu.zeros(3, **i32)
    ring, ends = gpu.arange(12, **i32), gpu.tensor([0, 12], device="cuda")
    def extend(table=table, lens=lens, news=news, page=16, ring=ring, ends=ends, tokens=5, **kw):
        return ops.cache4_extend(table, lens, news, page, ring, ends, tokens, **kw)
    extend()
    for bad, text in ((dict(table=table.long()), "page_table"), (dict(table=table.t()), "page_table"),
                      (dict(table=table[:1].expand(3, 4)), "overlaps"), (dict(lens=lens[:2]), "lens"),
                      (dict(news=news.long()), "news"), (dict(ends=ends.int()), "ends"),
                      (dict(ring=ring[:0]), "ring"), (dict(ring=ring[::2]), "ring"), (dict(tokens=-1), "negative"),
                      (dict(lens=lens.cpu()), "is on cpu"), (dict(parents=gpu.zeros(5, **i32)), "max_new"),
                      (dict(parents=gpu.zeros(4, **i32), max_new=3), "parents"),
                      (dict(news=table[0, :3]), "share memory"), (dict(ring=table[0]), "share memory")):
        with pytest.raises(ValueError, match=text):
            extend(**bad)
    for page in (8, 48, 1 << 16):
        with pytest.raises(Exception, match="page size"):
            extend(page=page)

    plan = ops.rotary_plan(32, [1.0, 0.5], [0, 1])
    x, pos = gpu.zeros((4, 2, 32), device="cuda"), gpu.zeros((2, 4), **i32)
    ops.rotary(x, pos, plan)
    for args, text in (((x.double(), pos), "float64"), ((x[..., :30], pos), "32"), ((x[0], pos), "32"),
                       ((x, pos.float()), "int32 or int64"), ((x, pos[:1]), "positions"),
                       ((x, pos[:, :3]), "positions"), ((x.cpu(), pos), "is on cpu"), ((x, pos.cpu()), "is on cpu"),
                       ((x.clone().requires_grad_(), pos), "gradient")):
        with pytest.raises(ValueError, match=text):
            ops.rotary(*args, plan)
    for out, text in ((x.half(), "out is"), (x[:3], "must be"), (x.flip(0)[:, :1].expand(4, 2, 32), "overlaps"),
                      (gpu.zeros((5, 2, 32), device="cuda")[1:], None)):
        if text:
            with pytest.raises(ValueError, match=text):
                ops.rotary(x, pos, plan, out=out)
        else:
            ops.rotary(x, pos, plan, out=out)
    base = gpu.zeros((5, 2, 32), device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        ops.rotary(base[:4], pos, plan, out=base[1:])
    for args in ((32, []), (32, [1.0] * 17), (32, [1.0], [0, 1]), (32, [math.inf]), (32, [1.0], [-1])):
        with pytest.raises(ValueError):
            ops.rotary_plan(*args)
    with pytest.raises(AttributeError):
        plan.turns = plan.turns.clone()

    c = ops.cache4(4, 16, 2, 64)
    at = gpu.arange(3, device="cuda")
    for args in ((at.int(), at), (at, at[:2]), (at[:, None], at), (at.cpu(), at), (at, at.cpu())):
        with pytest.raises(ValueError):
            ops.cache4_move(c, *args)
