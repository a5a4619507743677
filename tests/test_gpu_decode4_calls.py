"""The 4-bit operators' calls that a program makes in less usual ways (other default
types, scores and values of any size, bounds far from the work, in place), against
the same definitions in 64 bits as the other tests of these operators."""
import math

import numpy as np
import pytest

from test_gpu_decode4 import (DTYPES, attend_row, close, half_step, host, make_cache, numbers,
                              tables)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("default", ["bfloat16", "float64"])
@pytest.mark.parametrize("lens", [[20, 5, 33], [3000, 17, 2041]])
def test_lse_under_another_default_type(gpu, default, lens):
    """The sums' logarithms are float32 whatever torch's default type is."""
    from qppocr_amd import ops
    print("lse", default, lens, flush=True)
    rng = np.random.default_rng(2)
    pages = sum((n + 31) // 32 for n in lens) + 1
    c = make_cache(gpu, rng, pages, 32, 2, 64)
    q = gpu.from_numpy(rng.standard_normal((3, 4, 64)).astype(np.float32)).cuda().bfloat16()
    table = gpu.tensor(tables(rng, pages, 32, lens), dtype=gpu.int32, device="cuda")
    ln = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    y, s = ops.attention_cache4(q, c, table, ln, 0.125, lse=True)
    was = gpu.get_default_dtype()
    gpu.set_default_dtype(getattr(gpu, default))
    try:
        y2, s2 = ops.attention_cache4(q, c, table, ln, 0.125, lse=True)
    finally:
        gpu.set_default_dtype(was)
    assert s2.dtype == gpu.float32 and (host(y) == host(y2)).all() and (host(s) == host(s2)).all()


# -------------------------------------------------- scores of any finite size

# batch of one kernel form: cache heads, group, page, new tokens and lengths, rows checked
FORMS = {
    "short": (2, 2, 16, [1, 1, 3], [40, 7, 33], None),
    "split": (1, 4, 64, [1, 2], [3000, 1700], None),
    "rows": (8, 16, 32, [70, 64, 66, 69], [71, 200, 66, 150],
             [(0, 0), (0, 35), (0, 69), (1, 13), (1, 63), (2, 1), (2, 40), (3, 25), (3, 68)]),
}


def form_cache(torch, rng, form, dh, blocks):
    """A cache of the form whose keys are made by blocks(rng, shape) -> codes (one a
    byte), scale bytes, and its table."""
    heads, group, page, news, lens, _ = FORMS[form]
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(torch, rng, pages, page, heads, dh)
    code, scale = blocks(rng, (pages, heads, page, dh))
    c.k_codes.copy_(torch.from_numpy((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)))
    c.k_scales.copy_(torch.from_numpy(scale.astype(np.uint8)))
    return c, tables(rng, pages, page, lens)


def run_form(torch, c, form, table, q, scale):
    """The causal attention, and its rows as (out, lse, q, keys, values) per query
    head, in 64 bits."""
    from qppocr_amd import ops
    heads, group, page, news, lens, rows = FORMS[form]
    st = [0] + list(np.cumsum(news))
    i32 = dict(dtype=torch.int32, device="cuda")
    y, sums = ops.attention_cache4(q, c, torch.tensor(table, **i32), torch.tensor(lens, **i32), scale,
                                   starts=torch.tensor(st, **i32), max_new=max(news), max_len=max(lens),
                                   lse=True)
    y, sums, qd = host(y), host(sums), host(q)
    k, v = numbers(c)
    for b, i in rows or [(b, i) for b in range(len(news)) for i in range(news[b])]:
        pos = np.arange(lens[b] - news[b] + i + 1)
        pg = np.array(table[b])[pos // page]
        for h in range(heads * group):
            yield (f"token {b} {i} head {h}", y[st[b] + i, h], sums[st[b] + i, h], qd[st[b] + i, h],
                   k[pg, pos % page, h // group], v[pg, pos % page, h // group], (b, i))


def mean_of_values(p, off, v, kept):
    """The mean of v by the terms p, whose logarithms are off by at most `off`; what the
    sum's logarithm and the mean may then be off by (each addition a unit at most).
    Numbers below 2^-126 count as zeros: a term, each of its three bfloat16 parts and
    each of their products with a value (so four times 2^-126, times |v| or 1, a key)."""
    off = np.expm1(np.minimum(off, 1.0)) * p
    add = (len(p) / 32 + 100) * 2.0 ** -23
    d = off.sum() / p.sum() + add
    want = p @ v / p.sum()
    under = 4 * 2.0 ** -126 * (1 + np.abs(v)).sum(0)
    return want, d, (off @ np.abs(v) + (p @ np.abs(v)) * (d + kept + add) + under) / p.sum()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("power,scale", [
    (12, 0.5), (16, -0.5), (20, 0.5), (24, -1.0), (28, 0.125), (31, 0.5), (33, 0.3), (40, -0.5),
    (64, 0.25), (100, 0.5), (115, 4.0)])
def test_attention_large_scores(gpu, dtype, form, power, scale):
    """Whole and half numbers times 2^power, so that scores are exact and either
    equal or further apart than any exponential reaches: a row is the mean of the
    values of its largest score, however large that is."""
    print("attention large scores", dtype, form, power, scale, flush=True)
    rng = np.random.default_rng(power)
    heads, group, page, news, lens, _ = FORMS[form]
    dh = 64
    qp = min(power // 2, 12)                       # 7 2^12 fits float16
    t = getattr(gpu, dtype)

    def keys(rng, shape):
        return rng.integers(0, 16, shape), np.full(shape[:-1] + (shape[-1] // 32,), 127 + power - qp)
    c, table = form_cache(gpu, rng, form, dh, keys)
    q = rng.integers(-7, 8, (sum(news), heads * group, dh)) * 2.0 ** qp
    q[1::3] *= 2.0 ** -min(power, 34)              # rows of ordinary scores, and rows of none
    q[2::7] = 0.0
    q = gpu.from_numpy(q.astype(np.float32)).cuda().to(t)
    kept = 2.0 ** -23 if dtype == "float32" else 2.0 ** -16
    far = 0
    for name, y, lse, qd, k, v, _ in run_form(gpu, c, form, table, q, scale):
        z = (k @ qd) * float(np.float32(scale))    # exact in 64 bits but for the scale
        top = z.max()
        gap = top - z[z != top].max() if (z != top).any() else np.inf
        if gap < 200.0:
            # ordinary: exact scores; the constant's and the difference's own rounding
            p = np.exp(z - top)
            off = 2.0 ** -22 * (1 + np.abs(z - top))
        else:
            p, off, far = (z == top).astype(float), 0.0 * z, far + 1
        want, d, tol = mean_of_values(p, off, v, kept)
        close(y, want, tol + half_step(gpu, t, want) * 1.001, name)
        with np.errstate(over="ignore"):
            ref = np.float64(np.float32(top + np.log(p.sum())))
        close(np.array(lse), np.array(ref), 2.0 ** -21 * max(1.0, min(abs(ref), 3e38)) + d, name + " lse")
    assert far


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("common", [2 ** 15, -2 ** 18, 2 ** 19, 2 ** 20, -2 ** 21, 2 ** 22, -2 ** 23])
def test_attention_scores_with_a_large_common_part(gpu, dtype, form, common):
    """Scores that are whole numbers below 2^24, all of them near one large number:
    their differences count, and are exact."""
    print("attention common part", dtype, form, common, flush=True)
    rng = np.random.default_rng(abs(common) % 1000)
    heads, group, page, news, lens, _ = FORMS[form]
    dh, t = 64, getattr(gpu, dtype)

    def keys(rng, shape):
        code = np.zeros(shape, dtype=np.int64)
        code[..., 0] = 2                           # 1.0, times 2^11
        code[..., 32:] = rng.choice([0, 2, 4, 10, 12], shape[:-1] + (32,))      # 0, 1, 2, -1, -2
        scale = np.full(shape[:-1] + (2,), 127)
        scale[..., 0] = 127 + 11
        return code, scale
    c, table = form_cache(gpu, rng, form, dh, keys)
    q = np.zeros((sum(news), heads * group, dh))
    q[..., 0] = common / 2.0 ** 11
    q[..., 32:] = rng.integers(-1, 2, q[..., 32:].shape)
    q = gpu.from_numpy(q.astype(np.float32)).cuda().to(t)
    kept = 2.0 ** -23 if dtype == "float32" else 2.0 ** -16
    for name, y, lse, qd, k, v, _ in run_form(gpu, c, form, table, q, 1.0):
        z = k @ qd
        top = z.max()
        p = np.exp(z - top)
        want, d, tol = mean_of_values(p, 2.0 ** -22 * (1 + np.abs(z - top)), v, kept)
        close(y, want, tol + half_step(gpu, t, want) * 1.001, name)
        ref = top + np.log(p.sum())
        close(np.array(lse), np.array(ref), 2.0 ** -22 * abs(ref) + 2.0 ** -21 + d, name + " lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("common", [2 ** 10, 2 ** 19])
def test_attention_far_scores_before_ordinary_ones(gpu, dtype, form, common):
    """Rows whose first keys' scores lie far below zero (so far that the terms of
    their own running maximum overflow) and whose later ones do not, in every wave
    and split; neighbouring rows see no such keys' part of q."""
    print("attention far before", dtype, form, common, flush=True)
    rng = np.random.default_rng(common % 1000)
    heads, group, page, news, lens, _ = FORMS[form]
    dh, t = 64, getattr(gpu, dtype)
    where = {}

    def keys(rng, shape):
        code = np.zeros(shape, dtype=np.int64)
        code[..., 0] = 2                           # 1.0, times 2^20
        code[..., 32:] = rng.choice([0, 2, 4, 10, 12], shape[:-1] + (32,))      # 0, 1, 2, -1, -2
        scale = np.full(shape[:-1] + (2,), 127)
        scale[..., 0] = 127 + 20
        where.update(code=code)
        return code, scale
    c, table = form_cache(gpu, rng, form, dh, keys)
    code, step = where["code"], 128 if form == "split" else 16
    for b, n in enumerate(lens):                   # every other 128 (16) keys, from the first on
        for j in range(n):
            if j // step % 2 == 0:
                code[table[b][j // page], :, j % page, 1] = 15 if j % 3 else 14     # -6 or -4, times 2^20
    c.k_codes.copy_(gpu.from_numpy((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)))
    q = np.zeros((sum(news), heads * group, dh))
    q[..., 0] = common / 2.0 ** 20
    q[..., 1] = 2.0 ** 15
    q[1::2, :, 1] = 0.0
    q[..., 32:] = rng.integers(-1, 2, q[..., 32:].shape)
    q = gpu.from_numpy(q.astype(np.float32)).cuda().to(t)
    kept = 2.0 ** -23 if dtype == "float32" else 2.0 ** -16
    for name, y, lse, qd, k, v, _ in run_form(gpu, c, form, table, q, 1.0):
        z = k @ qd
        if z.max() < -2.0 ** 30:
            continue                               # (only such keys are seen: another test's)
        p = np.exp(z - z.max())
        want, d, tol = mean_of_values(p, np.where(p > 0, 2.0 ** -22 * (1 + np.abs(z - z.max())), 0.0), v, kept)
        close(y, want, tol + half_step(gpu, t, want) * 1.001, name)
        ref = z.max() + np.log(p.sum())
        close(np.array(lse), np.array(ref), 2.0 ** -22 * abs(ref) + 2.0 ** -21 + d, name + " lse")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", list(FORMS))
def test_attention_values_near_the_largest_number(gpu, dtype, form):
    """Values whose plain sum of n terms of at most 1 stays in float32's range, with
    scores that grow along the keys: no term is above 1."""
    print("attention large values", dtype, form, flush=True)
    rng = np.random.default_rng(5)
    heads, group, page, news, lens, _ = FORMS[form]
    dh, t = 64, getattr(gpu, dtype)
    c, table = form_cache(gpu, rng, form, dh, lambda rng, shape: (
        np.full(shape, 2), np.full(shape[:-1] + (2,), 127)))
    power = 127 - 3 - math.ceil(math.log2(max(lens)))        # 6 2^power, the longest sequence's times: below 2^127
    c.v_scales.fill_(127 + power)
    c.v_codes.bitwise_and_(0x33).bitwise_or_(0x44)           # 2 to 6, none negative
    code = np.full(c.k_codes.shape[:3] + (dh,), 2)           # 1.0
    for b, n in enumerate(lens):
        for j in range(n):                                   # 5.4 powers of two more every 32 keys, ...
            code[table[b][j // page], :, j % page, :j // 32 % 12] = 6        # ... 4.0 in place of 1.0
    c.k_codes.copy_(gpu.from_numpy((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)))
    q = gpu.full((sum(news), heads * group, dh), 1.25, device="cuda").to(t)
    kept = 2.0 ** -23 if dtype == "float32" else 2.0 ** -16
    for name, y, lse, qd, k, v, _ in run_form(gpu, c, form, table, q, 1.0):
        z = k @ qd
        p = np.exp(z - z.max())
        want, d, tol = mean_of_values(p, 2.0 ** -22 * (1 + np.abs(z - z.max())), v, kept)
        close(y, want, tol + half_step(gpu, t, want) * 1.001, name)
        ref = z.max() + np.log(p.sum())
        close(np.array(lse), np.array(ref), 2.0 ** -22 * abs(ref) + 2.0 ** -21 + d, name + " lse")


@pytest.mark.parametrize("dh,group,bound", [(256, 4, 1 << 17), (64, 2, 1 << 17), (64, 16, 1 << 20)])
def test_attention_bounds_far_past_the_new_tokens(gpu, dh, group, bound):
    """64 sequences of a few new tokens under a bound as one long prompt among them
    would need it (once 2^24 workgroups and more, which cannot be launched)."""
    print("attention bound", dh, group, bound, flush=True)
    rng = np.random.default_rng(dh)
    page, heads = 32, 8
    lens = [int(x) for x in rng.integers(1, 50, 64)]
    news = [int(x) for x in rng.integers(0, 4, 64)]
    news[5], lens[5] = 40, 60
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(gpu, rng, pages, page, heads, dh)
    table = tables(rng, pages, page, lens)
    st = [0] + list(np.cumsum(news))
    i32 = dict(dtype=gpu.int32, device="cuda")
    q = gpu.from_numpy(rng.standard_normal((st[-1], heads * group, dh)).astype(np.float32)).cuda().bfloat16()
    from qppocr_amd import ops
    args = q, c, gpu.tensor(table, **i32), gpu.tensor(lens, **i32), dh ** -0.5
    y, s = ops.attention_cache4(*args, starts=gpu.tensor(st, **i32), max_new=bound, lse=True)
    y, s, qd = host(y), host(s), host(q)
    k, v = numbers(c)
    for b in (0, 5, 6, 20, 63):
        for i in range(news[b]):
            pos = np.arange(max(0, lens[b] - news[b] + i + 1))
            pg = np.array(table[b])[pos // page]
            want, tol, (lse, ltol) = attend_row(qd[st[b] + i], k[pg, pos % page], v[pg, pos % page],
                                                dh ** -0.5, 1, group)
            close(y[st[b] + i], want, tol + half_step(gpu, q.dtype, want) * 1.001, f"token {b} {i}")
            close(s[st[b] + i], lse, ltol, f"lse of token {b} {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", list(FORMS))
def test_attention_in_place(gpu, dtype, form):
    """out may be q itself, packed among other rows: the same bits as apart from it."""
    from qppocr_amd import ops
    print("attention in place", dtype, form, flush=True)
    rng = np.random.default_rng(41)
    heads, group, page, news, lens, _ = FORMS[form]
    dh = 64
    c = make_cache(gpu, rng, sum((n + page - 1) // page for n in lens) + 1, page, heads, dh)
    table = tables(rng, c.pages, page, lens)
    st, i32 = [0] + list(np.cumsum(news)), dict(dtype=gpu.int32, device="cuda")
    packed = gpu.from_numpy(rng.standard_normal((st[-1], heads * group + 3, dh)).astype(np.float32))
    packed = packed.cuda().to(getattr(gpu, dtype))
    kept = packed.clone()
    q = packed[:, 2:2 + heads * group]
    args = c, gpu.tensor(table, **i32), gpu.tensor(lens, **i32), 0.125
    kw = dict(starts=gpu.tensor(st, **i32), max_new=max(news), max_len=max(lens))
    want = ops.attention_cache4(q, *args, **kw)
    assert ops.attention_cache4(q, *args, out=q, **kw) is q
    assert (host(q) == host(want)).all()
    assert (packed[:, :2] == kept[:, :2]).all() and (packed[:, 2 + heads * group:] == kept[:, 2 + heads * group:]).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", list(FORMS))
def test_attention_scores_past_the_largest_number(gpu, dtype, form):
    """Scores that overflow float32: minus infinity weighs nothing, plus infinity makes
    its row NaN; rows beside them do not change by a bit."""
    from qppocr_amd import ops
    print("attention overflowing scores", dtype, form, flush=True)
    rng = np.random.default_rng(19)
    heads, group, page, news, lens, _ = FORMS[form]
    dh, t = 64, getattr(gpu, dtype)

    def keys(rng, shape):
        code = np.zeros(shape, dtype=np.int64)
        code[..., 0] = rng.choice([0, 0, 15], shape[:-1])            # 0 or -6
        code[..., 32:] = rng.choice([0, 2, 4, 10, 12], shape[:-1] + (32,))
        return code, np.full(shape[:-1] + (2,), 127)
    c, table = form_cache(gpu, rng, form, dh, keys)
    q = np.zeros((sum(news), heads * group, dh))
    q[..., 32:] = rng.integers(-1, 2, q[..., 32:].shape)
    plain = gpu.from_numpy(q.astype(np.float32)).cuda().to(t)
    q[0::3, :, 0], q[1::3, :, 0] = 3e38, -3e38
    q = gpu.from_numpy(q.astype(np.float32)).cuda().to(t)
    st, i32 = [0] + list(np.cumsum(news)), dict(dtype=gpu.int32, device="cuda")
    ordinary = host(ops.attention_cache4(plain, c, gpu.tensor(table, **i32), gpu.tensor(lens, **i32), 1.0,
                                         starts=gpu.tensor(st, **i32), max_new=max(news), max_len=max(lens)))
    kept = 2.0 ** -23 if dtype == "float32" else 2.0 ** -16
    for name, y, lse, qd, k, v, (b, i) in run_form(gpu, c, form, table, q, 1.0):
        h = int(name.split()[-1])
        hidden = k[:, 0] < 0
        if qd[0] < 0 and hidden.any():
            assert np.isnan(y).all() and np.isnan(lse), name
        elif qd[0] > 0 and hidden.all():
            assert (y == 0).all() and lse == -np.inf, name
        elif qd[0] > 0:
            z = np.where(hidden, -np.inf, k[:, 32:] @ qd[32:])
            p = np.exp(z - z.max())
            off = np.where(hidden, 0.0, 2.0 ** -22 * (1 + np.abs(np.where(hidden, 0.0, z - z.max()))))
            want, d, tol = mean_of_values(p, off, v, kept)
            close(y, want, tol + half_step(gpu, t, want) * 1.001, name)
        else:
            assert (y == ordinary[st[b] + i, h]).all(), name
