"""The forms of the 4-bit operators' kernels that only particular sizes reach (many
tokens, splits of different numbers, rows of other groups, more new tokens than the
bound, wide linears of deep k), each activation, and the residual in place."""
import ctypes
import math

import numpy as np
import pytest

from test_gpu_decode4 import (DTYPES, HEAD_DIMS, attend_row, check_attention, close, decode, encode,
                              half_step, host, linear_reference, make_cache, numbers, tables)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- many tokens at once

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dh,page,tokens", [
    (8, 128, 64, 8192 + 3), (3, 64, 32, 81920 + 27), (1, 32, 16, 524288 + 4 * 64 + 1)])
def test_cache_many_tokens(gpu, dtype, heads, dh, page, tokens):
    """Long writes, and reads with four tokens in flight a thread (from 8192 workgroups'
    tokens on), the last group ragged, padded and bad slots among them: the bits of
    the same tokens in short calls; some of them against the definition."""
    from qppocr_amd import ops
    print("cache4 many", dtype, heads, dh, tokens, flush=True)
    t = getattr(gpu, dtype)
    g = gpu.Generator(device="cuda")
    g.manual_seed(tokens)
    pages = tokens // page + 2
    pool = [gpu.randint(0, 256, (pages, heads, page, dh // 2), generator=g, device="cuda", dtype=gpu.uint8),
            gpu.randint(121, 128, (pages, heads, page, dh // 32), generator=g, device="cuda", dtype=gpu.uint8)]
    pool += [x.flip(0).contiguous() for x in pool]
    c, d = ops.Cache4(*[x.clone() for x in pool]), ops.Cache4(*[x.clone() for x in pool])
    kv = gpu.randn((tokens, 2, heads, dh), generator=g, device="cuda").to(t)
    slots = gpu.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[5::97], slots[7::89], slots[-1] = -1, pages * page, -(1 << 40)
    slots[8:12] = -1                               # all four of a thread
    kv[5::97] = math.nan                           # a padded token may hold anything
    ops.cache4_write(c, kv[:, 0], kv[:, 1], slots)
    for i in range(0, tokens, 4000):
        ops.cache4_write(d, kv[i:i + 4000, 0], kv[i:i + 4000, 1], slots[i:i + 4000])
    for a, b in zip((c.k_codes, c.k_scales, c.v_codes, c.v_scales), (d.k_codes, d.k_scales, d.v_codes, d.v_scales)):
        assert gpu.equal(a, b)
    ok = (slots >= 0) & (slots < pages * page)
    assert not ok[-1] and ok[-2]
    some = gpu.cat([gpu.arange(0, 40, device="cuda"), gpu.arange(tokens - 40, tokens, device="cuda"),
                    gpu.randint(0, tokens, (200,), generator=g, device="cuda")])
    some = some[ok[some]]
    at, sh = host(slots[some]), host(kv[some])
    for i, (codes, scales) in enumerate(((c.k_codes, c.k_scales), (c.v_codes, c.v_scales))):
        code, scale = encode(sh[:, i])
        want = decode((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), scale)
        p, o = gpu.from_numpy(at // page).cuda(), gpu.from_numpy(at % page).cuda()
        close(decode(host(codes[p, :, o]), host(scales[p, :, o])), want, 0.0, f"stored {'kv'[i]}")
    k, v = ops.cache4_read(c, slots, t)
    for i in range(0, tokens, 4000):
        k2, v2 = ops.cache4_read(c, slots[i:i + 4000], t)
        assert gpu.equal(k[i:i + 4000], k2) and gpu.equal(v[i:i + 4000], v2)
    assert not k[~ok].any() and not v[~ok].any()
    for y, codes, scales in ((k, c.k_codes, c.k_scales), (v, c.v_codes, c.v_scales)):
        p, o = gpu.from_numpy(at // page).cuda(), gpu.from_numpy(at % page).cuda()
        want = gpu.from_numpy(decode(host(codes[p, :, o]), host(scales[p, :, o]))).to(t)
        close(host(y[some]), host(want), 0.0, "read")


# ------------------------------------------------------------------ attention

def sampled(torch, c, q, table, lens, news, scale, bound, rows, causal=True, max_len=None):
    """A call under the bound, its rows (sequence, new token) against the definition."""
    from qppocr_amd import ops
    st, i32 = [0] + list(np.cumsum(news)), dict(dtype=torch.int32, device="cuda")
    y, s = ops.attention_cache4(q, c, torch.tensor(table, **i32), torch.tensor(lens, **i32), scale,
                                starts=torch.tensor(st, **i32), max_new=bound, max_len=max_len or max(lens),
                                causal=causal, lse=True)
    y, s, qd = host(y), host(s), host(q)
    k, v = numbers(c)
    terms = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[q.dtype]
    for b, i in rows:
        pos = np.arange(max(0, lens[b] - news[b] + i + 1) if causal else lens[b])
        pg = np.array(table[b])[pos // c.page_size]
        want, tol, (lse, ltol) = attend_row(qd[st[b] + i], k[pg, pos % c.page_size], v[pg, pos % c.page_size],
                                            scale, terms, q.shape[1] // c.heads)
        close(y[st[b] + i], want, tol + half_step(torch, q.dtype, want) * 1.001, f"token {b} {i}")
        close(s[st[b] + i], lse, ltol, f"lse of token {b} {i}")


def chunks(torch, dtype, dh, heads, group, page, lens, news, seed):
    rng = np.random.default_rng(seed)
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(torch, rng, pages, page, heads, dh)
    q = torch.from_numpy(rng.standard_normal((sum(news), heads * group, dh)).astype(np.float32)).cuda()
    return c, q.to(getattr(torch, dtype)), tables(rng, pages, page, lens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("group,most", [(3, 350), (7, 150), (1, 1030)])
def test_attention_32_rows_of_odd_groups(gpu, dtype, dh, group, most):
    """Chunks long enough for 32 rows a wave (most new tokens a sequence times the
    group 1024 and more, in 512 waves and more), whose tokens' heads straddle the
    tiles.  (float32 past 64 elements a head: the other form.)"""
    print("attention 32 rows", dtype, dh, group, flush=True)
    news = [most, 3 * most // 4 + 1, most - 1, most // 2]
    lens = [most, most + 77, most + 160, most // 2 - 5]
    c, q, table = chunks(gpu, dtype, dh, 8, group, 32, lens, news, dh + group)
    rows = [(b, i) for b in range(4) for i in (0, 1, 10, 31, 33, news[b] // 2, news[b] - 2, news[b] - 1)]
    for causal in (True, False):
        sampled(gpu, c, q, table, lens, news, dh ** -0.5, most, rows, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh,group,news,lens,bound,max_len", [
    # four waves share 16 rows: a workgroup takes several tiles in turn
    (64, 4, [40, 3, 29], [50, 3, 100], 1, None), (128, 3, [33, 70], [90, 70], 2, None),
    (256, 2, [25], [61], 0, None), (96, 5, [50, 1], [200, 7], 1, 10),
    # the same with the keys split between workgroups
    (64, 2, [20, 9], [3000, 2100], 1, None), (192, 1, [37], [5000], 3, None),
    # 32 rows a wave
    (64, 4, [700, 512, 260, 300], [700, 600, 300, 300], 257, None),
    (128, 3, [800, 401, 100, 350], [900, 401, 120, 390], 345, 100)])
def test_attention_more_new_tokens_than_bound(gpu, dtype, dh, group, news, lens, bound, max_len):
    """max_new (and max_len) too small: slower, never wrong."""
    print("attention past its bound", dtype, dh, group, news, flush=True)
    heads = 8 if len(news) == 4 else 2
    c, q, table = chunks(gpu, dtype, dh, heads, group, 32, lens, news, dh + bound)
    rows = [(b, i) for b in range(len(news)) for i in sorted({0, 1, 5, 17, news[b] // 2, news[b] - 1}) if i < news[b]]
    sampled(gpu, c, q, table, lens, news, dh ** -0.5, bound, rows, max_len=max_len)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
@pytest.mark.parametrize("lens", [[1100, 0, 5], [4000, 3990, 17], [7000, 513], [40000]])
def test_attention_splits(gpu, dtype, dh, lens):
    """Keys split between few and many workgroups (joined by a wave or a workgroup a
    row), at every head dimension."""
    print("attention splits", dtype, dh, lens, flush=True)
    rng = np.random.default_rng(dh + len(lens))
    page = 128
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(gpu, rng, pages, page, 2, dh)
    q = gpu.from_numpy(rng.standard_normal((len(lens), 6, dh)).astype(np.float32)).cuda()
    q = q.to(getattr(gpu, dtype))
    check_attention(gpu, c, q, tables(rng, pages, page, lens), lens, dh ** -0.5, [1] * len(lens))


# --------------------------------------------------------------------- linear

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [
    (1, 2100, 4100), (3, 2100, 12300), (16, 1900, 8200), (9, 1100, 30001), (20, 2100, 17000), (25, 1100, 10000),
    (32, 1030, 8193), (17, 4100, 12288), (40, 2050, 4200), (64, 1300, 12300)])
def test_linear_wide_and_deep(gpu, dtype, rows, k, n):
    """More column tiles a workgroup with k for all of its waves."""
    from qppocr_amd import ops
    print("linear4 wide and deep", dtype, rows, k, n, flush=True)
    t = getattr(gpu, dtype)
    g = gpu.Generator(device="cuda")
    g.manual_seed(n + k)
    def r(*s):
        return gpu.randn(s, generator=g, device="cuda").to(t)
    w, x, b, e = ops.quantize4(r(k, n) / math.sqrt(k)), r(rows, k), r(n), r(rows, n)
    want, tol = linear_reference(gpu, x, w, b, 0, e)
    close(host(ops.linear4(x, w, b, 0, e)), want, tol + half_step(gpu, t, want) * 1.001, "linear4")


def call_linear4(torch, x, w, bias, act, residual, y):
    """qph_linear4 on torch's stream, as a C program calls it."""
    from qppocr_amd import _lib, ops
    p = lambda t: None if t is None else t.data_ptr()       # noqa: E731
    ops._enqueue(0, _lib.load().qph_linear4, x.data_ptr(), ops._DTYPES[x.dtype], x.stride(0), p(w.codes),
                 p(w.scales), p(bias), x.shape[0], w.k, w.n, None if act is None else ctypes.byref(act),
                 p(residual), p(y))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(1, 300, 77), (16, 1000, 5000), (30, 520, 130), (64, 640, 9001), (200, 300, 1000)])
def test_linear_residual_in_place(gpu, dtype, rows, k, n):
    """y may be the residual: the same bits as apart from it."""
    from qppocr_amd import ops
    print("linear4 in place", dtype, rows, k, n, flush=True)
    t = getattr(gpu, dtype)
    g = gpu.Generator(device="cuda")
    g.manual_seed(rows)
    w = ops.quantize4(gpu.randn((k, n), generator=g, device="cuda"))
    x, b = gpu.randn((rows, k), generator=g, device="cuda").to(t), gpu.randn(n, generator=g, device="cuda").to(t)
    e = gpu.randn((rows, n), generator=g, device="cuda").to(t)
    want = ops.linear4(x, w, b, 2, e)
    call_linear4(gpu, x, w, b, ops.act(2), e, e)
    assert gpu.equal(e, want)


ACTS = {
    "none": (0, 0.0, 0.0, 0.0), "gelu": (1, 1.4142135, 1.0, 0.5), "relu": (2, 0.0, 0.0, 0.0),
    "hardswish": (3, 1 / 6, 0.5, 0.0), "sigmoid": (4, 0.0, 0.0, 0.0), "hardsigmoid": (5, 0.2, 0.5, 0.0),
    "clip": (6, -0.75, 1.25, 0.0), "hardswish_clip": (7, 3.0, 6.0, 6.0)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(ACTS))
@pytest.mark.parametrize("rows", [3, 90])
def test_linear_activations(gpu, dtype, name, rows):
    """Every activation of the library, with its constants, in both kernels."""
    from qppocr_amd import _lib, ops
    print("linear4 activation", dtype, name, rows, flush=True)
    kind, *consts = ACTS[name]
    a, b, c = (float(np.float32(v)) for v in consts)
    t, k, n = getattr(gpu, dtype), 260, 150
    g = gpu.Generator(device="cuda")
    g.manual_seed(rows + kind)
    w = ops.quantize4(3.0 * gpu.randn((k, n), generator=g, device="cuda") / math.sqrt(k))
    x = gpu.randn((rows, k), generator=g, device="cuda").to(t)
    y = gpu.empty((rows, n), device="cuda", dtype=t)
    call_linear4(gpu, x, w, None, _lib.Act(kind, *consts), None, y)
    v, tol = linear_reference(gpu, x, w, None, 0, None)
    u = 2.0 ** -23
    # slope of the function times the sum's error, and the function's own roundings
    if kind == 0:
        want = v
    elif kind == 1:
        z = gpu.from_numpy(v)
        want = (z * 0.5 * gpu.erfc(-z / math.sqrt(2.0))).numpy()
        # (the constant is sqrt 2 to 24 bits, erfc good to a few units)
        tol = 1.13 * tol + (8 + 2 * np.abs(v) ** 2) * np.abs(want) * u + 2.0 ** -126
    elif kind == 2:
        want = np.maximum(v, 0.0)
    elif kind == 3:
        h = np.clip(v * a + b, 0, 1)
        want, tol = v * h, (1 + np.abs(v) * a) * tol + 4 * np.abs(v) * u
    elif kind == 4:
        want = 1.0 / (1.0 + np.exp(-v))
        # the exponential by six terms of its series past the power of two: r^7 / 5040 at
        # r = ln 2 / 2, 2^-22.5 of it, and its steps' roundings
        tol = tol / 4 + 8 * u * want
    elif kind == 5:
        want, tol = np.clip(v * a + b, 0, 1), a * tol + u * (np.abs(v * a) + 1)
    elif kind == 6:
        want = np.clip(v, a, b)
    else:
        want = v * np.clip(v + a, 0, b) / c
        tol = (b + np.abs(v)) / c * tol + 4 * u * np.abs(v) * (np.abs(v) + a + b) / c
    close(host(y), want, tol + half_step(gpu, t, want) * 1.001, name)


def test_cache_write_of_more_tokens_than_a_launch(gpu):
    """More workgroups than one launch takes (2^24 - 1, a token each): one row of keys
    and values for all tokens, all but a few at both sides of the border skipped."""
    from qppocr_amd import ops
    heads, dh, page, border = 64, 256, 16, (1 << 24) - 1
    print("cache4 write, two launches", flush=True)
    rng = np.random.default_rng(7)
    c = make_cache(gpu, rng, 2, page, heads, dh)
    want = [x.reshape(2 * page, heads, dh).copy() for x in numbers(c)]
    kv = gpu.from_numpy(rng.standard_normal((2, heads, dh)).astype(np.float32)).cuda().half()
    n = border + 5
    slots = gpu.full((n,), -1, dtype=gpu.int64, device="cuda")
    for t, slot in ((0, 3), (border - 1, 30), (border, 9), (n - 1, 17)):
        slots[t] = slot
    ops.cache4_write(c, kv[0].expand(n, heads, dh), kv[1].expand(n, heads, dh), slots)
    for i, x in enumerate(numbers(c)):
        code, scale = encode(host(kv[i]))
        want[i][[3, 30, 9, 17]] = decode((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), scale)
        close(x.reshape(2 * page, heads, dh), want[i], 0.0, f"stored {'kv'[i]}")
