"""The 4-bit operators against their definitions in 64 bits: quantising, the
paged cache's writes and reads (equal bit for bit), the linear and the
attention (within the roundings that their comments name), at the sizes, masks
and orders where they can go wrong; and a decoder's steps that use all of them.

Tolerances.  A float32 sum of n terms in any order that rounds (or cuts) each
addition is off by at most n 2^-23 of the sum of magnitudes; products with the
stored numbers are exact; an output is rounded once, by eps / 2 of its value.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6] + [-0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
DTYPES = ["float32", "float16", "bfloat16"]
HEAD_DIMS = [32, 64, 96, 128, 192, 256]


# ------------------------------------------------------------------ oracle

def encode(x):
    """Codes [..., k] and scale bytes [..., k / 32] of float64 x."""
    b = x.reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(b).all(-1)
    b = np.where(np.isfinite(b), b, 0.0)
    top = np.abs(b).max(-1)
    e = np.full(top.shape, -100)
    for _ in range(225):
        e = np.where((6.0 * np.ldexp(1.0, e) < top) & (e < 125), e + 1, e)
    y = np.abs(b) / np.ldexp(1.0, e)[..., None]
    # nearest level, ties to the even code: distances in the order of the codes,
    # even codes first
    order = [0, 2, 4, 6, 1, 3, 5, 7]
    d = np.abs(y[..., None] - LEVELS[order])
    code = np.array(order)[d.argmin(-1)]
    code = np.where(np.signbit(b) & (code > 0), code + 8, code)
    code[bad] = 0
    return code.reshape(x.shape), np.where(bad, 255, e + 127)


def decode(packed, scales):
    """Numbers of packed codes [..., k / 2] and scale bytes [..., k / 32]."""
    code = np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[:-1] + (-1,))
    two = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return LEVELS[code] * np.repeat(two, 32, -1)


def host(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def half_step(torch, dtype, y):
    """What rounding y to dtype may change, overflow and underflow aside."""
    f = torch.finfo(dtype)
    return np.maximum(np.abs(y) * f.eps / 2, f.tiny * f.eps / 2)


def close(got, want, tol, name):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{name}: NaN at {np.argwhere(np.isnan(got) != nan)[:4]}"
    same = (got == want) | nan
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= tol)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        pytest.fail(f"{name}: {bad.sum()} of {bad.size} off; at {i} {got[i]} for {want[i]}, "
                    f"tolerance {np.broadcast_to(tol, got.shape)[i]:.3g}")


# ---------------------------------------------------------------- quantise

def hard_blocks():
    """Blocks at the format's borders, [rows, 32] float32."""
    rng = np.random.default_rng(0)
    rows = [np.zeros(32), -np.zeros(32)]
    for e in (-110, -100, -99, -30, 0, 1, 60, 125):
        two = math.ldexp(1.0, e)
        ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
        near = np.concatenate([np.nextafter(ties.astype(np.float32), np.float32(0)),
                               np.nextafter(ties.astype(np.float32), np.float32(9))])
        rows.append(np.concatenate([ties, -ties, near]) * two)
        rows[-1][np.abs(rows[-1]) > 6 * two] = 6 * two      # (the step past 6 is a block of its own)
        for top in (6.0, np.nextafter(np.float32(6), np.float32(7)), 3.0,
                    np.nextafter(np.float32(3), np.float32(4)), 4.0):
            r = rng.uniform(-3, 3, 32) * two
            r[7] = -top * two
            rows.append(r)
    for v in (3.0e38, np.finfo(np.float32).max, 1e-38, 1e-45):
        r = rng.uniform(-1, 1, 32)
        r[3] = v
        rows += [r, np.full(32, -v)]
    for v in (np.inf, -np.inf, np.nan):
        r = rng.uniform(-1, 1, 32)
        r[31] = v
        rows.append(r)
    with np.errstate(over="ignore"):
        return np.stack(rows).astype(np.float32)


def check_weight(torch, w, got, k):
    """A Weight4 against the definition, w float64 [n, k] as quantised."""
    n, kp = w.shape[0], (k + 127) // 128 * 128
    full = np.zeros((n, kp))
    full[:, :k] = w
    code, scale = encode(full)
    assert tuple(got.codes.shape) == (n, kp // 2) and tuple(got.scales.shape) == (n, kp // 32)
    assert (host(got.scales) == scale).all()
    want = decode((code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8), scale)
    close(decode(host(got.codes), host(got.scales)), want, 0.0, "quantize4")


def test_quantize_borders(gpu):
    from qppocr_amd import ops
    x = gpu.from_numpy(hard_blocks())
    for name in DTYPES:
        print("quantize4 borders", name, flush=True)
        w = x.to(getattr(gpu, name)).cuda()
        check_weight(gpu, host(w), ops.quantize4(w.t()), 32)
        check_weight(gpu, host(w), ops.quantize4(w.t().contiguous()), 32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(1, 1), (31, 5), (33, 17), (128, 64), (129, 3), (1000, 250)])
def test_quantize_shapes(gpu, dtype, k, n):
    """Any layout of w [K, N]: contiguous, transposed, a slice of a larger one."""
    from qppocr_amd import ops
    print("quantize4", dtype, k, n, flush=True)
    rng = np.random.default_rng(k)
    big = gpu.from_numpy(rng.standard_normal((k + 3, 2 * n + 1)).astype(np.float32)).cuda()
    big = big.to(getattr(gpu, dtype))
    for w in (big[:k, :n].contiguous(), big[:k, :n].t().contiguous().t(), big[2:k + 2, 1:2 * n:2]):
        check_weight(gpu, host(w).T, ops.quantize4(w), k)


# ------------------------------------------------------------------- cache

def make_cache(torch, rng, pages, page, heads, dh, fill=True):
    """A Cache4 of random numbers, and (k, v) float64 [pages, page, heads, dh]."""
    from qppocr_amd import ops
    c = ops.cache4(pages, page, heads, dh)
    if fill:
        for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)):
            codes.copy_(torch.from_numpy(rng.integers(0, 256, codes.shape, dtype=np.uint8)))
            scales.copy_(torch.from_numpy(rng.integers(121, 128, scales.shape).astype(np.uint8)))
    return c


def numbers(c):
    """The cache's keys and values, float64 [pages, page, heads, dh]."""
    return [decode(host(a), host(b)).transpose(0, 2, 1, 3)
            for a, b in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh,heads,page,tokens", [
    (32, 1, 16, 1), (32, 5, 16, 33), (64, 3, 32, 40), (96, 2, 16, 7), (128, 8, 64, 130),
    (128, 1, 16, 300), (192, 3, 32, 21), (256, 16, 16, 19), (64, 40, 256, 3)])
def test_cache_write_read(gpu, dtype, dh, heads, page, tokens):
    """Writes out of a packed projection, padded and bad slots among them; the
    rest of the pool stays; reads give what is stored, in each type."""
    from qppocr_amd import ops
    print("cache4", dtype, dh, heads, page, tokens, flush=True)
    rng = np.random.default_rng(dh + tokens)
    t = getattr(gpu, dtype)
    pages = tokens // page + 3
    c = make_cache(gpu, rng, pages, page, heads, dh)
    before = [x.copy() for x in numbers(c)]
    qkv = gpu.from_numpy(rng.standard_normal((tokens, 3, heads, dh)).astype(np.float32) *
                         np.exp(rng.standard_normal((1, 3, heads, dh))).astype(np.float32))
    qkv = qkv.cuda().to(t)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 5:
        slots[1], slots[2], slots[4] = -1, pages * page, -(1 << 40)
        qkv[1] = math.nan              # a padded token may hold anything
        qkv[2] = math.inf
    ops.cache4_write(c, qkv[:, 1], qkv[:, 2], gpu.from_numpy(slots).cuda())
    ok = (slots >= 0) & (slots < pages * page)
    now = numbers(c)
    for i in range(2):
        want = before[i].reshape(pages * page, heads, dh)
        code, scale = encode(host(qkv[:, i + 1])[ok])
        want[slots[ok]] = decode((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), scale)
        close(now[i].reshape(want.shape), want, 0.0, f"stored {'kv'[i]}")
    for out_t in DTYPES:
        k, v = ops.cache4_read(c, gpu.from_numpy(slots).cuda(), getattr(gpu, out_t))
        for i, y in enumerate((k, v)):
            flat = now[i].reshape(pages * page, heads, dh)
            want = np.where(ok[:, None, None], flat[np.where(ok, slots, 0)], 0.0)
            want = host(gpu.from_numpy(want).to(getattr(gpu, out_t)))
            close(host(y), want, 0.0, f"read {'kv'[i]}")


def test_cache_hard_numbers(gpu):
    """Infinities, NaN, the largest and the smallest numbers, through the cache."""
    from qppocr_amd import ops
    x = gpu.from_numpy(hard_blocks()).cuda()
    n = x.shape[0]
    c = ops.cache4((n + 15) // 16, 16, 1, 32)
    slots = gpu.arange(n, device="cuda")
    ops.cache4_write(c, x.view(n, 1, 32), x.flip(0).reshape(n, 1, 32), slots)
    code, scale = encode(host(x))
    want = decode((code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8), scale)
    k, v = ops.cache4_read(c, slots)
    close(host(k)[:, 0], want, 0.0, "k")
    close(host(v)[:, 0], want[::-1], 0.0, "v")
    # an element is off by at most the block's scale
    fine = np.isfinite(want).all(1) & (np.abs(host(x)).max(1) <= 6 * 2.0 ** 125)
    two = np.ldexp(1.0, scale[fine] - 127)
    assert (np.abs(want[fine] - host(x)[fine]) <= two).all()


def test_cache_nothing_to_do(gpu):
    from qppocr_amd import ops
    rng = np.random.default_rng(1)
    c = make_cache(gpu, rng, 2, 16, 2, 64)
    before = numbers(c)
    none = gpu.empty((0,), dtype=gpu.int64, device="cuda")
    ops.cache4_write(c, gpu.empty((0, 2, 64), device="cuda"), gpu.empty((0, 2, 64), device="cuda"), none)
    k, v = ops.cache4_read(c, none)
    assert tuple(k.shape) == tuple(v.shape) == (0, 2, 64)
    skip = gpu.full((9,), -1, dtype=gpu.int64, device="cuda")
    ops.cache4_write(c, gpu.ones((9, 2, 64), device="cuda"), gpu.ones((9, 2, 64), device="cuda"), skip)
    for a, b in zip(before, numbers(c)):
        assert (a == b).all()


def test_cache_past_32_bits(gpu):
    """A pool whose codes and scales lie past 4 GiB, written, read and attended to there."""
    from qppocr_amd import ops
    page, heads, dh = 1024, 8, 256
    pages = (1 << 32) // (page * heads * dh // 2) + 40
    c = ops.cache4(pages, page, heads, dh)
    assert c.k_codes.numel() > 1 << 32
    rng = np.random.default_rng(3)
    n = 300
    kv = gpu.from_numpy(rng.standard_normal((2, n, heads, dh)).astype(np.float32)).cuda()
    order = np.array([pages - 1, 3, pages - 7])
    slots = order[np.arange(n) // 128] * page + np.arange(n) % 128
    ops.cache4_write(c, kv[0], kv[1], gpu.from_numpy(slots).cuda())
    code, scale = encode(host(kv))
    want = decode((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), scale)
    k, v = ops.cache4_read(c, gpu.from_numpy(slots).cuda())
    close(host(k), want[0], 0.0, "k")
    close(host(v), want[1], 0.0, "v")
    q = gpu.from_numpy(rng.standard_normal((1, heads, dh)).astype(np.float32)).cuda()
    table = gpu.tensor([[pages - 1]], dtype=gpu.int32, device="cuda")
    lens = gpu.tensor([128], dtype=gpu.int32, device="cuda")
    out = ops.attention_cache4(q, c, table, lens, dh ** -0.5)
    y, tol, _ = attend_row(host(q)[0], want[0][:128], want[1][:128], dh ** -0.5, 3, 1)
    close(host(out)[0], y, tol + half_step(gpu, gpu.float32, y), "attention")


# ------------------------------------------------------------------ linear

def linear_reference(torch, x, w4, bias, act, res):
    """float64 result and the tolerance before the output's rounding."""
    w = decode(host(w4.codes), host(w4.scales))[:, :w4.k]
    xd = host(x)
    with np.errstate(invalid="ignore"):
        y = xd @ w.T
        tol = (w4.k + 24) * 2.0 ** -23 * (np.abs(xd) @ np.abs(w).T)
    if bias is not None:
        y = y + host(bias)
        tol = tol + np.abs(y) * 2.0 ** -24
    if act == 1:
        t = torch.from_numpy(y)
        y = (t * 0.5 * torch.erfc(-t / math.sqrt(2.0))).numpy()
        # GELU's slope is below 1.13; erfc is good to a few units, its argument to one
        tol = 1.13 * tol + (8 + 2 * np.abs(t.numpy()) ** 2) * np.abs(y) * 2.0 ** -23 + 2.0 ** -126
    elif act == 2:
        y = np.where(y > 0, y, 0.0)
    elif act == 3:
        a = np.clip(y / 6.0 + 0.5, 0, 1)
        tol = 2 * tol + np.abs(y) * 2.0 ** -22
        y = y * a
    if res is not None:
        y = y + host(res)
        tol = tol + np.abs(y) * 2.0 ** -24
    return y, tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n,act,bias,res", [
    (1, 1, 1, 0, True, False), (1, 32, 16, 0, False, False), (2, 100, 17, 1, True, True),
    (15, 128, 33, 2, True, False), (16, 129, 250, 3, False, True), (17, 1000, 40, 0, True, False),
    (33, 256, 65, 1, False, False), (64, 384, 31, 0, False, True), (65, 640, 130, 2, True, True),
    (130, 96, 257, 0, True, True), (3, 4100, 48, 0, True, False), (5, 2048, 1023, 1, True, True),
    (200, 520, 100, 0, False, False)])
def test_linear(gpu, dtype, rows, k, n, act, bias, res):
    from qppocr_amd import ops
    print("linear4", dtype, rows, k, n, act, flush=True)
    t = getattr(gpu, dtype)
    rng = np.random.default_rng(rows * 1000 + k)
    def r(*s):
        return gpu.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().to(t)
    w = ops.quantize4(r(k, n) / math.sqrt(k))
    x = r(rows, k + 5)[:, 3:3 + k]              # rows apart, and off every wide load's border
    b, e = (r(n) if bias else None), (r(rows, n) if res else None)
    y = ops.linear4(x, w, b, act, e)
    assert y.dtype == t
    want, tol = linear_reference(gpu, x, w, b, act, e)
    close(host(y), want, tol + half_step(gpu, t, want) * 1.001, "linear4")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(1, 256, 64), (16, 1024, 48), (40, 640, 130), (100, 2000, 96)])
def test_linear_whole_numbers(gpu, dtype, rows, k, n):
    """Whole numbers whose sums stay below 2^24: exact in any order."""
    from qppocr_amd import ops
    t = getattr(gpu, dtype)
    rng = np.random.default_rng(k)
    x = gpu.from_numpy(rng.integers(-3, 4, (rows, k)).astype(np.float32)).cuda().to(t)
    code = rng.integers(0, 16, (n, (k + 127) // 128 * 128))
    code[:, k:] = 0
    packed = (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)
    scales = rng.integers(128, 131, (n, code.shape[1] // 32)).astype(np.uint8)
    w = ops.Weight4(gpu.from_numpy(packed).cuda(), gpu.from_numpy(scales).cuda(), k)
    want = host(x) @ decode(packed, scales)[:, :k].T
    assert np.abs(want).max() < 1 << 24 and (np.abs(host(x)) @ np.abs(decode(packed, scales)[:, :k]).T).max() < 1 << 24
    y = ops.linear4(x, w)
    assert (host(y) == host(gpu.from_numpy(want).to(t))).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [
    (130, 300, 8330), (200, 70, 5500), (64, 200, 16500), (70, 520, 6100), (32, 260, 13000),
    (20, 140, 17000), (321, 1100, 4227), (64, 1030, 6200), (49, 513, 16421), (9, 700, 16999)])
def test_linear_more_than_a_round(gpu, dtype, rows, k, n):
    """Rows and columns at both sides of where the workgroups of a form no
    longer go into one round."""
    from qppocr_amd import ops
    print("linear4 rounds", dtype, rows, k, n, flush=True)
    t = getattr(gpu, dtype)
    rng = np.random.default_rng(n + k)
    def r(*s):
        return gpu.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().to(t)
    w, x, b, e = ops.quantize4(r(k, n) / math.sqrt(k)), r(rows, k + 1)[:, 1:], r(n), r(rows, n)
    want, tol = linear_reference(gpu, x, w, b, 0, e)
    close(host(ops.linear4(x, w, b, 0, e)), want, tol + half_step(gpu, t, want) * 1.001, "linear4")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [
    (1, 96, 4100), (16, 130, 8200), (3, 40, 12300), (30, 257, 4112), (25, 384, 12290), (60, 300, 2500),
    (48, 520, 16400), (47, 260, 16385), (66, 768, 8260), (129, 1100, 500), (70, 2600, 64)])
def test_linear_wide(gpu, dtype, rows, k, n):
    """Shapes that take more columns a workgroup, more rows, and more parts of
    k than are in flight at once."""
    from qppocr_amd import ops
    print("linear4 wide", dtype, rows, k, n, flush=True)
    t = getattr(gpu, dtype)
    rng = np.random.default_rng(n + k)
    def r(*s):
        return gpu.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().to(t)
    w, x, b, e = ops.quantize4(r(k, n) / math.sqrt(k)), r(rows, k), r(n), r(rows, n)
    want, tol = linear_reference(gpu, x, w, b, 0, e)
    close(host(ops.linear4(x, w, b, 0, e)), want, tol + half_step(gpu, t, want) * 1.001, "linear4")


@pytest.mark.parametrize("rows", [1, 20, 70])
@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** -22, 2.0 ** -12, 2.0 ** 12, 2.0 ** 20, 0.0])
def test_linear_weights_of_any_size(gpu, rows, size):
    """float16 x against weights inside and outside of float16's range, mixed
    with ordinary ones and with blocks of zeros."""
    from qppocr_amd import ops
    print("linear4 sizes", rows, size, flush=True)
    rng = np.random.default_rng(rows)
    k, n = 700, 90
    x = gpu.from_numpy((rng.standard_normal((rows, k)) * np.exp(rng.uniform(-9, 3, (rows, k))))
                       .astype(np.float32)).cuda().half()
    x[0, 5] = 2.0 ** -24                 # the smallest of all
    for mixed in (False, True):
        w = rng.standard_normal((k, n)) * size
        if mixed:
            w[64:96, ::3] = rng.standard_normal((32, 30)) * 0.1
            w[300:400] = 0.0
        w4 = ops.quantize4(gpu.from_numpy(w.astype(np.float32)).cuda())
        want, tol = linear_reference(gpu, x, w4, None, 0, None)
        got = ops.linear4(x, w4)
        big = gpu.from_numpy(want).half()           # (past 65504: an infinity, as rounding gives)
        assert (gpu.isinf(got).cpu() == gpu.isinf(big)).all() or size >= 2.0 ** 12
        fine = np.abs(want) < 6.0e4
        close(np.where(fine, host(got), 0), np.where(fine, want, 0),
              tol + half_step(gpu, gpu.float16, want) * 1.001, f"size {size} {mixed}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_keeps_every_bit(gpu, dtype):
    """A weight that picks one input times 1: the input itself, all its bits,
    the largest and infinities among them."""
    from qppocr_amd import ops
    t = getattr(gpu, dtype)
    rng = np.random.default_rng(8)
    k = n = 64
    x = rng.standard_normal((20, k)) * np.exp(rng.uniform(-12, 9, (20, k)))
    x = gpu.from_numpy(x).cuda().to(t)
    f = gpu.finfo(t)
    x[3, 5], x[4, 6], x[5, 7] = f.max, -f.max, f.tiny
    pick = rng.permutation(k)
    w = gpu.zeros((k, n), device="cuda")
    w[gpu.from_numpy(pick).cuda(), gpu.arange(n, device="cuda")] = 1.0
    y = ops.linear4(x, ops.quantize4(w))
    assert (host(y) == host(x)[:, pick]).all()


def test_linear_infinities_stay_in_their_rows(gpu):
    from qppocr_amd import ops
    rng = np.random.default_rng(9)
    for dtype in DTYPES:
        t = getattr(gpu, dtype)
        x = gpu.from_numpy(rng.standard_normal((21, 130)).astype(np.float32)).cuda().to(t)
        wf = gpu.from_numpy(rng.uniform(0.5, 1.0, (130, 37)).astype(np.float32)).cuda()
        w = ops.quantize4(wf)
        clean = host(ops.linear4(x, w))
        x[2, 129], x[7, 0], x[20, 64] = math.inf, math.nan, -math.inf
        got = host(ops.linear4(x, w))
        assert (got[2] == math.inf).all() and np.isnan(got[7]).all() and (got[20] == -math.inf).all()
        rest = [i for i in range(21) if i not in (2, 7, 20)]
        assert (got[rest] == clean[rest]).all()
        wf[40, 3] = math.nan            # a weight's block of NaN: its output column only
        got2 = host(ops.linear4(x, ops.quantize4(wf)))
        cols = [j for j in range(37) if j != 3]
        assert np.isnan(got2[:, 3]).all() and (got2[rest][:, cols] == got[rest][:, cols]).all()


def test_linear_forms(gpu):
    """Leading dimensions, one row as a vector, no rows, the residual in place."""
    from qppocr_amd import ops
    rng = np.random.default_rng(10)
    w = ops.quantize4(gpu.from_numpy(rng.standard_normal((96, 50)).astype(np.float32)).cuda())
    x = gpu.from_numpy(rng.standard_normal((3, 4, 96)).astype(np.float32)).cuda()
    y = ops.linear4(x, w)
    assert tuple(y.shape) == (3, 4, 50)
    assert (host(ops.linear4(x[1, 2], w)) == host(y)[1, 2]).all()
    assert (host(ops.linear4(x.transpose(0, 1), w)) == host(y).transpose(1, 0, 2)).all()
    assert tuple(ops.linear4(x[:0], w).shape) == (0, 4, 50)
    assert tuple(ops.linear4(x[0, :, :1].expand(4, 96), w).shape) == (4, 50)


# --------------------------------------------------------------- attention

def attend_row(q, k, v, scale, terms, group):
    """One token's attention in float64: q [heads, dh], visible k, v [n, cache
    heads, dh]: out, tolerance, log of the sums and its tolerance."""
    heads, dh = q.shape
    out, tol = np.zeros((heads, dh)), np.zeros((heads, dh))
    lse, ltol = np.full(heads, -np.inf), np.zeros(heads)
    n = k.shape[0]
    for h in range(heads if n else 0):
        kh, vh = k[:, h // group], v[:, h // group]
        s = kh @ q[h] * scale
        big = (np.abs(kh) @ np.abs(q[h]) * abs(scale))
        # a score's sum of dh terms (of each of the split's products), the
        # scaling, the exponent's argument and the exponential's own unit
        if np.isnan(s).all():
            out[h] = lse[h] = np.nan
            continue
        d = ((dh * terms + 8) * 2.0 ** -23 * np.nanmax(big) + 2.0 ** -21 * np.nanmax(np.abs(s)) +
             2.0 ** -22)
        top = s.max()
        p = np.exp(s - top)
        lse[h] = top + np.log(p.sum())
        p /= p.sum()
        # additions: a key enters a chain of at most n / 32 tiles and 64 joins
        add = (n / 32 + 96) * 2.0 ** -23
        kept = 2.0 ** -16 if terms < 3 else 2.0 ** -23
        with np.errstate(invalid="ignore"):
            out[h] = p @ vh
            tol[h] = (2 * np.expm1(d) + kept + 2 * add) * (p @ np.abs(vh))
        ltol[h] = d + add + 2.0 ** -22 * max(1.0, abs(lse[h]))
    return out, tol, (lse, ltol)


def check_attention(torch, c, q, table, lens, scale, news, causal=True, window=0, starts=None,
                    use_max_len=None, out=None, name="attention"):
    """Runs and checks a call; table, lens, news are host lists."""
    from qppocr_amd import ops
    k, v = numbers(c)
    t = q.dtype
    terms = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[t]
    group = q.shape[1] // c.heads
    tab = torch.tensor(table, dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if starts is None:
        starts = [0] + list(np.cumsum(news))
    uniform = len(set(news)) == 1 and starts[0] == 0 and starts[-1] == q.shape[0]
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    outs = []
    calls = [dict(starts=st, max_new=max(news))]
    if uniform:
        calls.append({})
    for kw in calls:
        if use_max_len:
            kw["max_len"] = use_max_len
        y, sums = ops.attention_cache4(q, c, tab, ln, scale, causal=causal, window=window, lse=True,
                                       out=None if out is None else out, **kw)
        outs.append((host(y), host(sums)))
    qd = host(q)
    page, seen_rows = c.page_size, 0
    for b, n in enumerate(lens):
        n = min(n, len(table[b]) * page)
        pos = np.arange(n)
        pg = np.array(table[b] + [-1], dtype=np.int64)[pos // page] if n else np.zeros(0, np.int64)
        there = (pg >= 0) & (pg < c.pages)
        for i in range(news[b]):
            p, row = n - news[b] + i, starts[b] + i
            see = there & (pos < n)
            if causal:
                see &= pos <= p
            if window:
                see &= pos > p - window
            kk = k[pg[see], pos[see] % page]
            vv = v[pg[see], pos[see] % page]
            want, tol, (lse, ltol) = attend_row(qd[row], kk, vv, scale, terms, group)
            for y, sums in outs:
                close(y[row], want, tol + half_step(torch, t, want) * 1.001, f"{name}: row {row}")
                close(sums[row], lse, ltol, f"{name}: lse of row {row}")
            seen_rows += 1
    return outs[0]


def tables(rng, pages, page, lens, width=None):
    """A page table of distinct pages in random order, -1 past each sequence's."""
    need = [(n + page - 1) // page for n in lens]
    width = width or max(1, max(need))
    order, at, out = list(rng.permutation(pages)), 0, []
    for m in need:
        out.append([int(x) for x in order[at:at + m]] + [-1] * (width - m))
        at += m
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", HEAD_DIMS)
def test_attention_steps(gpu, dtype, dh):
    """One token of each sequence: lengths at the borders of pages and tiles,
    slots without a sequence, groups of one and more query heads."""
    rng = np.random.default_rng(dh)
    t = getattr(gpu, dtype)
    lens = [1, 0, 15, 16, 17, 31, 33, 64, 127, 128, 129, 300, 700]
    for page, heads, group in ((16, 2, 1), (32, 1, 4), (256, 3, 7)):
        print("attention step", dtype, dh, page, heads, group, flush=True)
        pages = sum((n + page - 1) // page for n in lens) + 2
        c = make_cache(gpu, rng, pages, page, heads, dh)
        q = gpu.from_numpy(rng.standard_normal((len(lens), heads * group, dh)).astype(np.float32))
        q = q.cuda().to(t)
        check_attention(gpu, c, q, tables(rng, pages, page, lens), lens, dh ** -0.5, [1] * len(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh,heads,group,news,lens,causal,window", [
    (64, 2, 4, [5, 1, 8], [40, 1, 8], True, 0),
    (128, 1, 1, [3, 7, 2], [2, 7, 0], True, 0),          # more new tokens than cached ones
    (32, 2, 3, [33, 1, 20], [33, 200, 64], True, 17),
    (96, 1, 16, [2, 2], [100, 31], False, 0),
    (64, 1, 2, [4, 9], [90, 9], False, 13),
    (192, 1, 2, [40], [130], True, 64),
    (256, 2, 1, [17, 3], [40, 400], True, 1),
    (128, 1, 8, [50, 0, 70], [300, 9, 70], True, 0)])
def test_attention_chunks(gpu, dtype, dh, heads, group, news, lens, causal, window):
    print("attention chunk", dtype, dh, heads, group, news, lens, causal, window, flush=True)
    rng = np.random.default_rng(dh + sum(news))
    page = 16
    pages = sum((n + page - 1) // page for n in lens) + 2
    c = make_cache(gpu, rng, pages, page, heads, dh)
    q = gpu.from_numpy(rng.standard_normal((sum(news), heads * group, dh)).astype(np.float32))
    q = q.cuda().to(getattr(gpu, dtype))
    check_attention(gpu, c, q, tables(rng, pages, page, lens), lens, 0.7 * dh ** -0.5, news, causal,
                    window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
def test_attention_many_rows(gpu, dtype, dh):
    """Chunks of enough sequences and heads that a wave takes more rows alone."""
    rng = np.random.default_rng(dh)
    heads, group, page = 64, 2, 32
    news, lens = [64, 37, 64, 50, 64, 61, 63, 64], [64, 80, 70, 50, 96, 61, 100, 65]
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(gpu, rng, pages, page, heads, dh)
    print("attention many rows", dtype, dh, flush=True)
    q = gpu.from_numpy(rng.standard_normal((sum(news), heads * group, dh)).astype(np.float32))
    q = q.cuda().to(getattr(gpu, dtype))
    from qppocr_amd import ops
    table = tables(rng, pages, page, lens)
    st = [0] + list(np.cumsum(news))
    y = host(ops.attention_cache4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                  gpu.tensor(lens, dtype=gpu.int32, device="cuda"), dh ** -0.5,
                                  starts=gpu.tensor(st, dtype=gpu.int32, device="cuda"), max_new=64))
    k, v = numbers(c)
    terms = {"float32": 3, "float16": 2, "bfloat16": 1}[dtype]
    qd = host(q)
    for b, i in ((0, 0), (0, 31), (0, 63), (1, 5), (1, 36), (3, 49), (4, 17), (6, 62), (7, 0)):
        n = lens[b] - news[b] + i + 1
        pos = np.arange(n)
        pg = np.array(table[b])[pos // page]
        want, tol, _ = attend_row(qd[st[b] + i], k[pg, pos % page], v[pg, pos % page], dh ** -0.5, terms,
                                  group)
        close(y[st[b] + i], want, tol + half_step(gpu, q.dtype, want) * 1.001, f"token {b} {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 40), (False, 0)])
def test_attention_rows_of_their_own(gpu, dtype, dh, causal, window):
    """Chunks long enough that a wave takes 32 rows alone (float32: up to 64
    elements): odd lengths, a hole in the pages, a key's and a value's block of
    NaN, garbage behind the last token, rows before the first key."""
    from qppocr_amd import ops
    rng = np.random.default_rng(dh + window)
    heads, group, page = 8, 16, 32
    news, lens = [70, 64, 0, 66, 69], [71, 200, 40, 64, 150]
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(gpu, rng, pages, page, heads, dh)
    table = tables(rng, pages, page, lens)
    table[4][1] = -1                                   # keys 32 to 63 of the last sequence
    for p, n in ((table[0][2], 71 % page), (table[1][6], 200 % page)):
        c.k_scales[p, :, n:], c.v_scales[p, :, n:] = 255, 255
    c.v_scales[table[1][4], 3, 20, 0] = 255            # value 148 of head 3, sequence 1
    c.k_scales[table[4][3], 5, 10, 0] = 255            # key 106 of head 5, sequence 4
    print("attention rows of their own", dtype, dh, causal, window, flush=True)
    q = gpu.from_numpy(rng.standard_normal((sum(news), heads * group, dh)).astype(np.float32))
    q = q.cuda().to(getattr(gpu, dtype))
    st = [0] + list(np.cumsum(news))
    y, sums = ops.attention_cache4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                   gpu.tensor(lens, dtype=gpu.int32, device="cuda"), dh ** -0.5,
                                   starts=gpu.tensor(st, dtype=gpu.int32, device="cuda"), max_new=70,
                                   causal=causal, window=window, lse=True)
    y, sums, qd = host(y), host(sums), host(q)
    k, v = numbers(c)
    terms = {"float32": 3, "float16": 2, "bfloat16": 1}[dtype]
    for b, i in ((0, 0), (0, 35), (0, 69), (1, 0), (1, 11), (1, 12), (1, 13), (1, 63), (3, 0), (3, 1),
                 (3, 2), (3, 40), (3, 65), (4, 0), (4, 24), (4, 25), (4, 26), (4, 68)):
        p = lens[b] - news[b] + i
        pos = np.arange(lens[b])
        pg = np.array(table[b])[pos // page]
        see = pg >= 0
        if causal:
            see &= pos <= p
        if window:
            see &= pos > p - window
        want, tol, (lse, ltol) = attend_row(qd[st[b] + i], k[pg[see], pos[see] % page],
                                            v[pg[see], pos[see] % page], dh ** -0.5, terms, group)
        close(y[st[b] + i], want, tol + half_step(gpu, q.dtype, want) * 1.001, f"token {b} {i}")
        close(sums[st[b] + i], lse, ltol, f"lse of token {b} {i}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_long(gpu, dtype):
    """Contexts that many workgroups share, and bounds that are too small or
    too large for them."""
    rng = np.random.default_rng(77)
    lens, page = [9000, 3, 0, 4097], 64
    pages = sum((n + page - 1) // page for n in lens) + 1
    c = make_cache(gpu, rng, pages, page, 1, 128)
    q = gpu.from_numpy(rng.standard_normal((4, 4, 128)).astype(np.float32)).cuda()
    q = q.to(getattr(gpu, dtype))
    table = tables(rng, pages, page, lens)
    got = []
    for bound in (9000, 300, 5000, 1 << 20):
        print("attention long", dtype, bound, flush=True)
        got.append(check_attention(gpu, c, q, table, lens, 128 ** -0.5, [1] * 4, use_max_len=bound))
    check_attention(gpu, c, q, table, lens, 128 ** -0.5, [1] * 4, window=2500)
    check_attention(gpu, c, q, table, lens, -(128 ** -0.5), [1] * 4)
    # the same call gives the same bits
    again = check_attention(gpu, c, q, table, lens, 128 ** -0.5, [1] * 4, use_max_len=9000)
    assert (again[0] == got[0][0]).all() and (again[1] == got[0][1]).all()


def test_attention_bad_pages(gpu):
    """Page numbers outside the pool hold no keys, wherever they stand; lengths
    past the table are cut at it; a negative length is none."""
    rng = np.random.default_rng(5)
    page, pages = 16, 12
    c = make_cache(gpu, rng, pages, page, 2, 64)
    table = [[3, -1, 5, 7], [pages, 1, 2, 1 << 30], [-1, -1, -1, -1], [8, 9, 10, 11], [0, 4, 6, -5],
             [-(1 << 31), 0, 2, 2]]
    lens = [60, 64, 50, 1 << 20, 49, 33]
    for dtype in DTYPES:
        q = gpu.from_numpy(rng.standard_normal((6, 6, 64)).astype(np.float32)).cuda()
        q = q.to(getattr(gpu, dtype))
        check_attention(gpu, c, q, table, lens, 0.125, [1] * 6)
        check_attention(gpu, c, q, table, lens, 0.125, [1] * 6, window=20)
    from qppocr_amd import ops
    y, s = ops.attention_cache4(q, c, gpu.tensor(table, dtype=gpu.int32, device="cuda"),
                                gpu.full((6,), -7, dtype=gpu.int32, device="cuda"), 0.125, lse=True)
    assert (host(y) == 0).all() and (host(s) == -math.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dh", [32, 96, 128, 192])
def test_attention_nan_stays_with_its_rows(gpu, dtype, dh):
    """Blocks of NaN in masked places (behind the last token, later keys, keys
    before the window) reach no row; in visible ones, only the rows that see
    them: all of a row for a key's, the block's elements for a value's."""
    rng = np.random.default_rng(6 + dh)
    page, lens, news = 16, [50, 20], [30, 20]
    pages = 8
    c = make_cache(gpu, rng, pages, page, 1, dh)
    table = [[1, 4, 2, 6], [0, 3, -1, -1]]
    # behind the last token of either sequence: everything
    for s in (c.k_scales, c.v_scales):
        s[6, :, 2:], s[3, :, 4:], s[5], s[7] = 255, 255, 255, 255
    c.k_scales[4, 0, 9, 0] = 255           # key 25 of sequence 0
    c.v_scales[2, 0, 3, (dh // 32) - 1] = 255   # value 35, its last block
    q = gpu.from_numpy(rng.standard_normal((50, 3, dh)).astype(np.float32)).cuda()
    q = q.to(getattr(gpu, dtype))
    for causal, window in ((True, 0), (True, 8), (False, 0), (False, 5)):
        print("attention NaN", dtype, dh, causal, window, flush=True)
        y, _ = check_attention(gpu, c, q, table, lens, dh ** -0.5, news, causal, window)
        assert np.isfinite(y[30:]).all()
        if causal:
            assert np.isfinite(y[:5]).all() and np.isnan(y[5]).all()
    # one key, and it is NaN
    y, s = check_attention(gpu, c, q[:1], [[4]], [10], dh ** -0.5, [1], True, 1)
    assert np.isnan(y).all() and np.isnan(s).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_over_memory_never_written(gpu, dtype):
    """A pool whose unwritten tokens hold any bytes at all (scales that overflow
    among them): only the written ones count, in short and in split walks."""
    from qppocr_amd import ops
    rng = np.random.default_rng(31)
    t = getattr(gpu, dtype)
    for dh, heads, group, news, lens, window in ((64, 2, 3, [1, 1, 1], [17, 64, 31], 0),
                                                 (128, 1, 4, [5, 2], [1500, 1239], 0),
                                                 (96, 1, 1, [3], [70], 40),
                                                 (32, 8, 16, [66, 65, 64, 64], [66, 90, 70, 100], 0)):
        print("attention never written", dtype, dh, lens, flush=True)
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
        q = gpu.from_numpy(rng.standard_normal((sum(news), heads * group, dh)).astype(np.float32)).cuda().to(t)
        y, s = check_attention(gpu, c, q, table, lens, dh ** -0.5, news, window=window)
        assert np.isfinite(y).all() and np.isfinite(s).all()


def test_attention_widest_window(gpu):
    """The largest window hides nothing, rows before the first key included."""
    rng = np.random.default_rng(33)
    c = make_cache(gpu, rng, 3, 32, 1, 64)
    q = gpu.from_numpy(rng.standard_normal((9, 2, 64)).astype(np.float32)).cuda()
    for causal in (False, True):
        check_attention(gpu, c, q, [[2, 0]], [4], 0.2, [9], causal, (1 << 31) - 1)


def test_first_call_inside_a_capture(gpu):
    """Nothing is set up by a first call that a capture would not allow: a new
    process captures its first call of either kind (after torch's own start)."""
    import subprocess
    import sys
    code = """
import torch
from qppocr_amd import ops
x = torch.randn(2, 64, device="cuda")
w = ops.Weight4(torch.zeros((8, 64), dtype=torch.uint8, device="cuda") + 0x22,
                torch.zeros((8, 4), dtype=torch.uint8, device="cuda") + 127, 64)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.linear4(x, w)
for _ in range(3):
    x.normal_()
    g.replay()
    torch.cuda.synchronize()
    want = x.double().sum(1, keepdim=True).expand(2, 8)
    assert (y.double() - want).abs().max() < 1e-4, (y, want)
print("captured")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout[-500:] + r.stderr[-1500:]


def test_attention_strides_and_rows_left_alone(gpu):
    """q out of a packed projection, out with a stride of its own; rows before
    the first and behind the last sequence keep what they hold."""
    from qppocr_amd import ops
    rng = np.random.default_rng(12)
    page, lens, news = 32, [70, 33], [3, 6]
    c = make_cache(gpu, rng, 6, page, 2, 96)
    for dtype in DTYPES:
        t = getattr(gpu, dtype)
        qkv = gpu.from_numpy(rng.standard_normal((14, 8, 97)).astype(np.float32)).cuda().to(t)
        q = qkv[:, 1:5, 1:]
        hold = gpu.full((14, 7, 100), 5.0, device="cuda", dtype=t)
        out = hold[:, 2:6, 3:99]
        starts = [2, 5, 11]
        check_attention(gpu, c, q, tables(rng, 6, page, lens), lens, 0.1, news, starts=starts, out=out)
        left = host(hold)
        assert (left[:2] == 5).all() and (left[11:] == 5).all()
        assert (left[:, :2] == 5).all() and (left[:, 6:] == 5).all() and (left[:, :, :3] == 5).all()
        assert (left[:, :, 99] == 5).all()
        # the same where the keys are split between workgroups
        big = [(i * 5 + j) % 6 for i in range(1) for j in range(40)]
        check_attention(gpu, c, q, [big, big], [1200, 900], 0.1, news, starts=starts, out=out)
        left = host(hold)
        assert (left[:2] == 5).all() and (left[11:] == 5).all()


def test_attention_nothing_to_do(gpu):
    from qppocr_amd import ops
    c = ops.cache4(2, 16, 1, 64)
    i32 = dict(dtype=gpu.int32, device="cuda")
    y = ops.attention_cache4(gpu.empty((0, 2, 64), device="cuda"), c, gpu.zeros((0, 1), **i32),
                             gpu.zeros((0,), **i32), 1.0)
    assert tuple(y.shape) == (0, 2, 64)
    out = gpu.full((3, 2, 64), 9.0, device="cuda")
    ops.attention_cache4(gpu.ones((3, 2, 64), device="cuda"), c, gpu.zeros((0, 1), **i32),
                         gpu.zeros((0,), **i32), 1.0, starts=gpu.zeros((1,), **i32), max_new=1, out=out)
    assert (host(out) == 9).all()
    # sequences without new tokens, and a table without pages
    ops.attention_cache4(gpu.ones((3, 2, 64), device="cuda"), c, gpu.zeros((2, 1), **i32),
                         gpu.ones((2,), **i32), 1.0, starts=gpu.zeros((3,), **i32), max_new=0, out=out)
    assert (host(out) == 9).all()
    y = ops.attention_cache4(gpu.ones((3, 2, 64), device="cuda"), c, gpu.zeros((3, 0), **i32),
                             gpu.ones((3,), **i32), 1.0)
    assert (host(y) == 0).all()


# ----------------------------------------------------- refusals on the device

def test_refusals(gpu):
    from qppocr_amd import ops
    from qppocr_amd._lib import QphError
    c = ops.cache4(4, 16, 2, 64)
    f = lambda *s, **k: gpu.zeros(s, device="cuda", **k)     # noqa: E731
    i32 = dict(dtype=gpu.int32)
    i64 = dict(dtype=gpu.int64)
    w = ops.quantize4(f(64, 8))
    bad = [
        (lambda: ops.linear4(f(2, 63), w), "against a weight"),
        (lambda: ops.linear4(f(2, 64, dtype=gpu.float64), w), "float32, float16"),
        (lambda: ops.linear4(f(2, 64), w, f(9)), "bias"),
        (lambda: ops.linear4(f(2, 64), w, f(8, dtype=gpu.float16)), "bias"),
        (lambda: ops.linear4(f(2, 64), w, residual=f(2, 9)), "residual"),
        (lambda: ops.linear4(gpu.zeros(2, 64), w), "is on cpu"),
        (lambda: ops.Weight4(w.codes[:, :32], w.scales, 64), "codes"),
        (lambda: ops.Weight4(w.codes, w.scales[:, :2], 64), "scales"),
        (lambda: ops.quantize4(f(64)), "weight"),
        (lambda: ops.quantize4(f(0, 4)), "empty"),
        (lambda: ops.cache4(4, 24, 2, 64), "page size 24"),
        (lambda: ops.cache4(0, 16, 2, 64), "empty"),
        (lambda: ops.Cache4(c.k_codes, c.k_scales, c.v_codes, c.v_scales[:3]), "v_scales"),
        (lambda: ops.Cache4(c.k_codes, c.k_scales.int(), c.v_codes, c.v_scales), "k_scales"),
        (lambda: ops.cache4_write(c, f(3, 2, 64), f(3, 2, 64, dtype=gpu.float16), f(3, **i64)), "one type"),
        (lambda: ops.cache4_write(c, f(3, 2, 64), f(3, 2, 64), f(3, **i32)), "slots"),
        (lambda: ops.cache4_write(c, f(3, 2, 64), f(3, 2, 64), f(4, **i64)), "slots"),
        (lambda: ops.cache4_write(c, f(3, 3, 64), f(3, 2, 64), f(3, **i64)), "k must be"),
        (lambda: ops.cache4_write(c, f(3, 64, 2).transpose(1, 2), f(3, 2, 64), f(3, **i64)), "neighbouring"),
        (lambda: ops.cache4_read(c, f(3, **i32)), "slots"),
        (lambda: ops.cache4_read(c, f(3, **i64), gpu.float64), "float32, float16"),
        (lambda: ops.attention_cache4(f(3, 3, 64), c, f(3, 1, **i32), f(3, **i32), 1.0), "multiple"),
        (lambda: ops.attention_cache4(f(3, 2, 32), c, f(3, 1, **i32), f(3, **i32), 1.0), "q must be"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(3, 1, **i64), f(3, **i32), 1.0), "page_table"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(3, 1, **i32), f(2, **i32), 1.0), "lens"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(2, 1, **i32), f(2, **i32), 1.0), "need starts"),
        (lambda: ops.attention_cache4(f(4, 2, 64), c, f(2, 1, **i32), f(2, **i32), 1.0, max_new=3), "max_new"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(3, 1, **i32), f(3, **i32), 1.0, starts=f(4, **i32)),
         "max_new"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(3, 1, **i32), f(3, **i32), 0.0), "scale"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(3, 1, **i32), f(3, **i32), 1.0, window=-2), "negative"),
        (lambda: ops.attention_cache4(f(3, 2, 64), c, f(3, 1, **i32), f(3, **i32), 1.0,
                                      out=f(3, 2, 64, dtype=gpu.float16)), "out is"),
    ]
    for i, (call, text) in enumerate(bad):
        with pytest.raises((ValueError, QphError), match=text):
            call()
            print("not refused:", i, text)


# ------------------------------------------------ streams, graphs, a decoder

class Decoder:
    """Two layers of a small decoder on the 4-bit operators, and the same in
    float64 with the stored numbers: x + attend(qkv(x)), then + MLP(x), and the
    framework's own head (linear + softmax + argmax)."""

    def __init__(self, torch, dtype, batch, heads=2, group=2, dh=32, page=16, pages=40, hidden=128,
                 classes=300):
        from qppocr_amd import ops
        self.torch, self.t, self.ops = torch, dtype, ops
        self.batch, self.heads, self.group, self.dh, self.page = batch, heads, group, dh, page
        rng = np.random.default_rng(21)
        self.q, self.kv = heads * group * dh, heads * dh
        def w(k, n):
            return torch.from_numpy((rng.standard_normal((k, n)) / math.sqrt(k)).astype(np.float32)).cuda()
        self.layers = [dict(qkv=ops.quantize4(w(hidden, self.q + 2 * self.kv)), out=ops.quantize4(w(self.q, hidden)),
                            up=ops.quantize4(w(hidden, 200)), down=ops.quantize4(w(200, hidden)),
                            cache=ops.cache4(pages, page, heads, dh)) for _ in range(2)]
        self.bias = torch.from_numpy(rng.standard_normal(200).astype(np.float32)).cuda().to(dtype)
        self.head = w(hidden, classes)
        order = rng.permutation(pages)
        self.table_host = order[:batch * (pages // batch)].reshape(batch, -1)
        self.table = torch.from_numpy(self.table_host.astype(np.int32)).cuda()
        self.rows = torch.from_numpy(rng.standard_normal((batch * 9, hidden)).astype(np.float32)).cuda().to(dtype)

    def step(self, x, pos, news):
        """x [batch * news, hidden] at positions pos .. (device tensor [batch])."""
        torch, ops = self.torch, self.ops
        n = x.shape[0]
        at = pos[:, None] + torch.arange(news, device="cuda")
        slots = (self.table.gather(1, (at // self.page)).long() * self.page + at % self.page).reshape(-1)
        lens = (pos + news).int()
        for l in self.layers:
            qkv = ops.linear4(x, l["qkv"])
            heads = qkv.view(n, -1, self.dh)
            hq = self.heads * self.group
            ops.cache4_write(l["cache"], heads[:, hq:hq + self.heads], heads[:, hq + self.heads:], slots)
            y = ops.attention_cache4(heads[:, :hq], l["cache"], self.table, lens, self.dh ** -0.5)
            x = ops.linear4(y.view(n, -1), l["out"], residual=x)
            h = ops.linear4(x, l["up"], self.bias, 1)
            x = ops.linear4(h, l["down"], residual=x)
        return x

    def reference(self, x, pos, news, stored):
        """The step in float64 from x, with the keys and values as stored."""
        xd = host(x)
        for l, (k, v) in zip(self.layers, stored):
            w = {n: decode(host(l[n].codes), host(l[n].scales))[:, :l[n].k] for n in ("qkv", "out", "up", "down")}
            q = (xd @ w["qkv"].T)[:, :self.q].reshape(-1, self.heads * self.group, self.dh)
            y = np.zeros_like(q)
            for r in range(q.shape[0]):
                b, i = r // news, r % news
                p = np.arange(pos + i + 1)
                pg = self.table_host[b][p // self.page]
                y[r] = attend_row(q[r], k[pg, p % self.page], v[pg, p % self.page], self.dh ** -0.5, 3,
                                  self.group)[0]
            xd = xd + y.reshape(len(xd), -1) @ w["out"].T
            h = self.torch.from_numpy(xd @ w["up"].T + host(self.bias))
            h = (h * 0.5 * self.torch.erfc(-h / math.sqrt(2.0))).numpy()
            xd = xd + h @ w["down"].T
        return xd


@pytest.mark.parametrize("dtype", DTYPES)
def test_decoder_steps(gpu, dtype):
    """A prompt of 20 tokens, then single tokens across a page's border."""
    t = getattr(gpu, dtype)
    d = Decoder(gpu, t, 3)
    rng = np.random.default_rng(4)
    pos, unit = 0, gpu.finfo(t).eps / 2
    for news in (20, 1, 1, 5, 7, 1):
        print("decoder", dtype, pos, news, flush=True)
        x = gpu.from_numpy(rng.standard_normal((3 * news, 128)).astype(np.float32)).cuda().to(t)
        y = d.step(x, gpu.full((3,), pos, device="cuda"), news)
        stored = [numbers(l["cache"]) for l in d.layers]
        want = d.reference(x, pos, news, stored)
        # every linear, attention and addition rounds to the type: ten of them,
        # each passed on by weights of unit gain to a handful of values; a
        # float32 run's own sums are off by up to 2^-23 of some 200 terms
        tol = (60 * unit + 2000 * 2.0 ** -23 * (dtype == "float32")) * (1 + np.abs(want).max())
        close(host(y), want, tol, f"decoder at {pos}")
        pos += news
    pairs = d.ops.linear_softmax_argmax(y.float(), d.head)
    logits = host(y) @ host(d.head)
    best = d.ops.pairs_ids(pairs).cpu().numpy()
    top = logits.max(1)
    assert (top - logits[np.arange(len(best)), best] < 1e-3).all()


def test_decoder_captured_steps(gpu):
    """A step captured once and replayed for every further token, the program's
    own work between the replays; two graphs that are alive together; each
    replay against an eager run, bit for bit."""
    t = gpu.bfloat16
    a, b = Decoder(gpu, t, 4), Decoder(gpu, t, 4)
    rng = np.random.default_rng(14)
    prompt = gpu.from_numpy(rng.standard_normal((4 * 6, 128)).astype(np.float32)).cuda().to(t)
    for d in (a, b):
        d.step(prompt, gpu.zeros(4, dtype=gpu.int64, device="cuda"), 6)
    x = gpu.zeros((4, 128), device="cuda", dtype=t)
    pos = gpu.full((4,), 6, device="cuda")
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        a.step(x, pos, 1)
    gpu.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(a.step(x, pos, 1))
        graphs.append(g)
    for i in range(12):
        tok = gpu.from_numpy(rng.standard_normal((4, 128)).astype(np.float32)).cuda().to(t)
        x.copy_(tok)
        pos.fill_(6 + i)
        graphs[i % 2].replay()
        want = b.step(tok, gpu.full((4,), 6 + i, device="cuda"), 1)      # eager, own buffers
        gpu.cuda.synchronize()
        assert (host(outs[i % 2]) == host(want)).all(), f"replay {i}"
        (want @ want.t()).float().softmax(-1).sum().item()
    for la, lb in zip(a.layers, b.layers):
        for p, q in zip(numbers(la["cache"]), numbers(lb["cache"])):
            assert (p == q).all()


def test_captured_split_attention(gpu):
    """Two captured attentions whose keys many workgroups share, replayed in turn
    and in flight together on two streams: a workspace each."""
    from qppocr_amd import ops
    rng = np.random.default_rng(15)
    c = make_cache(gpu, rng, 130, 64, 2, 128)
    table = gpu.from_numpy(rng.permutation(128)[None].astype(np.int32)).cuda()
    lens = gpu.tensor([8000], dtype=gpu.int32, device="cuda")
    qs = [gpu.zeros((1, 8, 128), device="cuda", dtype=gpu.float16) for _ in range(2)]
    graphs, outs = [], []
    for q in qs:
        ops.attention_cache4(q, c, table, lens, 0.1)
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(ops.attention_cache4(q, c, table, lens, 0.1, lse=True))
        graphs.append(g)
    side = gpu.cuda.Stream()
    for i in range(6):
        new = [gpu.from_numpy(rng.standard_normal((1, 8, 128)).astype(np.float32)).cuda().half() for _ in qs]
        for q, v in zip(qs, new):
            q.copy_(v)
        lens.fill_(8000 - 1111 * i)
        gpu.cuda.synchronize()
        graphs[0].replay()
        with gpu.cuda.stream(side):
            graphs[1].replay()
        gpu.cuda.synchronize()
        for v, (y, s) in zip(new, outs):
            y2, s2 = ops.attention_cache4(v, c, table, lens, 0.1, max_len=8192, lse=True)
            assert (host(y) == host(y2)).all() and (host(s) == host(s2)).all()


def test_other_streams_and_threads(gpu):
    """Calls from several threads, each on a stream of its own, in its order."""
    import threading
    from qppocr_amd import ops
    rng = np.random.default_rng(16)
    w = [ops.quantize4(gpu.from_numpy((rng.standard_normal((256, 256)) / 16).astype(np.float32)).cuda())
         for _ in range(3)]
    x0 = [gpu.from_numpy(rng.standard_normal((5, 256)).astype(np.float32)).cuda() for _ in range(4)]
    def chain(x):
        for i in range(60):
            x = ops.linear4(x, w[i % 3])
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
    for _ in range(3):
        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        for a, b in zip(got, want):
            assert (a == b).all()
