"""The Python calls of the 4-bit operators as the library gets them, on the host:
the device's check and the library's call are replaced, the tensors are host
tensors, and nothing is computed."""
import copy
import os
import pickle

import pytest
import torch

from qppocr_amd import _lib, ops

TYPES = [torch.float32, torch.float16, torch.bfloat16]


class Lib:
    """Every entry point's name in its place, but the plan's (it needs no GPU)."""

    def __init__(self, real):
        self.qph_attention_cache4_workspace = real.qph_attention_cache4_workspace

    def __getattr__(self, name):
        return name


@pytest.fixture
def calls(monkeypatch):
    """The library's calls as they come: (device, name, arguments)."""
    if not os.path.exists(_lib.LIB_PATH):
        from qppocr_amd import build
        build.build()
    lib, got = Lib(_lib.load()), []
    monkeypatch.setattr(ops, "_on", lambda *a: None)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_enqueue", lambda device, fn, *a: got.append((device, fn, a)))
    return got


def cache(pages=4, page=16, heads=2, dh=64):
    return ops.cache4(pages, page, heads, dh, device="cpu")


def attend(c, tokens=3, heads=4, dtype=torch.float32, pages=4, **kw):
    q = kw.pop("q", None)
    q = torch.zeros((tokens, heads, c.dh), dtype=dtype) if q is None else q
    return ops.attention_cache4(q, c, torch.zeros((tokens, pages), dtype=torch.int32),
                                torch.ones(tokens, dtype=torch.int32), 0.125, **kw)


@pytest.mark.parametrize("default", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("dtype", TYPES)
def test_every_buffer_has_its_own_type(calls, default, dtype):
    """What the calls allocate does not follow torch's default type: the sums of
    the attention are float32 always."""
    was = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        c = cache()
        out, sums = attend(c, dtype=dtype, lse=True)
        assert out.dtype == dtype and sums.dtype == torch.float32 and tuple(sums.shape) == (3, 4)
        k, v = ops.cache4_read(c, torch.zeros(5, dtype=torch.int64), dtype)
        assert k.dtype == v.dtype == dtype
        w = ops.quantize4(torch.zeros((64, 8), dtype=dtype))
        assert w.codes.dtype == w.scales.dtype == torch.uint8
        assert ops.linear4(torch.zeros((2, 64), dtype=dtype), w).dtype == dtype
    finally:
        torch.set_default_dtype(was)


def test_first_call_leaves_the_callers_device(monkeypatch):
    """The context that a device's first call makes leaves the thread's device as it was."""
    now, log = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, now[0] = now[0], self.index

        def __exit__(self, *a):
            now[0] = self.was

    class Library:
        def qph_ctx_create(self, device, out):
            now[0] = device                # as the library does
            return 0

        def qph_ctx_set_stream(self, ctx, stream):
            return 0
    monkeypatch.setattr(ops, "_queued", {})
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 64)
    monkeypatch.setattr(_lib, "load", lambda: Library())
    monkeypatch.setattr(torch.cuda, "device", Device)
    for device in (3, 3, 0, 1):
        ops._enqueue(device, lambda ctx, *a: log.append(a) or 0, "x")
        assert now[0] == 0
    assert log == [("x",)] * 4 and sorted(ops._queued) == [0, 1, 3]


@pytest.mark.parametrize("name", ["codes", "scales", "n", "k", "device"])
def test_a_weights_memory_is_fixed(calls, name):
    """A call reads the memory a Weight4 was made of, so another tensor in its place
    is refused rather than not looked at."""
    w = ops.quantize4(torch.zeros((100, 8)))
    with pytest.raises(AttributeError, match=name):
        setattr(w, name, getattr(w, name))
    with pytest.raises(AttributeError, match=name):
        delattr(w, name)
    w.note = "mine"
    w.note = "other"
    ops.linear4(torch.zeros((2, 100)), w)
    assert calls[-1][2][3:5] == (w.codes.data_ptr(), w.scales.data_ptr())


@pytest.mark.parametrize("name", ["k_codes", "k_scales", "v_codes", "v_scales", "pages", "heads",
                                  "page_size", "dh", "device"])
def test_a_caches_memory_is_fixed(calls, name):
    c = cache()
    with pytest.raises(AttributeError, match=name):
        setattr(c, name, getattr(c, name))
    with pytest.raises(AttributeError, match=name):
        delattr(c, name)
    assert c._c.k_codes == c.k_codes.data_ptr() and c._c.v_scales == c.v_scales.data_ptr()


@pytest.mark.parametrize("how", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))], ids=["deepcopy", "pickle"])
def test_copies_have_their_own_memory(calls, how):
    w, c = ops.quantize4(torch.zeros((100, 8))), cache()
    w2, c2 = how(w), how(c)
    assert (w2.n, w2.k, w2.device) == (w.n, w.k, w.device) and w2.codes.data_ptr() != w.codes.data_ptr()
    assert w2._ptrs == (w2.codes.data_ptr(), w2.scales.data_ptr())
    assert (c2.pages, c2.heads, c2.page_size, c2.dh) == (c.pages, c.heads, c.page_size, c.dh)
    assert c2._c.k_codes == c2.k_codes.data_ptr() != c.k_codes.data_ptr()
    assert c2._c.v_scales == c2.v_scales.data_ptr() != c.v_scales.data_ptr()
    w3 = copy.copy(w)
    assert w3._ptrs == w._ptrs


def views(dtype=torch.float32):
    """(k, v, the pair does not overlap) of 5 tokens, 2 heads of 64."""
    z = torch.zeros
    both = z((5, 2, 2, 64), dtype=dtype)
    packed = z((5, 7, 64), dtype=dtype)
    long = z(5 * 2 * 2 * 64 + 640, dtype=dtype)

    def at(offset, *strides):
        return long.as_strided((5, 2, 64), strides + (1,), offset)
    yield both[:, 0], both[:, 1], True
    yield both[:, 1], both[:, 0], True
    yield both[:, :, 0], both[:, :, 1], True
    yield packed[:, 1:3], packed[:, 4:6], True
    yield packed[:, 4:6], packed[:, 2:4], True
    yield z((5, 2, 64), dtype=dtype), z((2, 5, 64), dtype=dtype).transpose(0, 1), True
    yield at(0, 128, 64), at(640, 64, 320), True
    yield packed[:, 1:3], packed[:, 2:4], False
    yield both[:, 0], both[:, 0], False
    yield at(0, 128, 64), at(64, 128, 64), False
    yield at(0, 128, 64), at(639, 64, 320), False
    yield z((1, 2, 64), dtype=dtype).expand(5, 2, 64), z((5, 2, 64), dtype=dtype), False
    yield z((5, 2, 64), dtype=dtype), z((5, 1, 64), dtype=dtype).expand(5, 2, 64), False
    yield at(0, 100, 64), at(1000, 128, 64), False
    yield at(0, 128, 63), at(1000, 128, 64), False


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(15))
def test_outputs_that_overlap(calls, dtype, i):
    k, v, good = list(views(dtype))[i]
    slots = torch.zeros(5, dtype=torch.int64)
    if good:
        assert ops.cache4_read(cache(), slots, out=(k, v)) == (k, v)
        assert attend(cache(), 5, 2, dtype, q=k, out=v) is v
    else:
        with pytest.raises(ValueError, match="overlaps itself|share memory"):
            ops.cache4_read(cache(), slots, out=(k, v))
        if k.data_ptr() != v.data_ptr():           # (out may be q itself)
            # v as out, and k where only that overlaps itself
            q, out = (v, k) if k.stride() in ((0, 64, 1), (100, 64, 1), (128, 63, 1)) else (k, v)
            with pytest.raises(ValueError, match="overlaps itself|share memory"):
                attend(cache(), 5, 2, dtype, q=q, out=out)


def test_an_output_that_is_the_query(calls):
    q = torch.zeros((5, 2, 64))
    assert attend(cache(), 5, 2, q=q, out=q) is q
    # one token, or one head: nothing of theirs can overlap, whatever the stride says
    one = torch.zeros((1, 2, 64))
    attend(cache(), 1, 2, q=one, out=torch.zeros(128).as_strided((1, 2, 64), (0, 64, 1)))
    none = torch.zeros((0, 2, 64))
    ops.cache4_read(cache(), torch.zeros(0, dtype=torch.int64), out=(none, none))


def test_no_gradient_is_dropped(calls):
    """The operators compute no gradients: an input that requires one is refused while
    gradients are recorded, and taken under no_grad; a weight to quantise is taken."""
    p = lambda *s: torch.zeros(s, requires_grad=True)      # noqa: E731
    z, slots = torch.zeros, torch.zeros(3, dtype=torch.int64)
    c = cache()
    w = ops.quantize4(p(64, 8))
    refused = [
        lambda: ops.linear4(p(2, 64), w), lambda: ops.linear4(z(2, 64), w, p(8)),
        lambda: ops.linear4(z(2, 64), w, None, 0, p(2, 8)),
        lambda: ops.linear4(p(2, 64) * 2, w),
        lambda: ops.cache4_write(c, p(3, 2, 64), z(3, 2, 64), slots),
        lambda: ops.cache4_write(c, z(3, 2, 64), p(3, 2, 64), slots),
        lambda: ops.cache4_read(c, slots, out=(z(3, 2, 64), p(3, 2, 64))),
        lambda: attend(c, q=p(3, 4, 64)), lambda: attend(c, out=p(3, 4, 64)),
    ]
    for call in refused:
        n = len(calls)
        with pytest.raises(ValueError, match="no gradient"):
            call()
        assert len(calls) == n
        with torch.no_grad():
            call()
        assert len(calls) == n + 1


def test_bounds_past_32_bits(calls):
    """Bounds that no sequence can reach mean what they say: the widest window, the
    longest sequences; negative ones are refused however small."""
    starts = torch.arange(4, dtype=torch.int32)
    top = (1 << 31) - 1
    for big in (top, 1 << 31, (1 << 32) - 1, 1 << 32, (1 << 32) + 5, 1 << 70):
        attend(cache(), window=big)
        assert calls[-1][2][1]._obj.window == top
        attend(cache(), max_len=big, max_new=big, starts=starts)
        a = calls[-1][2][1]._obj
        assert a.max_len == a.max_new == top and a.window == 0
    for low in (-1, -(1 << 31) - 1, -(1 << 32), -(1 << 32) + 5):
        for kw in (dict(window=low), dict(max_len=low), dict(max_new=low, starts=starts)):
            with pytest.raises(ValueError, match="negative"):
                attend(cache(), **kw)
