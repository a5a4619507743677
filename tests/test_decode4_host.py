"""The 4-bit operators' refusals, on the host: every bad argument is an error
that names the operator before any device work (no GPU, no context), and the
attention's workspace depends on the arguments alone."""
import ctypes
import glob
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SAN_LIB = os.path.join(ROOT, "qppocr_amd", "_build", "sanitize", "libqppocr_hip.so")
EINVAL, EUNSUPPORTED = -1, -3
A = 1 << 20                       # an aligned address that no host code follows


@pytest.fixture(scope="module")
def lib():
    from qppocr_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from qppocr_amd import build
        build.build()
    return _lib.load()


def cache(**kw):
    from qppocr_amd import _lib
    d = dict(k_codes=A, k_scales=A, v_codes=A, v_scales=A, n_pages=4, page_size=16, heads=2, dh=64)
    d.update(kw)
    return _lib.Cache4(**d)


def attn(**kw):
    from qppocr_amd import _lib
    d = dict(q=A, out=A, lse=None, tokens=3, batch=3, page_table=A, table_stride=4, max_pages=4,
             lens=A, starts=A, dtype=0, heads=4, max_new=1, max_len=64, scale=0.125, causal=1,
             window=0, workspace=A, workspace_bytes=1 << 40)
    d.update(kw)
    a = _lib.Attn4(**d)
    a.q_token, a.q_head, a.out_token, a.out_head = 4 * 64, 64, 4 * 64, 64
    return a


def refused(lib, rc, code, text):
    assert rc == code, (rc, lib.qph_last_error())
    assert text.encode() in lib.qph_last_error(), lib.qph_last_error()


CACHES = [
    (dict(k_codes=None), EINVAL, "NULL cache memory"), (dict(v_scales=None), EINVAL, "NULL cache memory"),
    (dict(n_pages=0), EINVAL, "empty cache"), (dict(heads=0), EINVAL, "empty cache"),
    (dict(heads=-2), EINVAL, "empty cache"), (dict(heads=5000), EUNSUPPORTED, "4096 heads"),
    (dict(page_size=8), EUNSUPPORTED, "page size 8"), (dict(page_size=48), EUNSUPPORTED, "page size 48"),
    (dict(page_size=1 << 16), EUNSUPPORTED, "page size"), (dict(dh=0), EUNSUPPORTED, "head dimension 0"),
    (dict(dh=80), EUNSUPPORTED, "head dimension 80"), (dict(dh=288), EUNSUPPORTED, "head dimension"),
    (dict(n_pages=1 << 31), EUNSUPPORTED, "pages"), (dict(k_codes=A + 8), EINVAL, "16-byte aligned"),
]


@pytest.mark.parametrize("kw,code,text", CACHES)
def test_bad_caches(lib, kw, code, text):
    c = cache(**kw)
    st = (ctypes.c_int64 * 2)(128, 64)
    for fn in ("qph_cache4_write", "qph_cache4_read"):
        refused(lib, getattr(lib, fn)(None, ctypes.byref(c), A, A, 0, 3, st, st, A), code, text)
        assert fn[4:].encode() in lib.qph_last_error()
    n = ctypes.c_size_t()
    refused(lib, lib.qph_attention_cache4_workspace(ctypes.byref(c), ctypes.byref(attn()),
                                                    ctypes.byref(n)), code, text)
    refused(lib, lib.qph_attention_cache4(None, ctypes.byref(c), ctypes.byref(attn())), code, text)


def test_bad_cache_calls(lib):
    c, st = cache(), (ctypes.c_int64 * 2)(128, 64)
    for fn in (lib.qph_cache4_write, lib.qph_cache4_read):
        refused(lib, fn(None, None, A, A, 0, 3, st, st, A), EINVAL, "NULL cache")
        refused(lib, fn(None, ctypes.byref(c), A, A, 3, 3, st, st, A), EINVAL, "element type")
        refused(lib, fn(None, ctypes.byref(c), A, A, 0, -1, st, st, A), EINVAL, "negative")
        refused(lib, fn(None, ctypes.byref(c), None, A, 0, 3, st, st, A), EINVAL, "NULL argument")
        refused(lib, fn(None, ctypes.byref(c), A, A, 0, 3, None, st, A), EINVAL, "NULL argument")
        refused(lib, fn(None, ctypes.byref(c), A, A, 0, 3, st, st, None), EINVAL, "NULL argument")
        refused(lib, fn(None, ctypes.byref(c), A, A, 0, 3, st, st, A), EINVAL, "null context")
        refused(lib, fn(None, ctypes.byref(c), None, None, 0, 0, None, None, None), EINVAL, "null context")


ATTNS = [
    (dict(dtype=7), EINVAL, "element type"), (dict(tokens=-1), EINVAL, "negative"),
    (dict(batch=-1), EINVAL, "negative"), (dict(window=-1), EINVAL, "negative"),
    (dict(max_len=-1), EINVAL, "negative"), (dict(max_pages=-1), EINVAL, "negative"),
    (dict(heads=3), EINVAL, "multiple"), (dict(heads=0), EINVAL, "multiple"),
    (dict(heads=1 << 17), EUNSUPPORTED, "65536"), (dict(scale=0.0), EINVAL, "scale"),
    (dict(scale=float("nan")), EINVAL, "scale"), (dict(scale=float("inf")), EINVAL, "scale"),
    (dict(starts=None, tokens=4), EINVAL, "without starts"),
    (dict(tokens=1 << 32), EUNSUPPORTED, "too many rows"),
    (dict(batch=1 << 31), EUNSUPPORTED, "sequences"), (dict(batch=1 << 62), EUNSUPPORTED, "sequences"),
    (dict(tokens=1 << 62), EUNSUPPORTED, "too many rows"),
]


@pytest.mark.parametrize("kw,code,text", ATTNS)
def test_bad_attention(lib, kw, code, text):
    c, a, n = cache(), attn(**kw), ctypes.c_size_t()
    refused(lib, lib.qph_attention_cache4_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(n)),
            code, text)
    refused(lib, lib.qph_attention_cache4(None, ctypes.byref(c), ctypes.byref(a)), code, text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "NULL argument"), (dict(out=None), "NULL argument"),
    (dict(page_table=None), "NULL argument"), (dict(lens=None), "NULL argument"),
    (dict(max_len=100000, max_pages=7000, workspace=None), "workspace"),
    (dict(max_len=100000, max_pages=7000, workspace_bytes=100), "workspace of 100 bytes"),
    (dict(workspace=A + 8), "16-byte aligned"), (dict(), "null context"),
    (dict(tokens=0, q=None, out=None), "null context")])
def test_bad_attention_call(lib, kw, text):
    refused(lib, lib.qph_attention_cache4(None, ctypes.byref(cache()), ctypes.byref(attn(**kw))),
            EINVAL, text)


def _workspace(lib, c, a):
    n = ctypes.c_size_t()
    assert lib.qph_attention_cache4_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(n)) == 0
    return n.value


def test_workspace(lib):
    assert _workspace(lib, cache(), attn(max_len=1)) == 0
    assert _workspace(lib, cache(), attn(tokens=0, batch=0)) == 0
    long = attn(max_len=100000, max_pages=7000)
    n = _workspace(lib, cache(), long)
    row = 3 * 4 * (64 + 2) * 4               # one split of 3 tokens, 4 heads: sums and dh numbers
    assert n and n % row == 0 and 2 <= n // row <= 64
    # a window bounds the keys that are read
    assert _workspace(lib, cache(), attn(max_len=100000, max_pages=7000, window=100)) == 0
    for w in (1, 5, 31, 32, 1000, 16384 - 33):
        for m in (1, 3, 40):
            n = _workspace(lib, cache(), attn(max_len=1 << 20, max_pages=70000, window=w, max_new=m))
            assert n % row == 0 and n // row <= 64
    assert lib.qph_attention_cache4_workspace(ctypes.byref(cache()), ctypes.byref(long), None) == EINVAL


def test_workspace_of_the_largest_arguments(lib):
    """No product of sizes overflows in the plan (the sanitizer run says so)."""
    top = (1 << 31) - 1
    n = ctypes.c_size_t()
    a = attn(tokens=1 << 20, batch=top // 2, max_new=top, max_len=top, max_pages=top, heads=1 << 12,
             window=top)
    assert lib.qph_attention_cache4_workspace(ctypes.byref(cache()), ctypes.byref(a), ctypes.byref(n)) == 0
    refused(lib, lib.qph_attention_cache4(None, ctypes.byref(cache()), ctypes.byref(a)), EUNSUPPORTED,
            "batch too large")


def test_bad_linears(lib):
    def call(dtype=0, x=A, xs=64, codes=A, scales=A, rows=2, k=64, n=8, act=None, y=A):
        return lib.qph_linear4(None, x, dtype, xs, codes, scales, None, rows, k, n, act, None, y)
    from qppocr_amd import _lib
    refused(lib, call(dtype=-1), EINVAL, "element type")
    for kw in (dict(rows=-1), dict(k=0), dict(n=0)):
        refused(lib, call(**kw), EINVAL, "bad shape")
    refused(lib, call(act=ctypes.byref(_lib.Act(9, 0, 0, 0))), EINVAL, "activation")
    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(y=None)):
        refused(lib, call(**kw), EINVAL, "NULL argument")
    refused(lib, call(codes=A + 4), EINVAL, "aligned")
    refused(lib, call(scales=A + 2), EINVAL, "aligned")
    refused(lib, call(n=1 << 40), EUNSUPPORTED, "2^30")
    refused(lib, call(k=1 << 40), EUNSUPPORTED, "2^30")
    refused(lib, call(rows=1 << 30), EUNSUPPORTED, "rows")
    refused(lib, call(), EINVAL, "null context")
    refused(lib, call(rows=0, x=None, y=None), EINVAL, "null context")


def test_bad_quantize(lib):
    def call(x=A, dtype=0, rows=2, k=64, codes=A, scales=A):
        return lib.qph_quantize4(None, x, dtype, rows, k, 64, 1, codes, scales)
    refused(lib, call(dtype=3), EINVAL, "element type")
    refused(lib, call(rows=-1), EINVAL, "bad shape")
    refused(lib, call(k=0), EINVAL, "bad shape")
    refused(lib, call(k=1 << 40), EUNSUPPORTED, "2^30")
    refused(lib, call(rows=1 << 50), EUNSUPPORTED, "blocks")
    refused(lib, call(x=None), EINVAL, "NULL argument")
    refused(lib, call(codes=A + 1), EINVAL, "aligned")
    refused(lib, call(), EINVAL, "null context")


def test_python_refuses_host_tensors(lib):
    import torch
    from qppocr_amd import ops
    with pytest.raises(ValueError, match="is on cpu"):
        ops.quantize4(torch.zeros(64, 8))
    with pytest.raises(ValueError, match="is on cpu"):
        ops.Weight4(torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 4), dtype=torch.uint8), 128)
    with pytest.raises(ValueError, match="is on cpu"):
        ops.cache4(2, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        ops.quantize4(torch.zeros((64, 8), dtype=torch.float64))
    with pytest.raises(ValueError, match="head dimension 80"):
        ops.cache4(2, 16, 1, 80, device="cpu")


def test_host_checks_under_asan_ubsan():
    if os.environ.get("QPPOCR_HIP_LIB"):
        pytest.skip("this is the sanitizer run")
    rt = sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not rt or not os.path.exists(SAN_LIB):
        pytest.skip("no ASan runtime or sanitizer build")
    env = dict(os.environ, QPPOCR_HIP_LIB=SAN_LIB, LD_PRELOAD=rt[-1],
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "-m",
                        "not gpu", "tests/test_decode4_host.py"], cwd=ROOT, env=env,
                       capture_output=True, text=True, timeout=600)
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    assert "passed" in r.stdout and "runtime error" not in tail
