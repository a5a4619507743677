"""The host side of a step that checks drafted trees: every bad argument of the C calls
is an error that names the operator before any device work, workspaces depend on the
sizes alone, and the Python calls hand the library what the tensors are (no GPU, no
context; addresses that no host code follows)."""
import copy
import ctypes
import pickle

import pytest
import torch

from test_decode4_host import A, CACHES, EINVAL, EUNSUPPORTED, attn, cache, lib, refused  # noqa: F401

MASK = "attention_mask4"


def mask(**kw):
    from qppocr_amd import _lib
    return _lib.Attn4Mask(**dict(dict(sinks=4, tree=A, tree_words=1), **kw))


def mask_calls(lib, c, a, m):
    n = ctypes.c_size_t()
    return (lib.qph_attention_mask4_workspace(c, a, m, ctypes.byref(n)), lib.qph_attention_mask4(None, c, a, m))


@pytest.mark.parametrize("kw,code,text", CACHES)
def test_bad_caches(lib, kw, code, text):  # noqa: F811
    c = cache(**kw)
    for rc in mask_calls(lib, ctypes.byref(c), ctypes.byref(attn()), ctypes.byref(mask())):
        refused(lib, rc, code, text)
        assert MASK.encode() in lib.qph_last_error()
    n = ctypes.c_size_t()
    for rc in (lib.qph_cache4_move_workspace(ctypes.byref(c), 3, ctypes.byref(n)),
               lib.qph_cache4_move(None, ctypes.byref(c), A, A, 3, A, 1 << 40)):
        refused(lib, rc, code, text)
        assert b"cache4_move" in lib.qph_last_error()


@pytest.mark.parametrize("args,more,code,text", [
    (dict(dtype=7), {}, EINVAL, "element type"), (dict(tokens=-1), {}, EINVAL, "negative"),
    (dict(heads=3), {}, EINVAL, "multiple"), (dict(scale=0.0), {}, EINVAL, "scale"),
    (dict(window=-1), {}, EINVAL, "negative"), (dict(starts=None, tokens=4), {}, EINVAL, "without starts"),
    (dict(tokens=1 << 62), {}, EUNSUPPORTED, "too many rows"),
    ({}, dict(sinks=-1), EINVAL, "negative"), ({}, dict(tree_words=-1), EINVAL, "negative"),
    ({}, dict(tree_words=1 << 21), EUNSUPPORTED, "words"), (dict(max_new=65), {}, EINVAL, "1 words for up to 65"),
    (dict(max_new=(1 << 31) - 1), dict(tree_words=1 << 20), EINVAL, "words")])
def test_bad_attention(lib, args, more, code, text):  # noqa: F811
    for rc in mask_calls(lib, ctypes.byref(cache()), ctypes.byref(attn(**args)), ctypes.byref(mask(**more))):
        refused(lib, rc, code, text)


def test_attention_arguments(lib):  # noqa: F811
    c, a = ctypes.byref(cache()), ctypes.byref(attn())
    for rc in mask_calls(lib, c, a, None) + mask_calls(lib, c, None, ctypes.byref(mask())):
        refused(lib, rc, EINVAL, "NULL")
    refused(lib, lib.qph_attention_mask4_workspace(c, a, ctypes.byref(mask()), None), EINVAL, "NULL")
    def call(m=None, **kw):
        return lib.qph_attention_mask4(None, c, ctypes.byref(attn(**kw)), ctypes.byref(m or mask()))
    for kw in (dict(q=None), dict(out=None), dict(lens=None), dict(page_table=None)):
        refused(lib, call(**kw), EINVAL, "NULL argument")
    refused(lib, call(mask(tree=None)), EINVAL, "NULL argument")
    refused(lib, call(mask(tree=None, tree_words=0)), EINVAL, "null context")
    refused(lib, call(workspace=A + 4), EINVAL, "16-byte")
    for part in ("k_scales", "v_scales"):
        odd = cache(**{part: A + 2})
        refused(lib, lib.qph_attention_mask4(None, ctypes.byref(odd), ctypes.byref(attn()), ctypes.byref(mask())),
                EINVAL, "scales are not 4-byte aligned")
    refused(lib, call(), EINVAL, "null context")
    refused(lib, call(tokens=0, batch=0, q=None, out=None, lens=None), EINVAL, "null context")
    # a call that is split needs its workspace
    long = dict(tokens=1, batch=1, max_len=100000, max_pages=1 << 16, starts=A)
    refused(lib, call(workspace=None, workspace_bytes=0, **long), EINVAL, "needs")
    refused(lib, call(workspace_bytes=100, **long), EINVAL, "workspace of 100 bytes")


@pytest.mark.parametrize("sinks", [0, 1, 1 << 40, (1 << 63) - 1])
def test_workspace_and_most_sequences(lib, sinks):  # noqa: F811
    """Sizes at their types' ends neither overflow nor make more workgroups than can be
    launched."""
    c = cache(heads=8)
    n, m = ctypes.c_size_t(), mask(sinks=sinks, tree=None, tree_words=0)
    for window in (0, 1, (1 << 31) - 1):
        for new in (1, 9, 5000, (1 << 31) - 1):
            for batch, code, text in (((1 << 21) - 1, EINVAL, "null context"), (1 << 21, EUNSUPPORTED, "batch too large")):
                a = attn(batch=batch, heads=32, max_new=new, max_len=(1 << 31) - 1, window=window)
                refused(lib, lib.qph_attention_mask4(None, ctypes.byref(c), ctypes.byref(a), ctypes.byref(m)), code, text)
            a = attn(batch=1, tokens=100, heads=32, max_new=new, max_len=(1 << 31) - 1, window=window)
            assert lib.qph_attention_mask4_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(m), ctypes.byref(n)) == 0
            assert n.value <= 64 * 100 * 32 * 66 * 4
    # a window of few keys is not split, however long the bound
    a = attn(batch=1, heads=32, max_len=1 << 30, window=64)
    assert lib.qph_attention_mask4_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(mask(sinks=4)),
                                             ctypes.byref(n)) == 0 and n.value == 0


def extend(**kw):
    from qppocr_amd import _lib
    d = dict(page_table=A, table_stride=4, max_pages=4, batch=3, lens=A, news=A, ring=A, ring_n=12, ends=A,
             tokens=5, parents=None, tree_words=0, out_starts=A, out_lens=A, out_slots=A, out_positions=A,
             out_ends=A, out_tree=None, page_size=16, workspace=None, workspace_bytes=0)
    d.update(kw)
    return _lib.Extend4(**d)


@pytest.mark.parametrize("kw,code,text", [
    (dict(batch=-1), EINVAL, "negative"), (dict(tokens=-1), EINVAL, "negative"), (dict(ring_n=-1), EINVAL, "negative"),
    (dict(max_pages=-1), EINVAL, "negative"), (dict(page_size=8), EUNSUPPORTED, "page size 8"),
    (dict(page_size=48), EUNSUPPORTED, "page size 48"), (dict(page_size=0), EUNSUPPORTED, "page size"),
    (dict(batch=(1 << 24) + 1), EUNSUPPORTED, "2^24"), (dict(tokens=(1 << 30) + 1), EUNSUPPORTED, "2^30"),
    (dict(max_pages=1 << 30, table_stride=1 << 30), EUNSUPPORTED, "pages"),
    (dict(ring_n=1 << 31), EUNSUPPORTED, "pages"), (dict(ring_n=0), EINVAL, "empty ring"),
    (dict(table_stride=3), EINVAL, "overlap"), (dict(table_stride=-4), EINVAL, "overlap"),
    (dict(page_table=None), EINVAL, "NULL"), (dict(lens=None), EINVAL, "NULL"), (dict(news=None), EINVAL, "NULL"),
    (dict(ring=None), EINVAL, "NULL"), (dict(ends=None), EINVAL, "NULL"), (dict(out_starts=None), EINVAL, "NULL"),
    (dict(out_lens=None), EINVAL, "NULL"), (dict(out_slots=None), EINVAL, "NULL"),
    (dict(out_positions=None), EINVAL, "NULL"), (dict(out_ends=None), EINVAL, "NULL"),
    (dict(parents=A), EINVAL, "parents without masks"), (dict(parents=A, out_tree=A), EINVAL, "parents without masks"),
    (dict(parents=A, out_tree=A, tree_words=1 << 21), EUNSUPPORTED, "words"),
    (dict(batch=3000), EINVAL, "workspace of 0 bytes, needs 36012"),
    (dict(batch=3000, workspace=A, workspace_bytes=36011), EINVAL, "needs 36012"),
    (dict(batch=3000, workspace=A, workspace_bytes=36012), EINVAL, "null context"), ({}, EINVAL, "null context"),
    (dict(batch=0, max_pages=0, page_table=None, lens=None, news=None, out_lens=None), EINVAL, "null context"),
    (dict(tokens=0, out_slots=None, out_positions=None), EINVAL, "null context")])
def test_extend(lib, kw, code, text):  # noqa: F811
    refused(lib, lib.qph_cache4_extend(None, ctypes.byref(extend(**kw))), code, text)


def test_extend_workspace(lib):  # noqa: F811
    n = ctypes.c_size_t()
    for batch, want in ((0, 0), (2048, 0), (2049, 2050 * 12)):
        assert lib.qph_cache4_extend_workspace(batch, ctypes.byref(n)) == 0 and n.value == want
    refused(lib, lib.qph_cache4_extend_workspace(-1, ctypes.byref(n)), EINVAL, "negative")
    refused(lib, lib.qph_cache4_extend_workspace(1, None), EINVAL, "NULL")
    refused(lib, lib.qph_cache4_extend(None, None), EINVAL, "NULL")


def test_move(lib):  # noqa: F811
    c, n = ctypes.byref(cache()), ctypes.c_size_t()
    for tokens, want in ((0, 0), (2048, 0), (2049, 2049 * 8 * 17), (1 << 31, (1 << 31) * 8 * 17)):
        assert lib.qph_cache4_move_workspace(c, tokens, ctypes.byref(n)) == 0 and n.value == want
    refused(lib, lib.qph_cache4_move_workspace(c, 1, None), EINVAL, "NULL")
    def call(src=A, dst=A, tokens=3, ws=None, size=0):
        return lib.qph_cache4_move(None, c, src, dst, tokens, ws, size)
    refused(lib, call(tokens=-1), EINVAL, "negative")
    refused(lib, call(tokens=(1 << 31) + 1), EUNSUPPORTED, "2^31")
    refused(lib, call(src=None), EINVAL, "NULL argument")
    refused(lib, call(dst=None), EINVAL, "NULL argument")
    refused(lib, call(tokens=4000), EINVAL, "needs")
    refused(lib, call(tokens=4000, ws=A, size=4000 * 8 * 17 - 1), EINVAL, "needs")
    refused(lib, call(tokens=4000, ws=A + 8, size=1 << 40), EINVAL, "16-byte")
    refused(lib, call(tokens=4000, ws=A, size=1 << 40), EINVAL, "null context")
    refused(lib, call(src=None, dst=None, tokens=0), EINVAL, "null context")


def rot(**kw):
    from qppocr_amd import _lib
    d = dict(x=A, out=2 * A, x_token=64, x_head=32, out_token=64, out_head=32, tokens=3, positions=A, p_axis=0,
             p_token=1, turns=A, axes=A, dtype=0, heads=2, dh=32, pairs=16, n_axes=1)
    d.update(kw)
    return _lib.RotaryArgs(**d)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=3), EINVAL, "element type"), (dict(tokens=-1), EINVAL, "negative"), (dict(heads=-1), EINVAL, "negative"),
    (dict(dh=0), EINVAL, "pairs"), (dict(pairs=0), EINVAL, "pairs"), (dict(pairs=17), EINVAL, "17 pairs"),
    (dict(n_axes=0), EINVAL, "0 axes"), (dict(dh=1 << 21), EUNSUPPORTED, "2^20"), (dict(heads=1 << 21), EUNSUPPORTED, "2^20"),
    (dict(x=None), EINVAL, "NULL"), (dict(out=None), EINVAL, "NULL"), (dict(positions=None), EINVAL, "NULL"),
    (dict(turns=None), EINVAL, "NULL"), (dict(axes=None), EINVAL, "NULL"),
    (dict(out=A, out_token=65), EINVAL, "other strides"), (dict(out=A, out_head=33), EINVAL, "other strides"),
    (dict(tokens=1 << 62), EUNSUPPORTED, "tokens"), ({}, EINVAL, "null context"), (dict(out=A), EINVAL, "null context"),
    (dict(tokens=0, x=None, out=None), EINVAL, "null context"), (dict(heads=0, x=None, out=None), EINVAL, "null context")])
def test_rotary(lib, kw, code, text):  # noqa: F811
    refused(lib, lib.qph_rotary(None, ctypes.byref(rot(**kw))), code, text)
    refused(lib, lib.qph_rotary(None, None), EINVAL, "NULL")


# --------------------------------------------- the Python calls, on host tensors

class Lib:
    """Every entry point's name in its place, but those that need no GPU."""

    def __init__(self, real):
        for name in ("qph_attention_cache4_workspace", "qph_attention_mask4_workspace",
                     "qph_cache4_extend_workspace", "qph_cache4_move_workspace"):
            setattr(self, name, getattr(real, name))

    def __getattr__(self, name):
        return name


@pytest.fixture
def calls(lib, monkeypatch):  # noqa: F811
    from qppocr_amd import _lib, ops
    got, fake = [], Lib(lib)
    monkeypatch.setattr(ops, "_on", lambda *a: None)
    monkeypatch.setattr(_lib, "load", lambda: fake)
    monkeypatch.setattr(ops, "_enqueue", lambda device, fn, *a: got.append((fn, a)))
    return got


def attend(fn, words=1, tokens=3, **kw):
    from qppocr_amd import ops
    c = ops.cache4(8, 16, 2, 64, device="cpu")
    q = torch.zeros((tokens, 4, 64), dtype=torch.float32)
    table, lens = torch.zeros((tokens, 8), dtype=torch.int32), torch.ones(tokens, dtype=torch.int32)
    if fn == "tree":
        return ops.attention_tree4(q, c, table, lens, 0.1, torch.ones((tokens, words), dtype=torch.int64), **kw)
    return ops.attention_cache4(q, c, table, lens, 0.1, **kw)


def test_which_attention_is_called(calls):
    """Sinks without a window, or none of them, are the plain call."""
    for kw in ({}, dict(sinks=5), dict(window=3), dict(window=3, sinks=0)):
        attend("plain", **kw)
        assert calls[-1][0] == "qph_attention_cache4"
    attend("plain", window=3, sinks=1 << 50)
    fn, args = calls[-1]
    assert fn == "qph_attention_mask4"
    assert args[2]._obj.sinks == 0x7fffffff and args[2]._obj.tree is None and args[2]._obj.tree_words == 0
    attend("tree", words=3, window=7, sinks=2)
    fn, args = calls[-1]
    assert fn == "qph_attention_mask4" and args[2]._obj.tree_words == 3 and args[2]._obj.tree
    assert args[1]._obj.window == 7 and args[1]._obj.max_new == 1


@pytest.mark.parametrize("default", [torch.float32, torch.bfloat16, torch.float64])
def test_every_buffer_has_its_own_type(calls, default):
    from qppocr_amd import ops
    was = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        out, sums = attend("tree", lse=True)
        assert out.dtype == torch.float32 and sums.dtype == torch.float32
        i32 = dict(dtype=torch.int32)
        s = ops.cache4_extend(torch.zeros((3, 4), **i32), torch.zeros(3, **i32), torch.zeros(3, **i32), 16,
                              torch.zeros(12, **i32), torch.zeros(2, dtype=torch.int64), 70,
                              torch.zeros(70, **i32), 65)
        assert [t.dtype for t in s] == [torch.int32, torch.int32, torch.int64, torch.int32, torch.int64, torch.int64]
        assert [tuple(t.shape) for t in s] == [(4,), (3,), (70,), (70,), (2,), (70, 2)]
    finally:
        torch.set_default_dtype(was)


def test_turns_of_a_plan(calls):
    """Fixed-point turns a position: exact halves of a unit, whole turns taken off."""
    import fractions
    from qppocr_amd import ops
    two_pi = fractions.Fraction(628318530717958647692528676655900576839433879875021, 10 ** 50)
    freqs = [1.0, 0.1, 1e-5, 2.0 ** -60, 0.0, -1.0, 7.0, 1e6]
    plan = ops.rotary_plan(64, freqs, [0, 1, 2, 0, 0, 0, 5, 0], device="cpu")
    assert plan.n_axes == 6 and plan.pairs == 8 and plan.axes.tolist() == [0, 1, 2, 0, 0, 0, 5, 0]
    for f, t in zip(freqs, plan.turns.tolist()):
        off = (fractions.Fraction(f) / two_pi * 2 ** 64 - t) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= fractions.Fraction(1, 2)


def test_a_plan_is_fixed_and_copied_whole(calls):
    from qppocr_amd import ops
    plan = ops.rotary_plan(16, [1.0, 0.5], neighbours=True, device="cpu")
    for name in ("turns", "axes", "pairs", "_ptrs"):
        with pytest.raises(AttributeError):
            setattr(plan, name, None)
        with pytest.raises(AttributeError):
            delattr(plan, name)
    for other in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        assert other.turns.data_ptr() != plan.turns.data_ptr()
        assert other._ptrs == (other.turns.data_ptr(), other.axes.data_ptr())
        assert (other.turns == plan.turns).all() and other.neighbours and other.dh == 16


def test_rotary_arguments(calls):
    from qppocr_amd import ops
    plan = ops.rotary_plan(32, [1.0] * 8, [0, 1] * 4, device="cpu")
    x = torch.zeros((5, 3, 40))[:, :, 4:36]
    pos = torch.zeros((5, 2), dtype=torch.int64).t()
    y = ops.rotary(x, pos, plan, inverse=True)
    a = calls[-1][1][0]._obj
    assert (a.x_token, a.x_head, a.out_token, a.out_head) == (120, 40, 96, 32) and y.is_contiguous()
    assert (a.p_axis, a.p_token, a.positions_64, a.n_axes, a.pairs, a.inverse) == (1, 2, 1, 2, 8, 1)
    ops.rotary(x, torch.zeros(10, dtype=torch.int32)[::2], plan, out=x)
    a = calls[-1][1][0]._obj
    assert (a.p_axis, a.p_token, a.positions_64, a.inverse) == (0, 2, 0, 0) and a.x == a.out
    with torch.no_grad():
        ops.rotary(x.clone().requires_grad_(), pos, plan)
    n = len(calls)
    for bad in (dict(x=x.clone().requires_grad_()), dict(out=torch.zeros_like(x).requires_grad_()),
                dict(out=x[:, :2]), dict(out=x[:1].expand(5, 3, 32))):
        with pytest.raises(ValueError):
            ops.rotary(bad.get("x", x), pos, plan, out=bad.get("out"))
    assert len(calls) == n


def test_host_checks_under_asan_ubsan():
    """This file's checks again with the library's host code under sanitizers."""
    import glob
    import os
    import subprocess
    import sys
    from test_decode4_host import ROOT, SAN_LIB
    if os.environ.get("QPPOCR_HIP_LIB"):
        pytest.skip("this is the sanitizer run")
    rt = sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not rt or not os.path.exists(SAN_LIB):
        pytest.skip("no ASan runtime or sanitizer build")
    env = dict(os.environ, QPPOCR_HIP_LIB=SAN_LIB, LD_PRELOAD=rt[-1],
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "-m", "not gpu",
                        "tests/test_step4_host.py"], cwd=ROOT, env=env, capture_output=True, text=True,
                       timeout=600)
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    assert "passed" in r.stdout and "runtime error" not in tail
