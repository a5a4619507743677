"""Limits of the 4-bit operators' C calls, on the host: what a call may ask for
and still be launched, and what is refused (no GPU, no context)."""
import ctypes

import pytest

from test_decode4_host import A, EINVAL, EUNSUPPORTED, attn, cache, lib, refused  # noqa: F401


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("bad,good", [(1e-45, 1.18e-38), (1.17e-38, 1.18e-38), (2.36e38, 2.35e38), (3.4e38, 2.35e38)])
def test_smallest_and_largest_scale(lib, sign, bad, good):  # noqa: F811
    """The device's arithmetic takes a subnormal scale as zero, and multiplies
    scores by scale log2 e."""
    for scale, text in ((bad, "scale"), (good, "null context")):
        a = attn(scale=sign * scale)
        refused(lib, lib.qph_attention_cache4(None, ctypes.byref(cache()), ctypes.byref(a)), EINVAL, text)


def test_most_blocks_of_a_weight(lib):  # noqa: F811
    """A launch has fewer than 2^32 threads along an axis: 2^24 - 1 workgroups."""
    for k, groups in ((128, 4), (1 << 20, 1 << 15)):
        rows = ((1 << 24) - 1) * 256 // groups
        for n, code, text in ((rows, EINVAL, "null context"), (rows + 1, EUNSUPPORTED, "blocks")):
            refused(lib, lib.qph_quantize4(None, A, 1, n, k, 0, 1, A, A), code, text)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,k,columns,threads", [
    (1, 2048, 64, 512), (16, 4096, 64, 512), (1, 1024, 64, 256), (3, 512, 64, 128), (1, 256, 64, 64), (17, 2048, None, 512),
    (3000, 4096, 128, 512), (200, 64, 128, 512)])
def test_most_columns_of_a_linear(lib, dtype, rows, k, columns, threads):  # noqa: F811
    """Every column count whose workgroups (of 64 columns, with more rows 128) stay below
    2^32 threads, and 2^30 at most."""
    def call(n):
        return lib.qph_linear4(None, A, dtype, k, A, A, None, rows, k, n, None, None, A)
    if columns is None:                            # (48 or 128 by the type)
        columns = 128 if dtype == 0 else 48
    most = min(columns * (((1 << 32) - 1) // threads), 1 << 30)
    refused(lib, call(most), EINVAL, "null context")
    refused(lib, call(most + 1), EUNSUPPORTED, "columns")
    refused(lib, call(1 << 26), EINVAL, "null context")


def test_most_sequences_of_an_attention(lib):  # noqa: F811
    """Workgroups: one at least a sequence and cache head; bounds on new tokens and
    keys make no more of them than can be launched."""
    c = cache(heads=8)
    for batch, code, text in (((1 << 21) - 1, EINVAL, "null context"), (1 << 21, EUNSUPPORTED, "batch too large")):
        for new in (1, 5000, (1 << 31) - 1):
            a = attn(batch=batch, heads=32, max_new=new, max_len=(1 << 31) - 1)
            refused(lib, lib.qph_attention_cache4(None, ctypes.byref(c), ctypes.byref(a)), code, text)
