"""The 4-bit operators' calls that a program makes in less usual ways, and the
forms of their kernels that only particular sizes reach, against the same
definitions in 64 bits as the other tests of these operators."""
import numpy as np
import pytest

from test_gpu_decode4 import host, make_cache, tables

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
