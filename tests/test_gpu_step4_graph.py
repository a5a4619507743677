"""A whole step that checks drafted trees, captured once: pages, positions and masks from
the lengths, rotation, the cache's writes, attention, the accepted paths' move and the
pages given back, with nothing read by the host.  Every replay equals the same calls made
one after the other on a copy of the state."""
import numpy as np
import pytest

from test_gpu_decode4 import DTYPES, host
from test_gpu_mask4 import drafted, paths

pytestmark = pytest.mark.gpu

BATCH, MOST, HEADS, GROUP, DH, PAGE, WIDE = 6, 12, 2, 4, 64, 16, 8
TOKENS = BATCH * MOST


class State:
    def __init__(self, torch, rng, dtype, pages):
        from qppocr_amd import ops
        i32 = dict(dtype=torch.int32, device="cuda")
        self.cache = ops.cache4(pages, PAGE, HEADS, DH)
        self.table = torch.full((BATCH, WIDE), -1, **i32)
        self.ring = torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda()
        self.ends = torch.tensor([0, pages], device="cuda")
        self.lens, self.news = torch.zeros(BATCH, **i32), torch.zeros(BATCH, **i32)
        self.parents = torch.zeros(TOKENS, **i32)
        self.leaf = torch.zeros(BATCH, dtype=torch.int64, device="cuda")
        self.qkv = torch.zeros((TOKENS, HEADS * (GROUP + 2), DH), device="cuda", dtype=dtype)
        self.out = torch.zeros((TOKENS, HEADS * GROUP, DH), device="cuda", dtype=dtype)

    def tensors(self):
        c = self.cache
        return [self.table, self.ring, self.ends, self.lens, self.news, self.parents, self.leaf, self.qkv, self.out,
                c.k_codes, c.k_scales, c.v_codes, c.v_scales]


def step(torch, s, plan):
    """One step of the state; what was granted, and the tokens kept."""
    from qppocr_amd import ops
    grown = ops.cache4_extend(s.table, s.lens, s.news, PAGE, s.ring, s.ends, TOKENS, s.parents, MOST)
    granted = grown.lens - s.lens               # a sequence's new tokens, or none of them
    qk = ops.rotary(s.qkv[:, :HEADS * (GROUP + 1)], grown.positions, plan)
    q, k = qk.split([HEADS * GROUP, HEADS], 1)
    ops.cache4_write(s.cache, k, s.qkv[:, HEADS * (GROUP + 1):], grown.slots)
    ops.attention_tree4(q, s.cache, s.table, grown.lens, DH ** -0.5, grown.tree, starts=grown.starts,
                        max_new=MOST, out=s.out)
    # the path of each sequence's accepted leaf, from its mask
    i = torch.arange(MOST, device="cuda")
    first = grown.starts[:-1, None].long()
    leaf = (first[:, 0] + s.leaf).clamp(max=TOKENS - 1)
    path = (grown.tree[leaf, 0][:, None] >> i) & 1
    path = torch.where((granted > 0)[:, None], path, 0)
    rank = path.cumsum(1) - 1
    src = torch.where(path > 0, grown.slots[(first + i).clamp(max=TOKENS - 1)], -1)
    dst = torch.where(path > 0, grown.slots[(first + rank).clamp(0, TOKENS - 1)], -1)
    ops.cache4_move(s.cache, src.flatten(), dst.flatten())
    kept = (rank[:, -1] + 1).int()
    left = ops.cache4_extend(s.table, grown.lens, kept - granted, PAGE, s.ring, grown.ends, 0)
    s.lens.copy_(left.lens)
    s.ends.copy_(left.ends)
    return granted, kept


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pages", [11, 7])
def test_a_captured_step(gpu, dtype, pages):
    """Few pages: some steps' sequences are not granted, whose rows count for nothing."""
    rng = np.random.default_rng(11)
    from qppocr_amd import ops
    plan = ops.rotary_plan(DH, [1000.0 ** (-i / 32) for i in range(32)])
    a, b = State(gpu, rng, getattr(gpu, dtype), pages), State(gpu, rng, getattr(gpu, dtype), pages)

    def same_state():
        for x, y in zip(a.tensors(), b.tensors()):
            y.copy_(x)
    # (workspaces and contexts of a first call are made outside the graph)
    side = gpu.cuda.Stream()
    gpu.cuda.synchronize()
    with gpu.cuda.stream(side):
        step(gpu, b, plan)
    gpu.cuda.synchronize()
    same_state()
    g = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(g):
        granted, kept = step(gpu, a, plan)
    lens, refused = [0] * BATCH, 0
    for turn in range(12):
        print("captured step", dtype, pages, turn, flush=True)
        news = [int(x) for x in rng.integers(0, MOST + 1, BATCH)]
        trees = [drafted(rng, n, 3) for n in news]
        leaf = [int(rng.integers(0, n)) if n else 0 for n in news]
        if turn % 4 == 3:                       # a sequence ends
            gone = [0] * BATCH
            gone[turn % BATCH] = -lens[turn % BATCH]
            for s in (a, b):
                e = ops.cache4_extend(s.table, s.lens, gpu.tensor(gone, dtype=gpu.int32, device="cuda"), PAGE, s.ring,
                                      s.ends, 0)
                s.lens.copy_(e.lens)
                s.ends.copy_(e.ends)
            lens[turn % BATCH] = 0
        rows = [p for t in trees for p in t]
        qkv = gpu.from_numpy(rng.standard_normal(a.qkv.shape).astype(np.float32)).to(a.qkv.dtype)
        for s in (a, b):
            s.news.copy_(gpu.tensor(news, dtype=gpu.int32))
            s.leaf.copy_(gpu.tensor(leaf))
            s.parents[:len(rows)] = gpu.tensor(rows, dtype=gpu.int32, device="cuda")
            s.qkv.copy_(qkv)
        gpu.cuda.synchronize()
        g.replay()
        want = step(gpu, b, plan)
        gpu.cuda.synchronize()
        for name, x, y in (("granted", granted, want[0]), ("kept", kept, want[1])):
            assert x.tolist() == y.tolist(), (turn, name)
        for x, y in zip(a.tensors(), b.tensors()):
            assert (host(x) == host(y)).all(), turn
        # the definition of lengths; a sequence that is not granted keeps its own
        for i in range(BATCH):
            got = granted.tolist()[i]
            assert got in (0, news[i])
            refused += got != news[i]
            deep = int(paths(trees[i])[leaf[i]].sum()) if got else 0
            assert kept.tolist()[i] == deep
            lens[i] += deep
        assert a.lens.tolist() == lens
        # no page is held twice or lost
        tab, e = a.table.tolist(), a.ends.tolist()
        held = [tab[i][p] for i in range(BATCH) for p in range(-(-lens[i] // PAGE))]
        free = [int(a.ring[i % pages]) for i in range(*e)]
        assert sorted(held + free) == list(range(pages)), turn
    assert sum(lens) > 0 and (refused > 0 or pages > 7)
