"""The operators of a decoder's step that checks a tree of drafted tokens, as cases whose time is
measured.

A recogniser that writes a page's text token by token is fast when a cheap guess drafts several
continuations (a tree of tokens) and one pass of the decoder checks them all.  Beside its linears
and the cache of keys and values in 4 bits, such a step consists of

  extend   pages, slots, positions and the tree's masks of a batch, from its lengths
  rotary   the queries' and keys' rotation by positions of one or several axes (text; a page's
           sheet, row and column)
  tree     attention of drafted tokens over the cached context and the drafted ancestors
  sinks    attention to the last `window` tokens and to a sequence's first few
  move     the accepted tokens' keys and values to the places behind the context, and copies of
           cached tokens for a further continuation

The 4-bit format of the cache: 32 neighbouring elements share one scale byte s, an element is a
sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, and stands for that number times 2^(s - 127).
"""
import math
import random

import numpy as np
import torch

own = False

GPU = "cuda:0"
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a step of 48 sequences with a tree of drafted tokens each; some sequences end
        dict(name="extend_tree", op="extend", batch=48, context=4096, new=32, page=64, done=3,
             tree=True),
        # the prompts of many sequences at once
        dict(name="extend_prompts", op="extend", batch=384, context=512, new=4001, page=16,
             done=20, tree=False),
        # the queries and keys of a step, next to the values of the same projection
        dict(name="rotary_step", op="rotary", tokens=32, heads=40, dh=128, pairs=64, axes=1,
             dtype="f16", neighbours=False, inverse=False, index="i32"),
        # a page's patches and its text: sheet, row and column
        dict(name="rotary_page", op="rotary", tokens=20011, heads=40, dh=128, pairs=64, axes=3,
             dtype="bf16", neighbours=False, inverse=False, index="i64"),
        # keys turned back (to be turned anew, or a gradient), half of each head, far positions
        dict(name="rotary_back", op="rotary", tokens=4099, heads=8, dh=96, pairs=24, axes=2,
             dtype="f32", neighbours=True, inverse=True, index="i32"),
        # the accepted path of each of 48 drafted trees behind its context
        dict(name="move_accepted", op="move", tokens=190, heads=8, dh=128, page=64, pages=60,
             dtype="bf16"),
        # a context copied for another continuation
        dict(name="move_copy", op="move", tokens=16001, heads=8, dh=128, page=32, pages=1100,
             dtype="f16"),
        # a step of 32 sequences that see the last 4096 tokens and the first 4
        dict(name="sinks_step", op="attend", tree=0, batch=32, news=1, context=32768, least=1000,
             qheads=32, heads=8, dh=128, page=64, dtype="bf16", window=4096, sinks=4, lse=False),
        # a chunk of two prompts
        dict(name="sinks_chunk", op="attend", tree=0, batch=2, news=1024, context=8192, least=6001,
             qheads=32, heads=8, dh=128, page=64, dtype="bf16", window=2000, sinks=70, lse=False),
        # trees of 8 tokens for 32 lines at the rec encoder's heads
        dict(name="tree_lines", op="attend", tree=8, batch=32, news=8, context=136, least=20,
             qheads=8, heads=8, dh=32, page=16, dtype="f32", window=0, sinks=0, lse=True),
        # trees of up to 32 tokens for 32 sequences
        dict(name="tree_batch", op="attend", tree=8, batch=32, news=32, context=8192, least=300,
             qheads=32, heads=8, dh=128, page=64, dtype="bf16", window=0, sinks=0, lse=False),
        # a wide tree behind one very long context
        dict(name="tree_long", op="attend", tree=12, batch=1, news=100, context=131071,
             least=131071, qheads=32, heads=8, dh=128, page=128, dtype="f16", window=0, sinks=0,
             lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["extend", "rotary", "rotary", "move", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "extend":
        batch, tree = _log(rng, 1, 6000), rng.random() < 0.5
        new = _log(rng, 1, 200) if tree else _log(rng, 1, 6000)
        new = max(1, min(new, 700_000 // batch))
        return dict(op=op, batch=batch, context=_log(rng, 1, max(2, min(20000, 6_000_000 // batch))),
                    new=new, page=rng.choice([16, 32, 64, 128, 256]),
                    done=rng.choice([0, batch // 9]), tree=tree)
    dh = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256])
    heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    if op == "rotary":
        heads = rng.choice([1, 2, 5, 8, 12, 40])
        pairs = rng.choice([dh // 2, dh // 2, dh // 4, rng.randint(1, dh // 2)])
        axes = rng.randint(1, min(4, pairs))
        return dict(op=op, tokens=_log(rng, 1, 80_000_000 // (heads * dh)), heads=heads, dh=dh,
                    pairs=pairs, axes=axes, dtype=dtype, neighbours=rng.random() < 0.4,
                    inverse=rng.random() < 0.3, index=rng.choice(["i32", "i64"]))
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "move":
        tokens = _log(rng, 1, 16_000_000 // (heads * dh))
        pages = int(math.ceil(2 * tokens / page) * rng.uniform(1.0, 1.4)) + 1
        return dict(op=op, tokens=tokens, heads=heads, dh=dh, page=page, pages=pages, dtype=dtype)
    qheads = heads * rng.choice([1, 2, 3, 4, 7, 8, 16])
    qheads = qheads if qheads <= 128 else heads
    mode = rng.choice(["tree", "tree", "tree", "step", "chunk"])
    news = {"step": 1, "tree": _log(rng, 2, 200), "chunk": _log(rng, 16, 1500)}[mode]
    context = max(news, _log(rng, 16, 32768 if mode != "chunk" else 6000))
    batch = _log(rng, 1, 64)
    # no dearer than the listed ones: cached elements, and pairs of a chunk
    batch = max(1, min(batch, 120_000_000 // (context * heads * dh)))
    pairs = 220_000_000 * 128 // (dh * qheads * context)
    news = max(1, min(news, pairs))
    batch = max(1, min(batch, pairs // news))
    window = max(1, context // rng.choice([2, 5, 20]))
    if mode == "tree":
        window = rng.choice([0, 0, window])
    return dict(op=op, tree=rng.choice([1, 4, 16]) if mode == "tree" else 0, batch=batch, news=news,
                context=context, least=rng.choice([0, context // 4]), qheads=qheads, heads=heads,
                dh=dh, page=page, dtype=dtype, window=window,
                sinks=rng.choice([1, 4, 5, 33, 70]) if window else 0, lse=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

def _seeded(seed):
    g = torch.Generator(device=GPU)
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=GPU)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=GPU)


def _pool(case, g):
    """A cache's pages with normal keys and values, channels of different size, in them:
    [pages, heads, page, ...] codes and scales of keys and of values."""
    out = []
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=GPU)
    for _ in range(2):
        shape = (case["pages"], case["heads"], case["page"])
        codes = torch.empty(shape + (case["dh"] // 2,), dtype=torch.uint8, device=GPU)
        scales = torch.empty(shape + (case["dh"] // 32,), dtype=torch.uint8, device=GPU)
        size = torch.exp(0.5 * _normal(g, 1, case["heads"], 1, case["dh"]))
        step = max(1, (1 << 26) // (case["heads"] * case["page"] * case["dh"]))
        for p in range(0, case["pages"], step):
            q = min(case["pages"], p + step)
            x = (_normal(g, q - p, *shape[1:], case["dh"]) * size).unflatten(-1, (-1, 32))
            e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 6.0))
            c = torch.bucketize(x.abs() * torch.exp2(-e), grid).to(torch.uint8)
            c = torch.where(x < 0, c + 8, c).flatten(-2)
            codes[p:q] = c[..., 0::2] | (c[..., 1::2] << 4)
            scales[p:q] = (e[..., 0] + 127).to(torch.uint8)
        out += [codes, scales]
    return out


def _parents(rng, n, spread):
    """A drafted tree: each token's parent is one of the `spread` before it (-1: the context)."""
    return [rng.randint(max(-1, i - spread), i - 1) for i in range(n)]


def _ancestors(parents):
    """[n, n] truth values: token i's own path."""
    a = np.zeros((len(parents), len(parents)), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def _bits(a, words):
    """Rows of truth values as words of 64 bits, the first in the lowest."""
    wide = np.zeros((a.shape[0], 64 * words), dtype=bool)
    wide[:, :a.shape[1]] = a
    return np.packbits(wide, axis=1, bitorder="little").view(np.int64)


def _prepare_extend(case, seed, g, s):
    rng, page = random.Random(seed), case["page"]
    b, most = case["batch"], case["context"] + case["new"]
    lens = [rng.randint(0, case["context"]) for _ in range(b)]
    news = [case["new"] - 37 * i % max(1, case["new"] * 3 // 4) for i in range(b)]
    for k in range(case["done"]):
        # an ended sequence gives its pages back; others give back what was not accepted
        i = k * b // case["done"]
        news[i] = -lens[i] if k % 2 == 0 else -rng.randint(0, lens[i])
    wide = -(-most // page)
    held = [-(-n // page) for n in lens]
    pages = b * wide
    order = torch.randperm(pages, generator=g, device=GPU).int()
    at = np.concatenate([[0], np.cumsum(held)])
    col = torch.arange(wide, device=GPU)[None]
    table = order[(_i32(at[:-1])[:, None] + col).clamp(max=pages - 1).long()]
    s["table"] = torch.where(col < _i32(held)[:, None], table, -1).contiguous()
    # the ring of free pages, its head anywhere
    head = rng.randint(0, 10 * pages)
    ring = torch.full((pages,), -1, dtype=torch.int32, device=GPU)
    free = order[int(at[-1]):]
    ring[(head + torch.arange(free.numel(), device=GPU)) % pages] = free
    s["ring"] = ring
    s["ends"] = torch.tensor([head, head + free.numel()], dtype=torch.int64, device=GPU)
    s["lens"], s["news"] = _i32(lens), _i32(news)
    rows = [max(0, n) for n in news]
    # a padded batch: a few rows more than tokens
    s["tokens"], s["max_new"] = sum(rows) + 7, case["new"]
    s["parents"] = None
    if case["tree"]:
        p = [v for n in rows for v in _parents(rng, n, 8)]
        s["parents"] = _i32(p + [-1] * 7)


def _news(case, i):
    """New tokens of sequence i: they differ in a batch of chunks or trees."""
    m = case["news"]
    return m if m <= 8 else m - 37 * i % (m // 2)


def prepare(case, seed):
    g, rng = _seeded(seed), random.Random(seed)
    s = {"case": case}
    if case["op"] == "extend":
        _prepare_extend(case, seed, g, s)
        return s
    dtype = TYPES[case["dtype"]]
    heads, dh = case["heads"], case["dh"]
    if case["op"] == "rotary":
        t, r, n = case["tokens"], case["pairs"], case["axes"]
        # queries and keys in front of the values, as one projection leaves them
        packed = _normal(g, t, heads + 2, dh).to(dtype)
        s["x"] = packed[:, :heads]
        index = torch.int32 if case["index"] == "i32" else torch.int64
        i = torch.arange(t, device=GPU)
        side = max(1, int(math.sqrt(t)))
        grid = [i + rng.randint(0, 200_000), i // side, i % side, i // (3 * side) + 1000]
        s["pos"] = torch.stack(grid[:n]).to(index) if n > 1 else grid[0].to(index)
        s["freqs"] = [10000.0 ** (-k / r) for k in range(r)]
        s["axes"] = [k * n // r for k in range(r)]
        if own:
            from qppocr_amd import ops
            s["plan"] = ops.rotary_plan(dh, s["freqs"], s["axes"], case["neighbours"], device=GPU)
        return s
    if case["op"] == "attend":
        news = [_news(case, i) for i in range(case["batch"])]
        lens = [case["context"] if i == 0 else rng.randint(case["least"], case["context"])
                for i in range(case["batch"])]
        if case["tree"]:                  # the drafted tokens are cached behind the context
            lens = [max(n, m) for n, m in zip(lens, news)]
        if case["least"] == 0:            # slots of the batch that no sequence has
            lens = [0 if i and rng.random() < 0.08 else n for i, n in enumerate(lens)]
        s["lens_host"], s["news_host"] = lens, news
        need = [(v + case["page"] - 1) // case["page"] for v in lens]
        case = dict(case, pages=max(1, sum(need)) + 3)
    s["pool"] = _pool(case, g)
    page = case["page"]
    order = torch.randperm(case["pages"], generator=g, device=GPU)
    if case["op"] == "attend":
        table = torch.full((case["batch"], max(1, max(need))), -1, dtype=torch.int32, device=GPU)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = order[at:at + m].int()
            at += m
        s["table"], s["lens"] = table, _i32(lens)
        s["starts"] = _i32([0] + list(np.cumsum(news)))
        s["max_len"], s["max_new"] = max(lens), max(news)
        s["q"] = _normal(g, sum(news), case["qheads"], dh).to(dtype)
        if case["tree"]:
            words = -(-max(news) // 64)
            s["paths"] = [_ancestors(_parents(rng, n, case["tree"])) for n in news]
            bits = np.concatenate([_bits(a, words) for a in s["paths"]])
            s["tree"] = torch.from_numpy(bits).to(GPU)
            s["paths"] = [torch.from_numpy(a).to(GPU) for a in s["paths"]]
    else:
        # some tokens' places and others that they move to, in shuffled pages; a few stay
        t = torch.arange(case["pages"] * page, device=GPU)
        slots = order[t // page] * page + t % page
        n = case["tokens"]
        s["src"], s["dst"] = slots[n:2 * n].contiguous(), slots[:n].clone()
        s["dst"][::5] = s["src"][::5]
        s["all"] = t
    if own:
        from qppocr_amd import ops
        s["cache"] = ops.Cache4(*s["pool"])
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return {"extend": _run_extend, "rotary": _run_rotary, "move": _run_move,
            "attend": _run_attend}[s["case"]["op"]](s)


def _run_extend(s):
    page, tokens = s["case"]["page"], s["tokens"]
    table, ring = s["table"], s["ring"]
    if own:
        from qppocr_amd import ops
        step = ops.cache4_extend(table, s["lens"], s["news"], page, ring, s["ends"], tokens,
                                 parents=s["parents"], max_new=s["max_new"])
        out = [table, ring, step.lens, step.starts, step.slots, step.positions, step.ends]
        return out + ([step.tree] if s["parents"] is not None else [])
    lens, n = s["lens"].long(), s["news"].long()
    cap, wide = ring.numel(), table.shape[1]
    rows = n.clamp(min=0)
    ends = rows.cumsum(0)
    held, first = (lens + page - 1) // page, ends - rows
    after = torch.where(n < 0, (lens + n).clamp(min=0), lens + n)
    fits = (n >= 0) & (after <= wide * page) & (ends <= tokens)
    pages = (after + page - 1) // page
    need = torch.where(fits, pages - held, 0)
    taken = need.cumsum(0)
    head, tail = s["ends"][0], s["ends"][1]
    fits = fits & ((need == 0) | (taken <= tail - head))
    back = torch.where(n < 0, held - pages, 0)
    given = back.cumsum(0)
    # rows: the sequence of each, its page from the table or the ring
    r = torch.arange(tokens, device=GPU)
    b = torch.searchsorted(ends, r, right=True)
    live = b < ends.numel()
    b = b.clamp(max=ends.numel() - 1)
    i = r - first[b]
    at = lens[b] + i
    column = (at // page).clamp(max=wide - 1)
    fresh = ring[(head + (taken - need)[b] + column - held[b]).clamp(min=0) % cap]
    number = torch.where(column < held[b], table[b, column], fresh).long()
    ok = live & fits[b] & (number >= 0)
    slots = torch.where(ok, number * page + at % page, -1)
    positions = torch.where(live, at, 0)
    bits = None
    if s["parents"] is not None:
        # the paths of every sequence by squaring: one step, two steps, four, ...
        m = s["max_new"]
        k = torch.arange(m, device=GPU)
        have = k < rows[:, None]
        up = s["parents"][(first[:, None] + k).clamp(max=tokens - 1)]
        path = ((k == up.unsqueeze(-1)) | (k == k[:, None])) & have.unsqueeze(-1)
        path = path.float()
        for _ in range(max(1, m - 1).bit_length()):
            path = (torch.matmul(path, path) > 0).float()
        mine = torch.where(live.unsqueeze(-1), path[b, i.clamp(min=0, max=m - 1)], 0.0)
        positions = torch.where(live, lens[b] + mine.sum(-1).long() - 1, 0)
        words = (m + 63) // 64
        wide_bits = torch.zeros((tokens, 64 * words), dtype=torch.int64, device=GPU)
        wide_bits[:, :m] = mine.long()
        power = torch.arange(64, device=GPU)
        bits = (wide_bits.unflatten(-1, (words, 64)) << power).sum(-1)
    # the table's new pages, the ring's returned ones
    col = torch.arange(wide, device=GPU)[None]
    grown = fits[:, None] & (col >= held[:, None]) & (col < pages[:, None])
    new = ring[(head + (taken - need)[:, None] + col - held[:, None]).clamp(min=0) % cap]
    gone = (n < 0)[:, None] & (col >= pages[:, None]) & (col < held[:, None])
    place = (tail + (given - back)[:, None] + col - pages[:, None]).clamp(min=0) % cap
    # (places that get nothing: one behind the ring)
    held_ring = torch.cat([ring, ring[:1]])
    held_ring[torch.where(gone, place, cap).flatten()] = torch.where(gone, table, ring[0]).flatten()
    ring.copy_(held_ring[:cap])
    table.copy_(torch.where(grown, new, table))
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    most = torch.where(fits & (need > 0), taken, 0).amax()
    out = [table, ring, torch.where(fits | (n < 0), after, lens).int(), starts, slots,
           positions.int(), torch.stack([head + most, tail + given[-1]])]
    return out + ([bits] if bits is not None else [])


def _run_rotary(s):
    case, x = s["case"], s["x"]
    if own:
        from qppocr_amd import ops
        return ops.rotary(x, s["pos"], s["plan"], inverse=case["inverse"])
    r = case["pairs"]
    pos = s["pos"].double().view(-1, x.shape[0])
    axes = torch.tensor(s["axes"], device=GPU)
    turn = pos[axes].t() * torch.tensor(s["freqs"], dtype=torch.float64, device=GPU)
    cos, sin = torch.cos(turn).float().unsqueeze(1), torch.sin(turn).float().unsqueeze(1)
    if case["inverse"]:
        sin = -sin
    y = x.float().clone()
    if case["neighbours"]:
        a, b = y[..., 0:2 * r:2].clone(), y[..., 1:2 * r:2].clone()
        y[..., 0:2 * r:2], y[..., 1:2 * r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = y[..., :r].clone(), y[..., r:2 * r].clone()
        y[..., :r], y[..., r:2 * r] = a * cos - b * sin, a * sin + b * cos
    return y.to(x.dtype)


def _decode(packed, scale):
    """What packed codes [..., 16 m] and scale bytes [..., m] stand for."""
    level = torch.tensor(LEVELS + [-v for v in LEVELS], device=packed.device)
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    two = torch.exp2(scale.float() - 127.0)
    return level[code] * two.repeat_interleave(32, -1)


def _run_move(s):
    """The moves; then the pool's values, moved tokens and others."""
    case, pool = s["case"], s["pool"]
    dtype, page = TYPES[case["dtype"]], case["page"]
    if own:
        from qppocr_amd import ops
        ops.cache4_move(s["cache"], s["src"], s["dst"])
        return ops.cache4_read(s["cache"], s["all"], dtype)
    src, dst = s["src"], s["dst"]
    for t in pool:
        t[dst // page, :, dst % page] = t[src // page, :, src % page]
    kc, ks, vc, vs = pool
    return tuple(_decode(c, e).transpose(1, 2).reshape(-1, case["heads"], case["dh"]).to(dtype)
                 for c, e in ((kc, ks), (vc, vs)))


def _run_attend(s):
    case, q = s["case"], s["q"]
    scale = 1.0 / math.sqrt(case["dh"])
    if own:
        from qppocr_amd import ops
        more = dict(starts=s["starts"], max_new=s["max_new"], max_len=s["max_len"],
                    window=case["window"], sinks=case["sinks"], lse=case["lse"])
        if case["tree"]:
            return ops.attention_tree4(q, s["cache"], s["table"], s["lens"], scale, s["tree"],
                                       **more)
        return ops.attention_cache4(q, s["cache"], s["table"], s["lens"], scale, **more)
    kc, ks, vc, vs = s["pool"]
    heads, dh, qheads = case["heads"], case["dh"], case["qheads"]
    group, window, sinks = qheads // heads, case["window"], case["sinks"]
    out = torch.zeros(q.shape, device=GPU)
    sums = torch.full(q.shape[:2], -math.inf, device=GPU)
    at = 0
    for b, (n, m) in enumerate(zip(s["lens_host"], s["news_host"])):
        if n:
            # the tokens that some row sees: the first ones, and all from the window's start
            low = max(0, n - m - window) if window else 0
            key = torch.cat([torch.arange(min(sinks, low), device=GPU),
                             torch.arange(low, n, device=GPU)])
            pages = s["table"][b, key // case["page"]].long()
            place = key % case["page"]
            # [heads, tokens, dh]
            k = _decode(kc[pages, :, place], ks[pages, :, place]).transpose(0, 1).contiguous()
            v = _decode(vc[pages, :, place], vs[pages, :, place]).transpose(0, 1).contiguous()
            x = q[at:at + m].float().view(m, heads, group, dh)
            x = x.permute(1, 0, 2, 3).reshape(heads, -1, dh)
            w = torch.matmul(x, k.transpose(1, 2).contiguous()) * scale
            pos = torch.arange(m, device=GPU)[:, None] + (n - m)
            if case["tree"]:
                path = s["paths"][b]
                pos = n - m + path.sum(-1, keepdim=True) - 1
                drafted = path[:, (key - (n - m)).clamp(min=0)] & (key >= n - m)
                see = key < n - m
            else:
                drafted = torch.zeros((), dtype=torch.bool, device=GPU)
                see = key <= pos
            if window:
                see = see & ((key > pos - window) | (key < sinks))
            see = (see | drafted).expand(m, key.numel()).repeat_interleave(group, 0)
            w = torch.where(see, w, -math.inf)
            top = w.amax(-1, keepdim=True)
            none = top == -math.inf         # rows before the first key see nothing
            w = torch.exp(w - torch.where(none, 0.0, top))
            total = w.sum(-1, keepdim=True)
            y = torch.matmul(w, v) / torch.where(none, 1.0, total)
            out[at:at + m] = y.view(heads, m, group, dh).transpose(0, 1).reshape(m, qheads, dh)
            sums[at:at + m] = ((top + torch.log(total)).view(heads, m, group)
                               .transpose(0, 1).reshape(m, qheads))
        at += m
    out = out.to(q.dtype)
    return (out, sums) if case["lse"] else out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "extend":
        # (new tokens: those of the middle of the range)
        b = case["batch"]
        t = (b - case["done"]) * (case["new"] * 5 // 8 + 1)
        words = (case["new"] + 63) // 64
        # lengths and places of the batch, rows, parents and masks, pages from the ring
        byte = 16 * b + t * (12 + (4 + 8 * words if case["tree"] else 0)) + 8 * (t // case["page"])
        return {"bytes": byte, "flops": 4 * t}
    size, per = SIZE[case["dtype"]], case["heads"] * case["dh"]
    if case["op"] == "rotary":
        t = case["tokens"]
        index = (4 if case["index"] == "i32" else 8) * case["axes"]
        return {"bytes": t * (index + 2 * per * size), "flops": 6 * t * case["heads"] * case["pairs"]}
    held = 2 * (per // 2 + per // 32)           # a token's keys and values in the cache
    if case["op"] == "move":
        a = case["pages"] * case["page"]
        return {"bytes": case["tokens"] * (16 + 2 * held) + a * (8 + held + 2 * per * size),
                "flops": 2 * a * per}
    # lengths are drawn from the seed: those of the middle of the range
    ns = [case["context"]] + [(case["context"] + case["least"]) // 2] * (case["batch"] - 1)
    pairs = keys = rows = 0
    for i, n in enumerate(ns):
        m = _news(case, i)
        n = max(n, m)
        rows += m * case["qheads"] * case["dh"]
        window, sinks = case["window"] or n, case["sinks"]
        if case["tree"]:
            # (a path has a few tokens of the tree)
            c = n - m
            see = min(c, window + min(sinks, max(0, c - window)))
            pairs += m * (see + min(m, 8))
            keys += see + m
        else:
            for p in range(n - m, n):
                pairs += min(p + 1, window + min(sinks, max(0, p + 1 - window)))
            low = max(0, n - m - window + 1)
            keys += n - low + min(sinks, low)
    return {"bytes": keys * held + 2 * rows * size,
            "flops": 4 * pairs * case["qheads"] * case["dh"]}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_numbers(packed, scale):
    """The numbers of packed codes in 64 bits, from the fields of a code: sign, two bits of
    exponent (bias 1), one of mantissa."""
    c = torch.empty(packed.shape + (2,), dtype=torch.uint8, device=packed.device)
    c[..., 0], c[..., 1] = packed.remainder(16), packed.div(16, rounding_mode="floor")
    c = c.view(scale.shape + (32,))
    e, m = (c // 2) % 4, (c % 2).double()
    mag = torch.where(e == 0, 0.5 * m, (2.0 + m) * (1 << e.int()) / 4)
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.arange(256.0).double() - 127)
    two = s.to(packed.device)[scale.int()].unsqueeze(-1)
    return (torch.where(c >= 8, -mag, mag) * two).flatten(-2)


def _exact_extend(s):
    """Sequence by sequence, on the host."""
    page, tokens = s["case"]["page"], s["tokens"]
    table, ring = s["table"].cpu().numpy().copy(), s["ring"].cpu().numpy().copy()
    lens, news = s["lens"].cpu().numpy().copy(), s["news"].cpu().numpy()
    head, tail = (int(v) for v in s["ends"].cpu())
    free, limit = head, tail
    slots = np.full(tokens, -1, dtype=np.int64)
    positions = np.zeros(tokens, dtype=np.int32)
    starts = np.zeros(len(lens) + 1, dtype=np.int32)
    words = (s["max_new"] + 63) // 64
    tree = np.zeros((tokens, words), dtype=np.int64)
    parents = None if s["parents"] is None else s["parents"].cpu().numpy()
    was = ring.copy()
    for b in range(len(lens)):
        n, held = int(news[b]), -(-int(lens[b]) // page)
        r = int(starts[b])
        starts[b + 1] = r + max(n, 0)
        if n < 0:
            keep = -(-(int(lens[b]) + n) // page)
            for c in range(keep, held):
                ring[tail % len(ring)] = table[b, c]
                tail += 1
            lens[b] += n
            continue
        want = -(-(int(lens[b]) + n) // page)
        if free + want - held > limit:
            raise ValueError("the pool is too small")
        for c in range(held, want):
            table[b, c] = was[free % len(ring)]
            free += 1
        p = int(lens[b]) + np.arange(n)
        slots[r:r + n] = table[b, p // page].astype(np.int64) * page + p % page
        positions[r:r + n] = p
        if parents is not None:
            path = _ancestors(parents[r:r + n].tolist())
            tree[r:r + n] = _bits(path, words)
            positions[r:r + n] = lens[b] + path.sum(1) - 1
        lens[b] += n
    out = [table, ring, lens, starts, slots, positions, np.array([free, tail])]
    out += [tree] if parents is not None else []
    return [torch.from_numpy(np.ascontiguousarray(v)).to(GPU) for v in out]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "extend":
        return _exact_extend(s)
    if case["op"] == "rotary":
        # as a product of complex numbers, one pair of each head at a time
        x, r, dh = s["x"].double(), case["pairs"], case["dh"]
        y = x.clone()
        pos = s["pos"].double().reshape(-1, case["tokens"])
        sign = -1.0 if case["inverse"] else 1.0
        for i in range(r):
            a, b = (2 * i, 2 * i + 1) if case["neighbours"] else (i, i + r)
            angle = sign * pos[s["axes"][i]] * s["freqs"][i]
            z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(angle), angle)[:, None]
            y[..., a], y[..., b] = z.real, z.imag
        return y
    if case["op"] == "move":
        kc, ks, vc, vs = s["pool"]
        res = []
        for codes, scales in ((kc, ks), (vc, vs)):
            y = _exact_numbers(codes, scales).transpose(1, 2).flatten(0, 1)
            y[s["dst"]] = y[s["src"]]
            res.append(y)
        return tuple(res)
    # one sequence and one of the cache's heads at a time, in blocks of new tokens
    pool, at = s["pool"], 0
    heads, dh = case["heads"], case["dh"]
    group, window, sinks = case["qheads"] // heads, case["window"], case["sinks"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU)
    sums = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=GPU)
    for b, (n, m) in enumerate(zip(s["lens_host"], s["news_host"])):
        c = n - m
        for h in range(heads if n else 0):
            pages = s["table"][b, :-(-n // case["page"])].long()
            k, v = (_exact_numbers(pool[2 * i][pages, h], pool[2 * i + 1][pages, h])
                    .reshape(-1, dh)[:n] for i in (0, 1))
            kt = k.t().contiguous()
            key = torch.arange(n, device=GPU)
            for i in range(0, m, 256):
                j = min(m, i + 256)
                x = s["q"][at + i:at + j, h * group:(h + 1) * group].double()
                z = torch.mm(x.reshape(-1, dh), kt).view(j - i, group, n) / math.sqrt(dh)
                pos = torch.arange(c + i, c + j, device=GPU)[:, None]
                hide = key > pos
                if case["tree"]:
                    path = s["paths"][b][i:j]
                    pos = c - 1 + path.long().sum(1)[:, None]
                    hide = (key >= c).expand(j - i, n).clone()
                if window:
                    hide = hide | ((key + window <= pos) & (key >= sinks))
                if case["tree"] and c >= 0:
                    hide[:, c:] = ~path
                z = z.masked_fill(hide[:, None], -math.inf)
                lse = torch.logsumexp(z, -1)
                p = torch.exp(z - lse[..., None]).masked_fill(hide[:, None], 0.0).view(-1, n)
                out[at + i:at + j, h * group:(h + 1) * group] = torch.mm(p, v).view(j - i, group, dh)
                sums[at + i:at + j, h * group:(h + 1) * group] = lse
        at += m
    return (out, sums) if case["lse"] else out
