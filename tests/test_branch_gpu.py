"""Drafted trees, page copies and beams against plain restatements in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CUDA = "cuda"


def _ops():
    from inference_b200 import ops

    return ops


def _gen(seed):
    return torch.Generator(device=CUDA).manual_seed(seed)


def _trees(q_lens, seed, shape="bushy"):
    """Parents of each sequence's tokens."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in q_lens:
        back = {"bushy": 6, "chain": 1, "star": n}[shape]
        out.append([-1] + [max(0, i - 1 - int(torch.randint(0, back, (1,), generator=g))) if shape != "star" else 0 for i in range(1, n)] if n else [])
    return out


def _visible(trees, max_q):
    """sees [T, max_q] and depths [T] of trees."""
    rows, depths = [], []
    for tree in trees:
        mine = []
        for i, up in enumerate(tree):
            row = mine[up].clone() if 0 <= up < i else torch.zeros(max_q, dtype=torch.bool)
            row[i] = True
            mine.append(row)
            depths.append(int(row.sum()) - 1)
        rows += mine
    return (torch.stack(rows) if rows else torch.zeros(0, max_q, dtype=torch.bool)), torch.tensor(depths, dtype=torch.int32)


def _pack(sees):
    words = -(-sees.shape[1] // 32)
    wide = torch.zeros(sees.shape[0], words * 32, dtype=torch.int64)
    wide[:, :sees.shape[1]] = sees
    return (wide.view(-1, words, 32) << torch.arange(32)).sum(-1).to(torch.int32).to(CUDA)


class Step:
    """A paged cache whose pages lie in random order, NaN wherever no token of a sequence is, and a step's queries."""

    def __init__(self, base, q_lens, *, heads=8, kv_heads=2, D=128, Dv=None, bs=16, kind=torch.bfloat16, seed=0, extra_pages=2, ragged=True, front=0, behind=0, tight=False):
        g = _gen(seed)
        Dv = D if Dv is None else Dv
        self.base, self.q_lens, self.bs, self.kind, self.front = list(base), list(q_lens), bs, kind, front
        self.lens = [b + n for b, n in zip(base, q_lens)]
        B = len(self.lens)
        self.per = max(1, -(-max(self.lens) // bs)) + (0 if tight else extra_pages)
        self.blocks = B * self.per + 3
        self.k = torch.randn(self.blocks, kv_heads, bs, D, device=CUDA, generator=g).to(kind)
        self.v = torch.randn(self.blocks, kv_heads, bs, Dv, device=CUDA, generator=g).to(kind)
        self.table = torch.randperm(self.blocks, device=CUDA, generator=g)[:B * self.per].to(torch.int32).view(B, self.per)
        used = torch.zeros(self.blocks, bs, dtype=torch.bool, device=CUDA)
        for b, n in enumerate(self.lens):
            at = torch.arange(n, device=CUDA)
            used[self.table[b].long()[at // bs], at % bs] = True
        for t in (self.k, self.v):
            t.masked_fill_(~used[:, None, :, None], float("nan"))
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device=CUDA)
        self.T = sum(q_lens)
        rows = front + self.T + behind
        self.q = torch.randn(rows, heads + 1, D + 8, device=CUDA, generator=g).to(kind)[:, :heads, :D]      # strided tokens and heads
        self.heads, self.kv_heads, self.G = heads, kv_heads, heads // kv_heads
        self.max_q = max(1, max(q_lens))
        uniform = len(set(q_lens)) == 1 and not ragged and not behind and not front
        starts = [front]
        for n in q_lens:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.cu = None if uniform else torch.tensor(starts, dtype=torch.int32, device=CUDA)

    @property
    def step(self):
        return {"cu_q": self.cu, "max_q_len": self.max_q}

    def place(self, b, key):
        return int(self.table[b, key // self.bs]), key % self.bs

    def check(self, out, sees, scale, softcap=0.0, splits=64):
        """sees [T, max_q]: new tokens that each token sees."""
        Dv, D = self.v.shape[3], self.q.shape[2]
        out = out.view(out.shape[0], self.heads, Dv)
        for b, (c, n) in enumerate(zip(self.base, self.q_lens)):
            at = torch.arange(c + n, device=CUDA)
            k, v = (x[self.table[b].long()[at // self.bs], :, at % self.bs].transpose(0, 1).double() for x in (self.k, self.v))
            for i in range(n):
                t = self.starts[b] + i
                use = torch.cat([torch.arange(c), c + sees[t - self.front, :n].nonzero()[:, 0]]).to(CUDA)
                for h in range(self.kv_heads):
                    got = out[t, h * self.G:(h + 1) * self.G].double()
                    if use.numel() == 0:
                        assert (got == 0).all(), (t, h)
                        continue
                    q, kk, vv = self.q[t, h * self.G:(h + 1) * self.G].double(), k[h, use], v[h, use]
                    s = q @ kk.T * scale
                    size = float((q.abs() @ kk.abs().T * abs(scale)).max())
                    if softcap:
                        s = softcap * torch.tanh(s / softcap)
                    p = torch.softmax(s, -1)
                    o, pv = p @ vv, p @ vv.abs()
                    # A product of D terms in 32 bits is off by (D + 4) 2^-24 of the sum of their sizes, a capped score by 2^-19 of the cap more; the exponential of a score of which
                    # that much is uncertain, twice (numerator and sum), and sums over the keys and the splits.
                    ds = (D + 4) * 2.0 ** -24 * size + softcap * 2.0 ** -19
                    rel = math.expm1(2 * ds) + 2.0 ** -19 + (use.numel() + splits + 8) * 2.0 ** -23
                    tol = rel * pv + 1e-30
                    if self.kind == torch.bfloat16:     # the weights of a product and the result are rounded to bf16: half a step each
                        tol = tol + 2.0 ** -8 * pv * (1 + rel) + 2.0 ** -8 * o.abs()
                    assert ((got - o).abs() <= tol).all(), (t, b, h, float(((got - o).abs() / tol).max()))


def _run(c, mask, scale, **kw):
    return _ops().tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, mask, scale=scale, **c.step, **kw)


# ---- what trees see -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("q_lens,shape", [([1], "bushy"), ([7, 1, 40], "bushy"), ([33, 0, 32, 64], "chain"), ([100, 31], "star"), ([300, 2], "bushy"), ([257], "chain")])
def test_plans(q_lens, shape):
    trees = _trees(q_lens, 3, shape)
    sees, depths = _visible(trees, max(q_lens))
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device=CUDA)
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32, device=CUDA)
    got = _ops().plan_tree(parents, cu_q=cu, max_q_len=max(q_lens))
    assert torch.equal(got.mask, _pack(sees)) and torch.equal(got.depths.cpu(), depths)
    if len(q_lens) == 1:
        again = _ops().plan_tree(parents, cu_q=None, max_q_len=q_lens[0])
        assert torch.equal(again.mask, got.mask) and torch.equal(again.depths, got.depths)


def test_plans_of_parents_that_are_not_in_front():
    parents = torch.tensor([5, 1, -7, 0, 3, 2 ** 31 - 1], dtype=torch.int32, device=CUDA)
    got = _ops().plan_tree(parents, cu_q=None, max_q_len=6)
    assert got.depths.tolist() == [0, 0, 0, 1, 2, 0]
    assert got.mask[:, 0].tolist() == [1, 2, 4, 1 + 8, 1 + 8 + 16, 32]


# ---- attention ------------------------------------------------------------------------------------------------------------------------------------------
SHAPES = [
    # heads, kv heads, width, value width, page
    (8, 2, 128, 128, 16),
    (4, 4, 64, 64, 16),
    (12, 1, 96, 64, 32),
    (28, 4, 128, 128, 16),
    (5, 1, 40, 24, 16),
    (6, 3, 72, 120, 48),
]
ODD = [(8, 2, 33, 20, 5), (3, 1, 256, 200, 16), (2, 1, 10, 256, 1), (128, 1, 16, 8, 16)]


@pytest.mark.parametrize("shape", SHAPES + ODD, ids=str)
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("base,q_lens", [([0], [1]), ([130, 0, 61], [9, 5, 33]), ([1, 300], [17, 1]), ([127, 128, 129], [1, 1, 1]), ([500], [70])], ids=str)
def test_trees(shape, kind, base, q_lens):
    heads, kv_heads, D, Dv, bs = shape
    c = Step(base, q_lens, heads=heads, kv_heads=kv_heads, D=D, Dv=Dv, bs=bs, kind=kind, seed=len(base) + D, ragged=len(base) == 2)
    sees, _ = _visible(_trees(q_lens, 5), c.max_q)
    for splits in (None, 1, 3):
        c.check(_run(c, _pack(sees), D ** -0.5, num_splits=splits), sees, D ** -0.5)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("softcap,scale", [(0.0, 0.3), (30.0, 0.2), (5.0, 1.0)])
def test_softcaps_and_scales(kind, softcap, scale):
    c = Step([200, 13], [20, 6], kind=kind, seed=8)
    sees, _ = _visible(_trees(c.q_lens, 9), c.max_q)
    c.check(_run(c, _pack(sees), scale, softcap=softcap, num_splits=2), sees, scale, softcap)


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_that_are_not_positive(scale):
    c = Step([40], [6], seed=8)
    sees, _ = _visible(_trees(c.q_lens, 9), c.max_q)
    c.check(_run(c, _pack(sees), scale), sees, scale)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("base", [[0, 0], [3, 0], [250, 16]])
def test_any_mask_and_rows_that_see_nothing(kind, base):
    """Bits in any order, tokens that do not see themselves, rows without a bit: with nothing in front of them they get zeros."""
    c = Step(base, [45, 70], kind=kind, seed=11)
    sees = torch.rand(c.T, c.max_q, generator=torch.Generator().manual_seed(2)) < 0.3
    sees[::3] = False
    c.check(_run(c, _pack(sees), 0.1), sees, 0.1)
    c.check(_run(c, _pack(sees), 0.1, num_splits=4), sees, 0.1)


def test_mask_rows_that_are_short_or_strided():
    """Tokens that a row has no word for are not seen; a mask may be columns of a wider one."""
    c = Step([20], [50], seed=12)
    sees = torch.rand(50, 50, generator=torch.Generator().manual_seed(3)) < 0.5
    wide = torch.full((50, 5), -1, dtype=torch.int32, device=CUDA)
    wide[:, :2] = _pack(sees)
    c.check(_run(c, wide[:, :2], 0.1), sees, 0.1)
    sees[:, 32:] = False
    c.check(_run(c, wide[:, :1], 0.1), sees, 0.1)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("splits", [1, 3])
def test_numbers_that_a_token_does_not_see_do_not_reach_it(kind, what, value, splits):
    c = Step([100, 5], [12, 20], kind=kind, seed=13)
    sees, _ = _visible(_trees(c.q_lens, 4), c.max_q)
    for b, j in ((0, 7), (1, 11), (1, 19)):
        at, off = c.place(b, c.base[b] + j)
        getattr(c, what)[at, :, off] = value
    out = _run(c, _pack(sees), 0.1, num_splits=splits).view(c.T, -1)
    hit = torch.zeros(c.T, dtype=torch.bool)
    hit[:12], hit[12:] = sees[:12, 7], sees[12:, 11] | sees[12:, 19]
    assert 0 < hit.sum() < c.T
    assert torch.isfinite(out[(~hit).to(CUDA)]).all()
    if what == "v":         # and those that see it have what it is
        bad = out[hit.to(CUDA)]
        assert (bad.isnan() if math.isnan(value) else bad == value).all()
    keep = c.k.clone(), c.v.clone()
    for b, j in ((0, 7), (1, 11), (1, 19)):
        at, off = c.place(b, c.base[b] + j)
        getattr(c, what)[at, :, off] = 0.0
    clean = _run(c, _pack(sees), 0.1, num_splits=splits).view(c.T, -1)
    assert torch.equal(out[(~hit).to(CUDA)], clean[(~hit).to(CUDA)])
    c.k, c.v = keep


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_pages_that_are_not_there(kind):
    c = Step([100, 40], [9, 9], kind=kind, seed=14, ragged=False)
    sees, _ = _visible(_trees(c.q_lens, 4), c.max_q)
    want = Step([100, 40], [9, 9], kind=kind, seed=14, ragged=False)
    for b, page, number in ((0, 1, -1), (0, 3, c.blocks), (1, 2, 2 ** 31 - 1)):
        c.table[b, page] = number
    out = _run(c, _pack(sees), 0.1)
    for b in range(2):      # what is left of a sequence, row by row
        gone = {0: (1, 3), 1: (2,)}[b]
        for i in range(9):
            keys = [j for j in list(range(c.base[b])) + [c.base[b] + int(x) for x in sees[b * 9 + i].nonzero()[:, 0]] if j // 16 not in gone]
            at = torch.tensor(keys, device=CUDA)
            for h in range(2):
                q = want.q[b * 9 + i, h * 4:h * 4 + 4].double()
                k, v = (x[want.table[b].long()[at // 16], h, at % 16].double() for x in (want.k, want.v))
                o = torch.softmax(q @ k.T * 0.1, -1) @ v
                got = out[b * 9 + i].view(8, -1)[h * 4:h * 4 + 4].double()
                # bf16: weights and result each rounded by half a step, values up to 5
                assert (got - o).abs().max() <= (2.0 ** -8 * 2 * 5 if kind == torch.bfloat16 else 1e-5)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_lengths_behind_the_table_and_below_the_new_tokens(kind):
    """A length behind the table is the table's end; tokens that a short cache has no room for lie in front of it, and none of their keys is there."""
    c = Step([24], [8], kind=kind, seed=15, tight=True, bs=16)
    sees, _ = _visible(_trees([8], 6), 8)
    whole = _run(c, _pack(sees), 0.1)
    c.kv_lens += 1000
    assert torch.equal(_run(c, _pack(sees), 0.1), whole)
    c.kv_lens.fill_(5)          # keys 0 to 4 are tokens 3 to 7
    out = _run(c, _pack(sees), 0.1)
    short = Step([24], [8], kind=kind, seed=15, tight=True, bs=16)
    at = torch.arange(5, device=CUDA)
    for i in range(8):
        use = at[sees[i, 3:].to(CUDA)]
        for h in range(2):
            got = out[i].view(8, -1)[h * 4:h * 4 + 4].double()
            if use.numel() == 0:
                assert (got == 0).all()
                continue
            k, v = (x[short.table[0].long()[use // 16], h, use % 16].double() for x in (short.k, short.v))
            o = torch.softmax(short.q[i, h * 4:h * 4 + 4].double() @ k.T * 0.1, -1) @ v
            assert (got - o).abs().max() <= (2.0 ** -8 * 2 * 5 if kind == torch.bfloat16 else 1e-5)
    c.kv_lens.fill_(-3)
    assert (_run(c, _pack(sees), 0.1) == 0).all()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("splits", [1, 2])
def test_rows_of_no_sequence_stay(kind, splits):
    c = Step([70, 9, 30], [4, 0, 11], kind=kind, seed=16, front=3, behind=5)
    sees, _ = _visible(_trees(c.q_lens, 6), c.max_q)
    mask = torch.full((c.T + 8, 1), -1, dtype=torch.int32, device=CUDA)
    mask[3:-5] = _pack(sees)
    room = torch.full((c.T + 8, 8 * 128 + 24), 7.0, device=CUDA, dtype=kind)
    out = _run(c, mask, 0.1, num_splits=splits, out=room[:, :8 * 128])
    assert (room[:3] == 7).all() and (room[-5:] == 7).all() and (room[:, 8 * 128:] == 7).all()
    c.check(out, sees, 0.1)
    # tokens behind max_q_len are left too
    c.max_q = 6
    room.fill_(7.0)
    _run(c, mask, 0.1, num_splits=splits, out=room[:, :8 * 128])
    assert (room[3 + 4 + 6:] == 7).all() and (room[3:3 + 4 + 6, :8 * 128] != 7).any(1).all()


def test_a_long_cache():
    c = Step([20011, 3], [19, 2], heads=4, kv_heads=1, seed=17)
    sees, _ = _visible(_trees(c.q_lens, 6), c.max_q)
    c.check(_run(c, _pack(sees), 0.09), sees, 0.09)


def test_nothing_to_do():
    c = Step([5], [3], seed=1)
    q = c.q[:0]
    out = _ops().tree_attention(q, c.k, c.v, c.table[:0], c.kv_lens[:0], torch.zeros(0, 1, dtype=torch.int32, device=CUDA), cu_q=None, max_q_len=1, scale=1.0)
    assert out.shape == (0, 8 * 128)


# ---- acceptance -----------------------------------------------------------------------------------------------------------------------------------------
def _walk(tree, tokens, picks):
    path = [0] if tree else []
    while path:
        nxt = [i for i in range(len(tree)) if i > path[-1] and tree[i] == path[-1] and tokens[i] == picks[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])
    return path


@pytest.mark.parametrize("q_lens,base", [([1], [0]), ([25], [77]), ([9, 33, 0, 1, 64], [15, 0, 4, 31, 100]), ([130], [6]), ([16] * 7, list(range(7)))], ids=str)
@pytest.mark.parametrize("shape", ["bushy", "chain"])
@pytest.mark.parametrize("layout", ["pool", "layers", "odd"])
def test_accepted_paths(q_lens, base, shape, layout):
    g, cpu = _gen(21), torch.Generator().manual_seed(sum(q_lens) + len(layout))
    trees = _trees(q_lens, 22, shape)
    B, bs, T = len(q_lens), {"pool": 16, "layers": 8, "odd": 5}[layout], sum(q_lens)
    per = -(-max(a + b for a, b in zip(q_lens, base)) // bs) + 1
    blocks = B * per + 2
    table = torch.randperm(blocks, device=CUDA, generator=g)[:B * per].to(torch.int32).view(B, per)
    tokens = torch.randint(0, 6, (T,), generator=cpu)               # siblings share tokens: the first one counts
    picks = torch.randint(0, 6, (T,), generator=cpu)
    flat, at = tokens.tolist(), 0
    for tree in trees:
        for i in range(len(tree) - 1, 0, -1):
            if float(torch.rand(1, generator=cpu)) < 0.8:
                picks[at + tree[i]] = flat[at + i]
        at += len(tree)
    if layout == "pool":
        pages = torch.randn(3, 2, blocks, 2, bs, 24, device=CUDA, generator=g).bfloat16()
        tensors = [pages[i, j] for i in range(3) for j in range(2)]
    elif layout == "layers":        # what layered pools hold: keys and values of their own widths, latent rows, token ids
        pages = [torch.randn(blocks, 3, bs, 40, device=CUDA, generator=g).bfloat16(), torch.randn(blocks, 1, bs, 8, device=CUDA, generator=g),
                 torch.randn(blocks, bs, 72, device=CUDA, generator=g).bfloat16(), torch.randint(0, 1000, (blocks, bs), device=CUDA, generator=g, dtype=torch.int32)]
        tensors = pages
    else:                           # rows of odd sizes, more tensors than one launch takes
        pages = [torch.randint(0, 255, (blocks, 1, bs, 3), device=CUDA, generator=g, dtype=torch.uint8) for _ in range(100)]
        tensors = pages
    want = [t.clone() for t in tensors]
    lens = torch.tensor([a + b for a, b in zip(q_lens, base)], dtype=torch.int32, device=CUDA)
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32, device=CUDA)
    got = _ops().accept_tree(picks.to(CUDA), tokens.to(CUDA), torch.tensor(sum(trees, []), dtype=torch.int32, device=CUDA), pages, table, lens, cu_q=cu, max_q_len=max(q_lens))
    at = 0
    for b, tree in enumerate(trees):
        n = len(tree)
        path = _walk(tree, tokens[at:at + n].tolist(), picks[at:at + n].tolist())
        assert got.path[b].tolist() == path + [-1] * (max(q_lens) - len(path))
        assert int(got.counts[b]) == len(path) and int(got.kv_lens[b]) == base[b] + len(path)
        assert int(got.next_tokens[b]) == (int(picks[at + path[-1]]) if path else -1)
        for t, x in zip(tensors, want):
            rows = t.dim() - 2 if t.dim() == 4 else 1
            for d, i in enumerate(path):
                (to, o), (fro, f) = ((int(table[b, (base[b] + j) // bs]), (base[b] + j) % bs) for j in (d, i))
                if rows == 2:
                    x[to, :, o] = x[fro, :, f].clone()
                else:
                    x[to, o] = x[fro, f].clone()
        at += n
    for t, x in zip(tensors, want):
        assert torch.equal(t, x)


def test_accepting_moves_no_page_that_is_not_there_and_nothing_without_pages():
    tokens = torch.arange(5, device=CUDA)
    picks = torch.tensor([2, 9, 3, 4, 7], device=CUDA)               # 0 -> 2 -> 3 -> 4
    parents = torch.tensor([-1, 0, 0, 2, 3], dtype=torch.int32, device=CUDA)
    pool = torch.arange(1 * 2 * 3 * 1 * 4 * 8, device=CUDA, dtype=torch.float32).view(1, 2, 3, 1, 4, 8)
    table = torch.tensor([[2, 9]], dtype=torch.int32, device=CUDA)
    lens = torch.tensor([8], dtype=torch.int32, device=CUDA)          # tokens at 3 to 7: page 1 is not there
    before = pool.clone()
    got = _ops().accept_tree(picks, tokens, parents, pool, table, lens, cu_q=None, max_q_len=5)
    assert got.path.tolist() == [[0, 2, 3, 4, -1]] and got.next_tokens.tolist() == [7] and got.kv_lens.tolist() == [7] and torch.equal(pool, before)
    again = _ops().accept_tree(picks, tokens, parents, [], table, lens, cu_q=None, max_q_len=5)
    assert torch.equal(again.path, got.path)


# ---- copies of pages --------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("on_device", [False, True])
@pytest.mark.parametrize("n,blocks", [(1, 2), (7, 40), (300, 900), (600, 1900)])
def test_copies(on_device, n, blocks):
    g = _gen(31)
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(n)).tolist()
    dst, src = order[:n], [order[n + i * 2 // 3 % (blocks - n)] for i in range(n)]
    pool = torch.randn(2, 2, blocks, 2, 4, 24, device=CUDA, generator=g).bfloat16()
    many = [torch.randint(0, 255, (blocks, *s), device=CUDA, generator=g).to(t) for s, t in
            (((3, 5), torch.uint8), ((16,), torch.int32), ((2, 16, 64), torch.bfloat16), ((7,), torch.int16), ((4, 16, 129), torch.float32))] * 1
    many += [torch.randn(blocks, 6, device=CUDA, generator=g) for _ in range(95)]
    for pages in (pool, many):
        tensors = [pages.flatten(0, 1)[i] for i in range(4)] if pages is pool else pages
        want = [t.clone() for t in tensors]
        for t in want:
            t[dst] = t[src]
        a, b = src, dst
        if on_device:       # and pairs that are none
            a, b = (torch.tensor(x, dtype=torch.int32, device=CUDA) for x in (src + [-1, 0, blocks, 1], dst + [0, -1, 1, 2 ** 31 - 1]))
        _ops().copy_pages(pages, a, b)
        for t, x in zip(tensors, want):
            assert torch.equal(t, x)


def test_copies_of_nothing():
    pool = torch.randn(1, 2, 4, 1, 4, 8, device=CUDA)
    before = pool.clone()
    _ops().copy_pages(pool, [], [])
    _ops().copy_pages([], [], [])
    assert torch.equal(pool, before)


# ---- beams --------------------------------------------------------------------------------------------------------------------------------------------------
def _best(logits, scores, count):
    """In 64 bits, sequence by sequence: (score, beam, token), best first."""
    B, K = scores.shape
    x = logits.double().view(B, K, -1).cpu()
    out = []
    for b in range(B):
        rows = []
        for k in range(K):
            s, row = float(scores[b, k]), x[b, k]
            if not math.isfinite(s) or not (row < math.inf).all() or not (row > -math.inf).any():
                rows.append(torch.full_like(row, -math.inf))
            else:
                rows.append(s + (row - torch.logsumexp(row, 0)))
        flat = torch.cat(rows)
        order = torch.sort(flat, descending=True, stable=True).indices[:count].tolist()
        out.append([(float(flat[i]), i // x.shape[2], i % x.shape[2]) for i in order if flat[i] > -math.inf])
    return out


def _check_beams(logits, scores, count):
    got = _ops().beam_select(logits, scores, count=count)
    for b, want in enumerate(_best(logits, scores, count)):
        want = want + [(-math.inf, -1, -1)] * (count - len(want))
        assert got.beams[b].tolist() == [w[1] for w in want], b
        assert got.tokens[b].tolist() == [w[2] for w in want], b
        for a, w in zip(got.scores[b].tolist(), want):
            # rounded once to 32 bits; each exponential within 2^-29 of its value, and so the logarithm of their sum
            assert a == w[0] or abs(a - w[0]) <= 2.0 ** -24 * abs(w[0]) + 2.0 ** -29, (a, w)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,K,V,count", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 4, 1000, 8), (3, 3, 8192, 6), (1, 4, 8193, 128), (2, 5, 50257, 10), (1, 50, 9001, 100), (4, 2, 128256, 4), (1, 256, 70, 128)])
def test_beams(kind, B, K, V, count):
    g = _gen(V + K)
    logits = (torch.randn(B * K, V, device=CUDA, generator=g) * 3).to(kind)
    scores = -10 * torch.rand(B, K, device=CUDA, generator=g)
    _check_beams(logits, scores, count)
    wide = torch.full((B * K, V + 3), 99.0, device=CUDA, dtype=kind)       # rows that start anywhere
    wide[:, 1:V + 1] = logits
    _check_beams(wide[:, 1:V + 1], scores, count)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_beams_that_are_alike_and_ties(kind):
    """All logits alike, whole numbers, two alike beams: the order is that of beam and token."""
    for V in (40, 9000, 30000):
        scores = torch.tensor([[-1.0, -1.0, -1.0]], device=CUDA)
        _check_beams(torch.zeros(3, V, device=CUDA, dtype=kind), scores, 20)
        x = torch.randint(-3, 3, (3, V), device=CUDA, generator=_gen(V)).to(kind)
        x[2] = x[0]
        _check_beams(x, scores, 100)
        few = torch.full((3, V), -7.0, device=CUDA, dtype=kind)
        few[:, 11::V // 4] = 2.0
        _check_beams(few, scores, 64)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_tokens_that_are_not_allowed_and_beams_that_are_not_alive(kind):
    g = _gen(41)
    logits = (torch.randn(8, 20000, device=CUDA, generator=g) * 3).to(kind)
    scores = -10 * torch.rand(2, 4, device=CUDA, generator=g)
    scores[0, 1], scores[0, 3], scores[1, 0], scores[1, 1] = -math.inf, math.nan, math.inf, -0.0
    logits[0, 7:19990] = -math.inf          # most are not allowed, whole pieces of the row among them
    logits[2] = -math.inf                   # none
    logits[6, 15000] = math.nan             # not a distribution
    logits[7, 3] = math.inf
    logits[1] = math.nan                    # of a beam that is not alive
    _check_beams(logits, scores, 16)
    _check_beams(logits, scores, 128)       # the first prompt has 17 left
    _check_beams(logits, torch.full((2, 4), -math.inf, device=CUDA), 3)


def test_scores_near_each_other_are_told_apart():
    """Two beams whose best scores differ by less than 32-bit numbers of their size can say."""
    V = 5000
    row = torch.randn(V, device=CUDA, generator=_gen(5))
    logits = torch.stack([row, row])
    logits[1, 77] -= 3e-5                   # the second beam's sum is smaller by less than 1e-8 of it: all its other tokens are better
    _check_beams(logits, torch.full((1, 2), -30.0, device=CUDA), 40)


# ---- captured, and on other streams ---------------------------------------------------------------------------------------------------------------------------
def test_captured_steps_of_two_graphs():
    """A step of each operator, captured twice: the replays give what eager calls give on the inputs of the moment."""
    ops = _ops()
    c = Step([90, 33], [7, 12], seed=51)
    trees = _trees(c.q_lens, 52)
    parents = torch.tensor(sum(trees, []), dtype=torch.int32, device=CUDA)
    tokens, picks = torch.arange(c.T, device=CUDA), torch.randint(0, c.T, (c.T,), device=CUDA, generator=_gen(1))
    logits, scores = torch.randn(6, 30001, device=CUDA, generator=_gen(2)), -torch.rand(2, 3, device=CUDA, generator=_gen(3))
    src, dst = (torch.tensor(x, dtype=torch.int32, device=CUDA) for x in ([0, 1], [2, 3]))

    def step(pool):
        plan = ops.plan_tree(parents, **c.step)
        out = ops.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, plan.mask, scale=0.1, num_splits=3, **c.step)
        got = ops.accept_tree(picks, tokens, parents, pool, c.table, c.kv_lens, **c.step)
        ops.copy_pages(pool, src, dst)
        best = ops.beam_select(logits, scores, count=6)
        return plan.mask, plan.depths, out, got.path, got.counts, got.next_tokens, got.kv_lens, best.scores, best.beams, best.tokens

    blank = torch.randn(2, 2, c.blocks, 2, 16, 64, device=CUDA, generator=_gen(4))
    pools = [blank.clone(), blank.clone()]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            step(blank.clone())
    torch.cuda.synchronize()
    graphs, outs = [], []
    for pool in pools:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(pool))
        graphs.append(graph)
    for again in range(2):
        picks.copy_(torch.randint(0, c.T, (c.T,), device=CUDA, generator=_gen(60 + again)))
        logits.mul_(-1)
        eager = blank.clone()
        for p in pools:
            p.copy_(blank)
        for graph in graphs:
            graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        for pool, out in zip(pools, outs):
            assert torch.equal(pool, eager)
            for x, y in zip(out, want):
                assert torch.equal(x, y)


def test_results_repeat():
    c = Step([3000], [40], heads=8, kv_heads=2, seed=61)
    sees, _ = _visible(_trees(c.q_lens, 62), c.max_q)
    first = _run(c, _pack(sees), 0.1)
    for _ in range(5):
        assert torch.equal(_run(c, _pack(sees), 0.1), first)
    logits, scores = torch.randn(12, 60000, device=CUDA, generator=_gen(1)), torch.zeros(3, 4, device=CUDA)
    best = _ops().beam_select(logits, scores, count=30)
    for _ in range(5):
        again = _ops().beam_select(logits, scores, count=30)
        assert torch.equal(again.scores, best.scores) and torch.equal(again.tokens, best.tokens)


@pytest.mark.parametrize("n", [257, 700])
def test_long_paths_shift_in_place(n):
    """Every entry of the path moves one place to the front, onto what has been read before."""
    cu = torch.tensor([0, n], dtype=torch.int32, device=CUDA)
    parents = torch.tensor([-1, 0, 0] + list(range(2, n - 1)), dtype=torch.int32, device=CUDA)
    tokens = torch.arange(n, device=CUDA)
    picks = torch.tensor([2, -7] + list(range(3, n + 1)), device=CUDA)
    base, bs = 13, 16
    per = -(-(base + n) // bs)
    table = torch.randperm(per + 3, generator=torch.Generator().manual_seed(n))[:per].to(torch.int32)[None].to(CUDA)
    pool = torch.randn(60, 2, per + 3, 2, bs, 8, device=CUDA, generator=_gen(n))          # more tensors than a launch takes
    before = pool.clone()
    got = _ops().accept_tree(picks, tokens, parents, pool, table, torch.tensor([base + n], dtype=torch.int32, device=CUDA), cu_q=cu, max_q_len=n)
    path = [0] + list(range(2, n))
    assert got.path[0].tolist() == path + [-1] and int(got.next_tokens[0]) == n and int(got.kv_lens[0]) == base + n - 1
    where = lambda j: (table[0, torch.tensor(j, device=CUDA) // bs].long(), torch.tensor(j, device=CUDA) % bs)
    to, fro = where([base + d for d in range(n - 1)]), where([base + i for i in path])
    want = before.clone()
    want[:, :, to[0], :, to[1]] = before[:, :, fro[0], :, fro[1]]
    assert torch.equal(pool, want)


def test_copies_in_pools_of_many_layers():
    pool = torch.randn(60, 2, 9, 3, 4, 5, device=CUDA, generator=_gen(5))
    want = pool.clone()
    want[:, :, [7, 2]] = pool[:, :, [1, 1]]
    _ops().copy_pages(pool, [1, 1], [7, 2])
    assert torch.equal(pool, want)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_zeros_of_both_signs_are_equal(kind):
    """More ties at zero than a block takes notes of: the first tokens, whatever their signs."""
    V, count = 9001, 11
    logits = torch.zeros(2, V, dtype=kind, device=CUDA)
    logits[torch.rand(2, V, device=CUDA, generator=_gen(3)) < 0.5] = -0.0
    got = _ops().beam_select(logits, torch.zeros(1, 2, device=CUDA), count=count)
    assert got.beams[0].tolist() == [0] * count and got.tokens[0].tolist() == list(range(count))
