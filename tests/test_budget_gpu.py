"""Operators of long caches on a budget against plain restatements in 64 bits."""
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


class Cache:
    """Pages in random order, every place that no token of a sequence holds filled with `filler`, and the step's shape."""

    def __init__(self, lens, q_lens, *, heads=8, kv_heads=2, D=128, Dv=None, bs=16, kind=torch.bfloat16, seed=0, filler=float("nan"), extra_pages=2, ragged=False,
                 behind=0):
        g = _gen(seed)
        Dv = D if Dv is None else Dv
        self.lens, self.q_lens, self.bs, self.kind = list(lens), list(q_lens), bs, kind
        B, self.per = len(self.lens), max(1, -(-max(max(self.lens), 1) // bs)) + extra_pages
        self.blocks = B * self.per + 3
        self.k = torch.randn(self.blocks, kv_heads, bs, D, device=CUDA, generator=g).to(kind)
        self.v = torch.randn(self.blocks, kv_heads, bs, Dv, device=CUDA, generator=g).to(kind)
        self.table = torch.randperm(self.blocks, device=CUDA, generator=g)[:B * self.per].to(torch.int32).view(B, self.per)
        used = torch.zeros(self.blocks, bs, dtype=torch.bool, device=CUDA)
        for b, n in enumerate(self.lens):
            at = torch.arange(n, device=CUDA)
            used[self.table[b].long()[at // bs], at % bs] = True
        for t in (self.k, self.v):
            t.masked_fill_(~used[:, None, :, None], filler)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device=CUDA)
        self.T = sum(self.q_lens)
        wide = torch.randn(self.T + behind, heads + 1, D + 8, device=CUDA, generator=g).to(kind)
        self.q = wide[:, :heads, :D]                 # strided tokens and heads
        self.heads, self.kv_heads, self.G = heads, kv_heads, heads // kv_heads
        uniform = len(set(self.q_lens)) == 1 and not ragged and not behind
        self.cu = None if uniform else torch.tensor([0] + list(torch.tensor(self.q_lens).cumsum(0)), dtype=torch.int32, device=CUDA)
        self.max_q = max(self.q_lens)

    @property
    def step(self):
        return {"cu_q": self.cu, "max_q_len": self.max_q}

    def tokens(self):
        """(token, sequence, keys it sees) of every new token."""
        t = 0
        for b, (n, m) in enumerate(zip(self.lens, self.q_lens)):
            for i in range(m):
                yield t, b, max(0, n - (m - 1 - i))
                t += 1

    def row(self, name, b, key):
        """Rows of the keys `key` of sequence b in 64 bits [kv heads, keys, width]."""
        t = getattr(self, name)
        key = torch.as_tensor(key, device=CUDA, dtype=torch.long)
        return t[self.table[b].long()[key // self.bs], :, key % self.bs].transpose(0, 1).double()


def _attend(c, t, b, h, keys, scale, softcap):
    """Weights [G, keys], output [G, Dv], and what bounds their error: the largest sum |q k| and sum p |v|."""
    q = c.q[t, h * c.G:(h + 1) * c.G].double()
    k, v = c.row("k", b, keys)[h], c.row("v", b, keys)[h]
    s = q @ k.T * scale
    size = (q.abs() @ k.abs().T * abs(scale)).max()
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    p = torch.softmax(s, -1)
    return p, p @ v, size, p @ v.abs()


def _bounds(c, size, n, splits, softcap):
    """Relative error of a weight: a product of D terms in 32 bits is off by at most (D + 4) 2^-24 of the sum of the terms' sizes (4 more roundings: scale, cap, change of
    base), a capped score by 2^-19 of the cap more (tanhf, a division, a product), the exponential and its sum by 2^-20 + n 2^-24, and a score's
    error counts twice, in the numerator and in the sum."""
    ds = (c.q.shape[2] + 4) * 2.0 ** -24 * float(size) + softcap * 2.0 ** -19
    return math.expm1(2 * ds) + 2.0 ** -19 + (n + splits + 8) * 2.0 ** -23


def _check_attention(c, out, lists, scale, softcap=0.0, splits=64, weights=None, before=None):
    """lists[t][h]: the keys that token t sees in head h, in any order. out [T, Hq * Dv]."""
    Dv = c.v.shape[3]
    want_w = None if weights is None else before.double()
    tol_w = None if weights is None else torch.full_like(want_w, 2.0 ** -24) * want_w.abs() + 1e-12
    for t, b, seen in c.tokens():
        for h in range(c.kv_heads):
            keys = lists(t, b, h, seen)
            got = out[t].view(c.heads, Dv)[h * c.G:(h + 1) * c.G].double()
            if len(keys) == 0:
                assert (got == 0).all(), (t, h)
                continue
            p, o, size, pv = _attend(c, t, b, h, keys, scale, softcap)
            rel = _bounds(c, size, len(keys), splits, softcap)
            tol = rel * pv + 1e-30
            if c.kind == torch.bfloat16:             # the weights of a product and the result are rounded to bf16: half a step each
                tol = tol + 2.0 ** -8 * pv * (1 + rel) + 2.0 ** -8 * o.abs() + 1e-30
            assert ((got - o).abs() <= tol).all(), (t, b, h, float(((got - o).abs() / tol).max()))
            if weights is not None:
                at = torch.as_tensor(keys, device=CUDA, dtype=torch.long)
                want_w[b, h, at] += p.sum(0)
                tol_w[b, h, at] += rel * p.sum(0) + 2.0 ** -22 * want_w[b, h, at]
    if weights is not None:
        assert ((weights.double() - want_w).abs() <= tol_w).all(), float(((weights.double() - want_w).abs() - tol_w).max())


SHAPES = [
    # heads, kv heads, width, value width, page
    (8, 2, 128, 128, 16),
    (4, 4, 64, 64, 16),
    (12, 1, 96, 64, 32),
    (40, 1, 128, 128, 16),
    (6, 2, 40, 24, 16),
    (3, 1, 17, 33, 5),
    (4, 2, 192, 256, 48),
    (28, 4, 128, 120, 64),
]
STEPS = [
    # cached tokens with the new ones, new tokens
    ([1], [1]),
    ([0, 1, 15, 16, 17, 64, 65], [1] * 7),
    ([300, 33, 700], [1, 1, 1]),
    ([130, 9, 64], [5, 5, 5]),
    ([200, 20, 3, 90], [7, 0, 2, 16]),
    ([2], [4]),                 # more new tokens than cached ones: the first see nothing
]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_tracked_attention(shape, step, kind):
    ops = _ops()
    heads, kv, D, Dv, bs = shape
    c = Cache(*STEPS[step], heads=heads, kv_heads=kv, D=D, Dv=Dv, bs=bs, kind=kind, seed=step)
    room = torch.rand(len(c.lens), kv, c.per * bs + 5, device=CUDA, generator=_gen(9))
    for splits in (None, 1, 3):
        weights = room.clone()
        out = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=D ** -0.5, num_splits=splits, **c.step)
        _check_attention(c, out, lambda t, b, h, seen: range(seen), D ** -0.5, weights=weights, before=room)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_selected_attention(shape, step, kind):
    ops = _ops()
    heads, kv, D, Dv, bs = shape
    c = Cache(*STEPS[step], heads=heads, kv_heads=kv, D=D, Dv=Dv, bs=bs, kind=kind, seed=step + 50)
    N = 7
    g = _gen(step)
    # in any order, with pages that are not there or not seen
    pages = torch.randint(-2, c.per + 3, (c.T, kv, 64), device=CUDA, generator=g)
    pages = torch.stack([torch.stack([_distinct(r, N) for r in rows]) for rows in pages.cpu()]).to(CUDA, torch.int32)
    counts = torch.randint(0, N + 1, (c.T, kv), device=CUDA, generator=g).to(torch.int32)
    host, many = pages.cpu(), counts.cpu()

    def keys(t, b, h, seen):
        return [p * bs + i for p in host[t, h, :many[t, h]].tolist() if p >= 0 for i in range(bs) if p * bs + i < seen]

    for splits in (None, 1, 3):
        out = ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, ops.PageSelection(pages, counts), scale=D ** -0.5, num_splits=splits, **c.step)
        _check_attention(c, out, keys, D ** -0.5)


def _distinct(row, n):
    return torch.tensor(list(dict.fromkeys(row.tolist()))[:n] + [-1] * n)[:n]


def test_a_page_listed_twice_counts_twice():
    ops = _ops()
    c = Cache([64], [1], heads=4, kv_heads=1)
    pages = torch.tensor([[[2, 0, 2]]], dtype=torch.int32, device=CUDA)
    counts = torch.tensor([[3]], dtype=torch.int32, device=CUDA)
    out = ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, ops.PageSelection(pages, counts), scale=0.1, **c.step)
    _check_attention(c, out, lambda t, b, h, seen: [*range(32, 48), *range(16), *range(32, 48)], 0.1)


@pytest.mark.parametrize("softcap,scale", [(5.0, 0.3), (50.0, 0.0884), (0.0, -0.05), (0.0, 2.0)])
def test_caps_and_scales(softcap, scale):
    ops = _ops()
    c = Cache([100, 300], [1, 1])
    weights = torch.zeros(2, 2, c.per * 16, device=CUDA)
    out = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=scale, softcap=softcap, **c.step)
    _check_attention(c, out, lambda t, b, h, seen: range(seen), scale, softcap, weights=weights, before=torch.zeros_like(weights))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_pages_that_are_not_there_add_nothing(kind):
    ops = _ops()
    c = Cache([100], [1], kind=kind)
    whole = c.table.clone()
    c.table[0, 2], c.table[0, 4] = -5, c.blocks + 1000
    weights = torch.zeros(1, 2, c.per * 16, device=CUDA)
    out = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, **c.step)
    pages = torch.arange(7, dtype=torch.int32, device=CUDA).expand(1, 2, 7).contiguous()
    sel = ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, ops.PageSelection(pages, torch.full((1, 2), 7, dtype=torch.int32, device=CUDA)), scale=0.1, **c.step)
    c.table = whole
    left = [j for j in range(100) if j // 16 not in (2, 4)]
    _check_attention(c, out, lambda t, b, h, seen: left, 0.1, weights=weights, before=torch.zeros_like(weights))
    _check_attention(c, sel, lambda t, b, h, seen: left, 0.1)


def test_rows_behind_the_last_sequence_stay():
    ops = _ops()
    c = Cache([40, 70], [2, 3], behind=4)
    out = torch.full((c.T + 4, c.heads * 128), 7.0, dtype=torch.bfloat16, device=CUDA)
    weights = torch.zeros(2, 2, c.per * 16, device=CUDA)
    ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, out=out, **c.step)
    assert (out[c.T:] == 7).all()
    _check_attention(c, out, lambda t, b, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))
    pages = torch.arange(3, dtype=torch.int32, device=CUDA).expand(c.T + 4, 2, 3).contiguous()
    out.fill_(7)
    ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, ops.PageSelection(pages, torch.full((c.T + 4, 2), 3, dtype=torch.int32, device=CUDA)), scale=0.1, out=out,
                           **c.step)
    assert (out[c.T:] == 7).all()
    _check_attention(c, out, lambda t, b, h, seen: range(min(seen, 48)), 0.1)


def test_numbers_that_are_not_finite_reach_their_own_rows_only():
    ops = _ops()
    c = Cache([50, 50], [4, 4], heads=4, kv_heads=2)
    at = c.table[0, 48 // 16].long()
    c.v[at, 1, 48 % 16] = float("nan")               # key 48 of sequence 0, head 1: its tokens 2 and 3 (49 and 50 keys) see it
    weights = torch.zeros(2, 2, c.per * 16, device=CUDA)
    out = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, **c.step).view(8, 2, 2, 128)
    bad = torch.zeros(8, 2, 2, 128, dtype=torch.bool, device=CUDA)
    bad[2:4, 1] = True
    assert torch.equal(out.isnan(), bad) and weights.isfinite().all()
    c.k[at, 1, 48 % 16] = float("nan")
    weights.zero_()
    out = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, **c.step).view(8, 2, 2, 128)
    assert torch.equal(out.isnan(), bad)
    assert weights[0, 1, :50].isnan().all() and not weights[0, 0].isnan().any() and not weights[1].isnan().any()


# ---- summaries and selection --------------------------------------------------------------------------------------------------------------------------
def _summary(keys):
    """keys [bs, D] of one page and head -> codes, scale."""
    s = keys.double().sum(0)
    a = s.abs().max()
    if not torch.isfinite(s).all():
        return torch.zeros(len(s), dtype=torch.int8), float("nan")
    if a == 0:
        return torch.zeros(len(s), dtype=torch.int8), 0.0
    return torch.round(127.0 * s / a).to(torch.int8), float((a / (127.0 * len(keys))).float())


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,D,bs", [(2, 128, 16), (5, 64, 16), (1, 96, 32), (3, 17, 5), (2, 256, 16), (2, 136, 8), (1, 8, 128), (9, 40, 1)])
def test_page_summaries(kv, D, bs, kind):
    ops = _ops()
    lens, new = [0, 1, bs - 1, bs, bs + 1, 5 * bs, 7 * bs + 2, 3 * bs], [0, 1, bs - 1, 1, bs + 1, 3 * bs, 2, 3 * bs + 4]
    c = Cache(lens, [max(1, n) for n in new], heads=kv, kv_heads=kv, D=D, bs=bs, kind=kind, ragged=True)
    c.k[c.table[5, 3].long(), 0] = 0
    c.k[c.table[5, 4].long(), 0, 0, 0] = float("inf")
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=CUDA)
    sums = ops.PageSummaries.empty(c.k)
    sums.codes.fill_(99), sums.scales.fill_(-1)
    want_c, want_s = sums.codes.cpu().clone(), sums.scales.cpu().clone()
    for b, (n, m) in enumerate(zip(lens, new)):
        for page in range(c.per):
            if m and max(n - m, 0) < (page + 1) * bs <= n:
                at = int(c.table[b, page])
                for h in range(kv):
                    code, scale = _summary(c.k[at, h].cpu())
                    want_c[at, h], want_s[at, h] = code, scale
    ops.summarize_pages(c.k, c.table, c.kv_lens, sums, cu_q=cu, max_q_len=max(new))
    assert torch.equal(sums.values().nan_to_num(nan=-7.0), (sums.codes * sums.scales[..., None]).nan_to_num(nan=-7.0))
    assert torch.equal(sums.codes.cpu(), want_c) and torch.equal(sums.scales.cpu().nan_to_num(nan=-7.0), want_s.nan_to_num(nan=-7.0))


@pytest.mark.parametrize("D,bs", [(128, 16), (64, 32), (96, 4), (128, 80)])
def test_summaries_at_the_borders(D, bs):
    """Pages whose sums cancel, lie on halves of the step, differ by little, pass the range of 32 bits or have none."""
    ops = _ops()
    c = Cache([40 * bs], [1], heads=1, kv_heads=1, D=D, bs=bs)
    k, at = c.k, c.table[0].long()
    g = _gen(D)
    k[at[0]] *= 1e-3                                          # small numbers beside large ones that cancel
    k[at[0], 0, 0], k[at[0], 0, 1] = 300.0, -300.0
    k[at[1]] = 0
    k[at[1], 0, 0] = (torch.arange(D, device=CUDA) - D // 2).bfloat16()
    k[at[1], 0, 0, 0] = 254.0                                 # 127 x / 254: every odd number is a half
    k[at[2]] = 3e38
    k[at[2], 0, :, 1] = 1.5e38
    k[at[3]] = 0
    k[at[4]] = torch.randint(-2, 3, k[at[4]].shape, device=CUDA, generator=g).bfloat16() * 2.0 ** -130      # below the normal numbers of 32 bits
    k[at[5]] = 1.0
    k[at[5], 0, 0, 3] = 1.0 + 2.0 ** -7
    k[at[6], 0, bs - 1, D - 1] = float("nan")
    k[at[7], 0, 1, 1], k[at[7], 0, 2, 1] = float("inf"), float("-inf")
    k[at[8]] = torch.where(torch.rand(k[at[8]].shape, device=CUDA, generator=g) < 0.5, 1.0, 2.0 ** -20).bfloat16()
    sums = ops.PageSummaries.empty(k)
    ops.summarize_pages(k, c.table, c.kv_lens, sums, cu_q=None, max_q_len=40 * bs)
    for page in range(40):
        code, scale = _summary(k[at[page], 0].cpu())
        got = float(sums.scales[at[page], 0])
        assert torch.equal(sums.codes[at[page], 0].cpu(), code) and (got == scale or (math.isnan(got) and math.isnan(scale))), page


@pytest.mark.parametrize("bs", [16, 20, 3])
@pytest.mark.parametrize("low,high", [(0, 254), (0, 0), (0, 3), (250, 254), (100, 150)])
def test_summaries_of_any_finite_numbers(low, high, bs):
    """bf16 numbers of any sign and fraction whose exponents are `low` to `high`: below the normal range, near the end of it, and far apart."""
    ops = _ops()
    g = _gen(bs + low)
    bits = torch.randint(0, 2, (12, 2, bs, 64), device=CUDA, generator=g) << 15 | torch.randint(low, high + 1, (12, 2, bs, 64), device=CUDA, generator=g) << 7
    k = (bits | torch.randint(0, 128, bits.shape, device=CUDA, generator=g)).to(torch.int32).to(torch.int16).view(torch.bfloat16)
    table, lens = torch.randperm(12, device=CUDA, generator=g).to(torch.int32)[None], torch.tensor([12 * bs], dtype=torch.int32, device=CUDA)
    sums = ops.PageSummaries.empty(k)
    ops.summarize_pages(k, table, lens, sums, cu_q=None, max_q_len=12 * bs)
    for page in range(12):
        for h in range(2):
            code, scale = _summary(k[page, h].cpu())
            assert torch.equal(sums.codes[page, h].cpu(), code) and float(sums.scales[page, h]) == scale, (page, h)


def test_summaries_of_single_steps_are_those_of_the_prompt():
    ops = _ops()
    c = Cache([70], [1], kv_heads=2)
    whole, steps = ops.PageSummaries.empty(c.k), ops.PageSummaries.empty(c.k)
    ops.summarize_pages(c.k, c.table, c.kv_lens, whole, cu_q=None, max_q_len=70)
    for n in range(1, 71):
        ops.summarize_pages(c.k, c.table, torch.tensor([n], dtype=torch.int32, device=CUDA), steps, cu_q=None, max_q_len=1)
    assert torch.equal(whole.codes, steps.codes) and torch.equal(whole.scales, steps.scales) and whole.scales.count_nonzero() == 4 * 2
    mean = c.row("k", 0, range(64)).view(2, 4, 16, 128).mean(2)
    got = whole.values()[c.table[0, :4].long()].transpose(0, 1).double()
    # half a step of the codes, and the rounding of scale and product
    assert ((got - mean).abs() <= mean.abs().amax(-1, keepdim=True) * (0.5 / 127 + 2.0 ** -22)).all()


def _select(c, sums, t, b, h, seen, top, first, last):
    n, width = -(-seen // c.bs), first + top + last
    if n <= width:
        return list(range(n))
    q = c.q[t, h * c.G:(h + 1) * c.G].double().cpu()
    a = q.abs().max()
    qc = torch.round(127.0 * q / a) if torch.isfinite(q).all() and a > 0 else torch.zeros_like(q)
    rank = []
    for page in range(first, n - last):
        at = int(c.table[b, page])
        if not 0 <= at < c.blocks:
            rank.append((2, 0.0, page))
            continue
        dot = int((qc @ sums.codes[at, h].double().cpu()).max())
        score = float(torch.tensor(float(dot)) * sums.scales[at, h].cpu())
        rank.append((0, 0.0, page) if math.isnan(score) else (1, -score + 0.0, page))
    return [*range(first), *sorted(page for _, _, page in sorted(rank)[:top]), *range(n - last, n)]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,D,bs", [(8, 2, 128, 16), (4, 4, 64, 16), (12, 1, 96, 32), (40, 1, 128, 16), (6, 2, 40, 16), (3, 1, 17, 5), (16, 8, 256, 16), (16, 2, 128, 16),
                                           (6, 2, 128, 16), (5, 1, 128, 32), (4, 2, 128, 16)])
@pytest.mark.parametrize("top,first,last", [(3, 1, 2), (0, 2, 1), (20, 0, 1), (1, 0, 3)])
def test_select_pages(heads, kv, D, bs, top, first, last, kind):
    ops = _ops()
    lens, new = [1, 0, 40 * bs, 17 * bs + 3, 900, 6 * bs], [1, 2, 3, 5, 1, 2]
    c = Cache(lens, new, heads=heads, kv_heads=kv, D=D, bs=bs, kind=kind, seed=top, behind=3)
    g = _gen(top + 1)
    sums = ops.PageSummaries(torch.randint(-127, 128, c.k.shape[:2] + (D,), device=CUDA, generator=g).to(torch.int8),
                             torch.rand(c.k.shape[:2], device=CUDA, generator=g) * 0.01)
    sums.scales[c.table[2, 5].long(), 0] = float("nan")
    sums.scales[c.table[2, 20:30].long()] = 0.0              # ties
    c.q[3].zero_()
    c.q[4, 0, 0] = float("inf")
    c.q[6] *= 2.0 ** 124                                      # 127 of them pass the range of 32 bits
    c.q[7] *= 2.0 ** -128
    c.table[3, 4] = c.blocks + 7
    got = ops.select_pages(c.q, sums, c.table, c.kv_lens, block_size=bs, top=top, first=first, last=last, **c.step)
    pages, counts = got.pages.cpu(), got.counts.cpu()
    for t, b, seen in c.tokens():
        for h in range(kv):
            want = _select(c, sums, t, b, h, seen, top, first, last)
            assert pages[t, h].tolist() == want + [-1] * (first + top + last - len(want)), (t, b, h)
            assert counts[t, h] == len(want)


@pytest.mark.parametrize("G", [1, 2, 4, 7, 12])
@pytest.mark.parametrize("pages,top", [(5000, 60), (4097, 4090), (300, 299), (2049, 1)])
def test_selection_among_many_pages(pages, top, G):
    ops = _ops()
    g = _gen(pages)
    c = Cache([16], [1], heads=2 * G, kv_heads=2)
    c.lens, c.per, c.blocks = [pages * 16], pages, pages
    c.kv_lens, c.table = torch.tensor([pages * 16], dtype=torch.int32, device=CUDA), torch.randperm(pages, device=CUDA, generator=g).to(torch.int32)[None]
    # few codes: many scores are alike
    sums = ops.PageSummaries(torch.randint(-1, 2, (pages, 2, 128), device=CUDA, generator=g).to(torch.int8) * (torch.arange(128, device=CUDA) < 3).to(torch.int8),
                             torch.randint(1, 3, (pages, 2), device=CUDA, generator=g).float())
    got = ops.select_pages(c.q, sums, c.table, c.kv_lens, block_size=16, top=top, first=0, last=1, **c.step)
    q = c.q[0].double().view(2, G, 128)
    qc = torch.round(127 * q / q.abs().amax((1, 2), keepdim=True))
    score = (torch.einsum("hgd,phd->hgp", qc, sums.codes.double()).amax(1) * sums.scales.double().T)[:, c.table[0].long()]
    want = score[:, :-1].sort(dim=-1, descending=True, stable=True).indices[:, :top].sort(-1).values
    assert torch.equal(got.pages[0, :, :top].long(), want) and (got.pages[0, :, top] == pages - 1).all()


@pytest.mark.parametrize("G,tokens", [(4, 9), (8, 5), (2, 6)])
@pytest.mark.parametrize("pages,top", [(700, 63), (700, 64), (700, 65), (700, 128), (700, 129), (600, 256), (600, 257), (1300, 300)])
def test_selection_of_a_prompt_among_many_pages(pages, top, G, tokens):
    """Several tokens to a block, each chosen for by a part of its threads; many scores are alike, and the last tokens see other numbers of pages than the first."""
    ops = _ops()
    g = _gen(pages + top)
    n = pages * 16 - 13
    q = torch.randn(tokens, 2 * G, 128, device=CUDA, generator=g).bfloat16()
    lens, table = torch.tensor([n], dtype=torch.int32, device=CUDA), torch.randperm(pages, device=CUDA, generator=g).to(torch.int32)[None]
    sums = ops.PageSummaries(torch.randint(-1, 2, (pages, 2, 128), device=CUDA, generator=g).to(torch.int8) * (torch.arange(128, device=CUDA) < 3).to(torch.int8),
                             torch.randint(1, 3, (pages, 2), device=CUDA, generator=g).float())
    got = ops.select_pages(q, sums, table, lens, cu_q=None, max_q_len=tokens, block_size=16, top=top, first=1, last=2)
    grouped = q.double().view(tokens, 2, G, 128)
    qc = torch.round(127 * grouped / grouped.abs().amax((2, 3), keepdim=True))
    score = (torch.einsum("thgd,phd->thgp", qc, sums.codes.double()).amax(2) * sums.scales.double().T)[:, :, table[0].long()]
    for t in range(tokens):
        seen = -(-(n - (tokens - 1 - t)) // 16)
        best = score[t, :, 1:seen - 2].sort(dim=-1, descending=True, stable=True).indices[:, :top].sort(-1).values + 1
        ends = torch.tensor([seen - 2, seen - 1], device=CUDA).expand(2, 2)
        assert torch.equal(got.pages[t].long(), torch.cat((torch.zeros(2, 1, dtype=torch.long, device=CUDA), best, ends), 1)), t


# ---- eviction -----------------------------------------------------------------------------------------------------------------------------------------
def _evict(k, v, w, pos, n, nxt, keep, recent, first):
    """One head's rows [n, ...] as lists; the rule, entry by entry."""
    place = [p if p >= 0 else nxt - (n - i) for i, p in enumerate(pos[:n])]

    def rank(i):
        if place[i] < first or place[i] >= nxt - recent:
            return (0, 0.0, i)
        return (1, 0.0, i) if math.isnan(w[i]) else (2, -w[i] + 0.0, i)

    kept = set(sorted(range(n), key=rank)[:keep])
    holes = [i for i in range(keep) if i not in kept]
    sources = [i for i in range(keep, n) if i in kept]
    assert len(holes) == len(sources)
    k, v, w = list(k), list(v), list(w)
    for to, fro in zip(holes, sources):
        k[to], v[to], w[to], place[to] = k[fro], v[fro], w[fro], place[fro]
    return k, v, w[:keep], place[:keep]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,D,Dv,bs", [(2, 128, 128, 16), (3, 40, 24, 16), (1, 17, 33, 5), (2, 64, 256, 32)])
@pytest.mark.parametrize("keep,recent,first", [(1, 0, 0), (16, 4, 2), (33, 33, 0), (40, 0, 40), (70, 13, 5), (1000, 10, 10)])
def test_evict_tokens(kv, D, Dv, bs, keep, recent, first, kind):
    ops = _ops()
    lens = [0, 1, keep, keep + 1, keep + 2 * bs + 3, 5 * keep + 7, 90]
    c = Cache(lens, [1] * len(lens), heads=kv, kv_heads=kv, D=D, Dv=Dv, bs=bs, kind=kind, seed=keep, filler=1e9)
    B, N, g = len(lens), c.per * bs, _gen(keep)
    store = torch.rand(B, kv + 1, N + 3, device=CUDA, generator=g)
    w = store[:, :kv, :N]                                     # strided rows
    w.copy_((w * 20).round())                                 # many ties
    w[5, 0, 3], w[5, 0, 9], w[5, 0, 2] = float("nan"), float("inf"), -0.0
    pos = torch.full((B, kv, N), -1, dtype=torch.int32, device=CUDA)
    nxt = torch.tensor(lens, dtype=torch.int32, device=CUDA)
    nxt[4] += 50
    pos[4, :, :7] = torch.randperm(20, device=CUDA, generator=g)[:7].to(torch.int32)
    before = [t.clone() for t in (c.k, c.v, w, pos, store)]
    out = ops.evict_tokens(c.k, c.v, c.table, c.kv_lens, w, pos, nxt, keep=keep, recent=recent, first=first)
    assert out.tolist() == [min(n, keep) for n in lens]
    touched = torch.zeros(c.blocks, kv, bs, dtype=torch.bool, device=CUDA)
    for b, n in enumerate(lens):
        for h in range(kv):
            if n <= keep:
                assert torch.equal(w[b, h], before[2][b, h]) and torch.equal(pos[b, h], before[3][b, h])
                continue
            at = torch.arange(n, device=CUDA)
            page, off = c.table[b].long()[at // bs], at % bs
            old = [t[page, h, off].cpu() for t in before[:2]]
            k, v, ww, place = _evict(old[0], old[1], before[2][b, h].tolist(), before[3][b, h].tolist(), n, int(nxt[b]), keep, recent, first)
            assert torch.equal(c.k[page, h, off][:keep].cpu(), torch.stack(k[:keep])) and torch.equal(c.v[page, h, off][:keep].cpu(), torch.stack(v[:keep]))
            got = w[b, h, :keep].tolist()
            assert all(x == y or (math.isnan(x) and math.isnan(y)) for x, y in zip(got, ww))
            assert pos[b, h, :keep].tolist() == place
            assert (w[b, h, keep:n] == 0).all() and (pos[b, h, keep:] == -1).all() and torch.equal(w[b, h, n:], before[2][b, h, n:])
            touched[page[:keep], h, off[:keep]] = True
    for new, old in zip((c.k, c.v), before):
        assert torch.equal(new[~touched], old[~touched])       # nothing but kept entries is written
    assert torch.equal(store[:, kv:], before[4][:, kv:])


@pytest.mark.parametrize("n,keep", [(5000, 4096), (45000, 300), (41000, 40990), (3000, 2999)])
def test_evict_from_long_caches(n, keep):
    ops = _ops()
    c = Cache([n], [1], heads=1, kv_heads=1, D=8, seed=n, filler=0.0)
    w = torch.rand(1, 1, c.per * 16, device=CUDA, generator=_gen(n))
    pos = torch.full((1, 1, c.per * 16), -1, dtype=torch.int32, device=CUDA)
    old_w, rows = w.clone(), c.row("k", 0, range(n))[0]
    out = ops.evict_tokens(c.k, c.v, c.table, c.kv_lens, w, pos, c.kv_lens.clone(), keep=keep, recent=17, first=3)
    rank = old_w[0, 0, :n].clone()
    rank[:3], rank[n - 17:] = 9, 9
    stay = torch.zeros(n, dtype=torch.bool, device=CUDA)
    stay[rank.sort(dim=0, descending=True, stable=True).indices[:keep]] = True
    src = torch.arange(keep, device=CUDA)
    src[~stay[:keep]] = stay[keep:].nonzero()[:, 0] + keep
    assert out.tolist() == [keep] and torch.equal(pos[0, 0, :keep].long(), src) and torch.equal(w[0, 0, :keep], old_w[0, 0, src])
    assert torch.equal(c.row("k", 0, range(keep))[0], rows[src])


def test_eviction_from_a_graph():
    """One capture, replayed as the cache grows again: as the same calls one after the other."""
    ops = _ops()
    results = []
    for graphed in (False, True):
        c = Cache([200, 150], [1, 1], seed=11, extra_pages=1)
        g = _gen(12)
        weights = torch.rand(2, 2, c.per * 16, device=CUDA, generator=g)
        positions = torch.full((2, 2, c.per * 16), -1, dtype=torch.int32, device=CUDA)
        kv, nxt = c.kv_lens.clone(), c.kv_lens.clone()

        def body():
            return ops.evict_tokens(c.k, c.v, c.table, kv, weights, positions, nxt, keep=100, recent=8, first=2)

        state = [t.clone() for t in (c.k, c.v, weights, positions)]
        if graphed:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                body()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                lens = body()
            for t, old in zip((c.k, c.v, weights, positions), state):
                t.copy_(old)
        seen = []
        for step in range(4):
            if graphed:
                graph.replay()
            else:
                lens = body()
            seen += [lens.clone(), weights.clone(), positions.clone(), c.k.clone(), c.v.clone()]
            kv.copy_(lens + 37)                               # new tokens, with weights of their own
            nxt += 37
            weights[:, :, 100:137] = torch.rand(2, 2, 37, device=CUDA, generator=_gen(step))
        results.append(seen)
    for a, b in zip(*results):
        assert torch.equal(a.nan_to_num(nan=-7.0), b.nan_to_num(nan=-7.0)) if a.is_floating_point() else torch.equal(a, b)


# ---- together -----------------------------------------------------------------------------------------------------------------------------------------
def test_a_conversation_that_keeps_its_heavy_tokens():
    """A prompt's last tokens weigh the cache, and decode steps go on over what eviction leaves; a plain cache of lists does the same beside it. Weights that lie too
    near one another for 32 bits to order are not drawn: the plain cache takes the framework's own weights for its choice."""
    ops = _ops()
    G, H, D, bs, B = 4, 2, 64, 16, 2
    keep, recent, first = 48, 8, 4
    g = _gen(3)

    def rnd(*shape):
        return torch.randn(*shape, device=CUDA, generator=g).bfloat16()

    per, lens, nxt = 8, [90, 70], [90, 70]
    table = torch.randperm(B * per + 2, device=CUDA, generator=g)[:B * per].to(torch.int32).view(B, per)
    k, v = torch.full((B * per + 2, H, bs, D), float("nan"), device=CUDA).bfloat16(), torch.full((B * per + 2, H, bs, D), float("nan"), device=CUDA).bfloat16()
    plain = [[[] for _ in range(H)] for _ in range(B)]         # entries {position, k, v, w}

    def append(b, i, kk, vv, position):
        k[table[b, i // bs].long(), :, i % bs], v[table[b, i // bs].long(), :, i % bs] = kk, vv
        for h in range(H):
            plain[b][h].append([position, kk[h].double(), vv[h].double(), 0.0])

    for b in range(B):
        for i in range(lens[b]):
            append(b, i, rnd(H, D), rnd(H, D), i)
    weights = torch.zeros(B, H, per * bs, device=CUDA)
    positions = torch.full((B, H, per * bs), -1, dtype=torch.int32, device=CUDA)

    def attend(q, new):
        out = ops.tracked_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=CUDA), weights, cu_q=None, max_q_len=new, scale=D ** -0.5)
        for b in range(B):
            for i in range(new):
                for h in range(H):
                    seen = plain[b][h][:lens[b] - (new - 1 - i)]
                    qq = q[b * new + i, h * G:(h + 1) * G].double()
                    p = torch.softmax(qq @ torch.stack([e[1] for e in seen]).T * D ** -0.5, -1)
                    vv = torch.stack([e[2] for e in seen])
                    got = out[b * new + i].view(H, G, D)[h].double()
                    assert ((got - p @ vv).abs() <= 2.0 ** -8 * ((p @ vv).abs() + p @ vv.abs()) + 1e-3 * (p @ vv.abs())).all()
                    for e, x in zip(seen, p.sum(0).tolist()):
                        e[3] += x

    def evict():
        out = ops.evict_tokens(k, v, table, torch.tensor(lens, dtype=torch.int32, device=CUDA), weights, positions, torch.tensor(nxt, dtype=torch.int32, device=CUDA),
                               keep=keep, recent=recent, first=first)
        for b in range(B):
            lens[b] = int(out[b])
            for h in range(H):
                mine = {e[0]: e for e in plain[b][h]}
                place = positions[b, h, :lens[b]].tolist()
                assert len(set(place)) == lens[b] == keep and all(p in mine for p in place)
                safe = {p for p in mine if p < first or p >= nxt[b] - recent}
                gone = [mine[p][3] for p in mine if p not in place]
                assert safe <= set(place) and max(gone) <= min(mine[p][3] for p in place if p not in safe) + 1e-3
                plain[b][h] = [mine[p] for p in place]
                got = torch.tensor([e[3] for e in plain[b][h]], dtype=torch.float64, device=CUDA)
                assert (weights[b, h, :keep].double() - got).abs().max() <= 1e-3 and (weights[b, h, keep:] == 0).all()

    attend(rnd(B * 8, H * G, D), 8)
    evict()
    for step in range(70):
        for b in range(B):
            append(b, lens[b], rnd(H, D), rnd(H, D), nxt[b])
            lens[b], nxt[b] = lens[b] + 1, nxt[b] + 1
        attend(rnd(B, H * G, D), 1)
        if step % 32 == 31:
            evict()


def test_a_long_document_read_by_pages():
    """Prompt into the cache, summaries, and tokens that read the selected pages: as over the whole cache where the selection holds all pages, and near it where the rest carries
    no weight."""
    ops = _ops()
    c = Cache([700], [1], heads=8, kv_heads=2, D=128, seed=5)
    # two pages hold keys along the query: nearly all weight is theirs
    q = torch.randn(2, 128, device=CUDA, generator=_gen(1))
    q = (q / q.norm(dim=-1, keepdim=True) * 128 ** 0.5).bfloat16()
    c.q.copy_(q.repeat_interleave(4, 0)[None])
    for page in (7, 23):
        c.k[c.table[0, page].long()] = (q * 1.5)[:, None]
    sums = ops.PageSummaries.empty(c.k)
    ops.summarize_pages(c.k, c.table, c.kv_lens, sums, cu_q=None, max_q_len=700)
    weights = torch.zeros(1, 2, c.per * 16, device=CUDA)
    whole = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=128 ** -0.5, **c.step)
    every = ops.select_pages(c.q, sums, c.table, c.kv_lens, block_size=16, top=60, **c.step)
    assert every.counts.eq(44).all()
    _check_attention(c, ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, every, scale=128 ** -0.5, **c.step), lambda t, b, h, seen: range(seen), 128 ** -0.5)
    some = ops.select_pages(c.q, sums, c.table, c.kv_lens, block_size=16, top=2, first=1, last=2, **c.step)
    assert some.pages[0].tolist() == [[0, 7, 23, 42, 43]] * 2
    out = ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, some, scale=128 ** -0.5, **c.step)
    held = [j for p in (0, 7, 23, 42, 43) for j in range(p * 16, min(p * 16 + 16, 700))]
    lost = 4 - weights[0, :, held].sum(-1)                    # what the others weigh, of the four heads of a group
    assert (lost < 0.1).all()
    # dropping a share x of the weight moves the output by at most 2 x max |v|; both results and both products' weights are rounded, half a step each
    assert (out - whole).abs().max() <= (2 * lost.max() + 4 * 2.0 ** -8 + 1e-3) * c.row("v", 0, range(700)).abs().max()


def test_graphs_replay_with_other_lengths():
    """One capture of a decode step on a side stream, replayed as the sequence grows, beside a second graph on another cache."""
    ops = _ops()
    caches = [Cache([200, 90], [1, 1], seed=s) for s in (1, 2)]
    runs = []
    for c in caches:
        sums, weights, kv = ops.PageSummaries.empty(c.k), torch.zeros(2, 2, c.per * 16, device=CUDA), c.kv_lens.clone()
        ops.summarize_pages(c.k, c.table, kv, sums, cu_q=None, max_q_len=200)

        def body(c=c, sums=sums, weights=weights, kv=kv):
            ops.summarize_pages(c.k, c.table, kv, sums, cu_q=None, max_q_len=1)
            sel = ops.select_pages(c.q, sums, c.table, kv, block_size=16, top=2, first=1, last=1, **c.step)
            a = ops.selected_attention(c.q, c.k, c.v, c.table, kv, sel, scale=0.1, **c.step)
            return a, sel, ops.tracked_attention(c.q, c.k, c.v, c.table, kv, weights, scale=0.1, **c.step)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = body()
        weights.zero_()
        runs.append((c, graph, res, sums, weights, kv))
    for lens in ([150, 17], [200, 90], [48, 1]):
        for c, graph, res, sums, weights, kv in runs:
            kv.copy_(torch.tensor(lens, dtype=torch.int32))
            weights.zero_()
            graph.replay()
        for c, graph, (a, sel, b), sums, weights, kv in runs:
            c.lens = lens
            _check_attention(c, b, lambda t, s, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))
            host = sel.pages.cpu()
            _check_attention(c, a, lambda t, s, h, seen: [p * 16 + i for p in host[t, h].tolist() if p >= 0 for i in range(16) if p * 16 + i < seen], 0.1)
            for t, s, seen in c.tokens():
                for h in range(2):
                    want = _select(c, sums, t, s, h, seen, 2, 1, 1)
                    assert host[t, h].tolist() == want + [-1] * (4 - len(want))


def test_results_do_not_change_from_call_to_call():
    ops = _ops()
    c = Cache([5000, 777, 2300], [1, 1, 1], heads=32, kv_heads=8)
    first = None
    for _ in range(5):
        weights = torch.zeros(3, 8, c.per * 16, device=CUDA)
        got = [ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, **c.step), weights]
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(got, first))


@pytest.mark.parametrize("heads,kv", [(8, 2), (14, 2), (24, 2)])
def test_streams_beside_each_other(heads, kv):
    """The same calls on two streams at once, each with tensors of its own, give what they give one after the other."""
    ops = _ops()
    caches = [Cache([900, 300 + 40 * i], [3, 3], heads=heads, kv_heads=kv, seed=i) for i in range(2)]

    def work(c):
        sums = ops.PageSummaries.empty(c.k)
        ops.summarize_pages(c.k, c.table, c.kv_lens, sums, cu_q=None, max_q_len=900)
        sel = ops.select_pages(c.q, sums, c.table, c.kv_lens, block_size=16, top=5, **c.step)
        weights = torch.zeros(2, kv, c.per * 16, device=CUDA)
        return [sums.values().nan_to_num(), sel.pages, sel.counts, ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, sel, scale=0.1, **c.step),
                ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, **c.step), weights]

    want = [work(c) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    for _ in range(10):
        got = []
        for c, s in zip(caches, streams):
            with torch.cuda.stream(s):
                got.append(work(c))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))


def test_nothing_to_do():
    """No sequences, no new tokens, empty sequences."""
    ops = _ops()
    c = Cache([0, 40], [1, 1])
    none = torch.zeros(0, 8, 128, dtype=torch.bfloat16, device=CUDA)
    empty = {"cu_q": torch.zeros(3, dtype=torch.int32, device=CUDA), "max_q_len": 4}
    weights = torch.zeros(2, 2, c.per * 16, device=CUDA)
    sums = ops.PageSummaries.empty(c.k)
    ops.summarize_pages(c.k, c.table, c.kv_lens, sums, **empty)
    assert sums.scales.eq(0).all()
    sel = ops.select_pages(none, sums, c.table, c.kv_lens, block_size=16, top=2, **empty)
    assert sel.pages.shape == (0, 2, 7)
    assert ops.selected_attention(none, c.k, c.v, c.table, c.kv_lens, sel, scale=1.0, **empty).shape == (0, 1024)
    assert ops.tracked_attention(none, c.k, c.v, c.table, c.kv_lens, weights, scale=1.0, **empty).shape == (0, 1024) and weights.eq(0).all()
    lens = torch.zeros(0, dtype=torch.int32, device=CUDA)
    assert ops.tracked_attention(none, c.k, c.v, c.table[:0], lens, weights[:0], scale=1.0, cu_q=None, max_q_len=1).shape == (0, 1024)
    assert ops.evict_tokens(c.k, c.v, c.table[:0], lens, weights[:0], weights[:0].int(), lens, keep=4, recent=1).shape == (0,)
    pages = torch.full((2, 2, 3), -1, dtype=torch.int32, device=CUDA)
    out = ops.selected_attention(c.q, c.k, c.v, c.table, c.kv_lens, ops.PageSelection(pages, torch.zeros(2, 2, dtype=torch.int32, device=CUDA)), scale=1.0, **c.step)
    assert out.eq(0).all()


def test_lengths_behind_the_table_and_below_zero():
    """A length that the table has no pages for counts as the table's end; one below zero as none. New tokens that max_q_len does not cover are the caller's mistake, but nothing
    is read or written out of place for them."""
    ops = _ops()
    c = Cache([64, 64], [1, 1], extra_pages=0)
    kv = torch.tensor([1000, -5], dtype=torch.int32, device=CUDA)
    weights = torch.zeros(2, 2, 64, device=CUDA)
    out = ops.tracked_attention(c.q, c.k, c.v, c.table, kv, weights, scale=0.1, **c.step)
    c.lens = [64, 0]
    _check_attention(c, out, lambda t, b, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))
    sums = ops.PageSummaries.empty(c.k)
    ops.summarize_pages(c.k, c.table, kv, sums, cu_q=None, max_q_len=2000)
    sel = ops.select_pages(c.q, sums, c.table, kv, block_size=16, top=1, first=1, last=1, **c.step)
    assert sel.counts.tolist() == [[3, 3], [0, 0]]
    positions = torch.full((2, 2, 64), -1, dtype=torch.int32, device=CUDA)
    assert ops.evict_tokens(c.k, c.v, c.table, kv, weights, positions, kv.clone(), keep=50, recent=0).tolist() == [50, -5]
    assert (positions[0, :, :50] >= 0).all() and (positions[1] == -1).all()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_a_cache_behind_two_to_the_31_numbers(kind):
    """Pages whose first number lies behind 2^31: addresses are 64-bit."""
    ops = _ops()
    D, bs, kv = 128, 16, 2
    blocks = 2 ** 31 // (kv * bs * D) + 40
    k = torch.zeros(blocks, kv, bs, D, dtype=kind, device=CUDA)
    v = torch.zeros_like(k)
    g = _gen(8)
    tail = torch.arange(blocks - 20, blocks, device=CUDA)
    k[tail] = torch.randn(20, kv, bs, D, device=CUDA, generator=g).to(kind)
    v[tail] = torch.randn(20, kv, bs, D, device=CUDA, generator=g).to(kind)
    c = Cache([300], [1], heads=8, kv_heads=kv, kind=kind, extra_pages=1)
    c.k, c.v, c.blocks, c.table = k, v, blocks, tail[torch.randperm(20, device=CUDA, generator=g)].to(torch.int32)[None]
    weights = torch.zeros(1, kv, 320, device=CUDA)
    out = ops.tracked_attention(c.q, k, v, c.table, c.kv_lens, weights, scale=0.1, **c.step)
    _check_attention(c, out, lambda t, b, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))
    sums = ops.PageSummaries.empty(k)
    ops.summarize_pages(k, c.table, c.kv_lens, sums, cu_q=None, max_q_len=300)
    for page in (0, 17):
        code, scale = _summary(k[c.table[0, page].long(), 1].cpu())
        assert torch.equal(sums.codes[c.table[0, page].long(), 1].cpu(), code) and float(sums.scales[c.table[0, page].long(), 1]) == scale
    sel = ops.select_pages(c.q, sums, c.table, c.kv_lens, block_size=bs, top=4, **c.step)
    assert sel.pages[0, 0].tolist() == _select(c, sums, 0, 0, 0, 300, 4, 1, 4)
    rows = c.row("k", 0, range(300))
    positions = torch.full((1, kv, 320), -1, dtype=torch.int32, device=CUDA)
    ops.evict_tokens(k, v, c.table, c.kv_lens, weights, positions, c.kv_lens.clone(), keep=100, recent=10)
    for h in range(kv):
        assert torch.equal(c.row("k", 0, range(100))[h], rows[h, positions[0, h, :100].long()])


# ---- in the engine ------------------------------------------------------------------------------------------------------------------------------------
def _engine(budget, *, use_graphs=True, seed=0, **over):
    from inference_b200.engine.llm_engine import EngineConfig, LlmEngine
    from inference_b200.models import ModelConfig
    from inference_b200.models.llama import LlamaGpu

    cfg = ModelConfig.from_json({"hidden_size": 512, "intermediate_size": 1024, "num_hidden_layers": 3, "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": 128,
                                 "vocab_size": 2048, "rms_norm_eps": 1e-5, "rope_theta": 10000.0, **over})
    model = LlamaGpu(cfg, device=torch.device("cuda")).init_random(seed=seed)
    return LlmEngine(model, EngineConfig(max_batch=8, max_seq_len=1024, use_graphs=use_graphs, page_budget=budget))


def _prompts():
    g = torch.Generator().manual_seed(4)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (600, 37, 256, 15)]


@pytest.mark.parametrize("over", [{}, {"model_type": "gemma2", "attn_logit_softcapping": 50.0, "query_pre_attn_scalar": 128}])
def test_a_page_budget_that_holds_every_page_changes_nothing_but_roundings(over):
    ops = _ops()
    runs = []
    for budget in (None, ops.PageBudget(top=64)):
        eng = _engine(budget, **over)
        seqs = [eng.new_sequence() for _ in _prompts()]
        got = [eng.runner.prefill(seqs, _prompts(), want_logits=True)]
        for step in range(20):
            got.append(eng.runner.decode(seqs, [(7 * step + i) % 2048 for i in range(4)], want_logits=True).clone())
        runs.append(got)
    assert torch.equal(runs[0][0], runs[1][0])       # prompts read everything in either case
    for a, b in zip(*runs):
        assert (a - b).abs().max() <= 0.03 * a.abs().max()       # bf16 weights of the products are rounded in another order


def test_steps_on_a_page_budget_are_the_same_from_a_graph_and_without():
    ops = _ops()
    budget = ops.PageBudget(top=3, first=1, last=2)
    got = [_engine(budget, use_graphs=graphs).generate_batch(_prompts(), max_new_tokens=40).tokens for graphs in (True, False)]
    assert got[0] == got[1]
    assert all(len(t) == 40 for t in got[0])


def test_a_page_budget_reads_what_its_summaries_select():
    """Every layer's summaries are those of its pages after prompts, steps, a rollback and new steps; a fork finds them; and a step's attention is that of the pages they select."""
    ops = _ops()
    eng = _engine(ops.PageBudget(top=2, first=1, last=1))
    seq = eng.new_sequence()
    prompt = _prompts()[0]
    eng.runner.prefill([seq], [prompt])
    for i in range(30):
        eng.runner.decode([seq], [i])
    seq.truncate(603)                                 # within a page that was full
    eng.runner.prefill([seq], [[9] * 40], want_logits=True)
    seen = []
    real = ops.selected_attention

    def spy(q, k, v, table, lens, sel, **kw):
        out = real(q, k, v, table, lens, sel, **kw)
        seen.append((q.clone(), k, v, table, lens.clone(), sel, kw, out.clone()))
        return out

    eng.runner.use_graphs = False
    ops.selected_attention = spy
    try:
        eng.runner.decode([seq], [5])
    finally:
        ops.selected_attention = real
    assert len(seen) == 3
    full = seq.length // 16
    for layer, (q, k, v, table, lens, sel, kw, out) in enumerate(seen):
        for page in range(full):
            at = seq.blocks[page]
            for h in range(2):
                code, scale = _summary(eng.pool.data[layer, 0, at, h].cpu())
                assert torch.equal(eng.pool.summaries[layer].codes[at, h].cpu(), code) and float(eng.pool.summaries[layer].scales[at, h]) == scale
        c = Cache([seq.length], [1], heads=4, kv_heads=2)
        c.k, c.v, c.table, c.q, c.blocks = k, v, table, q, k.shape[0]
        for h in range(2):
            assert sel.pages[0, h].tolist() == _select(c, eng.pool.summaries[layer], 0, 0, h, seq.length, 2, 1, 1)
        host = sel.pages.cpu()
        _check_attention(c, out, lambda t, b, h, n: [p * 16 + i for p in host[t, h].tolist() for i in range(16) if p * 16 + i < n], kw["scale"])


def test_runners_of_one_pool_keep_its_summaries_up():
    """One runner with a budget, one without (made, and its step captured, before the pool had summaries): what the second one writes is summarised too."""
    from inference_b200.engine.runner import ModelRunner

    ops = _ops()
    eng = _engine(None)
    plain = eng.runner
    seq = eng.new_sequence()
    plain.prefill([seq], [_prompts()[1]])
    plain.decode([seq], [3])
    with pytest.raises(ValueError):
        ModelRunner(eng.model, eng.pool, max_batch=8, max_seq_len=1024, page_budget=ops.PageBudget(top=2))
    seq.release()
    short = ModelRunner(eng.model, eng.pool, max_batch=8, max_seq_len=1024, page_budget=ops.PageBudget(top=2))
    seq = eng.new_sequence()
    for i, run in enumerate((plain, short, plain)):
        run.prefill([seq], [_prompts()[i]])
        for token in range(20):
            run.decode([seq], [token])
    torch.cuda.synchronize()
    for layer in range(3):
        for page in range(seq.length // 16):
            at = seq.blocks[page]
            for h in range(2):
                code, scale = _summary(eng.pool.data[layer, 0, at, h].cpu())
                assert torch.equal(eng.pool.summaries[layer].codes[at, h].cpu(), code) and float(eng.pool.summaries[layer].scales[at, h]) == scale


def test_a_page_budget_needs_a_uniform_pool():
    from inference_b200.contracts.errors import Unsupported
    from inference_b200.engine.runner import ModelRunner

    ops = _ops()
    with pytest.raises(ops.KernelError):
        ops.PageBudget(top=1, last=0)
    with pytest.raises(Unsupported):
        ModelRunner(object(), object(), page_budget=ops.PageBudget(top=1))
