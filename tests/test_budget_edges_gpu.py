"""Operators of long caches on a budget where their definitions are easily missed: calls that the documentation allows and that differ from the usual ones."""
import pytest
import torch
from test_budget_gpu import CUDA, Cache, _check_attention, _engine, _gen, _ops, _prompts, _select, _summary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("splits", [1, 3, 9])
def test_pages_that_are_not_there_weigh_nothing_beside_a_key_that_is_no_number(splits, kind):
    """However a problem's splits are joined and its weights added up."""
    ops = _ops()
    c = Cache([100], [1], kind=kind)
    c.k[c.table[0, 0].long(), 1, 5] = float("nan")
    c.table[0, 2] = -5
    weights = torch.zeros(1, 2, c.per * 16, device=CUDA)
    ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, num_splits=splits, **c.step)
    there = torch.tensor([j // 16 != 2 for j in range(100)], device=CUDA)
    assert weights[0, 1, :100][there].isnan().all() and weights[0, 0].isfinite().all()
    assert weights[0, :, 32:48].eq(0).all() and weights[0, :, 100:].eq(0).all()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4), (24, 2)])
@pytest.mark.parametrize("q_lens", [(20, 7), (20, 20)])
def test_lengths_behind_the_table_of_several_tokens(q_lens, heads, kv, kind):
    """They count as the table's end: the last token sees all of it and the ones in front of it a key less each, in either type and however tokens share their keys."""
    ops = _ops()
    c = Cache([64, 30], q_lens, heads=heads, kv_heads=kv, kind=kind, extra_pages=0)
    lens = torch.tensor([1000, 30], dtype=torch.int32, device=CUDA)
    for splits in (None, 1, 3, 9):
        weights = torch.zeros(2, kv, 64, device=CUDA)
        out = ops.tracked_attention(c.q, c.k, c.v, c.table, lens, weights, scale=0.1, num_splits=splits, **c.step)
        _check_attention(c, out, lambda t, b, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))
    g = _gen(heads)
    sums = ops.PageSummaries(torch.randint(-127, 128, (c.blocks, kv, 128), device=CUDA, generator=g).to(torch.int8), torch.rand(c.blocks, kv, device=CUDA, generator=g))
    some = ops.select_pages(c.q, sums, c.table, lens, block_size=16, top=1, first=0, last=1, **c.step)
    for t, b, seen in c.tokens():
        for h in range(kv):
            want = _select(c, sums, t, b, h, seen, 1, 0, 1)
            assert some.pages[t, h].tolist() == want + [-1] * (2 - len(want)) and some.counts[t, h] == len(want)
    out = ops.selected_attention(c.q, c.k, c.v, c.table, lens, some, scale=0.1, **c.step)
    host = some.pages.cpu()
    _check_attention(c, out, lambda t, b, h, seen: [p * 16 + i for p in host[t, h].tolist() if p >= 0 for i in range(16) if p * 16 + i < seen], 0.1)


def test_the_largest_bound_of_a_step():
    """max_q_len is a bound, and the largest number is one."""
    ops = _ops()
    c = Cache([40, 70, 20], [2, 3, 1], heads=24, kv_heads=2)
    for kind in (torch.bfloat16, torch.float32):
        c.q, c.k, c.v, c.kind = c.q.to(kind), c.k.to(kind), c.v.to(kind), kind
        weights = torch.zeros(3, 2, c.per * 16, device=CUDA)
        out = ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, cu_q=c.cu, max_q_len=2 ** 31 - 1)
        _check_attention(c, out, lambda t, b, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [8, 24])
@pytest.mark.parametrize("splits", [1, 2, 9])
def test_rows_in_front_of_the_first_sequence_stay(splits, heads, kind):
    """As those behind the last one do: rows of no sequence."""
    ops = _ops()
    c = Cache([40, 70], [2, 3], heads=heads, kind=kind, behind=5)
    at, front = torch.full((10, 2), 3, dtype=torch.int32, device=CUDA), c.cu + 3
    pages = torch.arange(3, dtype=torch.int32, device=CUDA).expand(10, 2, 3).contiguous()
    q = c.q
    weights, out = torch.zeros(2, 2, c.per * 16, device=CUDA), torch.full((10, heads * 128), 7.0, dtype=kind, device=CUDA)
    some = out.clone()
    ops.tracked_attention(q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, num_splits=splits, out=out, cu_q=front, max_q_len=3)
    ops.selected_attention(q, c.k, c.v, c.table, c.kv_lens, ops.PageSelection(pages, at), scale=0.1, num_splits=splits, out=some, cu_q=front, max_q_len=3)
    for x in (out, some):
        assert x[:3].eq(7).all() and x[8:].eq(7).all()
    c.q = q[3:]
    _check_attention(c, out[3:], lambda t, b, h, seen: range(seen), 0.1, weights=weights, before=torch.zeros_like(weights))
    _check_attention(c, some[3:], lambda t, b, h, seen: range(min(seen, 48)), 0.1)


@pytest.mark.parametrize("cleared", [True, False])
def test_evictions_after_tokens_were_taken_back(cleared):
    """Weights of drafts that were taken back are the caller's to clear, whether or not the sequence shrinks then: an eviction leaves what lies behind a sequence's length, and
    the tokens that are appended there go on from it. Cleared, everything is as if the drafts had never been."""
    ops = _ops()
    keep, results = 60, []
    for drafts in (0, 7):
        c = Cache([100, 50], [1, 1], seed=3, filler=0.0)
        weights = torch.zeros(2, 2, c.per * 16, device=CUDA)
        positions = torch.full((2, 2, c.per * 16), -1, dtype=torch.int32, device=CUDA)
        lens = c.kv_lens.clone()

        def step(q, c=c, weights=weights, lens=lens):
            return ops.tracked_attention(q, c.k, c.v, c.table, lens, weights, scale=0.1, cu_q=None, max_q_len=q.shape[0] // 2)

        step(c.q)
        if drafts:
            lens += drafts
            step(torch.randn(2 * drafts, 8, 128, device=CUDA, generator=_gen(5)).bfloat16())
            lens -= drafts
            stale = weights.clone()
            at = torch.arange(c.per * 16, device=CUDA)
            assert (stale[0, :, 100:107] > 0).all() and (stale[1, :, 50:57] > 0).all()
            weights.copy_(seen)                        # what the drafts gave to the entries that stay is theirs: here only the rest is looked at
            weights += stale * (at >= lens[:, None, None])
            if cleared:
                weights.masked_fill_(at >= lens[:, None, None], 0)
        seen = weights.clone()
        lens.copy_(ops.evict_tokens(c.k, c.v, c.table, lens, weights, positions, torch.tensor([100, 50], dtype=torch.int32, device=CUDA), keep=keep, recent=5, first=2))
        assert lens.tolist() == [60, 50]
        assert weights[0, :, keep:100].eq(0).all() and positions[0, :, keep:].eq(-1).all() and positions[1].eq(-1).all()
        assert torch.equal(weights[0, :, 100:], seen[0, :, 100:]) and torch.equal(weights[1], seen[1])
        results.append((weights.clone(), positions.clone(), c.k.clone(), c.v.clone()))
    same = [torch.equal(a, b) for a, b in zip(*results)]
    assert same == [cleared, True, True, True]


@pytest.mark.parametrize("splits", [1, 3, 9])
def test_weights_below_the_normal_range_are_zeros_however_splits_are_joined(splits):
    """A key 90 below the largest has a weight of 2^-129.8, which 32 bits hold as a number below the normal range only."""
    ops = _ops()
    c = Cache([200], [1], filler=0.0)
    c.q.zero_(), c.k.zero_()
    c.q[..., 0] = 1
    c.k[..., 0] = -90
    c.k[c.table[0, 0].long(), :, 3, 0] = 0
    weights = torch.zeros(1, 2, c.per * 16, device=CUDA)
    ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=1.0, num_splits=splits, **c.step)
    assert weights[0, :, 3].eq(4).all() and weights.count_nonzero() == 2


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_columns_of_a_wide_table(kind):
    """What a caller with a table for long contexts gives for short ones: rows that lie apart, beside weights and positions of the whole width."""
    ops = _ops()
    got = []
    for wide in (0, 500):
        c = Cache([200, 90, 130], [1, 1, 1], kind=kind, seed=8, filler=0.0)
        whole = torch.full((3, c.per + wide), -7, dtype=torch.int32, device=CUDA)
        whole[:, :c.per] = c.table
        table, n = whole[:, :c.per], (c.per + wide) * 16
        weights, positions = torch.zeros(3, 2, n, device=CUDA), torch.full((3, 2, n), -1, dtype=torch.int32, device=CUDA)
        sums = ops.PageSummaries.empty(c.k)
        ops.summarize_pages(c.k, table, c.kv_lens, sums, cu_q=None, max_q_len=200)
        some = ops.select_pages(c.q, sums, table, c.kv_lens, block_size=16, top=2, first=1, last=1, **c.step)
        out = [ops.selected_attention(c.q, c.k, c.v, table, c.kv_lens, some, scale=0.1, **c.step), ops.tracked_attention(c.q, c.k, c.v, table, c.kv_lens, weights, scale=0.1, **c.step)]
        lens = ops.evict_tokens(c.k, c.v, table, c.kv_lens, weights, positions, c.kv_lens, keep=100, recent=8)
        m = c.per * 16
        assert weights[..., m:].eq(0).all() and positions[..., m:].eq(-1).all()
        got.append([*out, sums.codes, sums.scales, some.pages, some.counts, lens, weights[..., :m].clone(), positions[..., :m].clone(), c.k, c.v])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_pages_are_summarised_again_behind_an_eviction():
    ops = _ops()
    c = Cache([300, 90], [1, 1], seed=6, filler=0.0)
    sums = ops.PageSummaries.empty(c.k)
    ops.summarize_pages(c.k, c.table, c.kv_lens, sums, cu_q=None, max_q_len=300)
    weights = torch.zeros(2, 2, c.per * 16, device=CUDA)
    ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, **c.step)
    lens = ops.evict_tokens(c.k, c.v, c.table, c.kv_lens, weights, torch.full((2, 2, c.per * 16), -1, dtype=torch.int32, device=CUDA), c.kv_lens, keep=120, recent=8, first=2)
    old = sums.codes.clone()
    ops.summarize_pages(c.k, c.table, lens, sums, cu_q=None, max_q_len=120)
    assert not torch.equal(old, sums.codes)
    for b, n in enumerate(lens.tolist()):
        for at in c.table[b, :n // 16].tolist():
            for h in range(2):
                code, scale = _summary(c.k[at, h].cpu())
                assert torch.equal(sums.codes[at, h].cpu(), code) and float(sums.scales[at, h]) == scale
    c.lens = lens.tolist()
    some = ops.select_pages(c.q, sums, c.table, lens, block_size=16, top=2, first=1, last=1, **c.step)
    for t, b, seen in c.tokens():
        for h in range(2):
            want = _select(c, sums, t, b, h, seen, 2, 1, 1)
            assert some.pages[t, h].tolist() == want + [-1] * (4 - len(want))
    host = some.pages.cpu()
    _check_attention(c, ops.selected_attention(c.q, c.k, c.v, c.table, lens, some, scale=0.1, **c.step),
                     lambda t, b, h, seen: [p * 16 + i for p in host[t, h].tolist() if p >= 0 for i in range(16) if p * 16 + i < seen], 0.1)


# ---- in the engine ------------------------------------------------------------------------------------------------------------------------------------
@pytest.fixture
def read_by_pages(monkeypatch):
    """What selected_attention was called with, and gave."""
    ops, seen = _ops(), []
    real = ops.selected_attention

    def spy(q, k, v, table, lens, sel, **kw):
        out = real(q, k, v, table, lens, sel, **kw)
        seen.append((q.clone(), k, v, table.clone(), lens.clone(), sel, kw, out.clone()))
        return out

    monkeypatch.setattr(ops, "selected_attention", spy)
    return seen


def test_a_prompt_reads_everything_in_whatever_pieces_it_comes(read_by_pages):
    ops = _ops()
    pieces = [_prompts()[0], [5, 6, 7], _prompts()[1], [1, 2], [3, 4, 5, 6, 7, 8, 9, 10]]
    runs = []
    for budget in (None, ops.PageBudget(top=1, first=0, last=1)):
        eng = _engine(budget)
        seq = eng.new_sequence()
        runs.append([eng.runner.prefill([seq], [p], want_logits=True) for p in pieces])
        runs[-1].append(eng.runner.prefill([seq], [[11, 12, 13]], want=[[0, 2]]))
    assert all(torch.equal(a, b) for a, b in zip(*runs)) and not read_by_pages


def test_more_sequences_than_a_decode_batch_are_a_step_too(read_by_pages):
    from inference_b200.engine.backend import GpuBackend

    ops = _ops()
    eng = _engine(ops.PageBudget(top=1, first=1, last=1))
    backend = GpuBackend(eng.runner)
    seqs = [backend.new_sequence() for _ in range(9)]
    backend.forward(seqs, [[i + k for k in range(50 + 4 * i)] for i in range(9)])
    assert not read_by_pages
    backend.forward_greedy(seqs, [[i] for i in range(9)])
    assert len(read_by_pages) == 3 and all(x[0].shape[0] == 9 for x in read_by_pages)


@pytest.mark.parametrize("drafts", [0, 1, 4, 8, 20])
def test_verified_drafts_read_what_decode_steps_would(drafts, read_by_pages):
    """However many there are, of one sequence or of several with numbers of their own, in front of and behind the end of a page; and after a rollback."""
    ops = _ops()
    eng = _engine(ops.PageBudget(top=2, first=1, last=1))
    seqs = [eng.new_sequence(), eng.new_sequence()]
    eng.runner.prefill(seqs, [_prompts()[0], _prompts()[2]])
    ids = [[7 + i for i in range(drafts + 1)], [9, 8]]
    for group, new in ((seqs[:1], ids[:1]), (seqs, ids)):
        base = [s.length for s in group]
        read_by_pages.clear()
        got = eng.runner.prefill(group, new, all_positions=True)
        assert got.shape == (sum(map(len, new)), 2048) and len(read_by_pages) == 3
        for layer, (q, k, v, table, lens, sel, kw, out) in enumerate(read_by_pages):
            c = Cache([s.length for s in group], [len(n) for n in new], heads=4, kv_heads=2)
            c.k, c.v, c.table, c.q, c.blocks = k, v, table, q, k.shape[0]
            host = sel.pages.cpu()
            for t, b, seen in c.tokens():
                for h in range(2):
                    want = _select(c, eng.pool.summaries[layer], t, b, h, seen, 2, 1, 1)
                    assert host[t, h].tolist() == want + [-1] * (4 - len(want))
            _check_attention(c, out, lambda t, b, h, n: [p * 16 + i for p in host[t, h].tolist() if p >= 0 for i in range(16) if p * 16 + i < n], kw["scale"])
        for s, n in zip(group, base):
            s.truncate(n + 1)


def test_decode_steps_read_the_same_with_prompts_beside_them(read_by_pages):
    """A chunk of another sequence's prompt in the same call changes neither's result, and results keep the order of the call."""
    from inference_b200.engine.backend import GpuBackend

    ops = _ops()
    runs = []
    for together in (True, False):
        eng = _engine(ops.PageBudget(top=2, first=1, last=1))
        backend = GpuBackend(eng.runner)
        seqs = [backend.new_sequence() for _ in range(3)]
        backend.forward(seqs, [_prompts()[2], _prompts()[0], _prompts()[2][:100]])
        news, wants, got = [[5], _prompts()[1], [6]], [[0], [3, 36], [0, 0]], []
        order, call = range(3), [seqs, news]
        if together:
            got += [x.clone() for x in backend.forward(*call)]       # rows of a decode graph's own output, which the next step writes again
            got += [torch.tensor(backend.forward_greedy(*call))]
            got += [backend.forward_at(*call, wants)]
            assert backend.forward_at(*call, [[], [], []]) is None and backend.forward_at(*call, [[], [1], []]).shape == (1, 2048)
        else:
            steps, prompt = [0, 2], [1]

            def apart(f, *lists):
                return {i: x for part in (steps, prompt) for i, x in zip(part, f(*([y[i] for i in part] for y in lists)))}

            parts = apart(backend.forward, *call)
            got += [parts[i].clone() for i in order]
            parts = apart(backend.forward_greedy, *call)
            got += [torch.tensor([parts[i] for i in order])]
            one, more = backend.forward_at([seqs[0], seqs[2]], [news[0], news[2]], [wants[0], wants[2]]), backend.forward_at([seqs[1]], [news[1]], [wants[1]])
            got += [torch.cat([one[:1], more, one[1:]])]
        runs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


class _OneRank:
    """The row-parallel products and the sums over ranks of a fused prefill, where there is one rank: all rows are its own."""

    def __init__(self):
        self.partial, self.used = None, 0

    def my_rows(self, T):
        return 0, T

    def gemm_scatter_rows(self, x, w):
        self.partial = _ops().linear_any(x, w)

    def reduce_norm_gather(self, T, res, weight, eps, woff, reduce=True):
        self.used += 1
        return _ops().rmsnorm(self.partial, weight, eps, residual=res, w_offset=woff) if reduce else _ops().rmsnorm(res, weight, eps, w_offset=woff)


def test_the_fused_prefill_of_several_ranks_keeps_summaries_up(monkeypatch):
    """Prompts on a page budget take it as they do without one; what it writes is summarised."""
    ops = _ops()
    eng, ctx = _engine(ops.PageBudget(top=2, first=1, last=1)), _OneRank()
    monkeypatch.setattr(eng.model, "_use_tp_prefill", lambda T: T > 16)
    monkeypatch.setattr(eng.model, "_tp_prefill_context", lambda: ctx)
    seqs = [eng.new_sequence(), eng.new_sequence()]
    for new in ([_prompts()[0], _prompts()[1]], [_prompts()[1], _prompts()[2]]):
        eng.runner.prefill(seqs, new)
    assert ctx.used == 2 * (1 + 2 * 3)
    eng.runner.prefill(seqs, [list(range(12))] * 2, all_positions=True)      # reads by pages, which the fused prefill does not
    assert ctx.used == 2 * (1 + 2 * 3)
    torch.cuda.synchronize()
    for layer in range(3):
        sums = eng.pool.summaries[layer]
        for seq in seqs:
            for at in seq.blocks[:seq.length // 16]:
                for h in range(2):
                    code, scale = _summary(eng.pool.data[layer, 0, at, h].cpu())
                    assert torch.equal(sums.codes[at, h].cpu(), code) and float(sums.scales[at, h]) == scale


def test_contexts_that_grow_replay_the_graph_of_their_batch():
    """What a step on a page budget reads does not follow from the context's length, so neither do its graphs."""
    ops = _ops()
    eng = _engine(ops.PageBudget(top=1))
    seq = eng.new_sequence()
    for n in (30, 300, 500):
        eng.runner.prefill([seq], [list(range(n))])
        eng.runner.decode([seq], [1])
    assert eng.runner.captures == 1
    eng.runner.decode_multi([seq], [1], 2)
    eng.runner.prefill([seq], [list(range(100))])
    eng.runner.decode_multi([seq], [1], 2)
    assert eng.runner.captures == 2


def test_a_budget_beyond_the_table_takes_the_tables_room(read_by_pages):
    """A large number is the natural way to say everything: lists are as long as the table's pages ask for."""
    ops = _ops()
    runs = []
    for budget in (ops.PageBudget(top=64), ops.PageBudget(top=10 ** 6), ops.PageBudget(top=0, first=10 ** 6), ops.PageBudget(top=1, last=2 ** 40)):
        eng = _engine(budget, use_graphs=False)
        seq = eng.new_sequence()
        eng.runner.prefill([seq], [_prompts()[0]])
        read_by_pages.clear()
        runs.append(eng.runner.decode([seq], [3], want_logits=True).clone())
        assert len(read_by_pages) == 3
        for x in read_by_pages:
            assert x[5].pages.shape[2] <= 64 + 64 + 1 and x[5].counts.eq(38).all()
    assert all(torch.equal(x, runs[0]) for x in runs)


def test_summaries_of_forks_and_of_pages_that_are_taken_back():
    """Two sequences share a prompt's pages. One goes back into a page that was full, which it then has to itself, and writes other tokens there: the other one still finds its own
    page's summary, and both read what their summaries select."""
    ops = _ops()
    eng = _engine(ops.PageBudget(top=2, first=1, last=1), use_graphs=False)
    from inference_b200.engine.backend import GpuBackend

    backend = GpuBackend(eng.runner)
    one = backend.new_sequence()
    backend.forward([one], [_prompts()[0]])
    two = backend.fork(one, 592)
    assert two.blocks == one.blocks[:37]
    two.truncate(580)                                  # within the last shared page
    backend.forward([two], [[3 + i for i in range(40)]])
    assert two.blocks[:36] == one.blocks[:36] and two.blocks[36] != one.blocks[36]
    one.truncate(590)
    for token in range(20):
        backend.forward_greedy([one, two], [[token], [token + 5]])
    three = backend.fork(two, 48)                      # whole pages, then tokens of its own
    backend.forward([three], [_prompts()[2]])
    seqs, seen = [one, two, three], []
    real = ops.selected_attention

    def spy(q, k, v, table, lens, sel, **kw):
        out = real(q, k, v, table, lens, sel, **kw)
        seen.append((q.clone(), k, v, table.clone(), sel, kw, out.clone()))
        return out

    ops.selected_attention = spy
    try:
        backend.forward_greedy(seqs, [[1], [2], [3]])
    finally:
        ops.selected_attention = real
    assert len(seen) == 3
    for layer, (q, k, v, table, sel, kw, out) in enumerate(seen):
        for seq in seqs:
            for at in seq.blocks[:seq.length // 16]:
                for h in range(2):
                    code, scale = _summary(eng.pool.data[layer, 0, at, h].cpu())
                    assert torch.equal(eng.pool.summaries[layer].codes[at, h].cpu(), code) and float(eng.pool.summaries[layer].scales[at, h]) == scale
        c = Cache([s.length for s in seqs], [1, 1, 1], heads=4, kv_heads=2)
        c.k, c.v, c.table, c.q, c.blocks = k, v, table, q[:3], k.shape[0]
        host = sel.pages.cpu()
        for t, b, n in c.tokens():
            for h in range(2):
                assert host[t, h].tolist() == _select(c, eng.pool.summaries[layer], t, b, h, n, 2, 1, 1)
        _check_attention(c, out[:3], lambda t, b, h, n: [p * 16 + i for p in host[t, h].tolist() for i in range(16) if p * 16 + i < n], kw["scale"])
