"""Drafted trees, accepted paths and beams at the edges of what their calls allow."""
import math

import pytest
import torch

from test_branch_gpu import CUDA, Step, _check_beams, _gen, _ops, _pack, _run, _trees, _visible

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])


# ---- scores that are not numbers ------------------------------------------------------------------------------------------------------------------------
# Tokens x 4 heads of a group: 28 rows are one half of a block, whose tiles of 128 keys are dealt out by turns; 240 rows are both halves, which share the tiles.
@KINDS
@pytest.mark.parametrize("q_lens", [[7, 5], [60, 33]], ids=["half", "two"])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("base", [[300, 140], [100, 0], [131, 513]], ids=str)
@pytest.mark.parametrize("what", ["nan", "inf", "cancel", "nan, capped"])
def test_a_query_that_is_no_number_is_its_own_rows_matter(kind, q_lens, splits, base, what):
    """One head of one token has NaN, or infinities whose products are, or add up to, none: its result is NaN, all others are those of the clean run, bit by bit."""
    c = Step(base, q_lens, kind=kind, seed=71)
    sees, _ = _visible(_trees(q_lens, 72), c.max_q)
    mask, cap = _pack(sees), 20.0 if "capped" in what else 0.0
    clean = _run(c, mask, 0.1, softcap=cap, num_splits=splits)
    t, head = q_lens[0] - 1, 5          # sees more than one key
    if "nan" in what:
        c.q[t, head, 3] = math.nan
    elif what == "inf":
        c.q[t, head, 3] = math.inf      # products of both signs: of the larger ones none is a number
    else:
        c.q[t, head, 3], c.q[t, head, 4] = math.inf, -math.inf
    out = _run(c, mask, 0.1, softcap=cap, num_splits=splits)
    _ops().check_status()
    out, clean = (x.view(c.T, c.heads, -1) for x in (out, clean))
    assert out[t, head].isnan().all()
    rest = torch.ones(c.T, c.heads, dtype=torch.bool, device=CUDA)
    rest[t, head] = False
    assert torch.equal(out[rest], clean[rest])


@KINDS
@pytest.mark.parametrize("q_lens", [[7, 5], [64, 33]], ids=["half", "two"])
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("base,first,n", [(b, f, min(n, b - f)) for b in (100, 130, 300, 520) for f, n in ((0, 64), (64, 64), (0, 100), (128, 64), (192, 64), (128, 128), (256, 40)) if f < b])
@pytest.mark.parametrize("lone", [False, True], ids=["", "and a query"])
def test_keys_that_are_no_numbers_fill_half_a_tile(kind, q_lens, splits, base, first, n, lone):
    """64 cached keys and more of one key/value head are NaN, which all of its sequence's tokens see; with a query that is NaN too. Everything else is that of the clean run."""
    c = Step([base, 200], q_lens, kind=kind, seed=73)
    sees, _ = _visible(_trees(q_lens, 74), c.max_q)
    clean = _run(c, _pack(sees), 0.1, num_splits=splits)
    for key in range(first, first + n):
        page, at = c.place(0, key)
        c.k[page, 1, at] = math.nan
    bad = torch.zeros(c.T, c.heads, dtype=torch.bool, device=CUDA)
    bad[:q_lens[0], 4:] = True
    if lone:
        c.q[2, 1, 0] = math.nan
        bad[2, 1] = True
    out = _run(c, _pack(sees), 0.1, num_splits=splits)
    _ops().check_status()
    out, clean = (x.view(c.T, c.heads, -1) for x in (out, clean))
    assert out[bad].isnan().all() and torch.equal(out[~bad], clean[~bad])


@KINDS
@pytest.mark.parametrize("splits", [1, 2])
def test_everything_is_no_number(kind, splits):
    c = Step([700, 3], [70, 2], kind=kind, seed=75)
    sees, _ = _visible(_trees(c.q_lens, 76), c.max_q)
    c.q.fill_(math.nan)
    out = _run(c, _pack(sees), 0.1, num_splits=splits)
    _ops().check_status()
    assert out.isnan().all()


# ---- bounds of a step ---------------------------------------------------------------------------------------------------------------------------------------
@KINDS
def test_a_steps_bound_may_be_the_largest_number(kind):
    ops, c = _ops(), Step([70, 9], [9, 20], kind=kind, seed=81)
    parents = torch.tensor(sum(_trees(c.q_lens, 82), []), dtype=torch.int32, device=CUDA)
    near, far = ops.plan_tree(parents, cu_q=c.cu, max_q_len=20), ops.plan_tree(parents, cu_q=c.cu, max_q_len=2 ** 31 - 1)
    assert torch.equal(near.mask, far.mask) and torch.equal(near.depths, far.depths)
    out = _run(c, near.mask, 0.1, num_splits=2)
    c.max_q = 2 ** 31 - 1
    assert torch.equal(_run(c, far.mask, 0.1, num_splits=2), out)
    empty = ops.plan_tree(parents[:0], cu_q=torch.zeros(3, dtype=torch.int32, device=CUDA), max_q_len=5)
    assert empty.mask.shape == (0, 1) and empty.depths.shape == (0,)


# ---- logits far from zero -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shift", [300, 2000, 20000, 29900, 31000, -20000, -31000])
def test_logits_far_from_zero_lose_nothing(shift):
    """Two beams with the same logits, one of them moved by a whole number, whose scores differ by 2e-8: the better one is first at every token. (Logits are multiples of 1 / 64, so that
    the move is exact; a logarithm is off by 2^-28.5 at most, 3e-9.)"""
    V = 6000
    row = (torch.randn(V, device=CUDA, generator=_gen(91)) * 3 * 64).round() / 64
    logits = torch.stack([row + shift, row])
    assert torch.equal(logits[0] - shift, row)
    for scores in ([2e-8, 0.0], [0.0, 2e-8]):
        _check_beams(logits, torch.tensor([scores], device=CUDA), 60)


@KINDS
@pytest.mark.parametrize("V", [90, 9001, 70001])
def test_tokens_forbidden_by_a_finite_number(kind, V):
    """What is filled in for them is a logit like others: it ties, and comes behind what is allowed."""
    for fill in (-1e4, -1e9, float(torch.finfo(kind).min)):
        logits = torch.full((3, V), fill, device=CUDA, dtype=kind)
        allowed = torch.randperm(V, device=CUDA, generator=_gen(V))[:7]
        logits[0, allowed] = torch.randn(7, device=CUDA, generator=_gen(92)).to(kind)
        logits[1, 3 * V // 4:] = torch.randn(V - 3 * V // 4, device=CUDA, generator=_gen(93)).to(kind)
        _check_beams(logits, torch.tensor([[-1.0, -2.0, -0.5]], device=CUDA), 12)


@KINDS
def test_logits_that_pass_the_rounding_s_reach(kind):
    """Rows above and below it, and rows that cross it on the way, up and down."""
    V = 40000
    ramp = torch.linspace(-1, 1, V, device=CUDA) * 40000
    step = torch.where(torch.arange(V, device=CUDA) < V // 2, 29000.0, 31000.0) + torch.randn(V, device=CUDA, generator=_gen(94)) * 3
    near = torch.randn(V, device=CUDA, generator=_gen(95)) * 3
    rows = torch.stack([ramp, ramp.flip(0), step, step.flip(0), near + 40000, near - 40000, -step, near]).to(kind)
    _check_beams(rows, -10 * torch.rand(2, 4, device=CUDA, generator=_gen(96)), 20)
    _check_beams(rows, -10 * torch.rand(8, 1, device=CUDA, generator=_gen(97)), 100)


@KINDS
@pytest.mark.parametrize("count", [1, 9, 128])
def test_logits_that_rise_with_the_tokens_number(kind, count):
    """Every step's are above the bound that the ones before it gave: more candidates than a block takes notes of."""
    V = 128256
    rise = torch.arange(V, device=CUDA, dtype=torch.float32) / 4096
    _check_beams(torch.stack([rise, rise * 2, rise.flip(0)]).to(kind), torch.tensor([[-1.0, -1.5, -2.0]], device=CUDA), count)


# ---- more tokens than the step was told of ------------------------------------------------------------------------------------------------------------------
@KINDS
@pytest.mark.parametrize("splits", [1, 3])
def test_of_more_tokens_than_the_bound_the_first_are_computed(kind, splits):
    c = Step([90, 40], [12, 5], kind=kind, seed=83)
    sees, _ = _visible(_trees(c.q_lens, 84), c.max_q)
    whole = _run(c, _pack(sees), 0.1, num_splits=splits)
    c.max_q = 7
    out = torch.full_like(whole, 7.0)
    _run(c, _pack(sees), 0.1, num_splits=splits, out=out)
    left = torch.zeros(c.T, dtype=torch.bool, device=CUDA)
    left[7:12] = True
    assert (out[left] == 7).all()
    c.q_lens[0] = 7         # the definition for the first seven, which lie behind 90 keys as in the whole step
    c.check(out, sees, 0.1)


def test_of_more_tokens_than_the_bound_the_first_may_be_accepted():
    ops = _ops()
    tokens = torch.arange(8, device=CUDA)
    picks = torch.tensor([1, 3, 9, 4, 5, 6, 7, 2], device=CUDA)           # 0 -> 1 -> 3 -> 4 -> 5 ..
    parents = torch.tensor([-1, 0, 0, 1, 3, 4, 5, 6], dtype=torch.int32, device=CUDA)
    pool = torch.arange(2 * 4 * 4 * 8, device=CUDA, dtype=torch.float32).view(1, 2, 4, 1, 4, 8)
    table, lens = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=CUDA), torch.tensor([11], dtype=torch.int32, device=CUDA)      # tokens at 3 to 10
    want = pool.clone()
    for to, fro in ((5, 6), (6, 7)):                                        # 3 and 4 close up behind 0 and 1
        want[:, :, table[0, to // 4], :, to % 4] = pool[:, :, table[0, fro // 4], :, fro % 4]
    got = ops.accept_tree(picks, tokens, parents, pool, table, lens, cu_q=torch.tensor([0, 8], dtype=torch.int32, device=CUDA), max_q_len=5)
    assert got.path.tolist() == [[0, 1, 3, 4, -1]] and got.counts.tolist() == [4] and got.next_tokens.tolist() == [5] and got.kv_lens.tolist() == [7]
    assert torch.equal(pool, want)


# ---- alignment ----------------------------------------------------------------------------------------------------------------------------------------------
@KINDS
@pytest.mark.parametrize("D,Dv,bs", [(128, 128, 16), (256, 64, 16), (36, 20, 5), (33, 20, 16)])
@pytest.mark.parametrize("splits", [1, 2])
def test_queries_and_results_lie_anywhere(kind, D, Dv, bs, splits):
    """Rows that start on 16 bytes or on any number, far apart or side by side: the same results, bit by bit."""
    c = Step([70, 9], [9, 30], D=D, Dv=Dv, bs=bs, kind=kind, seed=85)
    sees, _ = _visible(_trees(c.q_lens, 86), c.max_q)
    whole = _run(c, _pack(sees), 0.1, num_splits=splits)
    c.check(whole, sees, 0.1)
    T, H, q = c.T, c.heads, c.q
    for shift, gap in ((0, 0), (1, 0), (2, 1), (4, 4), (8, 3)):
        room = torch.zeros(shift + T * H * (D + gap) + 8, dtype=kind, device=CUDA)
        c.q = room[shift:shift + T * H * (D + gap)].view(T, H, D + gap)[..., :D]
        c.q.copy_(q)
        to = torch.full((T, H * Dv + gap + 3), 7.0, dtype=kind, device=CUDA)
        got = _run(c, _pack(sees), 0.1, num_splits=splits, out=to[:, gap:gap + H * Dv])
        assert torch.equal(got, whole) and (to[:, :gap] == 7).all() and (to[:, gap + H * Dv:] == 7).all()


# ---- sums of many alike -------------------------------------------------------------------------------------------------------------------------------------
@KINDS
@pytest.mark.parametrize("apart", [1e-8, -1e-8])
def test_sums_of_many_logits_that_are_alike(kind, apart):
    """Two beams a prompt: all logits of one are c, all of the other 0, so that every continuation has -log V. Of as many rows as fill the SMs a thread adds up hundreds of
    equal exponentials, whose roundings all go one way: the better beam is first nevertheless. (A sum is off by 2^-28.5 of itself at most, 3e-9, however many it is of.)"""
    B, V, count = 300, 128256, 7
    c = (torch.randn(B, device=CUDA, generator=_gen(98)) * 3).to(kind)
    logits = torch.zeros(B, 2, V, device=CUDA, dtype=kind)
    logits[:, 0] = c[:, None]
    scores = torch.tensor([[apart, 0.0]], device=CUDA).expand(B, 2).contiguous()
    got = _ops().beam_select(logits.view(2 * B, V), scores, count=count)
    better = 0 if apart > 0 else 1
    wrong = (got.beams != better).any(1).nonzero()[:, 0].tolist()
    assert not wrong, (len(wrong), c[wrong[0]].item())
    assert (got.tokens == torch.arange(count, device=CUDA)).all()
    assert ((got.scores.double() - (float(scores[0, better]) - math.log(V))).abs() <= 2.0 ** -24 * 12 + 2.0 ** -28.5).all()

