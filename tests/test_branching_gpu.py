"""Drafted trees, beams and page copies through the engine on the GPU, against the 32-bit oracle on the same weights."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg(**kw):
    from inference_b200.models import ModelConfig

    base = dict(hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=128, vocab_size=2048, rms_norm_eps=1e-5,
                rope_theta=10000.0)
    base.update(kw)
    return ModelConfig.from_json(base)


def _build(cfg, seed=0, blocks=256, max_seq_len=512, std=0.05):
    from inference_b200.engine.backend import GpuBackend
    from inference_b200.engine.kv_pool import PagedKvPool
    from inference_b200.engine.runner import ModelRunner
    from inference_b200.models.llama import LlamaGpu
    from inference_b200.models.oracle import OracleLlama, random_llama_weights

    w = {k: v.bfloat16().float() for k, v in random_llama_weights(cfg, seed=seed, std=std).items()}
    oracle = OracleLlama(cfg, w, dtype=torch.float32, device="cuda")
    model = LlamaGpu(cfg, device=torch.device("cuda")).load_state_dict(w)
    pool = PagedKvPool(cfg.num_layers, blocks, model.hkv, cfg.head_dim, 16, device="cuda")
    return oracle, GpuBackend(ModelRunner(model, pool, max_batch=8, max_seq_len=max_seq_len))


def _logits(oracle, tokens):
    return oracle.decode_logits(torch.tensor([tokens], device="cuda"), oracle.make_cache(), 0)[0].float()


def _path(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def _near(got, ref):
    """Of the decoder in bf16, as its prefill and decode steps are held to."""
    err = (got - ref).abs().max().item()
    assert err < 0.08 * max(1.0, ref.abs().max().item()), err


TREES = [[-1, 0, 0, 1, 1, 2, 5, 3], [-1], [-1, 0, 1, 2, 3, 4], [-1, 0, 0, 0, 0, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13]]


@pytest.mark.parametrize("kw", [{}, dict(model_type="gemma2", attn_logit_softcapping=50.0, final_logit_softcapping=30.0, query_pre_attn_scalar=128), dict(model_type="qwen3")])
def test_logits_of_trees_and_steps_behind_them(kw):
    cfg = _cfg(**kw)
    oracle, be = _build(cfg, seed=2)
    g = torch.Generator().manual_seed(5)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
    prompts = [draw(n) for n in (37, 5, 16, 31)]
    seqs = [be.new_sequence() for _ in prompts]
    be.forward(seqs, prompts)
    tokens = [draw(len(p)) for p in TREES]
    rows = {}

    def choose(logits):
        """The model's picks are put in: of each tree the path to its last token."""
        at, picks = 0, []
        for prompt, toks, ups in zip(prompts, tokens, TREES):
            for i in range(len(toks)):
                _near(logits[at + i], _logits(oracle, prompt + [toks[j] for j in _path(ups, i)]))
            goal = _path(ups, len(ups) - 1)
            picks += [toks[goal[goal.index(i) + 1]] if i in goal[:-1] else cfg.vocab_size for i in range(len(toks))]
            at += len(toks)
        rows["n"] = at
        return torch.tensor(picks, dtype=torch.int64, device="cuda")

    got = be.step_trees(seqs, tokens, TREES, choose)
    assert rows["n"] == sum(map(len, TREES))
    texts = []
    for (path, nxt), prompt, toks, ups, s in zip(got, prompts, tokens, TREES, seqs):
        want = _path(ups, len(ups) - 1)
        # an earlier child with the same token is taken first; tokens are drawn from 2048, so that none is
        assert path == want and nxt == cfg.vocab_size and s.length == len(prompt) + len(path)
        texts.append(prompt + [toks[j] for j in path])
    # what the cache holds now is what a decode step and another tree see
    feed = draw(len(seqs))
    for lg, text, t in zip(be.forward(seqs, [[t] for t in feed]), texts, feed):
        _near(lg, _logits(oracle, text + [t]))
    texts = [a + [t] for a, t in zip(texts, feed)]
    again = [draw(3) for _ in seqs]

    def last(logits):
        for i, (text, toks) in enumerate(zip(texts, again)):
            for j in range(3):
                _near(logits[3 * i + j], _logits(oracle, text + toks[:1] + ([toks[j]] if j else [])))
        return torch.full((3 * len(seqs),), -5, device="cuda")

    assert be.step_trees(seqs, again, [[-1, 0, 0]] * len(seqs), last) == [([0], -5)] * len(seqs)
    for s, text in zip(seqs, texts):
        assert s.length == len(text) + 1
        be.release(s)
    assert be.runner.pool.allocator.live_blocks() == 0


def test_a_tree_is_a_sequences_first_step():
    cfg = _cfg()
    oracle, be = _build(cfg, seed=12)
    seqs = [be.new_sequence(), be.new_sequence()]
    be.forward([seqs[1]], [[9, 8]])
    tokens, ups = [[5, 6, 7, 6], [4, 3]], [[-1, 0, 0, 2], [-1, 0]]

    def choose(logits):
        for at, front, path in ((0, [], [5]), (1, [], [5, 6]), (2, [], [5, 7]), (3, [], [5, 7, 6]), (4, [9, 8], [4]), (5, [9, 8], [4, 3])):
            _near(logits[at], _logits(oracle, front + path))
        return torch.tensor([7, 0, 6, 2, 1, 1], device="cuda")

    assert be.step_trees(seqs, tokens, ups, choose) == [([0, 2, 3], 2), ([0], 1)]
    for lg, text in zip(be.forward(seqs, [[2], [1]]), ([5, 7, 6, 2], [9, 8, 4, 1])):
        _near(lg, _logits(oracle, text))


def test_tree_lookup_is_greedy():
    from inference_b200.engine.branching import TreeConfig, generate_tree_lookup
    from inference_b200.engine.decode import GenerationConfig

    cfg = _cfg()
    oracle, be = _build(cfg, seed=3)
    prompt = torch.randint(0, cfg.vocab_size, (9,), generator=torch.Generator().manual_seed(0)).tolist() * 3
    got, stats = generate_tree_lookup(be, prompt, GenerationConfig(max_new_tokens=40), TreeConfig())
    assert len(got.tokens) == 40
    for i in range(40):         # each token is the model's own, or one that bf16 cannot tell from it
        ref = _logits(oracle, prompt + got.tokens[:i])
        assert ref[got.tokens[i]] >= ref.max() - 0.08 * max(1.0, ref.abs().max().item())
    assert stats.forwards + stats.accepted >= 40
    assert be.runner.pool.allocator.live_blocks() == 0


def test_sampled_tree_lookup_runs_on_the_device():
    from inference_b200.engine.branching import generate_tree_lookup
    from inference_b200.engine.decode import GenerationConfig
    from inference_b200.policy.sampler import SamplingParams

    cfg = _cfg(vocab_size=64)
    _, be = _build(cfg, seed=4)
    for sp in (SamplingParams(temperature=0.8, top_k=8), SamplingParams(temperature=0.8, repetition_penalty=1.2)):
        got, stats = generate_tree_lookup(be, [1, 2, 3, 1, 2, 3, 1, 2], GenerationConfig(max_new_tokens=30, sampling=sp, seed=7))
        assert len(got.tokens) == 30 and all(0 <= t < 64 for t in got.tokens) and stats.proposed > 0
    assert be.runner.pool.allocator.live_blocks() == 0


@pytest.mark.parametrize("beams", [1, 4, 12])
def test_beams_have_the_scores_of_their_texts(beams):
    from inference_b200.engine.branching import BeamConfig, generate_beam
    from inference_b200.engine.decode import GenerationConfig

    cfg = _cfg()
    oracle, be = _build(cfg, seed=6)
    prompt = torch.randint(0, cfg.vocab_size, (27,), generator=torch.Generator().manual_seed(1)).tolist()
    got = generate_beam(be, prompt, GenerationConfig(max_new_tokens=13, stop_tokens=(5, 9)), BeamConfig(beams=beams))
    assert len(got) == beams and [g.score for g in got] == sorted((g.score for g in got), reverse=True)
    assert be.runner.pool.allocator.live_blocks() == 0
    for r in got:
        if r.finish_reason.name != "LENGTH":
            continue
        total, spread = 0.0, 0.0
        for i, t in enumerate(r.tokens):
            ref = _logits(oracle, prompt + r.tokens[:i])
            total += float(torch.log_softmax(ref.double(), -1)[t])
            spread += 2 * 0.08 * max(1.0, ref.abs().max().item())      # the token's logit and the sum's, each off by what a decode step may be
        assert abs(r.score * len(r.tokens) - total) < spread


def test_a_beams_entries_are_its_own():
    """After each reordering, sequences that share a prefix are decoded with other tokens: each of them sees its own text, and the shared pages stay as they were."""
    cfg = _cfg()
    oracle, be = _build(cfg, seed=8)
    g = torch.Generator().manual_seed(3)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
    prompt = draw(21)
    seqs, texts = [be.new_sequence()], [prompt]
    be.forward(seqs, [prompt])
    for parents in ([0, 0, 0, 0, 0], [4, 1, 1, 0, 4], [2, 2, 2, 2, 2], [3, 0, 3, 1, 1]) * 2:
        seqs = be.reorder(seqs, parents)
        feed = draw(len(parents))
        texts = [texts[p] + [t] for p, t in zip(parents, feed)]
        for lg, text in zip(be.forward(seqs, [[t] for t in feed]), texts):
            _near(lg, _logits(oracle, text))
    for s in seqs:
        be.release(s)
    assert be.runner.pool.allocator.live_blocks() == 0


def test_a_reordering_without_pages_holds_nothing():
    cfg = _cfg()
    _, be = _build(cfg, blocks=4)
    seq = be.new_sequence()
    be.forward([seq], [list(range(20))])
    alloc = be.runner.pool.allocator
    with pytest.raises(Exception):
        be.reorder([seq], [0] * 5)              # four copies of the last page, two pages free
    assert alloc.live_blocks() == 2 and seq.length == 20
    be.release(seq)
    assert alloc.live_blocks() == 0


def test_a_step_of_trees_that_fails_leaves_the_text():
    cfg = _cfg()
    oracle, be = _build(cfg)
    seq = be.new_sequence()
    be.forward([seq], [[3, 4, 5]])

    def fails(logits):
        raise KeyError("no choice")

    with pytest.raises(KeyError):
        be.step_trees([seq], [[1, 2, 3]], [[-1, 0, 0]], fails)
    assert seq.length == 3
    for bad in ([[0, 0, 0]], [[-1, 1, 0]], [[-1, 0]]):
        with pytest.raises(ValueError):
            be.step_trees([seq], [[1, 2, 3]], bad, fails)
    with pytest.raises(ValueError):
        be.step_trees([seq, seq], [[1], [1]], [[-1], [-1]], fails)
    _near(be.forward([seq], [[7]])[0], _logits(oracle, [3, 4, 5, 7]))


def test_two_clients_of_a_batching_backend():
    """A tree's client and a beams' client at once, each with the tokens that it has by itself."""
    import threading

    from inference_b200.engine.batching import BatchingBackend
    from inference_b200.engine.branching import BeamConfig, generate_beam, generate_tree_lookup
    from inference_b200.engine.decode import GenerationConfig

    cfg = _cfg()
    oracle, be = _build(cfg, seed=3)
    prompt = torch.randint(0, cfg.vocab_size, (9,), generator=torch.Generator().manual_seed(0)).tolist() * 3
    batch, out, errors = BatchingBackend(be), {}, []

    def client(name, run):
        try:
            with batch:
                out[name] = run()
        except BaseException as e:
            errors.append(e)

    try:
        jobs = [threading.Thread(target=client, args=("tree", lambda: generate_tree_lookup(batch, prompt, GenerationConfig(max_new_tokens=12))[0].tokens)),
                threading.Thread(target=client, args=("beam", lambda: generate_beam(batch, prompt, GenerationConfig(max_new_tokens=12), BeamConfig(beams=3))))]
        for j in jobs:
            j.start()
        for j in jobs:
            j.join(120)
    finally:
        batch.close()
    assert not errors and len(out["tree"]) == 12 and len(out["beam"]) == 3
    for i, t in enumerate(out["tree"]):
        ref = _logits(oracle, prompt + out["tree"][:i])
        assert ref[t] >= ref.max() - 0.08 * max(1.0, ref.abs().max().item())
    assert be.runner.pool.allocator.live_blocks() == 0


def test_states_and_pages_of_layered_pools_are_copied():
    from inference_b200.engine.kv_pool import KvGeometry, LatentGeometry, LayeredKvPool, StateGeometry, TokenGeometry, WindowGeometry

    pool = LayeredKvPool([KvGeometry(2, 24, 16), StateGeometry((3, 5), (7, 3)), LatentGeometry(40), WindowGeometry((9,)), TokenGeometry()], 9, 8, state_slots=6)
    for kv in pool.data:
        for t in kv:
            t.copy_(torch.randint(-1000, 1000, t.shape, device="cuda"))
    before = [[t.clone() for t in kv] for kv in pool.data]
    pool.copy_blocks([1, 1, 4], [0, 8, 2])
    pool.copy_states([5, 3], [1, 0])
    pool.copy_state(2, 2)
    for kv, old in zip(pool.data, before):
        for t, o in zip(kv, old):
            want = o.clone()
            src, dst = ([1, 1, 4], [0, 8, 2]) if t.shape[0] == 9 else ([5, 3], [1, 0])
            want[dst] = o[src]
            assert torch.equal(t, want)


def test_a_whole_step_captured_into_one_graph():
    """plan, attention, picks, acceptance, page copy and beam selection in one graph, replayed on other contents: the eager run's results each time."""
    from inference_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(11)
    n, q_len, Hk, G, D, bs, V = 3, 12, 2, 4, 64, 16, 500
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 7] * n, dtype=torch.int32, device="cuda")
    cu = torch.arange(0, n * q_len + 1, q_len, dtype=torch.int32, device="cuda")
    table = torch.randperm(24, device="cuda", generator=g).int().view(n, 8)
    kv_lens = torch.tensor([40, 100, 13], dtype=torch.int32, device="cuda")
    head = torch.randn(Hk * G * D, V, device="cuda", generator=g)
    q, pool = torch.empty(n * q_len, Hk * G, D, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 2, 26, Hk, bs, D, dtype=torch.bfloat16, device="cuda")
    tokens, sums = torch.empty(n * q_len, dtype=torch.int64, device="cuda"), torch.empty(n, q_len, device="cuda")
    src, dst = table[:2, 0].contiguous(), torch.tensor([24, 25], dtype=torch.int32, device="cuda")

    def fill(seed):
        g.manual_seed(seed)
        q.copy_(torch.randn(q.shape, device="cuda", generator=g))
        pool.copy_(torch.randn(pool.shape, device="cuda", generator=g))
        tokens.copy_(torch.randint(0, 3, tokens.shape, device="cuda", generator=g))
        sums.copy_(torch.randn(sums.shape, device="cuda", generator=g))

    def run():
        plan = ops.plan_tree(parents, cu_q=cu, max_q_len=q_len)
        a = ops.tree_attention(q, pool[0, 0], pool[0, 1], table, kv_lens, plan.mask, cu_q=cu, max_q_len=q_len, scale=0.125)
        logits = a.reshape(n * q_len, -1).float() @ head
        picks = ops.argmax(logits) % 3
        acc = ops.accept_tree(picks, tokens, parents, pool, table, kv_lens, cu_q=cu, max_q_len=q_len)
        ops.copy_pages(pool, src, dst)
        best = ops.beam_select(logits, sums, count=8)
        return [a, acc.path, acc.counts, acc.next_tokens, acc.kv_lens, best.scores, best.beams, best.tokens]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fill(0)
        run()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(1, 6):
        fill(seed)
        want, after = [t.clone() for t in run()], pool.clone()
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(pool, after)
    assert not math.isnan(float(out[0].float().sum()))
