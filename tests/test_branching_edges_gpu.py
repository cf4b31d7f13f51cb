"""Drafted trees, beams and page copies through the engine on the GPU, where their calls are easily missed."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_page_that_is_copied_to_itself_stays():
    from inference_b200.engine.kv_pool import KvGeometry, LayeredKvPool, PagedKvPool

    pool = PagedKvPool(2, 5, 1, 64, 16)
    pool.data.copy_(torch.randn(pool.data.shape))
    want = pool.data.clone()
    pool.copy_block(3, 3)
    assert torch.equal(pool.data, want)
    pool.copy_blocks([1, 2, 1], [1, 4, 0])
    want[:, :, [4, 0]] = want[:, :, [2, 1]]
    assert torch.equal(pool.data, want)
    layered = LayeredKvPool([KvGeometry(1, 8, 8)], 3, 16)
    layered.copy_block(1, 1)
    layered.copy_state(0, 1)        # it keeps none


def test_two_beam_searches_whose_steps_run_back_to_back():
    """Two clients of a batching proxy with as many beams each, one group behind the other: each has the texts and scores that it has by itself."""
    import threading

    from test_branching_gpu import _build, _cfg

    from inference_b200.engine.batching import BatchingBackend
    from inference_b200.engine.branching import BeamConfig, generate_beam
    from inference_b200.engine.decode import GenerationConfig

    _, be = _build(_cfg(), seed=21)
    draw = lambda seed: torch.randint(0, 2048, (19,), generator=torch.Generator().manual_seed(seed)).tolist()
    run = lambda backend, seed: [(r.tokens, r.score) for r in generate_beam(backend, draw(seed), GenerationConfig(max_new_tokens=24), BeamConfig(beams=4))]
    alone = [run(be, seed) for seed in (1, 2)]
    for _ in range(3):
        batch, got, errors, start = BatchingBackend(be, max_batch=1), {}, [], threading.Barrier(2)

        def client(seed):
            try:
                with batch:
                    start.wait(60)
                    got[seed] = run(batch, seed)
            except BaseException as e:
                errors.append(e)

        jobs = [threading.Thread(target=client, args=(seed,)) for seed in (1, 2)]
        for j in jobs:
            j.start()
        for j in jobs:
            j.join(120)
        batch.close()
        assert not errors and [got.get(1), got.get(2)] == alone
    assert be.runner.pool.allocator.live_blocks() == 0


def test_trees_on_a_pool_that_is_sized_for_the_text():
    from test_branching_gpu import _build, _cfg

    from inference_b200.engine.branching import TreeConfig, generate_tree_lookup
    from inference_b200.engine.decode import GenerationConfig, generate

    prompt = [3, 4, 5, 3, 4, 6, 3, 4, 7, 3, 4]
    _, be = _build(_cfg(vocab_size=64), seed=22, blocks=3)       # 11 tokens and 37 new ones, of which the last is not kept
    cfg = GenerationConfig(max_new_tokens=38)
    assert len(generate(be, prompt, cfg).tokens) == 38
    got, stats = generate_tree_lookup(be, prompt, cfg, TreeConfig(branches=8, depth=8))
    assert len(got.tokens) == 38 and stats.proposed > 0
    assert be.runner.pool.allocator.live_blocks() == 0


def test_a_client_chooses_while_another_ones_step_is_recorded(monkeypatch):
    """Steps of a new size are recorded by the proxy's worker; clients of others choose their beams meanwhile, take memory and wait for their results."""
    import threading

    from test_branching_gpu import _build, _cfg

    from inference_b200.engine.branching import best_continuations

    _, be = _build(_cfg(), seed=23)
    begun, chosen, errors, rows, plain = threading.Event(), threading.Event(), [], {}, be.runner.model.logits
    logits = torch.randn(5, 70001, device="cuda")
    want = best_continuations(logits, torch.zeros(5, device="cuda"), 10)

    def waits(hidden):
        got = plain(hidden)
        if torch.cuda.is_current_stream_capturing():
            begun.set()
            chosen.wait(60)
        return got

    monkeypatch.setattr(be.runner.model, "logits", waits)
    first, again = be.new_sequence(), be.new_sequence()
    be.forward([first, again], [[1, 2, 3], [1, 2, 3]])

    def record():
        try:
            rows["recorded"] = be.forward([first], [[7]])[0].clone()
            torch.cuda.synchronize()
        except BaseException as e:
            errors.append(e)
            begun.set()

    job = threading.Thread(target=record)
    job.start()
    try:
        assert begun.wait(60)
        room = torch.empty(1 << 29, dtype=torch.uint8, device="cuda")       # more than the allocator has at hand
        got = best_continuations(logits.clone(), torch.zeros(5, device="cuda"), 10)
    finally:
        chosen.set()
        job.join(60)
    assert not errors and got == want and room.numel() == 1 << 29
    assert torch.equal(rows["recorded"], be.forward([again], [[7]])[0])


MOE = dict(model_type="qwen2_moe", num_experts=8, num_experts_per_tok=2, moe_intermediate_size=256, shared_expert_intermediate_size=256)


@pytest.mark.parametrize("sizes", [[1], [5, 9, 1], [70, 33, 130]], ids=str)
@pytest.mark.parametrize("kw,fmt", [({}, None), ({}, "Q8_0"), (MOE, None)], ids=["dense", "packed", "experts"])
def test_chains_as_trees_have_the_logits_of_chains(kw, fmt, sizes):
    """Steps of up to 64 tokens and of more, dense, packed and routed weights: the tree of a chain against the step that verifies it, on one model. A second one, whose tokens part behind the
    third, against chains of its paths. (Not of many tokens on routed experts: of those one or two go to another expert in another batch, chains too.)"""
    from test_branching_gpu import _build, _cfg, _near

    if kw and max(sizes) > 64:
        sizes = sizes[1:2]
    _, be = _build(_cfg(vocab_size=1024, **kw), seed=24)
    if fmt:
        be.runner.model.quantize_(fmt)
    g = torch.Generator().manual_seed(len(sizes))
    draw = lambda n: torch.randint(0, 1024, (n,), generator=g).tolist()
    prompts, drafts = [draw(11 + 9 * i) for i in range(len(sizes))], [draw(n) for n in sizes]
    seqs, chains = [be.new_sequence() for _ in sizes], [be.new_sequence() for _ in sizes]
    be.forward(seqs + chains, prompts + prompts)
    want, got = torch.cat(be.forward(chains, drafts, all_positions=True)), {}

    def choose(logits):
        got["rows"] = logits.clone()
        return torch.full((logits.shape[0],), -1, device="cuda")

    assert be.step_trees(seqs, drafts, [list(range(-1, n - 1)) for n in sizes], choose) == [([0], -1)] * len(sizes)
    _near(got["rows"], want)
    for s, prompt in zip(seqs, prompts):
        be.truncate(s, len(prompt))
    parents = [[-1] + [i - 1 if i < 3 else max(2, i - 2) for i in range(1, n)] for n in sizes]       # two chains, token by token by turns
    be.step_trees(seqs, drafts, parents, choose)
    for side in (3, 4):
        at = 0
        for prompt, toks, ups, n in zip(prompts, drafts, parents, sizes):
            path = list(range(min(n, 3))) + list(range(side, n, 2))
            assert all(ups[b] == a for a, b in zip(path, path[1:]))
            seq = be.new_sequence()
            be.forward([seq], [prompt])
            _near(got["rows"][[at + i for i in path]], be.forward([seq], [[toks[i] for i in path]], all_positions=True)[0])
            be.release(seq)
            at += n
    for s in seqs + chains:
        be.release(s)
    assert be.runner.pool.allocator.live_blocks() == 0
