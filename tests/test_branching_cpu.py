"""Beam search and tree speculation on the CPU oracle backend, page sharing of beams, and lookup trees."""
import itertools

import pytest
import torch

from inference_b200.contracts.core_llm import CancelFlag, FinishReason
from inference_b200.contracts.errors import Unsupported
from inference_b200.engine.backend import OracleBackend
from inference_b200.engine.branching import BeamConfig, TreeConfig, best_continuations, generate_beam, generate_tree_lookup
from inference_b200.engine.decode import GenerationConfig, generate
from inference_b200.engine.kv_pool import PagedKvPool, PagedSequence, unshare_tails
from inference_b200.models import ModelConfig
from inference_b200.models.oracle import OracleLlama, random_llama_weights
from inference_b200.policy.sampler import SamplingParams
from inference_b200.policy.speculative import ngram_tree


def _model(seed=0, vocab=96, std=0.3):
    cfg = ModelConfig(hidden_size=32, intermediate_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=8, vocab_size=vocab, rope_theta=10000.0, tie_word_embeddings=True)
    return OracleBackend(OracleLlama(cfg, random_llama_weights(cfg, seed=seed, std=std)))


PROMPT = [1, 5, 9, 2, 7, 7, 3]


def _log_probability(be, prompt, text):
    seq, total, feed = be.new_sequence(), 0.0, prompt
    for t in text:
        total += float(torch.log_softmax(be.forward([seq], [feed])[0].double(), -1)[t])
        feed = [t]
    return total


def test_one_beam_is_greedy():
    be = _model()
    got, = generate_beam(be, PROMPT, GenerationConfig(max_new_tokens=9), BeamConfig(beams=1))
    assert got.tokens == generate(be, PROMPT, GenerationConfig(max_new_tokens=9)).tokens and got.finish_reason is FinishReason.LENGTH


def test_beams_that_hold_everything_find_the_best_texts():
    """With as many beams as there are texts of two tokens nothing is lost: the search is exhaustive."""
    be = _model(vocab=6, std=0.8)
    got = generate_beam(be, [1, 2, 3], GenerationConfig(max_new_tokens=3), BeamConfig(beams=36, length_penalty=0.0))
    texts = sorted(((_log_probability(be, [1, 2, 3], t), list(t)) for t in itertools.product(range(6), repeat=3)), reverse=True)[:36]
    assert [g.tokens for g in got] == [t for _, t in texts]
    for g, (score, _) in zip(got, texts):
        assert abs(g.score - score) < 1e-4        # the model's logits are 32-bit numbers, and so are the beams' sums


@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("penalty", [0.0, 1.0])
def test_scores_stops_and_order(early, penalty):
    be = _model(vocab=20, std=0.6)
    stops = (3, 11)
    got = generate_beam(be, PROMPT, GenerationConfig(max_new_tokens=6, stop_tokens=stops), BeamConfig(beams=5, length_penalty=penalty, early_stopping=early))
    assert len(got) == 5 and [g.score for g in got] == sorted((g.score for g in got), reverse=True)
    assert len({tuple(g.tokens) for g in got if g.finish_reason is FinishReason.LENGTH}) == sum(g.finish_reason is FinishReason.LENGTH for g in got)
    for g in got:
        assert not set(g.tokens) & set(stops) and len(g.tokens) <= 6
        endings = [[s] for s in stops] if g.finish_reason is FinishReason.STOP else [[]]
        scores = [_log_probability(be, PROMPT, g.tokens + e) / max(len(g.tokens), 1) ** penalty for e in endings]
        assert min(abs(g.score - s) for s in scores) < 1e-4


def test_beams_refuse_and_cancel():
    be = _model()
    with pytest.raises(Unsupported):
        generate_beam(be, PROMPT, GenerationConfig(), BeamConfig(beams=65))
    flag = CancelFlag()
    flag.cancel()
    assert generate_beam(be, PROMPT, GenerationConfig(max_new_tokens=4, cancel=flag))[0].finish_reason is FinishReason.CANCELLED
    assert generate_beam(be, PROMPT, GenerationConfig(max_new_tokens=0))[0].tokens == []


def test_continuations_in_the_order_of_beam_and_token():
    logits = torch.zeros(2, 4)
    assert [c[1:] for c in best_continuations(logits, torch.zeros(2), 6)] == [(0, 0), (0, 1), (0, 2), (0, 3), (1, 0), (1, 1)]
    assert [c[1] for c in best_continuations(logits, torch.tensor([-float("inf"), 0.0]), 6)] == [1] * 4


# ---- trees ----------------------------------------------------------------------------------------------------------------------------------------------
def test_lookup_trees():
    assert ngram_tree([1, 2, 3], 3, 4, 5) == ([3], [-1])
    # 7 8 came before twice, with other continuations, which share their first token; the latest is found first
    tokens, parents = ngram_tree([7, 8, 1, 2, 9, 7, 8, 1, 3, 9, 7, 8], 2, 4, 3)
    assert tokens == [8, 1, 3, 9, 2, 9] and parents == [-1, 0, 1, 2, 1, 4]
    assert ngram_tree([7, 8, 1, 2, 9, 7, 8, 1, 3, 9, 7, 8], 2, 1, 2) == ([8, 1, 3], [-1, 0, 1])
    assert ngram_tree([5, 5, 5], 2, 3, 0) == ([5], [-1])
    assert ngram_tree([5], 2, 3, 4) == ([5], [-1])


@pytest.mark.parametrize("prompt", [PROMPT, [4, 4, 8, 4, 4, 8, 4, 4], [2, 3, 2, 4, 2, 3, 2, 4, 2], [6]])
@pytest.mark.parametrize("spec", [TreeConfig(), TreeConfig(max_ngram=1, branches=8, depth=3), TreeConfig(branches=1)])
def test_greedy_trees_give_plain_greedy_tokens(prompt, spec):
    be = _model()
    cfg = GenerationConfig(max_new_tokens=17)
    got, stats = generate_tree_lookup(be, prompt, cfg, spec)
    assert got.tokens == generate(be, prompt, cfg).tokens and got.finish_reason is FinishReason.LENGTH
    assert stats.forwards + stats.accepted >= len(got.tokens) and stats.accepted <= stats.proposed


def test_trees_stop_where_plain_decoding_does():
    be = _model()
    plain = generate(be, PROMPT, GenerationConfig(max_new_tokens=20)).tokens
    for stop in set(plain[3:10]):
        cfg = GenerationConfig(max_new_tokens=20, stop_tokens=(stop,))
        got, _ = generate_tree_lookup(be, PROMPT, cfg, TreeConfig(max_ngram=1))
        want = generate(be, PROMPT, cfg)
        assert got.tokens == want.tokens and got.finish_reason is want.finish_reason
    seen = []
    got, _ = generate_tree_lookup(be, PROMPT, GenerationConfig(max_new_tokens=20), sink=lambda t: seen.append(t) or len(seen) < 5)
    assert got.tokens == seen == plain[:5] and got.finish_reason is FinishReason.STOP
    assert generate_tree_lookup(be, PROMPT, GenerationConfig(max_new_tokens=0))[0].tokens == []


def test_penalties_see_each_tokens_own_path():
    be = _model()
    cfg = GenerationConfig(max_new_tokens=14, sampling=SamplingParams(temperature=0.0, repetition_penalty=1.3))
    assert generate_tree_lookup(be, [4, 4, 8, 4, 4, 8, 4, 4], cfg, TreeConfig(max_ngram=2))[0].tokens == generate(be, [4, 4, 8, 4, 4, 8, 4, 4], cfg).tokens


def test_sampled_trees_draw_from_the_models_distribution():
    """The second token's frequencies over many seeds, with a tree that drafts some of them: within five standard deviations of the model's own."""
    be = _model(vocab=8, std=0.8)
    prompt = [1, 2, 1, 3, 1, 2, 1, 3, 1]
    sp = SamplingParams(temperature=1.0)
    counts, n = torch.zeros(8, 8), 1500
    for seed in range(n):
        got, _ = generate_tree_lookup(be, prompt, GenerationConfig(max_new_tokens=2, sampling=sp, seed=seed), TreeConfig(max_ngram=1, branches=4, depth=2))
        counts[got.tokens[0], got.tokens[1]] += 1
    first = torch.softmax(be.forward([be.new_sequence()], [prompt])[0].double(), -1)
    for a in range(8):
        second = torch.softmax(be.forward([be.new_sequence()], [prompt + [a]])[0].double(), -1)
        for b in range(8):
            p = float(first[a] * second[b])
            assert abs(float(counts[a, b]) - n * p) <= 5 * (n * p * (1 - p)) ** 0.5 + 1, (a, b, float(counts[a, b]), n * p)


# ---- pages of beams ---------------------------------------------------------------------------------------------------------------------------------------
def test_forks_share_pages_until_they_write():
    pool = PagedKvPool(2, 12, 2, 8, 4, device="cpu", dtype=torch.float32)
    a = PagedSequence(pool)
    a.reserve(10)
    pool.data.copy_(torch.randn(pool.data.shape))
    b, c = a.fork(), a.fork()
    assert a.blocks == b.blocks == c.blocks and pool.allocator.live_blocks() == 3
    unshare_tails([a, b, c])
    assert len({s.blocks[2] for s in (a, b, c)}) == 3 and a.blocks[:2] == b.blocks[:2] == c.blocks[:2] and pool.allocator.live_blocks() == 5
    for s in (b, c):
        assert torch.equal(pool.data[:, :, s.blocks[2]], pool.data[:, :, a.blocks[2]])
    before = pool.allocator.live_blocks()
    unshare_tails([a, b, c])
    assert pool.allocator.live_blocks() == before
    b.reserve(2)                # the page is full then: the next one is b's own
    unshare_tails([b])
    assert pool.allocator.live_blocks() == before
    for s in (a, b, c):
        s.release()
    assert pool.allocator.live_blocks() == 0
