"""Loops that carry several continuations, and the pools and proxies below them, where their calls are easily missed."""
import contextlib
import math
import random
import threading

import pytest
import torch

from inference_b200.contracts.core_llm import CancelFlag, FinishReason
from inference_b200.engine.backend import GpuBackend, OracleBackend
from inference_b200.engine.batching import BatchingBackend
from inference_b200.engine.branching import TreeConfig, best_continuations, generate_tree_lookup
from inference_b200.engine.decode import GenerationConfig, generate
from inference_b200.engine.kv_pool import KvGeometry, LayeredKvPool, PagedKvPool, PagedSequence, StateGeometry, copy_entries
from inference_b200.models import ModelConfig
from inference_b200.models.oracle import OracleLlama, random_llama_weights
from inference_b200.policy.speculative import NgramIndex, ngram_tree


def _oracle(seed=0, vocab=96, std=0.3):
    cfg = ModelConfig(hidden_size=32, intermediate_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=8, vocab_size=vocab, rope_theta=10000.0, tie_word_embeddings=True)
    return OracleBackend(OracleLlama(cfg, random_llama_weights(cfg, seed=seed, std=std)))


class _OneBuffer:
    """A backend whose steps write their logits into one buffer, as replays of a graph do."""
    max_context = 100

    def __init__(self):
        self.buffer = torch.zeros(4, 6)

    def forward(self, seqs, new_tokens, all_positions=False):
        for i, toks in enumerate(new_tokens):
            self.buffer[i] = float(toks[-1])
        return [self.buffer[i] for i in range(len(seqs))]


def test_a_clients_logits_outlive_the_steps_of_others():
    """Steps of two clients, one behind the other: what the first was handed is still its own when the second has run."""
    batch, got = BatchingBackend(_OneBuffer(), max_batch=1), {}

    def client(name, tokens):
        with batch:
            got[name] = batch.forward([name] * len(tokens), [[t] for t in tokens])

    try:
        for name, tokens in (("a", [3, 4]), ("b", [5, 6, 7]), ("c", [8])):
            job = threading.Thread(target=client, args=(name, tokens))
            job.start()
            job.join(60)
    finally:
        batch.close()
    for name, tokens in (("a", [3, 4]), ("b", [5, 6, 7]), ("c", [8])):
        assert [row.tolist() for row in got[name]] == [[float(t)] * 6 for t in tokens]


# ---- copies in pools ----------------------------------------------------------------------------------------------------------------------------------------
@pytest.fixture
def on_a_device(monkeypatch):
    """Copies as they are on the GPU: `ops.copy_pages` with its checks, its launch put in by elementary operations."""
    from inference_b200 import ops
    from inference_b200.ops import branch

    class Device:
        type = "cuda"

    class OnDevice(torch.Tensor):
        device = Device()

    def launch(pages, src, dst):
        _, _, _, _, _, blocks, held = branch._tensors(pages)
        assert min(*src, *dst) >= 0 and max(*src, *dst) < blocks and len(set(dst)) == len(dst) and not set(dst) & set(src)
        for t in held:
            t = t.flatten(0, 1) if isinstance(pages, torch.Tensor) else t[None]
            for a, b in zip(src, dst):
                t[:, b] = t[:, a].clone()

    monkeypatch.setattr(ops, "copy_pages", launch)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return lambda t: t.as_subclass(OnDevice)


def test_a_page_that_is_copied_to_itself_stays(on_a_device):
    pool = PagedKvPool(2, 5, 1, 4, 2, device="cpu", dtype=torch.float32)
    pool.data.copy_(torch.randn(pool.data.shape))
    want = pool.data.clone()
    pool.data = on_a_device(pool.data)
    pool.copy_block(3, 3)
    assert (torch.Tensor(pool.data) == want).all()
    pool.copy_blocks([1, 2, 1], [1, 4, 0])
    want[:, :, 4], want[:, :, 0] = want[:, :, 2].clone(), want[:, :, 1].clone()
    assert (torch.Tensor(pool.data) == want).all()


def test_pools_that_keep_no_states_or_no_pages():
    pages = LayeredKvPool([KvGeometry(1, 4, 4)], 3, 2, device="cpu", dtype=torch.float32)
    pages.copy_state(0, 1)
    states = LayeredKvPool([StateGeometry((2,), (3,))], 3, 2, device="cpu", dtype=torch.float32, state_slots=2)
    states.copy_block(0, 1)
    with pytest.raises(ValueError):
        copy_entries(pages.data[0], [0, 1], [2])


# ---- reorderings --------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("parents", [[-1], [0, -2], [2], [1, 0, 7]], ids=str)
def test_reorderings_by_numbers_of_no_sequence_touch_nothing(parents):
    oracle = _oracle()
    seqs = [oracle.new_sequence(), oracle.new_sequence()]
    oracle.forward(seqs, [[1, 2, 3], [4]])
    with pytest.raises(ValueError):
        oracle.reorder(seqs, parents)
    assert [oracle.length(s) for s in seqs] == [3, 1]
    pool = PagedKvPool(1, 9, 1, 4, 4, device="cpu", dtype=torch.float32)
    paged = GpuBackend.__new__(GpuBackend)
    paged.runner = type("Runner", (), {"pool": pool})()
    seqs = [PagedSequence(pool), PagedSequence(pool)]
    seqs[0].reserve(6)
    seqs[1].reserve(3)
    with pytest.raises(ValueError):
        paged.reorder(seqs, parents)
    assert [s.length for s in seqs] == [6, 3] and pool.allocator.live_blocks() == 3
    a, b, c = paged.reorder(seqs, [0, 0, 0])
    assert a is seqs[0] and (a.length, b.length, c.length) == (6, 6, 6) and seqs[1].length == 0 and pool.allocator.live_blocks() == 4


# ---- trees --------------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,parents", [([[1, 2]], [[0, 0]]), ([[1, 2]], [[-1, 1]]), ([[1, 2, 3]], [[-1, 2, 0]]), ([[1, 2]], [[-1]]), ([[]], [[]]), ([[1], [2]], [[-1], [-1]]), ([], [])], ids=str)
def test_trees_that_are_none_are_refused_on_the_oracle_too(tokens, parents):
    be = _oracle()
    seq = be.new_sequence()
    be.forward([seq], [[1, 2, 3]])
    with pytest.raises(ValueError):
        be.step_trees([seq], tokens, parents, lambda logits: torch.argmax(logits, -1))
    assert be.length(seq) == 3
    with pytest.raises(ValueError):
        be.step_trees([seq, seq], [[1], [1]], [[-1], [-1]], lambda logits: torch.argmax(logits, -1))


class _Full(OracleBackend):
    """A cache with room for so many tokens."""
    room = 0

    def forward(self, seqs, new_tokens, all_positions=False):
        assert all(self.length(s) + len(t) <= self.room for s, t in zip(seqs, new_tokens)), "no room"
        return super().forward(seqs, new_tokens, all_positions)

    def step_trees(self, seqs, tokens, parents, choose):
        assert all(self.length(s) + len(t) <= self.room for s, t in zip(seqs, tokens)), "no room"
        return super().step_trees(seqs, tokens, parents, choose)


@pytest.mark.parametrize("prompt", [[4, 4, 8, 4, 4, 8, 4, 4], [2, 3, 2, 4, 2, 3, 2, 4, 2]])
@pytest.mark.parametrize("new", [1, 2, 5, 13])
def test_trees_need_no_more_room_than_plain_decoding(prompt, new):
    be = _Full(_oracle().model)
    be.room = len(prompt) + new - 1
    cfg = GenerationConfig(max_new_tokens=new)
    assert generate_tree_lookup(be, prompt, cfg, TreeConfig(max_ngram=2, branches=8, depth=6))[0].tokens == generate(be, prompt, cfg).tokens


# ---- continuations --------------------------------------------------------------------------------------------------------------------------------------------
def test_beams_that_offer_nothing_on_the_host():
    """As `ops.beam_select` has it: scores that are not finite, logits with NaN or +inf, tokens that are not allowed."""
    logits = torch.zeros(6, 3)
    logits[3, 1], logits[4, 0], logits[5, :2] = math.nan, math.inf, -math.inf
    got = best_continuations(logits, torch.tensor([math.inf, -math.inf, math.nan, 0.0, 0.0, -1.0]), 20)
    assert got == [(-1.0, 5, 2)]


# ---- drafts -------------------------------------------------------------------------------------------------------------------------------------------------
def _scanned(tokens, max_ngram, branches, depth):
    """The definition, by going through the text: the continuations of the longest repeated runs that end it, the latest first, as one tree."""
    paths = []
    for n in range(min(max_ngram, len(tokens) - 1), 0, -1):
        for at in range(len(tokens) - n - 1, -1, -1):
            if len(paths) < branches and depth > 0 and tokens[at:at + n] == tokens[-n:] and tokens[at + n:at + n + depth] not in paths:
                paths.append(tokens[at + n:at + n + depth])
    nodes = [()]
    for p in paths:
        nodes += [tuple(p[:i]) for i in range(1, len(p) + 1) if tuple(p[:i]) not in nodes]
    return [n[-1] if n else tokens[-1] for n in nodes], [nodes.index(n[:-1]) if n else -1 for n in nodes]


@pytest.mark.parametrize("vocab", [1, 3, 40])
@pytest.mark.parametrize("max_ngram,branches,depth", [(3, 4, 8), (1, 8, 3), (2, 1, 1), (5, 3, 2), (0, 4, 4), (3, 0, 4)])
def test_an_index_that_grows_drafts_what_the_whole_text_offers(vocab, max_ngram, branches, depth):
    rng = random.Random(vocab)
    text = [rng.randrange(vocab) for _ in range(5)]
    index = NgramIndex(text, max_ngram)
    for _ in range(60):
        text.append(rng.randrange(vocab))
        index.append(text[-1])
        assert index.tree(branches, depth) == _scanned(text, max_ngram, branches, depth) == ngram_tree(text, max_ngram, branches, depth)


def test_a_draft_does_not_go_through_the_text():
    """Of a long text only the matches are looked at: 200 000 tokens in which the last one stood before once."""
    class Watched(list):
        read = 0

        def __getitem__(self, i):
            Watched.read += 1 if isinstance(i, int) else len(range(*i.indices(len(self))))
            return super().__getitem__(i)

    index = NgramIndex(list(range(200000)), 3)
    index.tokens = Watched(index.tokens)
    index.append(77)
    Watched.read = 0
    assert index.tree(4, 5) == ([77, 78, 79, 80, 81, 82], [-1, 0, 1, 2, 3, 4])
    assert Watched.read < 20


@pytest.mark.parametrize("after", [0, 1, 3, 6])
@pytest.mark.parametrize("prompt", [[4, 4, 8, 4, 4, 8, 4, 4], [2, 3, 2, 4, 2, 3, 2, 4, 2]])
def test_a_cancelled_text_ends_where_plain_decoding_ends_it(prompt, after):
    """No token behind the one at which it was cancelled, drafted and accepted ones neither."""
    def run(loop):
        flag, seen = CancelFlag(), []
        if after == 0:
            flag.cancel()

        def sink(token):
            seen.append(token)
            if len(seen) == after:
                flag.cancel()
            return True

        got = loop(_oracle(vocab=12), prompt, GenerationConfig(max_new_tokens=12, cancel=flag), sink=sink)
        got = got[0] if isinstance(got, tuple) else got
        assert got.tokens == seen and got.finish_reason is FinishReason.CANCELLED
        return seen

    assert run(generate_tree_lookup) == run(generate) and len(run(generate_tree_lookup)) == after
