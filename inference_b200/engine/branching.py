"""Generation loops that carry several continuations of a sequence: beam search, and speculation over trees of drafts.

Both run on any `DecodeBackend` with `reorder` and `step_trees`. On the GPU a beam step picks its continuations with `ops.beam_select` and parts pages with one `ops.copy_pages`; a tree is verified in one forward
with `ops.tree_attention`, and `ops.accept_tree` closes the accepted entries up. Law kept: greedy tree speculation gives the model's own largest logit at each place, sampled one draws each token from the
model's own distribution, whatever was drafted. On the oracle these are the tokens of plain decoding; in bf16 a tree's step and a decode step are different kernels, so that logits within its
rounding of one another may change places, as they may between a chain's verification and decoding. Routed experts, which such a change may switch, widen that.

Each loop serves one prompt: a beam step is a `beam_select` of one prompt, a tree step one tree. Trees of several sequences in one step are `step_trees`, several prompts' beams `ops.beam_select`."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ..contracts.core_llm.output import FinishReason
from ..contracts.errors import Unsupported
from ..policy import sampler as hs
from ..policy.speculative import NgramIndex
from .backend import DecodeBackend
from .decode import GenerationConfig, GenerationResult, SpeculativeStats, TokenSink, _pick

MAX_BEAMS, MAX_CONTINUATIONS = 64, 128


@dataclass
class BeamConfig:
    """length_penalty: a finished text's score is its tokens' summed log probability, the stop token's too, over (their number without it) ** length_penalty. early_stopping: the search ends with as many finished texts as beams."""
    beams: int = 4
    length_penalty: float = 1.0
    early_stopping: bool = False


@dataclass
class BeamResult:
    tokens: list[int]
    score: float
    finish_reason: FinishReason


def best_continuations(logits: torch.Tensor, scores: torch.Tensor, count: int) -> list[tuple[float, int, int]]:
    """(score, beam, token) of the best continuations of one prompt's beams, best first: logits [K, V], scores fp32 [K]. See `ops.beam_select`."""
    if logits.is_cuda:
        from .. import ops

        got = ops.beam_select(logits, scores[None], count=count)
        # scores and numbers to the host in one piece: 32-bit numbers and tokens are exact in 64 bits
        rows = torch.stack([got.scores[0].double(), got.beams[0].double(), got.tokens[0].double()]).tolist()
        return [(s, int(b), int(t)) for s, b, t in zip(*rows) if b >= 0]
    s = scores.double()[:, None] + torch.log_softmax(logits.double(), -1)
    s = torch.where(s.isfinite(), s, -math.inf).flatten()      # of a beam that is not alive, or whose logits are no distribution: nothing
    order = torch.sort(s, descending=True, stable=True).indices[:count].tolist()
    return [(float(s[i]), i // logits.shape[1], i % logits.shape[1]) for i in order if s[i] > -math.inf]


def generate_beam(backend: DecodeBackend, prompt: list[int], cfg: GenerationConfig, beam: BeamConfig | None = None) -> list[BeamResult]:
    """Beam search: the `beams` best texts that it finds, best first. cfg gives max_new_tokens, stop_tokens and cancel; sampling is not looked at."""
    beam = beam or BeamConfig()
    K, stops = beam.beams, set(cfg.stop_tokens)
    if not 1 <= K <= MAX_BEAMS:
        raise Unsupported(f"1 to {MAX_BEAMS} beams")
    # as many as there may be texts that end, and K that do not (many beams with many stop tokens: as many as there is room for, so that fewer may go on)
    count = min(MAX_CONTINUATIONS, K * (1 + len(stops)))
    done: list[BeamResult] = []
    seqs, texts, scores, why = [backend.new_sequence()], [[]], [0.0], FinishReason.LENGTH

    def rate(score: float, length: int) -> float:
        return score / max(length, 1) ** beam.length_penalty

    def ranked(results: list[BeamResult]) -> list[BeamResult]:
        return sorted(results, key=lambda r: -r.score)[:K]

    try:
        if cfg.max_new_tokens <= 0:
            return [BeamResult([], 0.0, FinishReason.LENGTH)]
        new = [list(prompt)]
        while True:
            if cfg.cancel is not None and cfg.cancel.is_cancelled():
                why = FinishReason.CANCELLED
                break
            rows = backend.forward(seqs, new)
            logits = torch.stack(list(rows)) if len(rows) > 1 else rows[0][None]
            best = best_continuations(logits, torch.tensor(scores, dtype=torch.float32).to(logits.device), count)
            live = []
            for rank, (score, b, token) in enumerate(best):
                if token in stops:
                    if rank < K:
                        done.append(BeamResult(texts[b], rate(score, len(texts[b])), FinishReason.STOP))
                elif len(live) < K:
                    live.append((score, b, token))
            done = ranked(done)
            if not live:
                texts, scores = [], []
                break
            parents = [b for _, b, _ in live]
            texts, scores = [texts[b] + [t] for _, b, t in live], [s for s, _, _ in live]
            if len(texts[0]) >= cfg.max_new_tokens:
                break
            if len(done) >= K and (beam.early_stopping or done[-1].score >= max(rate(scores[0], len(texts[0])), rate(scores[0], cfg.max_new_tokens))):
                texts, scores = [], []
                break
            seqs = backend.reorder(seqs, parents)
            new = [[t] for _, _, t in live]
        return ranked(done + [BeamResult(t, rate(s, len(t)), why) for t, s in zip(texts, scores)])
    finally:
        for s in seqs:
            backend.release(s)


@dataclass
class TreeConfig:
    """Trees of prompt lookup: up to `branches` continuations of up to `depth` tokens, found behind repeated runs of up to max_ngram tokens."""
    max_ngram: int = 3
    branches: int = 4
    depth: int = 8


def generate_tree_lookup(target: DecodeBackend, prompt: list[int], cfg: GenerationConfig, spec: TreeConfig | None = None, sink: TokenSink | None = None
                         ) -> tuple[GenerationResult, SpeculativeStats]:
    """Speculation without a draft model, over several continuations at once: each step verifies a tree of what followed the text's last tokens before."""
    spec = spec or TreeConfig()
    stats, rng, sp = SpeculativeStats(), hs.SplitMix64(cfg.seed), cfg.sampling
    seq, out, why = target.new_sequence(), [], FinishReason.LENGTH
    index = NgramIndex(prompt, spec.max_ngram)

    def choose(tokens: list[int], parents: list[int]):
        def run(logits: torch.Tensor) -> torch.Tensor:
            if sp.is_plain_greedy():
                if logits.is_cuda:
                    from .. import ops

                    return ops.argmax(logits)
                return torch.argmax(logits, -1)
            if logits.is_cuda and sp.temperature > 0 and sp.repetition_penalty == 1.0 and cfg.device_sampling is not False:
                from .. import ops

                u = torch.tensor([rng.next_f32() for _ in tokens], dtype=torch.float32).to(logits.device)
                return ops.sample_device(logits, sp.temperature, sp.top_k, sp.top_p, u)
            rows, picks = logits.detach().float().cpu().numpy(), []
            for i in range(len(tokens)):       # each behind its own path
                path, j = [], i
                while j > 0:
                    path.append(tokens[j])
                    j = parents[j]
                picks.append(hs.sample(rows[i], list(prompt) + out + path[::-1], sp, rng, None))
            return torch.tensor(picks, dtype=torch.int64, device=logits.device)
        return run

    def emit(token: int) -> bool:
        """Whether the text goes on behind this token."""
        nonlocal why
        if cfg.cancel is not None and cfg.cancel.is_cancelled():
            why = FinishReason.CANCELLED
            return False
        if token in cfg.stop_tokens:
            why = FinishReason.STOP
            return False
        out.append(token)
        index.append(token)
        if sink is not None and sink(token) is False:
            why = FinishReason.STOP
            return False
        return len(out) < cfg.max_new_tokens

    try:
        if cfg.max_new_tokens <= 0:
            return GenerationResult([], FinishReason.LENGTH, len(prompt)), stats
        if cfg.cancel is not None and cfg.cancel.is_cancelled():
            return GenerationResult([], FinishReason.CANCELLED, len(prompt)), stats
        logits = target.forward([seq], [list(prompt)])[0]
        stats.forwards += 1
        last = _pick(target, logits, list(prompt), cfg, rng, None)
        while emit(last):
            room = cfg.max_new_tokens - len(out)        # a tree takes no more of the cache than the text may
            tokens, parents = (x[:room] for x in index.tree(spec.branches, min(spec.depth, room - 1)))
            (path, last), = target.step_trees([seq], [tokens], [parents], choose(tokens, parents))
            stats.forwards += 1
            stats.proposed += len(tokens) - 1
            stats.accepted += len(path) - 1
            if not all(emit(tokens[i]) for i in path[1:]):
                break
        return GenerationResult(out, why, len(prompt)), stats
    finally:
        target.release(seq)
