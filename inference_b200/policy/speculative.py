"""Speculative-decoding policy: prompt-lookup n-gram proposer, greedy acceptance run, distribution-preserving
stochastic acceptance with residual resampling (core-llm/src/speculative.rs:32-156). RNG-free: uniform draws are
arguments, so the math is testable and the engine owns the random stream."""
from __future__ import annotations

import ctypes

from ._lib import f32_array, i32_array, lib


def ngram_propose(tokens: list[int], max_ngram: int, max_proposal: int) -> list[int]:
    out = (ctypes.c_int32 * max(1, max_proposal))()
    n = lib().swb_ngram_propose(i32_array(tokens), len(tokens), max_ngram, max_proposal, out)
    return list(out[:n])


def accept_greedy_run(target_argmax: list[int], drafts: list[int]) -> int:
    assert len(target_argmax) == len(drafts) + 1, "need a bonus slot past the drafts"
    return lib().swb_accept_greedy_run(i32_array(target_argmax), i32_array(drafts), len(drafts))


def sample_weighted(candidates: list[tuple[int, float]], u: float, fallback: int) -> int:
    ids = i32_array([c[0] for c in candidates])
    w = f32_array([c[1] for c in candidates])
    return lib().swb_sample_weighted(ids, w, len(candidates), u, fallback)


def accept_token(target: list[tuple[int, float]], draft: list[tuple[int, float]], proposed: int, u_accept: float,
                 u_resample: float) -> tuple[bool, int]:
    """Returns (accepted, token): the proposed token when accepted, else the residual resample."""
    tok = ctypes.c_int32()
    ok = lib().swb_accept_token(i32_array([t[0] for t in target]), f32_array([t[1] for t in target]), len(target),
                                i32_array([d[0] for d in draft]), f32_array([d[1] for d in draft]), len(draft),
                                proposed, u_accept, u_resample, ctypes.byref(tok))
    return bool(ok), tok.value


def check_trees(seqs: list, tokens: list[list[int]], parents: list[list[int]]) -> None:
    """A tree for each sequence, each sequence once: its first token the root (parent -1), the others behind their parents."""
    if not len(seqs) == len(tokens) == len(parents) or len({id(s) for s in seqs}) != len(seqs):
        raise ValueError("a tree for each sequence, and each sequence once")
    if any(len(t) != len(p) or not t or p[0] != -1 or any(not 0 <= up < j for j, up in enumerate(p) if j) for t, p in zip(tokens, parents)):
        raise ValueError("a tree has a root and tokens that hang on tokens in front of them")


class NgramIndex:
    """What followed each run of up to max_ngram tokens of a text, kept up as the text grows: a draft takes as long as there are matches, however long the text is."""

    def __init__(self, tokens: list[int], max_ngram: int):
        self.tokens: list[int] = []
        self._behind: list[dict[tuple[int, ...], list[int]]] = [{} for _ in range(max(max_ngram, 0))]      # of n + 1 tokens: places behind the run, ascending
        for t in tokens:
            self.append(t)

    def append(self, token: int) -> None:
        at = len(self.tokens)
        for n, behind in enumerate(self._behind[:at], 1):
            behind.setdefault(tuple(self.tokens[at - n:]), []).append(at)
        self.tokens.append(token)

    def tree(self, branches: int, depth: int) -> tuple[list[int], list[int]]:
        """Prompt lookup with several answers: what followed the earlier occurrences of the longest repeated run that ends the text (shorter runs while there is room), the latest first, up
        to `branches` different continuations of up to `depth` tokens, as one tree. Returns its tokens, the text's last one first, and each one's parent (-1 of the root)."""
        out, parents, children = [self.tokens[-1]], [-1], {}
        found, seen = 0, set()
        for n in range(min(len(self._behind), len(self.tokens) - 1), 0, -1):
            for at in reversed(self._behind[n - 1].get(tuple(self.tokens[-n:]), ())):
                if found >= branches or depth < 1:
                    return out, parents
                follow = tuple(self.tokens[at:at + depth])
                if follow in seen:
                    continue
                seen.add(follow)
                found += 1
                node = 0
                for t in follow:
                    if (node, t) not in children:
                        children[node, t] = len(out)
                        out.append(t)
                        parents.append(node)
                    node = children[node, t]
        return out, parents


def ngram_tree(tokens: list[int], max_ngram: int, branches: int, depth: int) -> tuple[list[int], list[int]]:
    """The tree of one text; see `NgramIndex.tree`. (A text that grows is better kept in an index: this one is made anew.)"""
    return NgramIndex(tokens, max_ngram).tree(branches, depth)
