"""Decoding with several continuations at once (csrc/kernels/attention_tree.cu, branch_ops.cu, beam_select.cu).

  a tree of drafts   `plan_tree` makes of its parents what each token sees, `tree_attention` reads the cache once for all of its tokens, `accept_tree` finds the path that the model
                     agrees with and closes its cache entries up
  beams              `beam_select` picks the best continuations, `copy_pages` gives beams that part pages of their own

Steps are described as in `paged_attention`: kv_lens int32 [num_seqs] counts a sequence's tokens with the new ones, cu_q int32 [num_seqs + 1] are the new tokens' ranges within the rows of the
step and max_q_len bounds a sequence's number (None: every sequence has max_q_len of them). Rows in front of the first range and behind the last are left as they were. Of a sequence that
has more than max_q_len of them the first max_q_len are computed, and may be accepted, where they lie among all of them; the rows behind these are left too. Lengths beyond a table's pages
count as the table's end, which lies in front of 2^31 - 1024 tokens; pages whose number is not in the cache are passed over.

Caches are bf16 or fp32, widths up to 256; the caches of all layers together are a pool's tensor [layers, 2, blocks, kv heads, block_size, width] or a list of tensors [blocks, ...]. Calls
run on the current stream, take no host reads and can be captured into graphs. Scores, the softmax and all sums are 32-bit numbers, those of `beam_select` 64-bit ones."""
from __future__ import annotations

import math
import struct
from dataclasses import dataclass

import torch

from .._native import kernels
from .budget import _check_cache, _check_rows, _check_step, _place, _require
from .runtime import check, ptr

MAX_SPLITS, MAX_PATH = 64, 8192
MAX_TOKENS = 2 ** 31 - 1025       # of a sequence in a table: places behind its end, up to 1024 of them, are whole numbers of 32 bits too
MAX_BEAMS, MAX_COUNT = 256, 128

_ONE = struct.Struct("q").pack
_DIMS = {n: struct.Struct(f"{n}i").pack for n in (8, 16)}
_STRIDES = struct.Struct("8q").pack


@dataclass
class TreePlan:
    """mask int32 [T, words]: bit j % 32 of word j / 32 says that the token sees its sequence's new token j. depths int32 [T]: tokens of the tree in front of it on its path."""
    mask: torch.Tensor
    depths: torch.Tensor


def plan_tree(parents: torch.Tensor, *, cu_q: torch.Tensor | None, max_q_len: int) -> TreePlan:
    """What the tokens of drafted trees see: themselves, and their parents up to the root. parents int32 [T]: the place of a token's parent among its sequence's new tokens, in front
    of its own; -1, or any other number: it continues the cache itself. A position is that of the first new token plus the depth. Once a step, for all of its layers."""
    stream = _place(parents, cu_q)
    _require(parents.dim() == 1 and parents.dtype == torch.int32 and parents.is_contiguous(), "parents are int32 [T]")
    T = parents.shape[0]
    n = _check_ranges(cu_q, max_q_len, T)
    most = max(1, min(max_q_len, T))               # no sequence has more tokens than the step, however loose the bound is
    words = (most + 31) // 32
    mask, depths = parents.new_zeros((T, words)), parents.new_zeros(T)
    check(kernels().swb_plan_tree(parents.data_ptr(), ptr(cu_q), n, most, T, words, mask.data_ptr(), depths.data_ptr(), stream), "swb_plan_tree")
    return TreePlan(mask, depths)


def _check_ranges(cu_q: torch.Tensor | None, max_q_len: int, tokens: int) -> int:
    """Sequences of a step that is described by its tokens' ranges alone."""
    _require(1 <= max_q_len < 2 ** 31, "1 <= max_q_len < 2^31")
    if cu_q is None:
        _require(tokens % max_q_len == 0, "without cu_q every sequence has max_q_len tokens")
        return tokens // max_q_len
    _require(cu_q.dim() == 1 and cu_q.shape[0] >= 1 and cu_q.dtype == torch.int32 and cu_q.is_contiguous(), "cu_q is int32 [num_seqs + 1]")
    return cu_q.shape[0] - 1


def tree_splits(problems: int, keys: int, tensor_cores: bool = True, sms: int = 148) -> int:
    """Blocks that share the keys of a tile of rows, of a tile of keys and more each.

    On tensor memory no more than all SMs hold at once, one each: beyond that a block's start and the sum of the parts cost more than the last wave's idle SMs (30 tokens x 32 heads, 4100 keys, us:
    4 sequences 33.0, 30.0 and 39.2 with 3, 4 and 6 splits, 8 sequences 58.2, 42.7 and 53.7 with 1, 2 and 3; 24 sequences of 48 tokens 109, 122 and 138). The plain kernel waits for its own
    steps and wants several blocks an SM and waves that blend: eight blocks an SM in all (16 heads, us: 8 x 20 tokens, 900 keys 125, 78, 68 and 69 with 2, 4, 6 and 12; 16 x 30 tokens, 2000 keys 589,
    360, 317 and 305 with 1, 2, 4 and 8; 40 x 30 tokens, 900 keys 441, 366 and 337 with 1, 2 and 4; 60 tokens, 20 000 keys 575, 739 and 637 with 12, 18 and 32)."""
    problems = max(1, problems)
    if tensor_cores:
        return max(1, min(MAX_SPLITS, (keys + 127) // 128, sms // problems))
    return max(1, min(MAX_SPLITS, (keys + 63) // 64, -(-8 * sms // problems)))


def tree_attention(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, mask: torch.Tensor, *,
                   cu_q: torch.Tensor | None, max_q_len: int, scale: float, softcap: float = 0.0, num_splits: int | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every new token over all keys in front of the step's tokens and those new tokens whose bit is set in its row of mask -> [T, Hq * Dv] in the type of q.

    q [T, Hq, D] and the caches of one type (token and head strides free); the new tokens' keys and values are in the cache already, in the tokens' order. mask int32 [T, words] as of
    `plan_tree`, or any other: bits of tokens that a row has no word for are not set. softcap > 0: scores s become softcap tanh(s / softcap). A token that sees no key gets zeros;
    what a token does not see adds nothing, infinities and NaN included. With bf16 caches each weight is rounded to bf16 in front of its product with the values, as in
    `paged_attention`; the softmax's sum is not."""
    stream = _place(q, kcache, vcache, block_table, kv_lens, mask, cu_q, out)
    blocks, heads, bs, D, Dv = _check_cache(kcache, vcache)
    T, G, tok, head = _check_rows(q, heads, D)
    n, per = _check_step(block_table, kv_lens, cu_q, max_q_len, T)
    _require(per * bs <= MAX_TOKENS, f"block_table has room for {MAX_TOKENS} tokens at most")
    most = max(1, min(max_q_len, T))
    kind, columns = q.dtype, G * heads * Dv
    _require(kind == kcache.dtype, "queries and cache have one type")
    _require(mask.dim() == 2 and mask.dtype == torch.int32 and mask.shape[0] == T and mask.shape[1] >= 1 and mask.stride(1) == 1, "mask is int32 [T, words], unit inner stride")
    if out is None:
        out = q.new_empty((T, columns))
    else:
        _require(out.shape == (T, columns) and out.dtype == kind and out.stride(1) == 1, "out is [T, heads * value width] in the type of q, unit inner stride")
        _require(out.stride(0) >= columns or T <= 1, "rows of out share memory")
    k_ptr, v_ptr = kcache.data_ptr(), vcache.data_ptr()
    fast = kind is torch.bfloat16 and (D | Dv) % 8 == 0 and D <= 128 and Dv <= 128 and bs % 16 == 0 and scale > 0 and (k_ptr | v_ptr) % 16 == 0 and blocks * heads * bs < 2 ** 31 - 1
    problems = n * heads * -(-most * G // (256 if fast else 32))
    splits = tree_splits(problems, per * bs, fast) if num_splits is None else num_splits
    _require(1 <= splits <= MAX_SPLITS, "1 to 64 splits")
    ws, nbytes = None, 0
    if splits > 1:
        nbytes = 4 * splits * T * G * heads * (Dv + 2) + 16
        ws = q.new_empty(nbytes, dtype=torch.uint8)        # the call's own: two streams or graphs share none
    dims = _DIMS[16](T, n, most, per, blocks, bs, heads, G, D, Dv, mask.shape[1], splits, kind == torch.float32, 0, 0, 0)
    strides = _STRIDES(tok, head, out.stride(0), block_table.stride(0), mask.stride(0), 0, 0, 0)
    check(kernels().swb_attn_tree(dims, strides, q.data_ptr(), out.data_ptr(), k_ptr, v_ptr, block_table.data_ptr(), ptr(cu_q), kv_lens.data_ptr(),
                                  mask.data_ptr(), scale, softcap, ptr(ws), nbytes, stream), "swb_attn_tree")
    return out


def _longs(numbers: list[int]) -> bytes:
    return _ONE(numbers[0]) if len(numbers) == 1 else struct.pack(f"{len(numbers)}q", *numbers)


def _tensors(pages) -> tuple[list[int], list[int], list[tuple], int, int, int, list]:
    """Bases, bytes of a page and shapes of a page, the number of tensors and the bytes between them (0: the lists tell each; else they tell the first), the number of pages, and what
    holds them."""
    if isinstance(pages, torch.Tensor):
        _require(pages.dim() == 6 and pages.is_contiguous(), "a pool's pages are one contiguous tensor [layers, 2, blocks, kv heads, block_size, width]")
        shape, n = pages.shape, pages.shape[0] * pages.shape[1]
        page = math.prod(shape[3:]) * pages.element_size()
        step = shape[2] * page
        return [pages.data_ptr()], [page], [tuple(shape[3:])], n if step else 0, step, shape[2], [pages]
    pages = list(pages)
    _require(all(t.dim() >= 2 and t.is_contiguous() for t in pages) and len({t.shape[0] for t in pages}) <= 1, "pages are contiguous tensors [blocks, ...] of one number of blocks")
    live = [t for t in pages if t.numel()]
    blocks = pages[0].shape[0] if pages else 0
    return [t.data_ptr() for t in live], [t.numel() // blocks * t.element_size() for t in live], [tuple(t.shape[1:]) for t in live], len(live), 0, blocks, pages


@dataclass
class Acceptance:
    """path int32 [num_seqs, width]: the accepted tokens' places within their sequence's new tokens, -1 behind the counts int32 [num_seqs]; next_tokens int64 [num_seqs]: the pick at
    the path's end (-1 of a sequence without new tokens); kv_lens int32 [num_seqs]: cached tokens with the accepted ones."""
    path: torch.Tensor
    counts: torch.Tensor
    next_tokens: torch.Tensor
    kv_lens: torch.Tensor


def accept_tree(picks: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, pages, block_table: torch.Tensor, kv_lens: torch.Tensor, *, cu_q: torch.Tensor | None,
                max_q_len: int) -> Acceptance:
    """The path of each sequence's tree that agrees with the model, whose cache entries move to the places behind the cache in front of the tree, in all of `pages`.

    picks int64 [T]: what the model would have behind each token (the largest logit, or a draw from its distribution: then the tokens that come out are such draws, whatever was drafted).
    tokens int64 [T] and parents int32 [T] as in `plan_tree`: the tree. The first new token is its root and always accepted (it was certain before); then, as long as there is one, the
    first child whose token is its parent's pick. Entries behind the path keep what they held; pages of a tree are its sequence's own. pages: a pool's tensor or a list of
    tensors [blocks, heads, block_size, width], [blocks, block_size, width] or [blocks, block_size]; an empty list moves nothing."""
    bases, sizes, shapes, count, step, blocks, held = _tensors(pages)
    stream = _place(picks, tokens, parents, block_table, kv_lens, cu_q, *held)
    _require(picks.dim() == 1 and picks.dtype == tokens.dtype == torch.int64 and parents.dtype == torch.int32 and picks.shape == tokens.shape == parents.shape
             and picks.is_contiguous() and tokens.is_contiguous() and parents.is_contiguous(), "picks and tokens are int64 [T], parents int32 [T]")
    T = picks.shape[0]
    n, per = _check_step(block_table, kv_lens, cu_q, max_q_len, T)
    _require(max_q_len <= MAX_PATH, f"trees of up to {MAX_PATH} tokens")
    heads = [s[0] if len(s) == 3 else 1 for s in shapes]
    rows = {s[-1] if len(s) == 1 else s[-2] for s in shapes}
    _require(max(map(len, shapes), default=1) <= 3 and len(rows) <= 1, "pages are [blocks, heads, block_size, width], [blocks, block_size, width] or [blocks, block_size], of one block_size")
    _require(len(set(bases)) == len(bases), "the same tensor twice")
    bs = rows.pop() if rows else 1
    got = Acceptance(kv_lens.new_empty((n, max_q_len)), torch.empty_like(kv_lens), picks.new_empty(n), torch.empty_like(kv_lens))
    dims = _DIMS[8](n, max_q_len, T, per, max(blocks, 1), bs, max_q_len, count)
    check(kernels().swb_accept_tree(dims, picks.data_ptr(), tokens.data_ptr(), parents.data_ptr(), _longs(bases), _longs(sizes),
                                    struct.pack(f"{len(bases)}i", *heads), step, block_table.data_ptr(), block_table.stride(0), ptr(cu_q), kv_lens.data_ptr(), got.path.data_ptr(),
                                    got.counts.data_ptr(), got.next_tokens.data_ptr(), got.kv_lens.data_ptr(), stream), "swb_accept_tree")
    return got


def copy_pages(pages, src, dst) -> None:
    """Page dst[i] of every tensor becomes a copy of its page src[i]. pages as in `accept_tree`, of any types and page shapes. src and dst: lists of whole numbers, or int32 tensors on the
    device, whose pairs are passed over where one of the two is no page. A page may be copied to several, but is written once and not copied from where it is: lists are
    checked for that, tensors are the caller's word."""
    bases, sizes, _, count, step, blocks, held = _tensors(pages)
    on_device = isinstance(src, torch.Tensor)
    _require(on_device == isinstance(dst, torch.Tensor), "src and dst are both lists or both tensors")
    stream = _place(*held, *((src, dst) if on_device else ()))
    n = len(src)
    _require(n == len(dst), "as many pages to copy to as to copy")
    if on_device:
        _require(src.dim() == dst.dim() == 1 and src.dtype == dst.dtype == torch.int32 and src.is_contiguous() and dst.is_contiguous(), "src and dst are int32 [n]")
        a, b = src.data_ptr(), dst.data_ptr()
    elif n:
        to = set(dst)
        _require(min(min(src), min(dst)) >= 0 and max(max(src), max(dst)) < blocks, f"pages are 0 to {blocks - 1}")
        _require(len(to) == n and to.isdisjoint(src), "a page is written once, and none that is copied")
        a, b = struct.pack(f"{n}i", *src), struct.pack(f"{n}i", *dst)
    if n == 0 or count == 0:
        return
    check(kernels().swb_copy_pages(_longs(bases), _longs(sizes), step, count, blocks, a, b, n, 0 if on_device else 1, stream), "swb_copy_pages")


@dataclass
class BeamChoice:
    """scores fp32, beams int32 and tokens int64 [B, count], best first; -inf, -1 and -1 behind the last one that there is."""
    scores: torch.Tensor
    beams: torch.Tensor
    tokens: torch.Tensor


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, count: int) -> BeamChoice:
    """The `count` best of all continuations of each prompt's beams by one token: scores[b, k] + log softmax(logits[b K + k])[v], equal ones in the order of beam and token.

    logits [B * K, V] bf16 or fp32 (row stride free), scores fp32 [B, K]: what the beams have added up so far. A beam whose score is not finite, or with a logit that is NaN or +inf,
    offers nothing, nor does a logit of -inf (a token that is not allowed; a finite number in its place ties with others like it, which takes up to eight times as long). A sum of
    exponentials is within 2^-28.5 of its value. A search that keeps K beams asks for 2 K: so many are left when each of K may end."""
    stream = _place(logits, scores)
    _require(logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32) and logits.shape[1] >= 1 and (logits.stride(1) == 1 or logits.shape[1] == 1),
             "logits are bf16 or fp32 [B * K, V], unit inner stride")
    _require(scores.dim() == 2 and scores.dtype == torch.float32 and scores.is_contiguous() and scores.numel() == logits.shape[0], "scores are contiguous fp32 [B, K]")
    B, K = scores.shape
    V = logits.shape[1]
    _require(1 <= K <= MAX_BEAMS and B * K < 65536, "1 to 256 beams, fewer than 65536 of all prompts")
    _require(1 <= count <= MAX_COUNT and V < 2 ** 31 - 65536, "1 to 128 continuations, a vocabulary below 2^31 - 65536")
    got = BeamChoice(scores.new_empty((B, count)), scores.new_empty((B, count), dtype=torch.int32), scores.new_empty((B, count), dtype=torch.int64))
    nbytes = kernels().swb_beam_workspace_bytes(B, K, V, count)
    ws = scores.new_empty(nbytes, dtype=torch.uint8)
    check(kernels().swb_beam_select(logits.data_ptr(), logits.stride(0), logits.dtype == torch.float32, scores.data_ptr(), B, K, V, count, got.scores.data_ptr(), got.beams.data_ptr(),
                                    got.tokens.data_ptr(), ws.data_ptr(), nbytes, stream), "swb_beam_select")
    return got
