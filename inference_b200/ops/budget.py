"""Long paged caches on a budget (csrc/kernels/page_select.cu, attention_budget.cu, cache_evict.cu).

Two ways to spend less than the whole cache on a new token, both beside `paged_attention`:

  read less    `summarize_pages` keeps an 8-bit summary of every full page, `select_pages` picks the pages that promise a token the most,
               `selected_attention` reads these alone
  keep less    `tracked_attention` reads the whole cache and adds up the weight that each entry receives, `evict_tokens` lets the entries of least
               weight go and closes their holes

Both go together as long as pages are summarised again behind an eviction.

Scores, the softmax and all sums are 32-bit numbers (a page's sum of keys a 64-bit one). With bf16 caches each weight is rounded to bf16 in front of its product with the values, as in
`paged_attention`; the softmax's sum and the weights that `tracked_attention` hands out are not. Weights below 2^-126 of a row's largest are zeros.

Caches are one layer's pages [blocks, kv heads, block_size, width] with the block tables of `PagedSequence`. bf16, or fp32 in the 32-bit mode; widths up to 256.
Calls run on the current stream, take no host reads and can be captured into graphs; buffers that a call fills (summaries, weights, positions, the cache) belong
to the caller. Steps are described as in `paged_attention`: kv_lens int32 [num_seqs] counts a sequence's tokens with the new ones, cu_q int32 [num_seqs + 1]
are the new tokens' ranges within the rows of q and max_q_len bounds a sequence's number (None: every sequence has max_q_len of them); rows in front of the first range
and behind the last are left as they were. Lengths beyond a table's pages count as the table's end (the last new token sees the whole table, the one before it a key less), and pages whose
number is not in the cache are passed over."""
from __future__ import annotations

import struct
from dataclasses import dataclass

import torch

from .._native import kernels
from .runtime import KernelError, check, ptr, require_cuda

MAX_WIDTH, MAX_GROUP, MAX_SPLITS = 256, 128, 64
MAX_PAGES = 40000         # of a selection: the scores of a token lie in one block's shared memory


@dataclass
class PageSummaries:
    """codes int8 [blocks, kv heads, D] and scales fp32 [blocks, kv heads]: codes * scale is a full page's mean key to within half a step, the
    largest code is 127. A page with a key that is not finite has the scale NaN and is selected before all others. Pages not summarised yet hold whatever the buffers held."""
    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def empty(cls, kcache: torch.Tensor) -> "PageSummaries":
        blocks, heads, _, width = kcache.shape
        return cls(torch.zeros((blocks, heads, width), dtype=torch.int8, device=kcache.device),
                   torch.zeros((blocks, heads), dtype=torch.float32, device=kcache.device))

    def values(self) -> torch.Tensor:
        """The mean keys that the summaries stand for, fp32 [blocks, kv heads, D]."""
        codes, scales = self.codes, self.scales
        stream = _place(codes, scales)
        _check_summaries(codes, scales)
        out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
        check(kernels().swb_page_values(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), scales.numel(), codes.shape[2], stream), "swb_page_values")
        return out


@dataclass(frozen=True)
class PageBudget:
    """How many pages a new token reads: the first ones, the last ones (its own among them) and the best of those between (`select_pages`)."""
    top: int
    first: int = 1
    last: int = 4

    def __post_init__(self):
        _require(self.top >= 0 and self.first >= 0 and self.last >= 1, "top >= 0, first >= 0, last >= 1")


@dataclass
class PageSelection:
    """pages int32 [T, kv heads, N]: places in the sequence (page p holds tokens p * block_size and on), -1 behind the first counts int32 [T, kv heads]."""
    pages: torch.Tensor
    counts: torch.Tensor


# A decode step calls these once a layer: what is checked is read from each tensor once, and host arrays go to the library as packed bytes.
_INTS = {n: struct.Struct(f"{n}i").pack for n in (9, 11, 14, 16)}
_LONGS = {n: struct.Struct(f"{n}q").pack for n in (5, 8)}
_KINDS = (torch.bfloat16, torch.float32)


def _require(ok: bool, what: str) -> None:
    if not ok:
        raise KernelError(what)


def _place(*tensors: torch.Tensor | None) -> int:
    """All operands on the current device; its current stream, which launches go to."""
    dev = torch.cuda.current_device() if torch.cuda.is_initialized() else 0
    for t in tensors:
        if t is not None and t.get_device() != dev:
            require_cuda(t)
            raise KernelError(f"operands lie on {t.device}, the current device is cuda:{dev}")
    return torch._C._cuda_getCurrentRawStream(dev)          # (a Stream object takes 3 us to make)


def _check_cache(kcache: torch.Tensor, vcache: torch.Tensor | None = None) -> tuple[int, int, int, int, int]:
    shape, kind = kcache.shape, kcache.dtype
    _require(len(shape) == 4 and kind in _KINDS and kcache.is_contiguous() and shape[3] <= MAX_WIDTH,
             "pages are contiguous [blocks, kv heads, block_size, width] in bf16 or fp32, at most 256 wide")
    blocks, heads, bs, D = shape
    if vcache is None:
        return blocks, heads, bs, D, 0
    other = vcache.shape
    _require(len(other) == 4 and vcache.dtype == kind and vcache.is_contiguous() and other[:3] == shape[:3] and other[3] <= MAX_WIDTH,
             "value pages match the key pages in type, number, heads and block_size")
    return blocks, heads, bs, D, other[3]


def _check_summaries(codes: torch.Tensor, scales: torch.Tensor) -> tuple[int, int, int]:
    shape = codes.shape
    _require(len(shape) == 3 and codes.dtype == torch.int8 and codes.is_contiguous() and scales.dtype == torch.float32 and scales.shape == shape[:2]
             and scales.is_contiguous() and shape[2] <= MAX_WIDTH, "summaries are contiguous int8 [blocks, kv heads, D] and fp32 [blocks, kv heads], at most 256 wide")
    return shape


def _check_step(table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor | None, max_q_len: int, tokens: int) -> tuple[int, int]:
    """Number of sequences and width of the table. tokens < 0: not known."""
    lens, rows = kv_lens.shape, table.shape
    _require(len(lens) == 1 and len(rows) == 2 and rows[0] == lens[0] < 65536 and rows[1] >= 1 and table.dtype == kv_lens.dtype == torch.int32 and table.stride(1) == 1
             and kv_lens.is_contiguous(), "block_table is int32 [num_seqs, pages] with rows of unit stride, kv_lens int32 [num_seqs], up to 65535 sequences of a page at least")
    n = lens[0]
    _require(max_q_len < 2 ** 31, "max_q_len is below 2^31")
    if cu_q is None:
        _require(max_q_len >= 1 and (tokens < 0 or tokens == n * max_q_len), "without cu_q every sequence has max_q_len >= 1 tokens")
    else:
        _require(max_q_len >= 1 and cu_q.dtype == torch.int32 and cu_q.shape == (n + 1,) and cu_q.is_contiguous(), "cu_q is int32 [num_seqs + 1], max_q_len >= 1")
    return n, rows[1]


def _check_rows(q: torch.Tensor, kv_heads: int, width: int) -> tuple[int, int, int, int]:
    """Tokens, heads of a group, token and head strides."""
    _require(q.dim() == 3, "q is [T, heads, width]")
    (T, heads, D), (tok, head, inner) = q.shape, q.stride()
    G = heads // max(kv_heads, 1)
    _require(inner == 1 and D == width and heads == G * kv_heads and 1 <= G <= MAX_GROUP, "q is [T, heads, width], unit inner stride, up to 128 heads to a key/value head")
    return T, G, tok, head


def summarize_pages(kcache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, summaries: PageSummaries, *, cu_q: torch.Tensor | None,
                    max_q_len: int) -> None:
    """Fills the summaries of the pages that the step's new tokens complete: the last tokens of each sequence, already in the cache (max_q_len bounds their
    number). s = sum of a page's keys, a = max |s|: codes rint(127 s / a), scale a / (127 block_size); sums and quotient in 64 bits."""
    codes, scales = summaries.codes, summaries.scales
    stream = _place(kcache, block_table, kv_lens, codes, scales, cu_q)
    blocks, heads, bs, D, _ = _check_cache(kcache)
    n, per = _check_step(block_table, kv_lens, cu_q, max_q_len, -1)
    _require(_check_summaries(codes, scales) == (blocks, heads, D), "summaries belong to these pages: [blocks, kv heads, D]")
    dims = _INTS[9](n, max_q_len, per, blocks, bs, heads, D, kcache.dtype == torch.float32, 0)
    check(kernels().swb_page_summaries(dims, kcache.data_ptr(), codes.data_ptr(), scales.data_ptr(), block_table.data_ptr(), block_table.stride(0), ptr(cu_q),
                                       kv_lens.data_ptr(), stream), "swb_page_summaries")


def select_pages(q: torch.Tensor, summaries: PageSummaries, block_table: torch.Tensor, kv_lens: torch.Tensor, *, cu_q: torch.Tensor | None, max_q_len: int,
                 block_size: int, top: int, first: int = 1, last: int = 4) -> PageSelection:
    """The pages that each new token reads, per key/value head: its first `first`, its last `last` (its own page among them, at least one) and between these the
    `top` of largest score, ties to the lowest page; all of them where that is no fewer. In ascending order.

    q [T, Hq, D] bf16 or fp32 (token and head strides free). The group's queries are rounded to 8-bit codes of one step, max |q| / 127; score = the page's scale * max over the
    group of the codes' dot product. A token whose queries are not all finite, or all zero, finds every page alike."""
    codes, scales = summaries.codes, summaries.scales
    stream = _place(q, codes, scales, block_table, kv_lens, cu_q)
    blocks, heads, D = _check_summaries(codes, scales)
    _require(q.dtype in _KINDS, "q is bf16 or fp32")
    T, G, tok, head = _check_rows(q, heads, D)
    n, per = _check_step(block_table, kv_lens, cu_q, max_q_len, T)
    _require(1 <= block_size < 2 ** 31 and top >= 0 and first >= 0 and last >= 1, "1 <= block_size < 2^31, top >= 0, first >= 0, last >= 1")
    _require(per <= MAX_PAGES, "a selection is made over at most 40000 pages")
    width, rows = first + top + last, T * heads
    _require(width < 2 ** 31, "a selection lists fewer than 2^31 pages")
    both = q.new_empty(rows * (width + 1), dtype=torch.int32)
    pages, counts = both.as_strided((T, heads, width), (heads * width, width, 1)), both.as_strided((T, heads), (heads, 1), rows * width)
    dims = _INTS[14](T, n, max_q_len, per, blocks, block_size, heads, G, D, first, top, last, q.dtype == torch.float32, 0)
    check(kernels().swb_page_select(dims, q.data_ptr(), tok, head, codes.data_ptr(), scales.data_ptr(), block_table.data_ptr(), block_table.stride(0), ptr(cu_q),
                              kv_lens.data_ptr(), pages.data_ptr(), counts.data_ptr(), stream), "swb_page_select")
    return PageSelection(pages, counts)


def budget_splits(problems: int, keys: int, even: bool, tensor_cores: bool = True, sms: int = 148) -> int:
    """Blocks that share a problem's keys (problems: tokens, or runs of a few of them, * kv heads; even: all have about as many keys). An SM holds two or three blocks of the
    kernel on tensor cores, more of the plain one.

    Fewer problems than fit at once: as many splits as fit, up to 8, which join within the launch; more, joined by a second one, where 8 would leave SMs idle over
    long caches (8 problems of 8192 keys: 21.0 us with 8 splits, 16.1 with 37; of 4096 keys 13.6 and 13.1; 16 of 16 384 keys: 39.4 with 8, 31.3 with 18). More problems: one block
    each, or where their lengths differ enough blocks of 512 keys and more to even out over seven rounds of the SMs (384 problems of 4096 to 8191 keys: 280 us with one block each,
    214 with 8, 218 with 16; 296 of 2048 to 4096, the border: 103 and 91; 512 of 512 to 1024: 48 with one, 53 with two). Cores without tensor instructions: eight blocks
    to an SM, of 64 keys and more (64 problems of 2000 to 4000 32-bit keys: 713 us with one block each, 118 with 9, 101 with 18)."""
    slots, problems = 2 * sms, max(1, problems)
    if not tensor_cores:
        return max(1, min(MAX_SPLITS, (keys + 63) // 64, 8 * sms // problems))
    fit = slots // problems
    if not even and problems * keys >= slots * 4096:
        return max(1, min(MAX_SPLITS, keys // 512, 21 * sms // problems))
    return max(1, min((keys + 63) // 64, MAX_SPLITS if fit > 8 and problems * 8 < sms and keys >= 8192 else 8, fit))


def _attention(q, kcache, vcache, block_table, kv_lens, cu_q, max_q_len, scale, softcap, num_splits, out, pages, counts, weights) -> torch.Tensor:
    stream = _place(q, kcache, vcache, block_table, kv_lens, cu_q, out, weights, pages, counts)
    blocks, heads, bs, D, Dv = _check_cache(kcache, vcache)
    T, G, tok, head = _check_rows(q, heads, D)
    n, per = _check_step(block_table, kv_lens, cu_q, max_q_len, T)
    kind, columns, width, keys = q.dtype, G * heads * Dv, 0, per * bs
    _require(kind == kcache.dtype, "queries and cache have one type")
    w_seq = w_head = 0
    if weights is not None:
        _check_entries(weights, torch.float32, n, heads, keys, "weights")
        w_seq, w_head, _ = weights.stride()
    else:
        listed = pages.shape
        _require(len(listed) == 3 and pages.dtype == counts.dtype == torch.int32 and listed[:2] == (T, heads) == counts.shape and listed[2] >= 1 and pages.is_contiguous()
                 and counts.is_contiguous(), "the selection is int32 [T, kv heads, N >= 1] and [T, kv heads], contiguous")
        width = listed[2]
        keys = min(width, per) * bs
    if out is None:
        out = q.new_empty((T, columns))
        out_stride = columns
    else:
        _require(out.shape == (T, columns) and out.dtype == kind and out.stride(1) == 1, "out is [T, heads * value width] in the type of q, unit inner stride")
        out_stride = out.stride(0)
        _require(out_stride >= columns or T <= 1, "rows of out share memory")
    k_ptr, v_ptr = kcache.data_ptr(), vcache.data_ptr()
    fast = kind is torch.bfloat16 and (D | Dv) % 8 == 0 and D <= 128 and Dv <= 128 and bs % 16 == 0 and (k_ptr | v_ptr) % 16 == 0 and blocks * heads * bs < 2 ** 31
    run = 1                                               # tokens of a sequence that share a problem
    while fast and weights is not None and run < max_q_len and run * 2 * G <= 16:
        run *= 2
    problems = (T if run == 1 else n * -(-max_q_len // run)) * heads * -(-G // 16)
    splits = budget_splits(problems, keys, weights is None, fast) if num_splits is None else num_splits
    _require(1 <= splits <= MAX_SPLITS, "1 to 64 splits")
    ws, nbytes = None, 0
    if weights is not None or not (splits == 1 or (fast and splits <= 8 and problems * splits <= 296)):      # else blocks finish their results, or clusters do
        nbytes = 4 * T * G * heads * (splits * (Dv + 2) + (0 if weights is None else per * bs)) + 16
        ws = q.new_empty(nbytes, dtype=torch.uint8)        # the call's own: two streams or graphs share none
    dims = _INTS[16](T, n, max_q_len, per, blocks, bs, heads, G, D, Dv, width, splits, kind == torch.float32, 0, 0, 0)
    strides = _LONGS[8](tok, head, out_stride, block_table.stride(0), w_seq, w_head, 0, 0)
    check(kernels().swb_attn_budget(dims, strides, q.data_ptr(), out.data_ptr(), k_ptr, v_ptr, block_table.data_ptr(), ptr(cu_q), kv_lens.data_ptr(),
                              ptr(pages), ptr(counts), ptr(weights), scale, softcap, ptr(ws), nbytes, stream), "swb_attn_budget")
    return out


def selected_attention(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, selection: PageSelection, *,
                       cu_q: torch.Tensor | None, max_q_len: int, scale: float, softcap: float = 0.0, num_splits: int | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every new token over the pages selected for it, causal within them -> [T, Hq * Dv] in the type of q.

    q [T, Hq, D] and the caches of one type. softcap > 0: scores s become softcap tanh(s / softcap). Lists may come from elsewhere than `select_pages`: in any order; pages that
    a token does not see, or that are not in the table, add nothing; a page listed twice counts twice. A token without keys gets zeros."""
    return _attention(q, kcache, vcache, block_table, kv_lens, cu_q, max_q_len, scale, softcap, num_splits, out, selection.pages, selection.counts, None)


def tracked_attention(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, weights: torch.Tensor, *,
                      cu_q: torch.Tensor | None, max_q_len: int, scale: float, softcap: float = 0.0, num_splits: int | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every new token over all keys that it sees -> [T, Hq * Dv], which also adds the softmax weights of the step, summed over its tokens and the query heads of
    a group, to weights fp32 [num_seqs, kv heads, >= table pages * block_size] (unit inner stride; entry j of a row belongs to cache entry j). Entries behind a sequence's
    length are not touched. A new token's entry starts from what the row holds: a caller who takes tokens back (drafts that were not accepted) sets their weights to 0, as
    `weights.masked_fill_(torch.arange(N) >= kv_lens[:, None, None], 0)` does for all sequences.

    For decode steps, and for the last tokens of a prompt: keys are read once for every 16 rows (tokens * heads of a group) of a sequence, and scores are kept until the sums
    are known, 4 bytes a token, query head and key of the table's width: give it the columns of a wide table that the longest
    sequence needs (`block_table[:, :n]`; weights may stay wider)."""
    return _attention(q, kcache, vcache, block_table, kv_lens, cu_q, max_q_len, scale, softcap, num_splits, out, None, None, weights)


def _check_entries(x: torch.Tensor, kind: torch.dtype, num_seqs: int, heads: int, entries: int, name: str) -> None:
    """x [num_seqs, heads, N] is written per (sequence, head): rows may be strided, but must not share memory (expanded or overlapping views)."""
    _require(x.dim() == 3 and x.dtype == kind, f"{name} are {kind} [num_seqs, kv heads, N]")
    (a, b, n), (sa, sb, inner) = x.shape, x.stride()
    _require(inner == 1 and a == num_seqs and b == heads and n >= entries, f"{name} have an entry for each that the block table has room for, unit inner stride")
    if sb * b > sa or sb < n:
        _require(not _overlaps(x), f"rows of {name} share memory")


def _overlaps(x: torch.Tensor) -> bool:
    """Whether two rows of x [A, B, N] share memory."""
    (a, sa), (b, sb) = sorted(((x.shape[i], x.stride(i)) for i in (0, 1)), key=lambda e: e[1])
    return (a > 1 and sa < x.shape[2]) or (b > 1 and sb < (a - 1) * sa + x.shape[2])


def evict_tokens(kcache: torch.Tensor, vcache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor,
                 next_positions: torch.Tensor, *, keep: int, recent: int, first: int = 0) -> torch.Tensor:
    """Shrinks every sequence of more than `keep` cached tokens to `keep`, per key/value head, and returns the new lengths int32 [num_seqs].

    A head keeps the entries whose position is below `first` or among the last `recent` in front of next_positions int32 [num_seqs] (the position of the
    sequence's next token), and of the others those of largest weight (fp32 [num_seqs, kv heads, N], as `tracked_attention` adds them up; ties: the lowest index). Entries that stay
    and lie behind `keep` move in order into the holes in front of it: their rows of both caches, weight and position. positions int32 [num_seqs, kv heads, N]: -1 for
    entries without a record, which stand in order in front of the next position (all of them before the first call); the call records those it keeps. Of a sequence that
    shrinks the weights of entries keep to L - 1 (L: its length) become 0 and the positions from `keep` to the table's end -1; weights behind L stay as they were, and so does all of a
    sequence of no more than `keep` tokens. Summaries of pages that entries move into are out of date then: `summarize_pages(kcache, block_table, new lengths, summaries, cu_q=None,
    max_q_len=keep)` makes those of all full pages anew. Everything is done in place. Pages must not be
    shared with a sequence that is not to lose tokens, nor between sequences of the call."""
    stream = _place(kcache, vcache, block_table, kv_lens, weights, positions, next_positions)
    blocks, heads, bs, D, Dv = _check_cache(kcache, vcache)
    n, per = _check_step(block_table, kv_lens, None, 1, -1)
    capacity, size = per * bs, 4 if kcache.dtype == torch.float32 else 2
    _check_entries(weights, torch.float32, n, heads, capacity, "weights")
    _check_entries(positions, torch.int32, n, heads, capacity, "positions")
    _require(next_positions.dtype == torch.int32 and next_positions.shape == (n,) and next_positions.is_contiguous(), "next_positions are int32 [num_seqs]")
    _require(1 <= keep < 2 ** 31 and recent >= 0 and first >= 0 and recent + first <= keep, "0 <= first, recent; 1 <= keep < 2^31; first + recent <= keep")
    device, room = kcache.device, 2 * n * heads * max(0, min(keep, capacity - keep))
    moves = torch.empty(room, dtype=torch.int32, device=device)
    lens = torch.empty(n, dtype=torch.int32, device=device)
    dims = _INTS[11](n, heads, per, blocks, bs, D * size, Dv * size, capacity, keep, recent, first)
    sizes = _LONGS[5](*weights.stride()[:2], *positions.stride()[:2], room)
    check(kernels().swb_evict(dims, sizes, kcache.data_ptr(), vcache.data_ptr(), block_table.data_ptr(), block_table.stride(0), kv_lens.data_ptr(), lens.data_ptr(),
                        next_positions.data_ptr(), weights.data_ptr(), positions.data_ptr(), moves.data_ptr(), stream), "swb_evict")
    return lens
