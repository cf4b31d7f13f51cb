"""Attention over long paged caches on a budget, as cases that can be timed and checked: one pass of each operator of `inference_b200.ops.budget`.

  summaries   int8 summaries of the pages that a step's new tokens complete
  select      the pages whose summaries promise a query the most, per query token and key/value head
  selected    attention over selected pages
  tracked     attention over the whole cache that adds up the weight each key receives
  evict       the cache entries of least weight leave, the others close the holes

Caches are paged as the engine keeps them (16 tokens a page, pages in random order, one layer), `context` is the longest sequence's length with its new tokens
and the others are between half of it and all of it. `new` tokens a sequence are the step's own."""
import math

import torch

own = False

BS = 16
FIRST, LAST = 1, 4          # pages that are always read: the first ones and the newest ones
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, batch, new, context, heads=32, kv_heads=8, dim=128, top=0, keep=0, recent=0, kind="bf16"):
    return {"name": name, "op": op, "batch": batch, "new": new, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim, "top": top,
            "keep": keep, "recent": recent, "type": kind}


def listed():
    return [
        # a decode step of a full server: one sequence in sixteen completes a page
        _case("summaries_step", "summaries", 64, 1, 501),
        # prompts on their way into the cache
        _case("summaries_prompts", "summaries", 8, 15000, 15000),
        # a decode step of a full server with long documents
        _case("select_server", "select", 64, 1, 16400, top=59),
        # a portion of a prompt on top of a long document, a selection for each of its tokens
        _case("select_prompt", "select", 1, 1000, 17000, top=59),
        # one user with a book in the cache
        _case("selected_chat", "selected", 1, 1, 131000, top=123),
        # a full server, a selection of 2 048 tokens each
        _case("selected_server", "selected", 64, 1, 16400, top=123),
        # a portion of a prompt, the heads of the sparse decoder
        _case("selected_prompt", "selected", 2, 250, 9001, heads=16, kv_heads=4, top=59),
        # a short conversation: latency counts
        _case("tracked_chat", "tracked", 1, 1, 2500),
        # a full server
        _case("tracked_server", "tracked", 48, 1, 8191),
        # the last tokens of two prompts, whose weights decide what stays of them
        _case("tracked_window", "tracked", 2, 16, 6001, heads=16, kv_heads=4),
        # a full server makes room for the next 512 tokens of each sequence
        _case("evict_step", "evict", 64, 0, 4608, keep=4096, recent=256),
        # two prompts shrink to their heavy part
        _case("evict_prompt", "evict", 2, 0, 30001, keep=4000, recent=64),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["summaries", "select", "selected", "tracked", "evict"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 4, 128), (32, 8, 64), (28, 4, 128), (8, 8, 96), (12, 1, 128)])
    kind = "fp32" if rng.random() < 0.15 else "bf16"
    batch, new, top, keep, recent = _log(rng, 1, 64), 1, 0, 0, 0
    if op == "summaries":
        batch, new = _log(rng, 1, 16), _log(rng, 1, 7000)
        context = new + rng.choice([0, rng.randrange(1, 500)])
    elif op == "evict":
        context = _log(rng, 200, min(30000, 290000 // batch))
        keep = max(64, int(context * rng.uniform(0.1, 0.95)))
        recent, new = rng.randrange(0, keep // 2), 0
    else:
        if op != "tracked" and rng.random() < 0.4:      # a portion of a prompt
            batch, new = rng.choice([1, 2, 3]), _log(rng, 2, 120)
        elif op == "tracked" and rng.random() < 0.3:
            batch, new = rng.choice([1, 2, 3]), rng.randrange(2, 17)
        limit = 390000 if op == "tracked" else 1000000
        context = _log(rng, new + 20, min(131000 if op != "tracked" else 32000, limit // (batch * 2)))
        top = rng.randrange(1, 124) if op != "tracked" else 0
        if kind == "fp32":
            batch, context = min(batch, 8), min(context, 20000)
    c = _case("", op, batch, new, context, heads, kv_heads, dim, top, keep, recent, kind)
    del c["name"]
    return c


def _lens(case, seed):
    """Cached tokens of each sequence, the step's new ones among them."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    low = max(case["new"], case["context"] // 2, 1)
    if case["op"] == "summaries":
        low = max(case["new"], case["context"] - 2 * BS)
    lens = torch.randint(low, case["context"] + 1, (case["batch"],), generator=g)
    lens[0] = case["context"]
    return lens.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 11 + 5)
    B, H, D, kind = case["batch"], case["kv_heads"], case["dim"], TYPES[case["type"]]
    lens = _lens(case, seed)
    per = -(-case["context"] // BS)
    blocks = B * per + 3
    st = {"case": case, "lens": lens.cuda(), "table": torch.randperm(blocks, device="cuda", generator=g)[:B * per].to(torch.int32).view(B, per)}

    def rnd(*shape):
        return torch.randn(*shape, device="cuda", dtype=kind, generator=g)

    T = B * case["new"]
    if case["op"] in ("select", "selected", "tracked"):
        st["q"] = rnd(T, case["heads"], D)
    if case["op"] != "select":
        st["k"] = rnd(blocks, H, BS, D)
    if case["op"] in ("selected", "tracked", "evict"):
        st["v"] = rnd(blocks, H, BS, D)
    if case["op"] in ("summaries", "select"):
        # what earlier steps left: codes up to +-127 and the scales of sums of 16 such keys
        st["codes"] = torch.randint(-127, 128, (blocks, H, D), device="cuda", generator=g).to(torch.int8)
        st["scales"] = torch.rand(blocks, H, device="cuda", generator=g) * 0.002 + 0.004
    if case["op"] == "selected":
        seen = _seen(st)
        pages = (seen + BS - 1) // BS
        most, want = -(-case["context"] // BS), FIRST + case["top"] + LAST
        at = torch.arange(most, device="cuda")
        pick = torch.rand(T, H, most, device="cuda", generator=g)
        pick = torch.where((at < FIRST) | (at >= pages[:, None, None] - LAST), 2.0, pick).masked_fill(at >= pages[:, None, None], -1.0)
        best = pick.topk(min(want, most), -1)
        chosen = torch.where(best.values < 0, most, best.indices).sort(-1).values.to(torch.int32)
        st["pages"] = torch.full((T, H, want), -1, dtype=torch.int32, device="cuda")
        st["pages"][..., :chosen.shape[-1]] = torch.where(chosen == most, -1, chosen)
        st["counts"] = (st["pages"] >= 0).sum(-1).to(torch.int32)
    if case["op"] in ("tracked", "evict"):
        # weights as steps have added them up: few large, most small
        w = torch.rand(B, H, per * BS, device="cuda", generator=g)
        old = torch.arange(per * BS, device="cuda")[None, :] < st["lens"][:, None]
        st["weights"] = (w ** 6 * 40 * old[:, None]).contiguous()
    if case["op"] == "evict":
        # every second sequence lost tokens before: its first entries are not in order any more
        gone = torch.arange(B, device="cuda") % 2 * 100
        st["next"] = (st["lens"] + gone).to(torch.int32)
        at = torch.arange(per * BS, device="cuda", dtype=torch.int32).expand(B, H, -1)
        st["positions"] = torch.where((gone > 0)[:, None, None] & (at < case["keep"] // 2), at + 7, -1).contiguous()
    return st


def _seen(st):
    """Keys that each of the step's tokens sees, its own among them."""
    new = st["case"]["new"]
    return (st["lens"][:, None].long() - new + 1 + torch.arange(new, device="cuda")).flatten()


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------------
def _softmax(s, mask):
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(s - top)
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_summaries(st):
    lens, new = st["lens"][:, None], st["case"]["new"]
    ends = (torch.arange(st["table"].shape[1], device="cuda") + 1)[None] * BS
    at = st["table"][(ends <= lens) & (ends > lens - new)].long()
    total = st["k"][at].double().sum(2)         # whether a code is rounded up or down is decided in 64 bits
    top = total.abs().amax(-1, keepdim=True)
    st["codes"][at] = torch.where(top > 0, torch.round(127 * total / top), 0.0).to(torch.int8)
    st["scales"][at] = (top[..., 0] / (127 * BS)).float()
    return st["codes"] * st["scales"][..., None], st["scales"]


def _plain_select(st):
    case, q = st["case"], st["q"].double()
    B, new, H, D = case["batch"], case["new"], case["kv_heads"], case["dim"]
    q = q.view(B, new, H, -1, D)
    top = q.abs().amax((-2, -1), keepdim=True)
    qc = torch.where(top > 0, torch.round(127 * q / top), 0.0).float()
    rows = st["table"].long()
    # products of whole numbers up to 127 and their sums stay below 2^24: exact in 32 bits
    dots = qc.permute(0, 2, 1, 3, 4).reshape(B, H, -1, D) @ st["codes"][rows].float().permute(0, 2, 3, 1)
    score = dots.view(B, H, new, -1, rows.shape[1]).amax(3) * st["scales"][rows].permute(0, 2, 1)[:, :, None]
    score = score.permute(0, 2, 1, 3).reshape(B * new, H, -1)
    pages = ((_seen(st) + BS - 1) // BS)[:, None, None]
    at = torch.arange(rows.shape[1], device="cuda")
    want = FIRST + case["top"] + LAST
    score = torch.where((at < FIRST) | (at >= pages - LAST), math.inf, score).masked_fill(at >= pages, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :want]
    chosen = torch.where(order < pages, order, 1 << 30).sort(-1).values
    out = torch.full((*score.shape[:2], want), -1, dtype=torch.int32, device="cuda")
    out[..., :chosen.shape[-1]] = torch.where(chosen == 1 << 30, -1, chosen)
    return out, (out >= 0).sum(-1).to(torch.int32)


def _plain_selected(st):
    case, q, pages = st["case"], st["q"].float(), st["pages"].long()
    T, Hq, D = q.shape
    H = case["kv_heads"]
    seq = torch.arange(T, device="cuda") // case["new"]
    at = st["table"][seq[:, None, None], pages.clamp_min(0)].long()
    heads = torch.arange(H, device="cuda")[None, :, None]
    key = pages[..., None] * BS + torch.arange(BS, device="cuda")
    seen = ((pages[..., None] >= 0) & (key < _seen(st)[:, None, None, None])).flatten(2)
    s = q.view(T, H, -1, D) @ st["k"][at, heads].float().flatten(2, 3).transpose(-1, -2) * D ** -0.5
    o = _softmax(s, seen[:, :, None]) @ st["v"][at, heads].float().flatten(2, 3)
    return o.reshape(T, Hq * D).to(st["q"].dtype)


def _plain_tracked(st):
    case, q = st["case"], st["q"].float()
    B, new, H, D = case["batch"], case["new"], case["kv_heads"], case["dim"]
    k, v = (st[n][st["table"].long()].permute(0, 2, 1, 3, 4).float().flatten(2, 3) for n in ("k", "v"))
    q = q.view(B, new, H, -1, D).transpose(1, 2).flatten(2, 3)
    seen = torch.arange(k.shape[2], device="cuda") < _seen(st).view(B, new, 1)
    p = _softmax(q @ k.transpose(-1, -2) * D ** -0.5, seen.repeat_interleave(case["heads"] // H, 1)[:, None])
    out = (p @ v).view(B, H, new, -1, D).transpose(1, 2).reshape(B * new, -1).to(st["q"].dtype)
    return out, st["weights"] + p.sum(2)


def _plain_evict(st):
    case, keep = st["case"], st["case"]["keep"]
    w, pos, lens = st["weights"].clone(), st["positions"].clone(), st["lens"][:, None, None]
    B, H, N = w.shape
    nxt = st["next"][:, None, None]
    at = torch.arange(N, device="cuda", dtype=torch.int32).expand(B, H, N)
    live = at < lens
    place = torch.where(pos >= 0, pos, nxt - lens + at)
    rank = torch.where((place < FIRST * BS) | (place >= nxt - case["recent"]), math.inf, w).masked_fill(~live, -math.inf)
    kept = torch.zeros_like(live).scatter(-1, torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep], True) & live
    full = lens > keep
    b, h, hole = (full & (at < keep) & ~kept).nonzero(as_tuple=True)        # in order, as many of a head as entries that move
    mover = (full & (at >= keep) & kept).nonzero(as_tuple=True)[2]
    to, fro = st["table"][b, hole // BS].long(), st["table"][b, mover // BS].long()
    for name in ("k", "v"):
        st[name][to, h, hole % BS] = st[name][fro, h, mover % BS]
    w[b, h, hole] = w[b, h, mover]
    place[b, h, hole] = place[b, h, mover]
    w = torch.where(full & (at >= keep), 0.0, w)
    pos = torch.where(full, torch.where(at < keep, place, -1), pos)
    return st["k"], st["v"], w, pos, st["lens"].clamp_max(keep)


# ---- what a user calls -------------------------------------------------------------------------------------------------------------------------------
def _own_summaries(st):
    from inference_b200 import ops

    summaries = ops.PageSummaries(st["codes"], st["scales"])
    ops.summarize_pages(st["k"], st["table"], st["lens"], summaries, cu_q=None, max_q_len=st["case"]["new"])
    return summaries.values(), st["scales"]


def _own_select(st):
    from inference_b200 import ops

    got = ops.select_pages(st["q"], ops.PageSummaries(st["codes"], st["scales"]), st["table"], st["lens"], cu_q=None, max_q_len=st["case"]["new"],
                           block_size=BS, top=st["case"]["top"], first=FIRST, last=LAST)
    return got.pages, got.counts


def _own_selected(st):
    from inference_b200 import ops

    return ops.selected_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], ops.PageSelection(st["pages"], st["counts"]), cu_q=None,
                                  max_q_len=st["case"]["new"], scale=st["case"]["dim"] ** -0.5)


def _own_tracked(st):
    from inference_b200 import ops

    weights = st["weights"].clone()         # the call adds to them
    out = ops.tracked_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], weights, cu_q=None, max_q_len=st["case"]["new"],
                                scale=st["case"]["dim"] ** -0.5)
    return out, weights


def _own_evict(st):
    from inference_b200 import ops

    case = st["case"]
    weights, positions = st["weights"].clone(), st["positions"].clone()     # the call closes their holes too
    lens = ops.evict_tokens(st["k"], st["v"], st["table"], st["lens"], weights, positions, st["next"], keep=case["keep"], recent=case["recent"],
                            first=FIRST * BS)
    return st["k"], st["v"], weights, positions, lens


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------------------
def work(case):
    B, new, Hq, H, D = (case[k] for k in ("batch", "new", "heads", "kv_heads", "dim"))
    size = 4 if case["type"] == "fp32" else 2
    T, op, mean = B * new, case["op"], (case["context"] * 0.75 if B > 1 else case["context"])
    if op == "summaries":
        pages = B * new / BS
        blocks = B * -(-case["context"] // BS) + 3      # the values come back for the whole pool
        return {"bytes": pages * H * (BS * D * size + D) + blocks * H * (5 * D + 4), "flops": pages * H * BS * D}
    if op == "select":
        pages = mean / BS
        want = FIRST + case["top"] + LAST
        return {"bytes": B * pages * H * (D + 4) + T * Hq * D * size + T * H * (want + 1) * 4, "flops": 2 * T * Hq * D * pages}
    if op == "selected":
        pages = min(mean / BS, FIRST + case["top"] + LAST)
        read = min(T * pages, B * mean / BS)            # several tokens of a sequence cannot need more than its cache
        return {"bytes": read * H * BS * D * 2 * size + T * H * (pages + 1) * 4 + 2 * T * Hq * D * size, "flops": 4 * T * Hq * D * pages * BS}
    if op == "tracked":
        return {"bytes": B * mean * H * (2 * D * size + 8) + 2 * T * Hq * D * size, "flops": 4 * T * Hq * D * mean}
    keep, low, high = case["keep"], max(case["context"] // 2, 1), case["context"]
    full = 1.0 if B == 1 else min(1.0, max(0.0, (high - max(low, keep)) / max(1, high - low)))      # share of the sequences that shrink
    length = high if B == 1 else (max(low, keep) + high) / 2
    safe = case["recent"] + FIRST * BS
    left = max(0.0, (keep - safe) / max(1.0, length - safe))        # of the unprotected
    moves = min(length - keep, case["recent"]) + max(0.0, length - keep - case["recent"]) * left
    return {"bytes": B * full * H * (length * 8 + moves * (4 * D * size + 16) + (length - keep) * 8) + B * 8, "flops": B * full * H * length}


# ---- the definition in 64 bits, sequence by sequence ---------------------------------------------------------------------------------------------------
def _rows(st, b, n, name):
    """The first n cached rows of sequence b in 64 bits [heads, n, width]."""
    got = st[name].index_select(0, st["table"][b, :-(-n // BS)].long())
    return got.transpose(0, 1).reshape(got.shape[1], -1, got.shape[3])[:, :n].double()


def exact(case, seed):
    st = prepare(case, seed)
    op, B, new, H, D = case["op"], case["batch"], case["new"], case["kv_heads"], case["dim"]
    lens, G = st["lens"].tolist(), case["heads"] // case["kv_heads"]
    if op == "select":
        return None             # whole numbers only
    if op == "summaries":
        values, scales = st["codes"].double() * st["scales"].double()[..., None], st["scales"].double()
        for b, n in enumerate(lens):
            lo, hi = (n - new) // BS, n // BS
            if hi > lo:
                at = st["table"][b, lo:hi].long()
                s = sum(st["k"][at, :, i].double() for i in range(BS))
                a = s.abs().max(-1, keepdim=True).values.clamp_min(1e-300)
                values[at], scales[at] = (s * 127 / a).round() * (a / BS / 127), a[..., 0] / BS / 127
        return values, scales
    if op == "evict":
        k, v, w, pos = st["k"].double(), st["v"].double(), st["weights"].double(), st["positions"].clone()
        for b, n in enumerate(lens):
            if n <= case["keep"]:
                continue
            nxt, rows = int(st["next"][b]), st["table"][b].long()
            for h in range(H):
                mine = pos[b, h, :n].long()
                mine = torch.where(mine < 0, torch.arange(nxt - n, nxt, device="cuda"), mine)
                order = w[b, h, :n].clone()
                order[(mine < FIRST * BS) | (mine >= nxt - case["recent"])] = 1e30
                stay = torch.zeros(n, dtype=torch.bool, device="cuda")
                stay[torch.argsort(-order, stable=True)[:case["keep"]]] = True
                hole = (~stay[:case["keep"]]).nonzero()[:, 0]
                move = stay[case["keep"]:].nonzero()[:, 0] + case["keep"]
                for t in (k, v):
                    t[rows[hole // BS], h, hole % BS] = t[rows[move // BS], h, move % BS]
                w[b, h, hole], mine[hole] = w[b, h, move], mine[move]
                w[b, h, case["keep"]:n] = 0
                pos[b, h, :case["keep"]], pos[b, h, case["keep"]:] = mine[:case["keep"]], -1
        return k, v, w, None, None
    q = st["q"].double().view(B, new, H, G, D)
    out = torch.zeros(B, new, H, G, D, dtype=torch.float64, device="cuda")
    if op == "tracked":
        weights = st["weights"].double()
        for b, n in enumerate(lens):
            k, v = _rows(st, b, n, "k"), _rows(st, b, n, "v")
            for i in range(new):
                m = n - new + 1 + i
                p = torch.softmax(q[b, i] @ k[:, :m].transpose(1, 2) / math.sqrt(D), -1)
                out[b, i] = p @ v[:, :m]
                weights[b, :, :m] += p.sum(1)
        return out.view(B * new, -1), weights
    for b, n in enumerate(lens):
        k, v = _rows(st, b, n, "k"), _rows(st, b, n, "v")
        for i in range(new):
            m = n - new + 1 + i
            use = torch.zeros(H, -(-m // BS) + 1, dtype=torch.bool, device="cuda")
            use.scatter_(1, torch.where(st["pages"][b * new + i] < 0, use.shape[1] - 1, st["pages"][b * new + i]).long(), True)
            use = use[:, :-1].repeat_interleave(BS, 1)[:, :m]
            s = (q[b, i] @ k[:, :m].transpose(1, 2) / math.sqrt(D)).masked_fill(~use[:, None], -math.inf)
            out[b, i] = torch.softmax(s, -1) @ v[:, :m]
    return out.view(B * new, -1)
