"""Decoding with several continuations at once, as cases that can be timed and checked: one pass of each operator of `inference_b200.ops.branch`.

  tree     attention of a tree of drafted tokens, behind a paged cache
  accept   the path of a drafted tree that the model agrees with; its cache entries close up, in every layer
  copy     copies of pages in every layer, for sequences that part
  beams    the best continuations over the beams of a prompt and the vocabulary

Caches are paged as the engine keeps them (16 tokens a page, pages in random order). `context` is what the longest sequence has cached in front of its tree, the others
half as much at least. A tree has `nodes` tokens, its root the last token that is certain; trees of a batch have between half as many and all."""
import math

import torch

own = False

BS = 16
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _tree(name, batch, nodes, context, heads=32, kv_heads=8, dim=128, kind="bf16"):
    return {"name": name, "op": "tree", "batch": batch, "nodes": nodes, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": kind}


def _accept(name, batch, nodes, context, layers=32, kv_heads=8, dim=128, kind="bf16"):
    return {"name": name, "op": "accept", "batch": batch, "nodes": nodes, "context": context, "layers": layers, "kv_heads": kv_heads, "dim": dim, "type": kind}


def _copy(name, pairs, blocks, layers=32, kv_heads=8, dim=128, kind="bf16"):
    return {"name": name, "op": "copy", "pairs": pairs, "blocks": blocks, "layers": layers, "kv_heads": kv_heads, "dim": dim, "type": kind}


def _beams(name, batch, beams, vocab, count, kind="fp32", first=False, allowed=1.0):
    return {"name": name, "op": "beams", "batch": batch, "beams": beams, "vocab": vocab, "count": count, "type": kind, "first": first, "allowed": allowed}


def listed():
    return [
        # one conversation, a few drafts: latency counts
        _tree("tree_chat", 1, 13, 1500),
        # one user with a book in the cache
        _tree("tree_book", 1, 64, 100001),
        # a full server
        _tree("tree_server", 48, 48, 4100),
        # the 32-bit mode, the heads of the sparse decoder
        _tree("tree_fp32", 2, 21, 900, heads=16, kv_heads=4, kind="fp32"),
        # one conversation: latency counts
        _accept("accept_chat", 1, 25, 77),
        # a full server
        _accept("accept_server", 64, 48, 150),
        # the beams of one prompt part in the middle of a page
        _copy("copy_beams", 5, 64),
        # beams of a full server
        _copy("copy_server", 190, 600),
        # one prompt, four beams
        _beams("beams_chat", 1, 4, 128256, 8),
        # the first step of a prompt: one of its beams is alive
        _beams("beams_first", 6, 10, 32768, 20, kind="bf16", first=True),
        # a full server
        _beams("beams_server", 32, 8, 128256, 16),
        # a wide search with an odd vocabulary, most of which a grammar forbids
        _beams("beams_wide", 3, 50, 50257, 100, allowed=0.02),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "accept", "copy", "beams"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 4, 128), (32, 8, 64), (28, 4, 128), (8, 8, 96), (12, 1, 128)])
    kind = "fp32" if rng.random() < 0.2 else "bf16"
    layers = rng.choice([4, 16, 28, 32])
    if op == "tree":
        batch, nodes = _log(rng, 1, 48), _log(rng, 1, 200)
        context = _log(rng, 1, min(100001, max(2, 9000000 // (batch * (nodes + 20)))))
        if kind == "fp32":
            batch, nodes, context = min(batch, 4), min(nodes, 40), min(context, 2000)
        c = _tree("", batch, nodes, context, heads, kv_heads, dim, kind)
    elif op == "accept":
        c = _accept("", _log(rng, 1, 64), _log(rng, 1, 100), rng.randrange(1, 150), layers, kv_heads, dim, kind)
    elif op == "copy":
        pairs = _log(rng, 1, 190)
        c = _copy("", pairs, 3 * pairs + rng.randrange(1, 60), layers, kv_heads, dim, kind)
    else:
        beams = _log(rng, 1, 50)
        batch, vocab = _log(rng, 1, max(1, 250 // beams)), _log(rng, 200, 128256)
        count = rng.choice([1, beams, 2 * beams, 2 * beams])
        c = _beams("", batch, beams, vocab, count, kind, rng.random() < 0.2, rng.choice([1.0, 1.0, 0.1, 0.01]))
    del c["name"]
    return c


def _grow(g, nodes):
    """Parents of a tree's tokens: each token hangs on one of the few in front of it, the first is the root."""
    u = torch.rand(nodes, generator=g).tolist()
    return [-1] + [max(0, i - 1 - int(u[i] ** 2 * 6)) for i in range(1, nodes)]


def _sizes(case, seed):
    """Tokens of each tree (the same of every seed: they are the outputs' shape), tokens cached in front of it, and parents."""
    nodes = torch.randint(max(1, case["nodes"] // 2), case["nodes"] + 1, (case["batch"],), generator=torch.Generator().manual_seed(case["nodes"]))
    g = torch.Generator().manual_seed(seed * 7 + 1)
    base = torch.randint(case["context"] // 2, case["context"] + 1, (case["batch"],), generator=g)
    nodes[0], base[0] = case["nodes"], case["context"]
    return nodes, base, [_grow(g, n) for n in nodes.tolist()], g


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 11 + 5)
    st = {"case": case}

    def rnd(*shape):
        return torch.randn(*shape, device="cuda", dtype=TYPES[case["type"]], generator=g)

    if case["op"] == "copy":
        # every page's copies go to pages that are free; some pages have several
        order = torch.randperm(case["blocks"], generator=torch.Generator().manual_seed(seed * 13 + 3)).tolist()
        st["dst"] = order[:case["pairs"]]
        from_ = order[case["pairs"]:]
        st["src"] = [from_[i * 2 // 3 % len(from_)] for i in range(case["pairs"])]
        st["pages"] = rnd(case["layers"], 2, case["blocks"], case["kv_heads"], BS, case["dim"])
        return st
    if case["op"] == "beams":
        B, K, V = case["batch"], case["beams"], case["vocab"]
        st["logits"] = rnd(B * K, V) * 2.5
        if case["allowed"] < 1.0:
            ok = torch.rand(B * K, V, device="cuda", generator=g) < case["allowed"]
            st["logits"].masked_fill_(~ok, -math.inf)
        st["scores"] = (-20 * torch.rand(B, K, device="cuda", generator=g)).sort(-1, descending=True).values.contiguous()
        if case["first"]:
            st["scores"][:, 0], st["scores"][:, 1:] = 0.0, -math.inf
        return st
    B, H, D = case["batch"], case["kv_heads"], case["dim"]
    nodes, base, trees, cpu = _sizes(case, seed)
    ends, lens = nodes.cumsum(0), nodes + base
    per = -(-int(lens.max()) // BS)
    blocks = B * per + 3
    st["table"] = torch.randperm(blocks, device="cuda", generator=g)[:B * per].to(torch.int32).view(B, per)
    st["cu"] = torch.cat([ends.new_zeros(1), ends]).to(torch.int32).cuda()
    st["lens"] = lens.to(torch.int32).cuda()
    T = int(ends[-1])
    if case["op"] == "accept":
        tokens = torch.randint(0, 50000, (T,), generator=cpu)
        picks = torch.randint(50000, 60000, (T,), generator=cpu)        # of nobody, unless a drafted token is picked below
        agrees = (torch.rand(T, generator=cpu) < 0.8).tolist()
        flat, at = tokens.tolist(), 0
        for tree in trees:
            for i in range(len(tree) - 1, 0, -1):                       # the last one written is the token's first child
                if agrees[at + tree[i]]:
                    picks[at + tree[i]] = flat[at + i]
            at += len(tree)
        st["tokens"], st["picks"] = tokens.cuda(), picks.cuda()
        st["parents"] = torch.tensor(sum(trees, []), dtype=torch.int32).cuda()
        st["pages"] = rnd(case["layers"], 2, blocks, H, BS, D)
        return st
    # what a token sees of its tree: itself and all in front of it on its path; packed as the framework takes it, bit j % 32 of word j / 32
    words = -(-case["nodes"] // 32)
    sees = torch.zeros(T, words * 32, dtype=torch.bool)
    at = 0
    for tree in trees:
        for i, parent in enumerate(tree):
            if parent >= 0:
                sees[at + i] = sees[at + parent]
            sees[at + i, i] = True
        at += len(tree)
    st["sees"] = sees.cuda()
    st["mask"] = (sees.view(T, words, 32).long() << torch.arange(32)).sum(-1).to(torch.int32).cuda()     # the highest bit is the sign
    st["q"], st["k"], st["v"] = rnd(T, case["heads"], D), rnd(blocks, H, BS, D), rnd(blocks, H, BS, D)
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------------
def _places(st, tokens):
    """Sequence of each of the step's tokens, its place within it, and the tokens of each sequence."""
    cu, t = st["cu"].long(), torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    return seq, t - cu[seq], cu[1:] - cu[:-1]


def _plain_tree(st):
    case, q = st["case"], st["q"].float()
    B, N, H, D = case["batch"], case["nodes"], case["kv_heads"], case["dim"]
    seq, place, n = _places(st, q.shape[0])
    k, v = (st[name][st["table"].long()].permute(0, 2, 1, 3, 4).float().flatten(2, 3) for name in ("k", "v"))
    qp = q.new_zeros(B, N, case["heads"], D)
    qp[seq, place] = q
    qp = qp.view(B, N, H, -1, D).transpose(1, 2).flatten(2, 3)
    rel = torch.arange(k.shape[2], device="cuda") - (st["lens"].long() - n)[:, None]        # place in the tree, below 0: in the cache in front of it
    tree = torch.zeros(B, N, st["sees"].shape[1], dtype=torch.bool, device="cuda")
    tree[seq, place] = st["sees"]
    seen = (rel < 0)[:, None] | (tree.gather(2, rel.clamp(0, tree.shape[2] - 1)[:, None].expand(-1, N, -1)) & (rel < n[:, None])[:, None])
    s = (qp @ k.transpose(-1, -2) * D ** -0.5).masked_fill(~seen.repeat_interleave(case["heads"] // H, 1)[:, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    o = (e / e.sum(-1, keepdim=True).clamp_min(1e-30)) @ v
    return o.view(B, H, N, -1, D).transpose(1, 2).reshape(B, N, -1)[seq, place].to(st["q"].dtype)


def _plain_accept(st):
    B, N = st["case"]["batch"], st["case"]["nodes"]
    seq, place, n = _places(st, st["picks"].numel())

    def padded(x):
        out = torch.full((B, N), -2, dtype=torch.int64, device="cuda")
        out[seq, place] = x.long()
        return out

    picks, tokens, parents = padded(st["picks"]), padded(st["tokens"]), padded(st["parents"])
    node, live = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.ones(B, dtype=torch.bool, device="cuda")
    path, last, counts = torch.full((B, N), -1, device="cuda"), node.clone(), node.clone()
    for d in range(N):
        path[:, d] = torch.where(live, node, -1)
        last = torch.where(live, node, last)
        counts += live
        fits = (parents == node[:, None]) & (tokens == picks.gather(1, node[:, None]))
        live = live & fits.any(1)
        node = fits.to(torch.int8).argmax(1)                # the first one
    base = st["lens"].long() - n
    b, d = (path >= 0).nonzero(as_tuple=True)
    fro, to = base[b] + path[b, d], base[b] + d
    pages = st["pages"]
    pages[:, :, st["table"][b, to // BS].long(), :, to % BS] = pages[:, :, st["table"][b, fro // BS].long(), :, fro % BS]
    nxt = picks.gather(1, last[:, None])[:, 0]
    return pages, path.to(torch.int32), counts.to(torch.int32), nxt, (base + counts).to(torch.int32)


def _plain_copy(st):
    st["pages"][:, :, st["dst"]] = st["pages"][:, :, st["src"]]
    return st["pages"]


def _plain_beams(st):
    case = st["case"]
    B, K, n = case["batch"], case["beams"], case["count"]
    x = st["logits"].double().view(B, K, -1)        # which of two near scores is the better one is decided in 64 bits
    V = x.shape[2]
    top = x.amax(-1, keepdim=True)
    scores = st["scores"].double()
    s = (scores.masked_fill(~scores.isfinite(), -math.inf)[..., None] + (x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))))).flatten(1)
    s = s.nan_to_num(nan=-math.inf, posinf=-math.inf, neginf=-math.inf)
    out = torch.full((B, n), -math.inf, dtype=torch.float64, device="cuda")
    flat = torch.full((B, n), -1, dtype=torch.int64, device="cuda")
    least = s.topk(min(n, K * V), -1).values[:, -1]
    for b in range(B):
        at = ((s[b] >= least[b]) & (s[b] > -math.inf)).nonzero()[:, 0]
        best = at[torch.sort(s[b, at], descending=True, stable=True).indices[:n]]
        out[b, :best.numel()], flat[b, :best.numel()] = s[b, best], best
    return out.float(), torch.where(flat < 0, -1, flat // V).to(torch.int32), torch.where(flat < 0, -1, flat % V)


# ---- what a user calls -------------------------------------------------------------------------------------------------------------------------------
def _own_tree(st):
    from inference_b200 import ops

    case = st["case"]
    return ops.tree_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["mask"], cu_q=st["cu"], max_q_len=case["nodes"], scale=case["dim"] ** -0.5)


def _own_accept(st):
    from inference_b200 import ops

    got = ops.accept_tree(st["picks"], st["tokens"], st["parents"], st["pages"], st["table"], st["lens"], cu_q=st["cu"], max_q_len=st["case"]["nodes"])
    return st["pages"], got.path, got.counts, got.next_tokens, got.kv_lens


def _own_copy(st):
    from inference_b200 import ops

    ops.copy_pages(st["pages"], st["src"], st["dst"])
    return st["pages"]


def _own_beams(st):
    from inference_b200 import ops

    got = ops.beam_select(st["logits"], st["scores"], count=st["case"]["count"])
    return got.scores, got.beams, got.tokens


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------------------
def work(case):
    size, op = 4 if case["type"] == "fp32" else 2, case["op"]
    if op == "beams":
        rows = case["batch"] * (1 if case["first"] else case["beams"])
        return {"bytes": rows * case["vocab"] * size + case["batch"] * (case["beams"] * 4 + case["count"] * 16), "flops": 4 * rows * case["vocab"]}
    row = case["kv_heads"] * case["dim"] * size
    if op == "copy":
        sources = -(-case["pairs"] * 2 // 3)
        return {"bytes": case["layers"] * 2 * BS * row * (sources + case["pairs"]), "flops": 0}
    nodes, base = (case[x] * (0.75 if case["batch"] > 1 else 1.0) for x in ("nodes", "context"))
    tokens = case["batch"] * nodes
    if op == "tree":
        cached = case["batch"] * (base + nodes) * 2 * row
        return {"bytes": cached + 2 * tokens * case["heads"] * case["dim"] * size + tokens * 4 * -(-case["nodes"] // 32),
                "flops": 4 * tokens * case["heads"] * case["dim"] * (base + 1)}
    # a path is some four tokens long, of which the first stays
    moved = case["batch"] * min(nodes - 1, 3)
    return {"bytes": case["layers"] * 2 * 2 * row * moved + tokens * 20 + case["batch"] * (case["nodes"] * 4 + 16), "flops": 0}


# ---- the definition in 64 bits, sequence by sequence ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("copy", "accept"):
        return None             # nothing is computed in numbers
    if case["op"] == "beams":
        B, K, V = case["batch"], case["beams"], case["vocab"]
        out = []
        for b in range(B):
            rows = torch.log_softmax(st["logits"][b * K:(b + 1) * K].double(), -1) + st["scores"][b].double()[:, None]
            best = rows.nan_to_num(nan=-math.inf).flatten().topk(min(case["count"], K * V)).values
            out.append(torch.cat([best, best.new_full((case["count"] - best.numel(),), -math.inf)]))
        return torch.stack(out), None, None
    nodes, base, trees, _ = _sizes(case, seed)
    H, D, G = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    out, at = [], 0
    for b, (n, c) in enumerate(zip(nodes.tolist(), base.tolist())):
        rows = st["table"][b, :-(-(n + c) // BS)].long()
        k, v = (st[x][rows].transpose(0, 1).reshape(H, -1, D).double() for x in ("k", "v"))
        seen = torch.zeros(n, n + c, dtype=torch.bool)
        seen[:, :c] = True
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, c + j], j = True, trees[b][j]
        q = st["q"][at:at + n].double().view(n, H, G, D).transpose(0, 1).flatten(1, 2)
        s = (q @ k[:, :n + c].transpose(1, 2) / math.sqrt(D)).masked_fill(~seen.cuda().repeat_interleave(G, 0), -math.inf)
        out.append((torch.softmax(s, -1) @ v[:, :n + c]).view(H, n, G, D).transpose(0, 1).reshape(n, -1))
        at += n
    return torch.cat(out)
