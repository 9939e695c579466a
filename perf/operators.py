"""Measured cases of the speculative-decoding operators.

A step that verifies drafted tokens runs four operators over the paged cache:

  tree     attention of a tree of drafted tokens over a sequence's pages
           (``paged_tree_fwd``)
  verify   acceptance of the drafted tokens against the target's
           probabilities, and the token that follows (``layer_verify``)
  compact  the accepted path's K/V rows moved together behind the context, in
           every layer (``cache_compact_paths``)
  copy     whole or partly filled pages copied in every layer, for forked
           sequences (``cache_copy_pages``)

With ``own`` false ``run`` computes them from elementary torch operations;
with ``own`` true it calls the library. Shapes are the ones the repository's
benchmark configurations use (16 or 32 or 64 query heads over 8 K/V heads of
128, 256-token pages, 28 layers, a vocabulary of 151,936) and generic ones.
"""
import math

import numpy as np
import torch

own = False

DIM = 128
PAGE = 256


def listed():
    return [
        # One user, a chain of three drafts behind the last token, a short chat: launch latency.
        dict(name="tree one chat", op="tree", batch=1, ctx_lo=200, ctx_hi=200, nodes_lo=4, nodes_hi=4, q_heads=16,
             kv_heads=8),
        # An engine's batch at ragged contexts, with drafts of different lengths (none for some).
        dict(name="tree engine batch", op="tree", batch=32, ctx_lo=128, ctx_hi=1024, nodes_lo=1, nodes_hi=9,
             q_heads=16, kv_heads=8),
        # A loaded server: many sequences of 4k tokens, small trees.
        dict(name="tree loaded server", op="tree", batch=64, ctx_lo=3900, ctx_hi=4200, nodes_lo=8, nodes_hi=16,
             q_heads=32, kv_heads=8),
        # Few users with long documents.
        dict(name="tree long documents", op="tree", batch=4, ctx_lo=32000, ctx_hi=32768, nodes_lo=16, nodes_hi=16,
             q_heads=64, kv_heads=8),
        # Wide trees at mixed lengths: several row tiles for a K/V head.
        dict(name="tree wide", op="tree", batch=16, ctx_lo=500, ctx_hi=8192, nodes_lo=33, nodes_hi=64, q_heads=32,
             kv_heads=8),
        # One user, a chain of four drafts from a draft model.
        dict(name="verify one user", op="verify", batch=1, nodes_lo=5, nodes_hi=5, vocab=151936, fan=1, draft=True,
             greedy_every=0),
        # A loaded server with trees from a draft model, a few greedy requests among them.
        dict(name="verify trees", op="verify", batch=64, nodes_lo=8, nodes_hi=8, vocab=151936, fan=3, draft=True,
             greedy_every=5),
        # Drafts looked up in the prompt (no draft probabilities), odd vocabulary.
        dict(name="verify lookup", op="verify", batch=32, nodes_lo=1, nodes_hi=9, vocab=32003, fan=2, draft=False,
             greedy_every=4),
        # One user: a tree of 8, a few rows to move.
        dict(name="compact one user", op="compact", batch=1, nodes_lo=8, nodes_hi=8, layers=28, kv_heads=8),
        # A loaded server: trees of up to 32 nodes.
        dict(name="compact batch", op="compact", batch=64, nodes_lo=8, nodes_hi=32, layers=28, kv_heads=8),
        # One fork: the parent's half-filled last page.
        dict(name="copy one fork", op="copy", pairs=1, layers=28, kv_heads=8, whole=False),
        # Sixteen pages copied whole.
        dict(name="copy pages", op="copy", pairs=16, layers=28, kv_heads=8, whole=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "verify", "verify", "compact", "copy"])
    if op == "tree":
        q_heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 1), (14, 2), (12, 12), (40, 8)])
        nodes = _log(rng, 1, 64)
        ctx = _log(rng, 1, 32768)
        nodes = min(nodes, max(1, 120_000_000 // (max(ctx, 128) * q_heads)))
        # bounded by the cache's size and, for wide trees, by the products
        most = min(96, 2_000_000 // (max(ctx, 128) * kv_heads), 120_000_000 // (max(ctx, 128) * nodes * q_heads))
        batch = _log(rng, 1, max(1, most))
        return dict(op=op, batch=batch, ctx_lo=rng.randint(max(0, ctx // 2), ctx), ctx_hi=ctx,
                    nodes_lo=rng.randint(1, nodes), nodes_hi=nodes, q_heads=q_heads, kv_heads=kv_heads)
    if op == "verify":
        vocab = _log(rng, 1000, 151936)
        nodes = _log(rng, 1, 24)
        batch = _log(rng, 1, max(1, min(64, 64 * 8 * 151936 // (nodes * vocab * 2))))
        return dict(op=op, batch=batch, nodes_lo=rng.randint(1, nodes), nodes_hi=nodes, vocab=vocab,
                    fan=rng.choice([1, 1, 2, 4]), draft=rng.random() < 0.6, greedy_every=rng.choice([0, 0, 2, 5]))
    if op == "compact":
        return dict(op=op, batch=_log(rng, 1, 64), nodes_lo=rng.randint(1, 8), nodes_hi=rng.randint(8, 32),
                    layers=rng.randint(1, 28), kv_heads=rng.choice([1, 2, 4, 8]))
    return dict(op=op, pairs=_log(rng, 1, 16), layers=rng.randint(1, 28), kv_heads=rng.choice([1, 2, 4, 8]),
                whole=rng.random() < 0.5)


# ------------------------------------------------------------- sizes of a case
def _sizes(case):
    """Node counts and contexts of a case's sequences: by the case alone, so that its work is one number."""
    r = np.random.RandomState((case.get("batch", 1) * 7919 + case.get("nodes_hi", 0) * 31 + case.get("ctx_hi", 0)) % (2 ** 31))
    b = case["batch"]
    nodes = r.randint(case["nodes_lo"], case["nodes_hi"] + 1, b)
    ctx = r.randint(case.get("ctx_lo", 0), case.get("ctx_hi", 0) + 1, b)
    accepted = (nodes * r.uniform(0.1, 0.7, b)).astype(np.int64)  # drafts kept by a step
    accepted = np.minimum(accepted, nodes - 1)
    return nodes.astype(np.int64), ctx.astype(np.int64), accepted


def _copy_rows(case):
    if case["whole"]:
        return np.full(case["pairs"], PAGE, np.int64)
    return np.random.RandomState(case["pairs"]).randint(1, PAGE, case["pairs"]).astype(np.int64)


def work(case):
    if case["op"] == "tree":
        nodes, ctx, _ = _sizes(case)
        kv = int((ctx + nodes).sum())
        rows = int(nodes.sum())
        qh, kvh = case["q_heads"], case["kv_heads"]
        words = (case["nodes_hi"] + 63) // 64
        visible = float((nodes * ctx).sum() + (nodes * (nodes + 1) / 2).sum())  # a chain's pairs
        return {"bytes": kv * kvh * DIM * 4 + rows * qh * (DIM * 4 + 4) + rows * words * 8,
                "flops": 4.0 * DIM * qh * visible}
    if case["op"] == "verify":
        # the target's and the draft's row of every node that has children, the target's alone where nothing was drafted
        nodes, _, _ = _sizes(case)
        inner = [len(set(p[1:].tolist())) for p in _topology(case)]
        read = sum(max(1, i) + (i if case["draft"] else 0) for i in inner)
        return {"bytes": read * case["vocab"] * 2 + int(nodes.sum()) * 24 + case["batch"] * (8 + 8 * case["nodes_hi"]),
                "flops": read * case["vocab"] * 4.0}
    if case["op"] == "compact":
        _, _, accepted = _sizes(case)
        row = case["kv_heads"] * DIM * 2
        return {"bytes": int(accepted.sum()) * case["layers"] * 2 * 2 * row + case["batch"] * 64, "flops": 0}
    return {"bytes": int(_copy_rows(case).sum()) * case["layers"] * 2 * 2 * case["kv_heads"] * DIM * 2, "flops": 0}


# ------------------------------------------------------------------- prepare
def _parents(rng, n, fan):
    """Parent of each node of a tree in an order where parents come first; fan 1 is a chain."""
    return np.array([-1] + [rng.randint(max(0, i - fan), i) for i in range(1, n)], np.int64)


def _topology(case):
    """The trees of a verify case: by the case alone, as its work goes by which nodes have children."""
    nodes, _, _ = _sizes(case)
    rng = np.random.RandomState(case["batch"] * 131 + case["nodes_hi"])
    return [_parents(rng, n, case["fan"]) for n in nodes]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _cu(nodes):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)).cuda()


def prepare(case, seed):
    return {"tree": _prepare_tree, "verify": _prepare_verify, "compact": _prepare_compact,
            "copy": _prepare_copy}[case["op"]](case, seed)


def _prepare_tree(case, seed):
    nodes, ctx, _ = _sizes(case)
    rng, g = np.random.RandomState(seed % (2 ** 31)), _generator(seed)
    b, qh, kvh = case["batch"], case["q_heads"], case["kv_heads"]
    words = (case["nodes_hi"] + 63) // 64
    pages = (ctx + nodes + PAGE - 1) // PAGE
    blocks, stride = int(pages.sum()), int(pages.max())
    order = rng.permutation(blocks)
    table, at = np.full((b, stride), -1, np.int32), 0
    for i in range(b):
        table[i, :pages[i]] = order[at:at + pages[i]]
        at += pages[i]
    rows = int(nodes.sum())
    mask, r = np.zeros((rows, words), np.uint64), 0
    for n in nodes:
        p = _parents(rng, n, 4)
        for i in range(n):
            if i:
                mask[r + i] = mask[r + p[i]]
            mask[r + i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
        r += n

    def values(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 0.5).to(torch.bfloat16)

    return dict(op="tree", case=case, q=values(rows, qh, DIM) * 4, k=values(blocks, PAGE, kvh, DIM),
                v=values(blocks, PAGE, kvh, DIM), table=torch.from_numpy(table).cuda(),
                mask=torch.from_numpy(mask.view(np.int64)).cuda(), cu_q=_cu(nodes),
                lens=torch.from_numpy((ctx + nodes).astype(np.int32)).cuda(), max_q=int(nodes.max()),
                max_k=int((ctx + nodes).max()), out=torch.zeros(rows, qh, DIM, dtype=torch.bfloat16, device="cuda"),
                lse=torch.zeros(rows, qh, device="cuda"))


def _prepare_verify(case, seed):
    nodes, _, _ = _sizes(case)
    rng, g = np.random.RandomState(seed % (2 ** 31)), _generator(seed)
    b, vocab, rows = case["batch"], case["vocab"], int(nodes.sum())
    parents = _topology(case)
    temps = rng.uniform(0.5, 1.2, b).astype(np.float32)
    temps[::2] = 1.0
    if case["greedy_every"]:
        temps[::case["greedy_every"]] = 0.0
    base = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
    logits = base.to(torch.bfloat16)
    draft = (base + torch.randn(rows, vocab, generator=g, device="cuda") * 0.7).to(torch.bfloat16)
    # The drafts of one node are drawn without replacement from the draft's probabilities: the highest of
    # logit / temperature + Gumbel noise, in that order (the highest logits where the temperature is 0).
    kids = max(1, int(max(np.bincount(p[1:]).max() if len(p) > 1 else 1 for p in parents)))
    row_t = torch.from_numpy(np.repeat(temps, nodes)).cuda()[:, None]
    noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)))
    top = torch.topk(draft.float() + noise * row_t, kids, dim=1).indices.cpu().numpy()
    tokens, depth, at = np.zeros(rows, np.int32), 0, 0
    for p in parents:
        seen, level = {}, np.zeros(len(p), np.int64)
        for i in range(1, len(p)):
            k = seen.get(p[i], 0)
            seen[p[i]] = k + 1
            tokens[at + i] = top[at + p[i], k]
            level[i] = level[p[i]] + 1
        depth = max(depth, int(level.max()))
        at += len(p)
    return dict(op="verify", case=case, logits=logits, draft=draft if case["draft"] else None,
                tokens=torch.from_numpy(tokens).cuda(),
                parents=torch.from_numpy(np.concatenate(parents).astype(np.int32)).cuda(),
                uniforms=torch.rand(rows, generator=g, device="cuda"),
                seeds=torch.randint(-2 ** 63, 2 ** 63 - 1, (rows,), generator=g, device="cuda"),
                temps=torch.from_numpy(temps).cuda(), cu_q=_cu(nodes), max_q=int(nodes.max()), kids=kids, depth=depth,
                out_tokens=torch.zeros(b, int(nodes.max()), dtype=torch.int32, device="cuda"),
                path=torch.zeros(b, int(nodes.max()), dtype=torch.int32, device="cuda"),
                counts=torch.zeros(b, dtype=torch.int32, device="cuda"),
                prob=torch.zeros(rows, device="cuda"))


def _caches(case, blocks, seed):
    """K and V caches of every layer, views of one allocation [layers, 2, blocks, page, kv_heads, 128], and the handle
    that a program makes of its caches once."""
    all_layers = torch.empty(case["layers"], 2, blocks, PAGE, case["kv_heads"], DIM, dtype=torch.bfloat16,
                             device="cuda")
    all_layers.normal_(generator=_generator(seed))
    handle = _package().CacheLayers([x[0] for x in all_layers], [x[1] for x in all_layers]) if own else None
    return all_layers, handle


def _prepare_compact(case, seed):
    nodes, _, accepted = _sizes(case)
    rng = np.random.RandomState(seed % (2 ** 31))
    b = case["batch"]
    # Every sequence shares the prompt's cached first page and writes in its own second one and, where the tree
    # crosses the border, its third.
    ctx = PAGE + rng.randint(0, PAGE, b)
    pages = (ctx + nodes + PAGE - 1) // PAGE
    blocks = 1 + 2 * b
    order, table = rng.permutation(blocks), np.full((b, 3), -1, np.int32)
    for i in range(b):
        table[i, :pages[i]] = [order[0], order[1 + 2 * i], order[2 + 2 * i]][:pages[i]]
    path = np.full((b, int(nodes.max())), -1, np.int32)
    for i in range(b):
        path[i, 0] = 0
        path[i, 1:1 + accepted[i]] = np.sort(rng.permutation(np.arange(1, nodes[i]))[:accepted[i]])
    whole, layers = _caches(case, blocks, seed)
    return dict(op="compact", case=case, whole=whole, layers=layers, table=torch.from_numpy(table).cuda(),
                cu_q=_cu(nodes), lens=torch.from_numpy((ctx + nodes).astype(np.int32)).cuda(),
                path=torch.from_numpy(path).cuda(), counts=torch.from_numpy((accepted + 1).astype(np.int32)).cuda(),
                blocks=blocks, new_lens=torch.zeros(b, dtype=torch.int32, device="cuda"))


def _prepare_copy(case, seed):
    rng, pairs = np.random.RandomState(seed % (2 ** 31)), case["pairs"]
    blocks = 2 * pairs + 3
    order = rng.permutation(blocks)
    whole, layers = _caches(case, blocks, seed)
    rows = None if case["whole"] else torch.from_numpy(_copy_rows(case).astype(np.int32)).cuda()
    return dict(op="copy", case=case, whole=whole, layers=layers, blocks=blocks, rows=rows,
                src=torch.from_numpy(order[:pairs].astype(np.int32)).cuda(),
                dst=torch.from_numpy(order[pairs:2 * pairs].astype(np.int32)).cuda())


# ----------------------------------------------------------------------- run
def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def run(st):
    if own:
        return {"tree": _own_tree, "verify": _own_verify, "compact": _own_compact, "copy": _own_copy}[st["op"]](st)
    return {"tree": _plain_tree, "verify": _plain_verify, "compact": _plain_compact, "copy": _plain_copy}[st["op"]](st)


def _own_tree(st):
    nvb, c = _package(), st["case"]
    stride, blocks = st["table"].shape[1], st["k"].shape[0]
    splits = nvb.tree_num_splits(c["batch"], st["max_q"], c["q_heads"], c["kv_heads"], st["max_k"])
    lse_accum, out_accum = nvb.tree_scratch(splits, st["q"].shape[0], c["q_heads"], st["q"].device)
    nvb.paged_tree_fwd(st["q"], st["k"], st["v"], st["out"], st["cu_q"], st["lens"], st["table"], st["mask"],
                       batch=c["batch"], max_q=st["max_q"], max_k=st["max_k"], q_heads=c["q_heads"],
                       kv_heads=c["kv_heads"], block_size=PAGE, table_stride=stride, num_blocks=blocks,
                       num_splits=splits, lse=st["lse"], lse_accum=lse_accum, out_accum=out_accum)
    return st["out"], st["lse"]


def _own_verify(st):
    model = _package().model
    model.layer_verify(st["logits"], st["draft"], st["tokens"], st["parents"], st["uniforms"], st["seeds"],
                       st["temps"], st["cu_q"], st["out_tokens"], st["path"], st["counts"], st["prob"])
    return st["out_tokens"], st["path"], st["counts"], st["prob"]


def _own_compact(st):
    _package().cache_compact_paths(st["layers"], st["cu_q"], st["lens"], st["table"], st["path"], st["counts"],
                                   st["new_lens"])
    return st["whole"], st["new_lens"]


def _own_copy(st):
    _package().cache_copy_pages(st["layers"], st["src"], st["dst"], st["rows"])
    return st["whole"]


# --------------------------------------------------------------- plain forms
def _sequence_of_rows(cu_q, rows):
    return torch.searchsorted(cu_q[1:], torch.arange(rows, device=cu_q.device, dtype=cu_q.dtype), right=True)


def _plain_tree(st):
    c, max_q = st["case"], st["max_q"]
    b, qh, kvh, rows = c["batch"], c["q_heads"], c["kv_heads"], st["q"].shape[0]
    group = qh // kvh
    n = (st["cu_q"][1:] - st["cu_q"][:-1]).long()
    ctx = st["lens"].long() - n
    span = st["table"].shape[1] * PAGE
    pages = st["table"].long().clamp_min(0)
    k = st["k"][pages].view(b, span, kvh, DIM).permute(0, 2, 3, 1).float()    # [b, kvh, dim, key]
    v = st["v"][pages].view(b, span, kvh, DIM).permute(0, 2, 1, 3).float()    # [b, kvh, key, dim]
    key = torch.arange(span, device="cuda")
    node = torch.arange(max_q, device="cuda")
    row = (st["cu_q"][:-1].long()[:, None] + node).clamp_max(rows - 1)         # [b, node]
    q = st["q"][row].float().view(b, max_q, kvh, group, DIM).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, DIM)
    # key `at` of the tree is visible where the row's mask has its bit
    at = key[None, :] - ctx[:, None]                                           # [b, key]
    word = st["mask"][row].gather(2, (at.clamp(0, max_q - 1) // 64)[:, None, :].expand(b, max_q, span))
    bit = (word >> (at.clamp_min(0) % 64)[:, None, :]) & 1
    seen = (at < 0)[:, None, :] | ((bit == 1) & (at >= 0)[:, None, :] & (at < n[:, None])[:, None, :])
    seen = seen & (st["table"] >= 0).repeat_interleave(PAGE, 1)[:, None, :]
    score = (q @ k) * (1.0 / math.sqrt(DIM))
    score = score.view(b, kvh, max_q, group, span).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    score = torch.exp_(score - top)
    total = score.sum(-1, keepdim=True)
    o = (score.view(b, kvh, -1, span) @ v).view(b, kvh, max_q, group, DIM) / total.clamp_min(1e-30)
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf))
    o = o.permute(0, 2, 1, 3, 4).reshape(b, max_q, qh, DIM)
    lse = lse.squeeze(-1).permute(0, 2, 1, 3).reshape(b, max_q, qh)
    real = node[None, :] < n[:, None]
    st["out"].copy_(o[real].to(torch.bfloat16))
    st["lse"].copy_(lse[real])
    return st["out"], st["lse"]


def _mix(x):
    """SplitMix64 of int64 words (products and sums wrap)."""
    def shift(v, n):
        return (v >> n) & ((1 << (64 - n)) - 1)

    x = x + (0x9e3779b97f4a7c15 - 2 ** 64)
    x = (x ^ shift(x, 30)) * (0xbf58476d1ce4e5b9 - 2 ** 64)
    x = (x ^ shift(x, 27)) * (0x94d049bb133111eb - 2 ** 64)
    return x ^ shift(x, 31)


def _gumbel(seeds, vocab):
    """The sampler's noise for each seed and token, in 64 bits: what is drawn goes by the highest of close scores."""
    token = torch.arange(vocab, device=seeds.device, dtype=torch.int64) * (0xd2b74407b1ce6e93 - 2 ** 64)
    bits = (_mix(seeds[:, None] ^ token[None, :]) >> 41) & (2 ** 23 - 1)
    return -torch.log(-torch.log((bits.double() + 0.5) / 2 ** 23))


def _softmax(logits, temperature):
    x = torch.exp((logits - logits.amax(1, keepdim=True)) / temperature)
    return x / x.sum(1, keepdim=True)


def _plain_verify(st):
    rows, vocab = st["logits"].shape
    b, dev = st["cu_q"].numel() - 1, st["logits"].device
    seq = _sequence_of_rows(st["cu_q"], rows)
    first = st["cu_q"][:-1].long()
    index = torch.arange(rows, device=dev)
    t = st["temps"][seq]
    greedy = t == 0
    scale = torch.where(greedy, torch.ones_like(t), t)[:, None]
    logits = st["logits"].float()
    p = _softmax(logits, scale)
    q = _softmax(st["draft"].float(), scale) if st["draft"] is not None else None
    best = logits.argmax(1)
    # child[r, i]: the row of r's child number i, or -1
    root = index == first[seq]
    parent = torch.where(root, torch.full_like(index, -1), first[seq] + st["parents"].long())
    same = (parent[:, None] == parent[None, :]) & (index[None, :] < index[:, None])
    child = torch.full((rows + 1, st["kids"]), -1, device=dev, dtype=torch.int64)
    child[parent, same.sum(1).clamp_max(st["kids"] - 1)] = index  # a root's goes into the row behind the last
    child = child[:rows]
    prob = torch.zeros(rows + 1, device=dev)  # what no child is tested for goes behind the last row
    winner = torch.full((rows,), -1, device=dev, dtype=torch.int64)
    rejected = torch.zeros(rows, device=dev, dtype=torch.int64)
    for i in range(st["kids"]):
        c = child[:, i]
        live = (c >= 0) & (winner < 0)
        token = st["tokens"][c.clamp_min(0)].long()[:, None]
        pt = p.gather(1, token)[:, 0]
        qt = q.gather(1, token)[:, 0] if q is not None else torch.ones_like(pt)
        a = torch.where(pt > 0, torch.where(qt > 0, (pt / qt).clamp_max(1.0), torch.ones_like(pt)), torch.zeros_like(pt))
        a = torch.where(greedy, (token[:, 0] == best).float(), a)
        prob[torch.where(live, c, torch.full_like(c, rows))] = a
        taken = live & (st["uniforms"][c.clamp_min(0)] < a)
        winner = torch.where(taken, c, winner)
        lost = live & ~taken
        rejected = rejected + lost
        left = (p - q).clamp_min_(0) if q is not None else p.scatter(1, token, 0.0)
        total = left.sum(1, keepdim=True)
        p = torch.where(lost[:, None] & (total > 0), left / total, p)
        if q is not None:
            rest = q.scatter(1, token, 0.0)
            mass = rest.sum(1, keepdim=True)
            q = torch.where(lost[:, None], torch.where(mass > 0, rest / mass, rest), q)
    # from the root along the accepted children
    at, alive = first.clone(), torch.ones(b, device=dev, dtype=torch.bool)
    st["path"].fill_(-1)
    st["out_tokens"].fill_(-1)
    st["path"][:, 0] = 0
    count = torch.ones(b, device=dev, dtype=torch.int64)
    for d in range(st["depth"]):
        nxt = winner[at]
        alive = alive & (nxt >= 0)
        at = torch.where(alive, nxt, at)
        count = count + alive
        st["path"][:, d + 1] = torch.where(alive, at - first, torch.full_like(at, -1)).int()
        st["out_tokens"][:, d] = torch.where(alive, st["tokens"][at], torch.full_like(at, -1).int())
    score = torch.where((rejected[at] == 0)[:, None], logits[at].double() / scale[at].double(), torch.log(p[at].double()))
    drawn = torch.where(greedy[at], best[at], (score + _gumbel(st["seeds"][at], vocab)).argmax(1))
    st["out_tokens"].scatter_(1, (count - 1)[:, None], drawn.int()[:, None])
    st["counts"].copy_(count)
    st["prob"].copy_(prob[:rows])
    return st["out_tokens"], st["path"], st["counts"], st["prob"]


def _plain_compact(st):
    c = st["case"]
    n = (st["cu_q"][1:] - st["cu_q"][:-1]).long()
    ctx = st["lens"].long() - n
    d = torch.arange(st["path"].shape[1], device="cuda")
    moved = (d[None, :] >= 1) & (d[None, :] < st["counts"][:, None])

    def slots(position):
        page = st["table"].gather(1, (position // PAGE).clamp_max(st["table"].shape[1] - 1)).long()
        return (page * PAGE + position % PAGE)[moved]

    src, dst = slots(ctx[:, None] + st["path"].long().clamp_min(0)), slots(ctx[:, None] + d[None, :])
    flat = st["whole"].view(c["layers"] * 2, -1, c["kv_heads"] * DIM)
    flat[:, dst] = flat[:, src]
    st["new_lens"].copy_(ctx + st["counts"])
    return st["whole"], st["new_lens"]


def _plain_copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    if st["rows"] is None:
        st["whole"][:, :, dst] = st["whole"][:, :, src]
        return st["whole"]
    part = torch.arange(PAGE, device="cuda")[None, :] < st["rows"][:, None]
    at = torch.arange(PAGE, device="cuda")[None, :]
    flat = st["whole"].view(st["whole"].shape[0] * 2, -1, st["case"]["kv_heads"] * DIM)
    flat[:, (dst[:, None] * PAGE + at)[part]] = flat[:, (src[:, None] * PAGE + at)[part]]
    return st["whole"]


# ------------------------------------------------------------ 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_tree, "verify": _exact_verify, "compact": _exact_compact, "copy": _exact_copy}[case["op"]](st)


def _exact_tree(st):
    c = st["case"]
    group = c["q_heads"] // c["kv_heads"]
    cu, lens, mask = st["cu_q"].tolist(), st["lens"].tolist(), st["mask"].cpu().numpy().view(np.uint64)
    outs, lses = [], []
    for s in range(c["batch"]):
        n, length = cu[s + 1] - cu[s], lens[s]
        pages = st["table"][s, :(length + PAGE - 1) // PAGE].long()
        k = st["k"][pages].reshape(-1, c["kv_heads"], DIM)[:length].double()
        v = st["v"][pages].reshape(-1, c["kv_heads"], DIM)[:length].double()
        q = st["q"][cu[s]:cu[s + 1]].double().reshape(n, c["kv_heads"], group, DIM)
        x = torch.einsum("nhgd,khd->nhgk", q, k) / math.sqrt(DIM)
        bits = np.unpackbits(mask[cu[s]:cu[s + 1]].view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        hidden = torch.zeros(n, length, dtype=torch.bool, device="cuda")
        hidden[:, length - n:] = ~torch.from_numpy(bits).cuda()
        x = x.masked_fill(hidden[:, None, None, :], -math.inf)
        lse = torch.logsumexp(x, -1)
        outs.append(torch.einsum("nhgk,khd->nhgd", torch.exp(x - lse[..., None]), v).reshape(n, -1, DIM))
        lses.append(lse.reshape(n, -1))
    return torch.cat(outs), torch.cat(lses)


def _exact_verify(st):
    """The probabilities of acceptance, node by node; the whole numbers go by comparison with the plain form."""
    cu, temps = st["cu_q"].tolist(), st["temps"].tolist()
    parents, tokens = st["parents"].tolist(), st["tokens"].tolist()
    uniforms = st["uniforms"].double().tolist()
    prob = [0.0] * len(tokens)
    for s, temperature in enumerate(temps):
        kids = {}
        for r in range(cu[s] + 1, cu[s + 1]):
            kids.setdefault(cu[s] + parents[r], []).append(r)
        for node, rows in kids.items():
            x = st["logits"][node].double()
            if temperature == 0:
                best = int((x == x.max()).nonzero()[0, 0])
                for r in rows:
                    prob[r] = float(tokens[r] == best)
                    if prob[r] == 1.0:
                        break
                continue
            p = torch.softmax(x / temperature, 0)
            q = torch.softmax(st["draft"][node].double() / temperature, 0) if st["draft"] is not None else None
            gone = []
            for r in rows:
                t = tokens[r]
                have, asked = float(p[t]), (0.0 if t in gone else float(q[t])) if q is not None else 1.0
                prob[r] = 0.0 if have <= 0 else (min(1.0, have / asked) if asked > 0 else 1.0)
                if uniforms[r] < prob[r]:
                    break
                if r == rows[-1]:
                    continue
                if q is None:
                    left = p.clone()
                    left[t] = 0
                else:
                    left = torch.relu(p - q)
                if float(left.sum()) > 0:
                    p = left / left.sum()
                gone.append(t)
                if q is not None:
                    q = q.clone()
                    q[t] = 0
                    q = q / q.sum() if float(q.sum()) > 0 else q
    return None, None, None, torch.tensor(prob, dtype=torch.float64)


def _exact_compact(st):
    cu, lens, table = st["cu_q"].tolist(), st["lens"].tolist(), st["table"].tolist()
    counts, path = st["counts"].tolist(), st["path"].tolist()
    source = torch.arange(st["blocks"] * PAGE)
    for s, count in enumerate(counts):
        ctx = lens[s] - (cu[s + 1] - cu[s])
        for d in range(1, count):
            a, z = ctx + path[s][d], ctx + d
            source[table[s][z // PAGE] * PAGE + z % PAGE] = table[s][a // PAGE] * PAGE + a % PAGE
    c = st["case"]
    flat = st["whole"].view(c["layers"] * 2, -1, c["kv_heads"] * DIM)
    return torch.index_select(flat, 1, source.cuda()).view(st["whole"].shape), None


def _exact_copy(st):
    source = torch.arange(st["blocks"] * PAGE).view(-1, PAGE)
    rows = st["rows"].tolist() if st["rows"] is not None else [PAGE] * len(st["src"])
    before = source.clone()
    for a, z, n in zip(st["src"].tolist(), st["dst"].tolist(), rows):
        source[z, :n] = before[a, :n]
    flat = st["whole"].view(st["case"]["layers"] * 2, -1, st["case"]["kv_heads"] * DIM)
    return torch.index_select(flat, 1, source.view(-1).cuda()).view(st["whole"].shape)
