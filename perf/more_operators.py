"""Measured cases of the latent-attention operators.

A cache with one latent vector a token holds, for every token, 512 normalised
latent values and 64 rotated key values shared by all heads. Four operators
write it and read it:

  store    a step's latents normalised, its key parts rotated, both appended
           to the pages; the queries' rotary parts rotated on the way
           (``latent_store``)
  gather   the cached rows of sequences made contiguous, for the projection
           that expands them into keys and values (``latent_gather``)
  latent   absorbed form: attention of a few queries a sequence over the pages
           themselves, keys 576 wide, values their first 512
           (``paged_latent_fwd``)
  prompt   expanded form: causal attention of prompts or chunks over expanded
           keys (128 a head and the shared 64) and values (128 a head)
           (``latent_prefill_fwd``)

With ``own`` false ``run`` computes them from elementary torch operations;
with ``own`` true it calls the library. Head counts, contexts and batches are
those of the repository's benchmark configurations (16, 32 and 64 query heads,
128 to 32,768 tokens) and generic ones.
"""
import math

import numpy as np
import torch

own = False

LATENT = 512          # latent values a token: the values, and the first part of the keys
ROPE = 64             # rotated values a token, and of each query head
WIDTH = LATENT + ROPE
NOPE = 128            # unrotated part of an expanded key; an expanded value is as wide
POSITIONS = 32768
SCALE = 1.0 / math.sqrt(NOPE + ROPE)


def listed():
    return [
        # One chat, a decode step: launch latency.
        dict(name="latent one chat", op="latent", batch=1, ctx_lo=500, ctx_hi=500, q_lo=1, q_hi=1, heads=16, page=256),
        # An engine's batch at ragged contexts.
        dict(name="latent engine batch", op="latent", batch=32, ctx_lo=128, ctx_hi=1024, q_lo=1, q_hi=1, heads=16,
             page=256),
        # A loaded server, all heads on one GPU.
        dict(name="latent loaded server", op="latent", batch=64, ctx_lo=3900, ctx_hi=4200, q_lo=1, q_hi=1, heads=64,
             page=64),
        # Few users with long documents.
        dict(name="latent long documents", op="latent", batch=4, ctx_lo=32000, ctx_hi=32700, q_lo=1, q_hi=1, heads=32,
             page=256),
        # Steps that verify drafted chains of different lengths, mixed contexts.
        dict(name="latent drafts", op="latent", batch=16, ctx_lo=500, ctx_hi=8000, q_lo=2, q_hi=6, heads=32, page=128),
        # One short prompt.
        dict(name="prompt short", op="prompt", batch=1, ctx_lo=0, ctx_hi=0, q_lo=300, q_hi=300, heads=16),
        # Prompts of mixed lengths.
        dict(name="prompts ragged", op="prompt", batch=32, ctx_lo=0, ctx_hi=0, q_lo=64, q_hi=2048, heads=16),
        # Chunks of long prompts behind their cached part.
        dict(name="prompt chunks", op="prompt", batch=4, ctx_lo=4000, ctx_hi=8000, q_lo=500, q_hi=512, heads=32),
        # A decode step's append.
        dict(name="store decode", op="store", rows=64, heads=16, interleaved=True, absorbed=True, page=256),
        # A prefill forward's append.
        dict(name="store prefill", op="store", rows=8191, heads=32, interleaved=False, absorbed=False, page=64),
        # One cached prefix.
        dict(name="gather one prefix", op="gather", batch=1, len_lo=1000, len_hi=1000, page=64),
        # The cached parts of a batch of chunks.
        dict(name="gather chunks", op="gather", batch=32, len_lo=1000, len_hi=8000, page=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["latent", "latent", "latent", "prompt", "prompt", "store", "gather"])
    page = rng.choice([64, 128, 256])
    if op == "latent":
        heads = rng.choice([16, 16, 32, 64, 128, 8, 20, 1])
        queries = _log(rng, 1, 8)
        ctx = _log(rng, 1, 32700)
        # bounded by the cache's size and by the products of the largest listed case
        queries = max(1, min(queries, 16_000_000 // (max(ctx, 64) * heads)))
        most = min(200, 250_000 // max(ctx, 64), 16_000_000 // (max(ctx, 64) * queries * heads))
        batch = _log(rng, 1, max(1, most))
        return dict(op=op, batch=batch, ctx_lo=rng.randint(ctx // 2, ctx), ctx_hi=ctx, q_lo=rng.randint(1, queries),
                    q_hi=queries, heads=heads, page=page)
    if op == "prompt":
        heads = rng.choice([16, 32, 64, 8, 5])
        queries = _log(rng, 1, 2048)
        ctx = rng.choice([0, 0, _log(rng, 1, 8000)])
        # bounded by the pairs of the largest listed case, and by the size of the expanded keys and values
        queries = max(1, min(queries, 300_000_000 // ((ctx + queries) * heads)))
        most = min(32, 300_000_000 // ((ctx + queries) * queries * heads), 700_000 // ((ctx + queries) * heads))
        batch = _log(rng, 1, max(1, most))
        return dict(op=op, batch=batch, ctx_lo=rng.randint(ctx // 2, ctx), ctx_hi=ctx,
                    q_lo=rng.randint((queries + 1) // 2, queries), q_hi=queries, heads=heads)
    if op == "store":
        return dict(op=op, rows=_log(rng, 1, 8191), heads=rng.choice([16, 32, 8, 5]),
                    interleaved=rng.random() < 0.5, absorbed=rng.random() < 0.5, page=page)
    most = _log(rng, 1, 8000)
    return dict(op=op, batch=_log(rng, 1, min(32, 140_000 // most)), len_lo=rng.randint(most // 2, most), len_hi=most,
                page=page)


# ------------------------------------------------------------- sizes of a case
def _sizes(case):
    """Query counts and contexts of a case's sequences: by the case alone, so that its work is one number."""
    r = np.random.RandomState((case["batch"] * 7919 + case.get("q_hi", 0) * 31 + case.get("ctx_hi", 0)
                               + case.get("len_hi", 0)) % (2 ** 31))
    b = case["batch"]
    if case["op"] == "gather":
        return None, r.randint(case["len_lo"], case["len_hi"] + 1, b).astype(np.int64)
    return (r.randint(case["q_lo"], case["q_hi"] + 1, b).astype(np.int64),
            r.randint(case["ctx_lo"], case["ctx_hi"] + 1, b).astype(np.int64))


def work(case):
    if case["op"] == "store":
        q_values = case["rows"] * case["heads"] * ROPE
        return {"bytes": case["rows"] * WIDTH * 4 + q_values * 4 + LATENT * 2 + case["rows"] * (8 + ROPE * 4),
                "flops": case["rows"] * LATENT * 4.0 + (q_values + case["rows"] * ROPE) * 3.0}
    n, ctx = _sizes(case)
    if case["op"] == "gather":
        return {"bytes": int(ctx.sum()) * WIDTH * 4, "flops": 0}
    pairs = float((n * ctx).sum() + (n * (n + 1) / 2).sum()) * case["heads"]
    rows, keys = int(n.sum()) * case["heads"], int((ctx + n).sum())
    if case["op"] == "latent":
        return {"bytes": keys * WIDTH * 2 + rows * (WIDTH * 2 + LATENT * 2 + 4), "flops": 2.0 * (WIDTH + LATENT) * pairs}
    return {"bytes": keys * (case["heads"] * 2 * NOPE + ROPE) * 2 + rows * ((NOPE + ROPE) * 2 + NOPE * 2 + 4),
            "flops": 2.0 * (2 * NOPE + ROPE) * pairs}


# ------------------------------------------------------------------- prepare
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _values(g, std, *shape):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _up(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _cu(counts):
    return _up(np.concatenate([[0], np.cumsum(counts)]))


def _pages(rng, lens, page):
    """Page table of sequences of these lengths, their pages in random order, and the number of pages."""
    pages = (lens + page - 1) // page
    blocks = int(pages.sum()) + 1
    order, at = rng.permutation(blocks), 0
    table = np.full((len(lens), max(1, int(pages.max()))), -1, np.int32)
    for i, m in enumerate(pages):
        table[i, :m] = order[at:at + m]
        at += m
    return table, blocks


def _rope_table():
    """cos | sin of every position and pair, positions stretched by 4 for long contexts, angles in 64 bits."""
    pair = torch.arange(ROPE // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None] / 4.0 * 10000.0 ** (-2.0 * pair / ROPE)
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def prepare(case, seed):
    return {"latent": _prepare_latent, "prompt": _prepare_prompt, "store": _prepare_store,
            "gather": _prepare_gather}[case["op"]](case, seed)


def _prepare_latent(case, seed):
    n, ctx = _sizes(case)
    rng, g = np.random.RandomState(seed % (2 ** 31)), _generator(seed)
    table, blocks = _pages(rng, ctx + n, case["page"])
    rows, heads = int(n.sum()), case["heads"]
    st = dict(op="latent", case=case, q=_values(g, 1.0, rows, heads, WIDTH),
              cache=_values(g, 1.0, blocks, case["page"], WIDTH), table=_up(table), cu_q=_cu(n), lens=_up(ctx + n),
              max_q=int(n.max()), out=torch.zeros(rows, heads, LATENT, dtype=torch.bfloat16, device="cuda"),
              lse=torch.zeros(rows, heads, device="cuda"))
    if own:
        st["scratch"] = _package().latent_scratch("cuda")  # as a program keeps it
    return st


def _prepare_prompt(case, seed):
    n, ctx = _sizes(case)
    g, heads = _generator(seed), case["heads"]
    rows, keys = int(n.sum()), int((ctx + n).sum())
    return dict(op="prompt", case=case, q=_values(g, 1.5, rows, heads, NOPE + ROPE),
                kv=_values(g, 1.0, keys, heads, 2 * NOPE), rope=_values(g, 1.0, keys, ROPE), cu_q=_cu(n),
                cu_k=_cu(ctx + n), max_q=int(n.max()),
                out=torch.zeros(rows, heads, NOPE, dtype=torch.bfloat16, device="cuda"),
                lse=torch.zeros(rows, heads, device="cuda"))


def _prepare_store(case, seed):
    rng, g = np.random.RandomState(seed % (2 ** 31)), _generator(seed)
    rows, heads, page = case["rows"], case["heads"], case["page"]
    blocks = (rows + page - 1) // page + 3
    slots = rng.permutation(blocks * page)[:rows]
    if not case["absorbed"]:  # a prompt's rows lie one behind the other within their pages
        slots = (rng.permutation(blocks)[:, None] * page + np.arange(page)[None, :]).reshape(-1)[:rows]
    positions = rng.randint(0, POSITIONS, rows) if case["absorbed"] else np.arange(rows) + rng.randint(0, POSITIONS // 2)
    width = WIDTH if case["absorbed"] else NOPE + ROPE
    return dict(op="store", case=case, kv=_values(g, 2.0, rows, WIDTH),
                weight=(1.0 + 0.2 * torch.randn(LATENT, generator=g, device="cuda")).to(torch.bfloat16),
                positions=_up(positions), slots=_up(slots), q=_values(g, 1.0, rows, heads, NOPE + ROPE),
                q_out=_values(g, 1.0, rows, heads, width), cache=_values(g, 1.0, blocks, page, WIDTH),
                rope_table=_rope_table())


def _prepare_gather(case, seed):
    _, lens = _sizes(case)
    rng, g = np.random.RandomState(seed % (2 ** 31)), _generator(seed)
    table, blocks = _pages(rng, lens, case["page"])
    keys = int(lens.sum())
    return dict(op="gather", case=case, cache=_values(g, 1.0, blocks, case["page"], WIDTH), table=_up(table),
                cu_k=_cu(lens), latent=torch.zeros(keys, LATENT, dtype=torch.bfloat16, device="cuda"),
                rope=torch.zeros(keys, ROPE, dtype=torch.bfloat16, device="cuda"))


# ----------------------------------------------------------------------- run
def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def run(st):
    if own:
        return {"latent": _own_latent, "prompt": _own_prompt, "store": _own_store, "gather": _own_gather}[st["op"]](st)
    return {"latent": _plain_latent, "prompt": _plain_prompt, "store": _plain_store,
            "gather": _plain_gather}[st["op"]](st)


def _own_latent(st):
    _package().paged_latent_fwd(st["q"], st["cache"], st["out"], st["cu_q"], st["lens"], st["table"],
                                max_q=st["max_q"], scale=SCALE, scratch=st["scratch"], lse=st["lse"])
    return st["out"], st["lse"]


def _own_prompt(st):
    _package().latent_prefill_fwd(st["q"], st["kv"], st["rope"], st["out"], st["cu_q"], st["cu_k"], max_q=st["max_q"],
                                  scale=SCALE, lse=st["lse"])
    return st["out"], st["lse"]


def _own_store(st):
    _package().latent_store(st["kv"], st["weight"], st["positions"], st["slots"], st["cache"],
                            q=st["q"][..., NOPE:], q_out=st["q_out"][..., -ROPE:], eps=1e-6,
                            rope_table=st["rope_table"], interleaved=st["case"]["interleaved"])
    return st["cache"], st["q_out"]


def _own_gather(st):
    _package().latent_gather(st["cache"], st["table"], st["cu_k"], st["latent"], st["rope"])
    return st["latent"], st["rope"]


# --------------------------------------------------------------- plain forms
def _softmax_rows(score, seen):
    """Probabilities, unnormalised, with their sums and the logarithm of the softmax's denominator."""
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    score = torch.exp_(score - top)
    total = score.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf))
    return score, total.clamp_min(1e-30), lse.squeeze(-1)


def _plain_latent(st):
    c, max_q = st["case"], st["max_q"]
    b, heads, rows, page = c["batch"], c["heads"], st["q"].shape[0], c["page"]
    n = (st["cu_q"][1:] - st["cu_q"][:-1]).long()
    span = st["table"].shape[1] * page
    keys = st["cache"][st["table"].long().clamp_min(0)].view(b, span, WIDTH).float()
    node, key = torch.arange(max_q, device="cuda"), torch.arange(span, device="cuda")
    row = (st["cu_q"][:-1].long()[:, None] + node).clamp_max(rows - 1)
    q = st["q"][row].float().view(b, max_q * heads, WIDTH)
    last = st["lens"].long()[:, None] - n[:, None] + node                       # [b, node]: the last key it sees
    seen = (key <= last[..., None]) & (st["table"] >= 0).repeat_interleave(page, 1)[:, None, :]
    score = ((q @ keys.transpose(1, 2)) * SCALE).view(b, max_q, heads, span)
    score, total, lse = _softmax_rows(score, seen[:, :, None, :])
    o = (score.view(b, -1, span) @ keys[..., :LATENT]).view(b, max_q, heads, LATENT) / total
    real = node[None, :] < n[:, None]
    st["out"].copy_(o[real].to(torch.bfloat16))
    st["lse"].copy_(lse[real])
    return st["out"], st["lse"]


def _plain_prompt(st):
    c, max_q = st["case"], st["max_q"]
    b, heads, rows, keys = c["batch"], c["heads"], st["q"].shape[0], st["kv"].shape[0]
    n, m = (st["cu_q"][1:] - st["cu_q"][:-1]).long(), (st["cu_k"][1:] - st["cu_k"][:-1]).long()
    max_k = c["ctx_hi"] + c["q_hi"]
    node, key = torch.arange(max_q, device="cuda"), torch.arange(max_k, device="cuda")
    row = (st["cu_q"][:-1].long()[:, None] + node).clamp_max(rows - 1)
    col = (st["cu_k"][:-1].long()[:, None] + key).clamp_max(keys - 1)
    q = st["q"][row].permute(0, 2, 1, 3).float()                                # [b, head, query, 192]
    kv = st["kv"][col].permute(0, 2, 1, 3).float()                              # [b, head, key, 256]
    rope = st["rope"][col][:, None].float()                                     # [b, 1, key, 64]
    seen = key[None, None, :] <= (m - n)[:, None, None] + node[None, :, None]
    score = q[..., :NOPE] @ kv[..., :NOPE].transpose(2, 3)
    score += q[..., NOPE:] @ rope.transpose(2, 3)
    score, total, lse = _softmax_rows(score.mul_(SCALE), seen[:, None])
    o = ((score @ kv[..., NOPE:]) / total).permute(0, 2, 1, 3)
    real = node[None, :] < n[:, None]
    st["out"].copy_(o[real].to(torch.bfloat16))
    st["lse"].copy_(lse.permute(0, 2, 1)[real])
    return st["out"], st["lse"]


def _rotate(x, cos, sin, interleaved):
    if interleaved:
        a, z = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - z * sin, z * cos + a * sin], -1).flatten(-2)
    a, z = x[..., :ROPE // 2], x[..., ROPE // 2:]
    return torch.cat([a * cos - z * sin, z * cos + a * sin], -1)


def _plain_store(st):
    table = st["rope_table"][st["positions"].long()]
    cos, sin = table[:, :ROPE // 2], table[:, ROPE // 2:]
    x = st["kv"].float()
    latent = x[:, :LATENT]
    latent = latent * torch.rsqrt((latent * latent).mean(1, keepdim=True) + 1e-6) * st["weight"].float()
    row = torch.cat([latent, _rotate(x[:, LATENT:], cos, sin, st["case"]["interleaved"])], 1)
    st["cache"].view(-1, WIDTH)[st["slots"].long()] = row.to(torch.bfloat16)
    q = st["q"][..., NOPE:].float()
    st["q_out"][..., -ROPE:] = _rotate(q, cos[:, None], sin[:, None], st["case"]["interleaved"]).to(torch.bfloat16)
    return st["cache"], st["q_out"]


def _plain_gather(st):
    page, keys = st["case"]["page"], st["latent"].shape[0]
    index = torch.arange(keys, device="cuda")
    seq = torch.searchsorted(st["cu_k"][1:].long(), index, right=True)
    at = index - st["cu_k"].long()[seq]
    slot = st["table"].long()[seq, at // page] * page + at % page
    row = st["cache"].view(-1, WIDTH)[slot]
    st["latent"].copy_(row[:, :LATENT])
    st["rope"].copy_(row[:, LATENT:])
    return st["latent"], st["rope"]


# ------------------------------------------------------------ 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    return {"latent": _exact_latent, "prompt": _exact_prompt, "store": _exact_store,
            "gather": _exact_gather}[case["op"]](st)


def _exact_attention(q, k, v):
    """q [n, h, d] over k [m, h or 1, d] and v [m, h or 1, e]: the last query sees every key."""
    n, m = q.shape[0], k.shape[0]
    x = torch.einsum("nhd,mhd->nhm", q, k.expand(-1, q.shape[1], -1)) / math.sqrt(NOPE + ROPE)
    ahead = torch.arange(m, device="cuda")[None, :] - (m - n) > torch.arange(n, device="cuda")[:, None]
    x = x.masked_fill(ahead[:, None, :], -math.inf)
    lse = torch.logsumexp(x, -1)
    return torch.einsum("nhm,mhe->nhe", torch.exp(x - lse[..., None]), v.expand(-1, q.shape[1], -1)), lse


def _exact_latent(st):
    cu, lens = st["cu_q"].tolist(), st["lens"].tolist()
    outs, lses = [], []
    for s, length in enumerate(lens):
        pages = st["table"][s, :(length + st["case"]["page"] - 1) // st["case"]["page"]].long()
        k = st["cache"][pages].reshape(-1, WIDTH)[:length].double()
        q = st["q"][cu[s]:cu[s + 1]].double()
        n, heads = q.shape[:2]
        x = (q.reshape(-1, WIDTH) @ k.T).view(n, heads, length) / math.sqrt(NOPE + ROPE)
        ahead = torch.arange(length, device="cuda")[None, :] - (length - n) > torch.arange(n, device="cuda")[:, None]
        x = x.masked_fill(ahead[:, None, :], -math.inf)
        lse = torch.logsumexp(x, -1)
        outs.append((torch.exp(x - lse[..., None]).view(-1, length) @ k[:, :LATENT]).view(n, heads, LATENT))
        lses.append(lse)
    return torch.cat(outs), torch.cat(lses)


def _exact_prompt(st):
    cu_q, cu_k = st["cu_q"].tolist(), st["cu_k"].tolist()
    outs, lses = [], []
    for s in range(len(cu_q) - 1):
        out, lse = [], []
        kv, rope = st["kv"][cu_k[s]:cu_k[s + 1]], st["rope"][cu_k[s]:cu_k[s + 1]].double()[:, None]
        for h in range(st["case"]["heads"]):
            one = kv[:, h:h + 1].double()
            o, x = _exact_attention(st["q"][cu_q[s]:cu_q[s + 1], h:h + 1].double(),
                                    torch.cat([one[..., :NOPE], rope], -1), one[..., NOPE:])
            out.append(o)
            lse.append(x)
        outs.append(torch.cat(out, 1))
        lses.append(torch.cat(lse, 1))
    return torch.cat(outs), torch.cat(lses)


def _exact_store(st):
    position, slots = st["positions"].tolist(), st["slots"].long()
    angles = st["rope_table"].double()[torch.tensor(position, device="cuda")]
    turn = torch.complex(angles[:, :ROPE // 2], angles[:, ROPE // 2:])

    def turned(x, by):
        if st["case"]["interleaved"]:
            return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * by).flatten(-2)
        z = torch.complex(x[..., :ROPE // 2].contiguous(), x[..., ROPE // 2:].contiguous()) * by
        return torch.cat([z.real, z.imag], -1)

    kv = st["kv"].double()
    norm = torch.sqrt(kv[:, :LATENT].square().sum(1, keepdim=True) / LATENT + 1e-6)
    cache = st["cache"].double()
    flat = cache.view(-1, WIDTH)
    flat[slots, :LATENT] = kv[:, :LATENT] / norm * st["weight"].double()
    flat[slots, LATENT:] = turned(kv[:, LATENT:], turn)
    q_out = st["q_out"].double()
    q_out[..., -ROPE:] = turned(st["q"][..., NOPE:].double(), turn[:, None])
    return cache, q_out


def _exact_gather(st):
    cu, page = st["cu_k"].tolist(), st["case"]["page"]
    rows = []
    for s in range(len(cu) - 1):
        length = cu[s + 1] - cu[s]
        pages = st["table"][s, :(length + page - 1) // page].long()
        rows.append(st["cache"][pages].reshape(-1, WIDTH)[:length])
    row = torch.cat(rows).double()
    return row[:, :LATENT], row[:, LATENT:]
