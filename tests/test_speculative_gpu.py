"""The speculative-decoding operators on the GPU against plain 64-bit forms.

Tree attention's tolerance, per element: the output is rounded to BF16 (half a
step, 2^-8 of the value); each probability may be rounded to BF16 before the
product with V (2^-8 of sum p |v|); the scores are FP32 sums of 128 products,
off by at most 128 steps of 2^-24 of sum |q k| (doubled: the tensor core's sums
truncate), which moves every probability by as much, relatively, and its sum
too. FP32 exponentials and sums of the probabilities add 2^-16 at most.

Verification's probabilities: an FP32 weight exp((l - max) / T) is off by its
argument's rounding, 2^-22.4 of up to 72 binary orders (9e-6), its sum by one
step of 2^-24 for each of the up to 300 terms of a thread (1.8e-5): 3e-5
together, carried through the tests of a node's children by spec_ref.verify.
"""
import math
from unittest import mock

import numpy as np
import pytest
import torch

import spec_ref

pytestmark = pytest.mark.gpu

BF16_HALF = 2.0 ** -8


# ------------------------------------------------------------- tree attention
def _mask_kind(kind, n, rng):
    if kind == "chain":
        return np.tril(np.ones((n, n), bool))
    if kind == "tree":
        return spec_ref.ancestors([-1] + [int(rng.randint(max(0, i - 4), i)) for i in range(1, n)])
    return rng.rand(n, n) < 0.4  # any mask: rows without a tree key, nodes that do not see themselves


class Case:
    def __init__(self, nodes, ctxs, qh, kvh, kind="tree", block_size=256, seed=0, words=None, spare_rows=3,
                 spare_pages=2, q_std=2.0):
        rng = np.random.RandomState(seed)
        g = torch.Generator().manual_seed(seed)
        self.nodes, self.qh, self.kvh, self.block_size = list(nodes), qh, kvh, block_size
        self.lens = [c + n for c, n in zip(ctxs, nodes)]
        pages = [(x + block_size - 1) // block_size for x in self.lens]
        self.blocks, self.stride = sum(pages) + spare_pages, max(max(pages), 1)
        order, at = rng.permutation(self.blocks), 0
        self.table = np.full((len(nodes), self.stride), -1, np.int32)
        for b, m in enumerate(pages):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.rows = int(self.cu[-1]) + spare_rows
        self.seens = [_mask_kind(kind, n, rng) for n in nodes]
        self.words = words or max(1, (max(nodes) + 63) // 64)
        self.mask = np.full((self.rows, self.words), -1, np.int64)  # what lies behind the rows says nothing
        for b, n in enumerate(nodes):
            self.mask[self.cu[b]:self.cu[b + 1]] = spec_ref.pack_bits(self.seens[b], self.words)

        def values(std, *shape):
            return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)

        self.q = values(q_std, self.rows, qh, 128)
        self.k = values(0.5, self.blocks, block_size, kvh, 128)
        self.v = values(0.5, self.blocks, block_size, kvh, 128)

    def args(self):
        up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        return dict(q=self.q.cuda(), k=self.k.cuda(), v=self.v.cuda(), cu_q=up(self.cu),
                    kv_lens=up(np.array(self.lens, np.int32)), block_table=up(self.table), tree_mask=up(self.mask))

    def shape(self):
        return dict(batch=len(self.nodes), max_q=max(max(self.nodes), 1), max_k=self.stride * self.block_size,
                    q_heads=self.qh, kv_heads=self.kvh, block_size=self.block_size, table_stride=self.stride,
                    num_blocks=self.blocks)

    def run(self, nvb, splits=1, args=None, stream=None, **shape):
        a = args or self.args()
        out = torch.full((self.rows, self.qh, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((self.rows, self.qh), 7.0, device="cuda")
        la, oa = nvb.tree_scratch(splits, self.rows, self.qh, "cuda")
        if la is not None:  # nothing may be taken from what the scratch held before
            la.fill_(math.nan)
            oa.fill_(math.nan)
        nvb.paged_tree_fwd(**a, out=out, lse=lse, num_splits=splits, lse_accum=la, out_accum=oa, stream=stream,
                           **{**self.shape(), **shape})
        torch.cuda.synchronize()
        assert nvb.device_error() == 0
        return out, lse

    def reference(self):
        f = spec_ref.as64
        return spec_ref.tree_attention(f(self.q), f(self.k), f(self.v), self.cu, self.lens, self.table, self.seens,
                                       self.block_size)


def close(case, out, lse, ref):
    o, s = spec_ref.as64(out), spec_ref.as64(lse)
    ro, rs, weight, size = ref
    n = case.cu[-1]
    assert (o[n:] == 7.0).all() and (s[n:] == 7.0).all(), "rows behind the last sequence were written"
    o, s, ro, rs, weight, size = o[:n], s[:n], ro[:n], rs[:n], weight[:n], size[:n]
    score = 2 * 128 * 2.0 ** -24 * size
    with np.errstate(invalid="ignore"):
        tol = BF16_HALF * np.abs(ro) + (BF16_HALF * (1 + BF16_HALF) + 2 * score[..., None] + 2.0 ** -16) * weight
        fine = np.isfinite(ro)
        assert np.array_equal(np.isnan(o), np.isnan(ro))
        assert np.array_equal(o[~fine & ~np.isnan(ro)], ro[~fine & ~np.isnan(ro)])
        assert (np.abs(o - ro)[fine] <= tol[fine]).all(), float((np.abs(o - ro) / tol)[fine].max())
        fine = np.isfinite(rs)
        assert np.array_equal(np.isnan(s), np.isnan(rs))
        assert np.array_equal(s[~fine & ~np.isnan(rs)], rs[~fine & ~np.isnan(rs)])
        tol = score + 2.0 ** -16 + 2.0 ** -22 * np.abs(rs)
        assert (np.abs(s - rs)[fine] <= tol[fine]).all(), float((np.abs(s - rs) / tol)[fine].max())


def check(nvb, case, splits=1, **kw):
    out, lse = case.run(nvb, splits, **kw)
    close(case, out, lse, case.reference())
    return out, lse


@pytest.mark.parametrize("kind", ["chain", "tree", "any"])
@pytest.mark.parametrize("nodes, ctxs", [([1], [0]), ([1], [1]), ([2], [0]), ([5], [123]), ([5], [124]), ([8], [256]),
                                         ([3], [254]), ([4, 1, 9, 2], [0, 700, 129, 40]), ([17], [300]), ([33], [95]),
                                         ([64], [64]), ([65], [511]), ([130, 7], [1, 200])])
def test_tree_attention(nvb, nodes, ctxs, kind):
    check(nvb, Case(nodes, ctxs, 4, 2, kind, seed=sum(nodes) + sum(ctxs)))


@pytest.mark.parametrize("qh, kvh", [(1, 1), (4, 4), (8, 1), (14, 2), (5, 1), (16, 8), (48, 1), (40, 8), (256, 2)])
@pytest.mark.parametrize("splits", [1, 3])
def test_tree_attention_head_layouts(nvb, qh, kvh, splits):
    check(nvb, Case([6, 19], [77, 300], qh, kvh, seed=qh), splits)


@pytest.mark.parametrize("splits", [2, 4, 7, 128])
def test_tree_attention_splits(nvb, splits):
    # empty ranges, ranges of one tile, a tree that crosses a range's end
    check(nvb, Case([9, 3, 64, 1], [1500, 0, 1000, 127], 8, 2, seed=splits), splits)


@pytest.mark.parametrize("block_size", [256, 512, 768])
def test_tree_attention_page_sizes(nvb, block_size):
    check(nvb, Case([12, 5], [block_size - 5, 2 * block_size], 4, 1, block_size=block_size, seed=3), 2)


def test_tree_attention_sequences_without_nodes(nvb):
    # a padded batch: its empty sequences are left alone, wherever they are
    check(nvb, Case([0, 4, 0, 0, 3, 0], [300, 20, 0, 5, 260, 0], 4, 2, seed=1), 2)


def test_tree_attention_rows_that_see_nothing(nvb):
    case = Case([6, 5], [0, 0], 4, 2, "chain", seed=2)
    case.seens[0][2] = False
    case.seens[1][:] = False
    for b in range(2):
        case.mask[case.cu[b]:case.cu[b + 1]] = spec_ref.pack_bits(case.seens[b], 1)
    for splits in (1, 3):
        out, lse = check(nvb, case, splits)
        assert (out[2] == 0).all() and (lse[2] == -math.inf).all() and (out[6:11] == 0).all()


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_tree_attention_ignores_what_a_node_does_not_see(nvb, splits, value):
    # two branches: the second one's K and V, the cache behind the sequence and the spare pages hold no numbers
    case = Case([6, 4], [150, 300], 4, 2, "chain", seed=5)
    parents = [-1, 0, 1, 0, 3, 4]
    case.seens[0] = spec_ref.ancestors(parents)
    case.mask[0:6] = spec_ref.pack_bits(case.seens[0], 1)
    for x in (case.k, case.v):
        for b, length in enumerate(case.lens):
            for at in range(length, len([p for p in case.table[b] if p >= 0]) * 256):
                x[case.table[b, at // 256], at % 256] = value
        used = set(case.table[case.table >= 0].tolist())
        for page in set(range(case.blocks)) - used:
            x[page] = value
    at = case.lens[0] - 2  # node 4: seen by nodes 4 and 5
    case.v[case.table[0, at // 256], at % 256] = value
    out, lse = check(nvb, case, splits)
    assert torch.isfinite(out[:4].float()).all() and torch.isfinite(lse[:10]).all()
    assert not torch.isfinite(out[4:6].float()).any()
    case.k[case.table[0, at // 256], at % 256] = math.nan
    out, lse = check(nvb, case, splits)
    assert torch.isfinite(out[:4].float()).all() and torch.isnan(out[4:6].float()).all()


@pytest.mark.parametrize("splits", [1, 2])
def test_tree_attention_one_infinite_dimension(nvb, splits):
    # an infinity of one sign in one dimension of a context key, both signs in another: inf and NaN there alone
    case = Case([5], [200], 4, 2, seed=6)
    case.v[case.table[0, 0], 10, 0, 3] = math.inf
    case.v[case.table[0, 0], 11, 0, 5] = -math.inf
    case.v[case.table[0, 0], 12, 0, 5] = math.inf
    out, _ = check(nvb, case, splits)
    assert (out[:5, :2, 3] == math.inf).all() and torch.isnan(out[:5, :2, 5].float()).all()


def test_tree_attention_bad_pages_mask_their_keys(nvb):
    case = Case([5, 3], [700, 300], 4, 2, seed=7)
    case.table[0, 1] = -1
    case.table[1, 0] = case.blocks  # past the cache
    for splits in (1, 3):
        check(nvb, case, splits)
    case.table[1, 1] = -5  # the page of the tree itself: nothing is left
    out, lse = check(nvb, case, 2)
    assert (out[5:8] == 0).all() and (lse[5:8] == -math.inf).all()


def test_tree_attention_lengths_that_do_not_fit(nvb):
    case = Case([4, 3, 2], [20, 30, 40], 4, 2, seed=8)
    case.lens[0] = 3    # fewer keys than nodes
    case.lens[1] = 300  # more than the table holds
    for splits in (1, 2):
        out, lse = check(nvb, case, splits)
        assert (out[:7] == 0).all() and (lse[:7] == -math.inf).all()


def test_tree_attention_large_scores(nvb):
    # scores of hundreds of orders: the running maximum moves, and one key takes all the weight
    check(nvb, Case([7, 20], [500, 130], 4, 2, seed=9, q_std=60.0), 2)


def test_tree_attention_equals_the_causal_and_decode_entry_points(nvb):
    # a chain is causal attention, one node is decode: within both kernels' roundings of each other
    case = Case([9, 20, 3], [300, 40, 129], 8, 2, "chain", seed=10, spare_rows=0)
    a = case.args()
    out, lse = case.run(nvb, 2, args=a)
    other = torch.empty_like(out)
    nvb.paged_fwd(a["q"], a["k"], a["v"], other, a["cu_q"], a["kv_lens"], a["block_table"], **case.shape())
    ref = case.reference()
    close(case, out, lse, ref)
    close(case, other, lse, ref)
    one = Case([1, 1], [300, 40], 8, 2, "chain", seed=11, spare_rows=0)
    a = one.args()
    out, lse = one.run(nvb, 1, args=a)
    other = torch.empty_like(out)
    nvb.paged_fwd(a["q"], a["k"], a["v"], other, a["cu_q"], a["kv_lens"], a["block_table"], **one.shape())
    ref = one.reference()
    close(one, out, lse, ref)
    close(one, other, lse, ref)


def test_tree_attention_twice_gives_the_same_bits(nvb):
    case = Case([33, 8], [900, 2000], 16, 2, seed=12)
    for splits in (1, 5):
        first, second = case.run(nvb, splits), case.run(nvb, splits)
        assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_tree_attention_without_lse_and_on_another_stream(nvb):
    case = Case([7, 20], [500, 130], 4, 2, seed=13)
    a = case.args()
    out, lse = case.run(nvb, 2, args=a)
    la, oa = nvb.tree_scratch(2, case.rows, 4, "cuda")
    other, side = torch.full_like(out, 7.0), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    nvb.paged_tree_fwd(**a, out=other, num_splits=2, lse_accum=la, out_accum=oa, stream=side, **case.shape())
    side.synchronize()
    assert torch.equal(out, other)


def test_tree_attention_captured_with_changing_lengths(nvb):
    # one capture serves steps whose node counts, lengths, tables and masks change on the device; two graphs with
    # scratch of their own run at the same time
    cases = [Case(n, c, 8, 2, seed=20 + i, words=1, spare_rows=24 - sum(n)) for i, (n, c) in enumerate(
        [([8, 8, 8], [500, 300, 90]), ([1, 8, 3], [20, 511, 255]), ([0, 2, 5], [0, 700, 100])])]
    shape = dict(cases[0].shape(), max_q=8, max_k=1024, table_stride=4, num_blocks=12)
    graphs = []
    for _ in range(2):
        a = dict(q=torch.zeros(24, 8, 128), k=torch.zeros(12, 256, 2, 128), v=torch.zeros(12, 256, 2, 128))
        a = {n: t.to(torch.bfloat16).cuda() for n, t in a.items()}
        a.update(cu_q=torch.zeros(4, dtype=torch.int32), kv_lens=torch.zeros(3, dtype=torch.int32),
                 block_table=torch.full((3, 4), -1, dtype=torch.int32), tree_mask=torch.zeros(24, 1, dtype=torch.int64))
        a = {n: t.cuda() for n, t in a.items()}
        la, oa = nvb.tree_scratch(3, 24, 8, "cuda")
        out, lse = torch.zeros(24, 8, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(24, 8, device="cuda")
        stream = torch.cuda.Stream()

        def step(a=a, out=out, lse=lse, la=la, oa=oa, stream=stream):
            nvb.paged_tree_fwd(**a, out=out, lse=lse, num_splits=3, lse_accum=la, out_accum=oa, stream=stream, **shape)

        torch.cuda.synchronize()
        step()
        stream.synchronize()
        graphs.append((nvb.capture(step, keep=[a, out, lse, la, oa], stream=stream), a, out, lse, stream))
    for i in range(4):
        for j, (graph, a, out, lse, stream) in enumerate(graphs):
            case = cases[(i + j) % 3]
            for name, t in case.args().items():
                a[name].zero_() if name != "block_table" else a[name].fill_(-1)
                a[name][tuple(slice(0, x) for x in t.shape)].copy_(t)
            out.fill_(7.0)
            lse.fill_(7.0)
        torch.cuda.synchronize()
        for graph, _, _, _, stream in graphs:
            graph.replay(stream)
        torch.cuda.synchronize()
        for j, (_, _, out, lse, _) in enumerate(graphs):
            case = cases[(i + j) % 3]
            close(case, out, lse, case.reference())


@pytest.mark.parametrize("splits", [11, 12, 24, 97])
def test_tree_attention_splits_that_leave_parts(nvb, splits):
    # clusters of 1, 6, 8 and 1, with 11, 2, 3 and 97 parts joined by the second kernel
    check(nvb, Case([9, 3, 40, 1], [1500, 0, 1000, 127], 8, 2, seed=splits), splits)


@pytest.mark.parametrize("splits", [1, 2, 11, 24, 128])
def test_tree_attention_scratch_of_its_parts_or_more(nvb, splits):
    # what lies behind the parts' rows is not written, fewer rows are refused, and a row for each split is enough
    case, parts = Case([9, 3], [1500, 40], 8, 2, seed=46), nvb.library().nvb_tree_parts(splits)
    want, want_lse = case.run(nvb, splits)
    a, f32 = case.args(), dict(dtype=torch.float32, device="cuda")
    for rows in {splits, parts + 1}:
        la, oa = torch.full((rows, case.rows, 8), 3.0, **f32), torch.full((rows, case.rows, 8, 128), 3.0, **f32)
        out, lse = torch.full_like(want, 7.0), torch.full_like(want_lse, 7.0)
        nvb.paged_tree_fwd(**a, out=out, lse=lse, num_splits=splits, lse_accum=la, out_accum=oa, **case.shape())
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        used = parts if parts > 1 else 0
        assert (la[used:] == 3.0).all() and (oa[used:] == 3.0).all()
    if parts > 1:
        la, oa = nvb.tree_scratch(splits, case.rows, 8, "cuda")
        for bad in (dict(lse_accum=la[1:], out_accum=oa), dict(lse_accum=la, out_accum=oa[1:]),
                    dict(lse_accum=la, out_accum=None), dict(lse_accum=None, out_accum=oa),
                    dict(lse_accum=la, out_accum=oa[:, 1:]), dict(lse_accum=la[0, 0, 0], out_accum=oa)):
            with pytest.raises(nvb.NvbError):
                nvb.paged_tree_fwd(**a, out=out, lse=lse, num_splits=splits, **bad, **case.shape())


@pytest.mark.parametrize("splits", [1, 2])
def test_tree_attention_the_largest_tree(nvb, splits):
    # 1,024 nodes of 16 words: 16 row tiles of 128 rows a head group
    check(nvb, Case([1024, 3], [70, 300], 4, 2, "tree", seed=40), splits)


@pytest.mark.parametrize("batch, kvh, splits", [(64, 4, 1), (64, 4, 2), (23, 8, 1), (65, 4, 1), (2, 80, 1)])
def test_tree_attention_of_ragged_batches(nvb, batch, kvh, splits):
    # more CTAs than SMs and long ranges: the sequences are taken in the order of their lengths. Equal lengths, empty
    # sequences, a length that does not fit and one below zero among them.
    rng = np.random.RandomState(batch)
    ctxs = rng.choice([0, 1, 60, 61, 200, 300], batch)
    nodes = rng.choice([0, 1, 3, 4], batch)
    ctxs[batch // 2], nodes[batch // 2] = 3900, 4
    case = Case(nodes.tolist(), ctxs.tolist(), 2 * kvh, kvh, seed=batch)
    a, want = case.args(), case.reference()
    close(case, *case.run(nvb, splits, args=a), want)
    if batch < 8:
        return
    nodes[[3, 5]] = 2
    case = Case(nodes.tolist(), ctxs.tolist(), 2 * kvh, kvh, seed=batch + 1)
    a, want = case.args(), case.reference()
    a["kv_lens"][3], a["kv_lens"][5] = -7, case.stride * 256 + 1
    for b in (3, 5):
        want[0][case.cu[b]:case.cu[b + 1]], want[1][case.cu[b]:case.cu[b + 1]] = 0, -math.inf
    close(case, *case.run(nvb, splits, args=a), want)


def test_tree_attention_lengths_below_zero(nvb):
    # a length that wraps around with the nodes subtracted is no length
    case = Case([4, 4, 4], [100, 100, 100], 4, 2, seed=41)
    a = case.args()
    a["kv_lens"] = torch.tensor([-2 ** 31, -1, case.lens[2]], dtype=torch.int32, device="cuda")
    for splits in (1, 3):
        out, lse = case.run(nvb, splits, args=a)
        assert (out[:8] == 0).all() and (lse[:8] == -math.inf).all() and torch.isfinite(lse[8:12]).all()


def test_tree_attention_between_the_other_kernels(nvb):
    # tree, causal and decode calls queued on one stream without a wait: kernels that are launched while the one before
    # them runs, and take tensor memory. Each leaves the bits that it leaves alone.
    case = Case([16] * 24, [700] * 24, 8, 2, "chain", seed=42, spare_rows=0)
    one = Case([1] * 24, [700] * 24, 8, 2, "chain", seed=43, spare_rows=0)
    a, d = case.args(), one.args()
    rows = lambda c: torch.zeros(c.rows, 8, 128, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    scratch = {s: nvb.tree_scratch(s, case.rows, 8, "cuda") for s in (1, 2, 11)}

    def tree(out, splits):
        la, oa = scratch[splits]
        nvb.paged_tree_fwd(**a, out=out, num_splits=splits, lse_accum=la, out_accum=oa, **case.shape())

    def causal(out, x, c):
        nvb.paged_fwd(x["q"], x["k"], x["v"], out, x["cu_q"], x["kv_lens"], x["block_table"], **c.shape())

    calls = [lambda o: tree(o, 1), lambda o: causal(o, a, case), lambda o: tree(o, 11), lambda o: causal(o, d, one),
             lambda o: tree(o, 2)]
    want = []
    for i, call in enumerate(calls):
        out = rows(one if i == 3 else case)
        call(out)
        torch.cuda.synchronize()
        want.append(out)
    outs = [[torch.zeros_like(w) for w in want] for _ in range(8)]
    torch.cuda.synchronize()
    for turn in outs:
        for call, out in zip(calls, turn):
            call(out)
    torch.cuda.synchronize()
    assert nvb.device_error() == 0
    for turn in outs:
        for w, out in zip(want, turn):
            assert torch.equal(w, out)


def test_tree_attention_parts_captured_and_at_the_same_time(nvb):
    # two graphs whose splits leave parts, with scratch of their own, replayed side by side over one cache
    case = Case([9, 3, 30], [1500, 0, 1000], 8, 2, seed=44)
    want, _ = case.run(nvb, 11)
    a, graphs = case.args(), []
    for _ in range(2):
        (la, oa), stream = nvb.tree_scratch(11, case.rows, 8, "cuda"), torch.cuda.Stream()
        out = torch.full_like(want, 7.0)
        torch.cuda.synchronize()

        def step(out=out, la=la, oa=oa, stream=stream):
            nvb.paged_tree_fwd(**a, out=out, num_splits=11, lse_accum=la, out_accum=oa, stream=stream, **case.shape())

        step()
        stream.synchronize()
        graphs.append((nvb.capture(step, keep=[a, out, la, oa], stream=stream), out, la, oa, stream))
    for _ in range(3):
        for _, out, la, oa, _ in graphs:
            out.fill_(7.0)
            la.fill_(math.nan)
            oa.fill_(math.nan)
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, _, _, _, stream in graphs:
                graph.replay(stream)
        torch.cuda.synchronize()
        for _, out, _, _, _ in graphs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("splits", [1, 2, 11])
def test_tree_attention_leaves_rows_before_the_first_sequence(nvb, splits):
    # a call on a slice of a larger batch: its first sequence starts behind others' rows, which are not its own
    case = Case([4, 9, 2], [300, 700, 40], 8, 2, seed=45, spare_rows=3)
    want, want_lse = case.run(nvb, splits)
    a = case.args()
    part = {**a, "cu_q": a["cu_q"][1:], "kv_lens": a["kv_lens"][1:], "block_table": a["block_table"][1:].contiguous()}
    out, lse = case.run(nvb, splits, args=part, batch=2)
    assert (out[:4] == 7.0).all() and (lse[:4] == 7.0).all() and (out[15:] == 7.0).all() and (lse[15:] == 7.0).all()
    assert torch.equal(out[4:15], want[4:15]) and torch.equal(lse[4:15], want_lse[4:15])


def test_tree_attention_in_a_cache_past_32_bit_offsets(nvb):
    # 8,704 pages of 256 x 8 x 128 elements: the last ones start past 2^31
    blocks = 8704
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 10 GB for the caches")
    case = Case([5, 9], [600, 300], 16, 8, seed=30)
    a = case.args()
    big = {n: torch.zeros(blocks, 256, 8, 128, dtype=torch.bfloat16, device="cuda") for n in "kv"}
    shift = blocks - case.blocks
    for n in "kv":
        big[n][shift:] = a[n]
    table = torch.where(a["block_table"] >= 0, a["block_table"] + shift, a["block_table"])
    out, lse = case.run(nvb, 2, args={**a, **big, "block_table": table}, num_blocks=blocks)
    close(case, out, lse, case.reference())


def test_tree_attention_refuses(nvb):
    case = Case([4], [20], 4, 2, seed=1)
    a = case.args()
    for bad in (dict(q=a["q"].float()), dict(q=a["q"].cpu()), dict(tree_mask=a["tree_mask"].int()),
                dict(tree_mask=a["tree_mask"][:3]), dict(cu_q=a["cu_q"].long()), dict(k=a["k"].transpose(1, 2)),
                dict(kv_lens=a["kv_lens"][:0])):
        with pytest.raises(nvb.NvbError):
            case.run(nvb, args={**a, **bad})
    with pytest.raises(nvb.NvbError):
        nvb.paged_tree_fwd(**a, out=a["q"], **case.shape())
    for bad in (dict(max_q=65), dict(block_size=128, num_blocks=2 * case.blocks, table_stride=1)):
        with pytest.raises(nvb.NvbError):
            case.run(nvb, args=a, **bad)


# ------------------------------------------------------------- verification
class Drafts:
    def __init__(self, sizes, vocab, fan, draft=True, temps=None, seed=0, noise=0.7, spread=2.5):
        rng, g = np.random.RandomState(seed), torch.Generator().manual_seed(seed)
        self.cu = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        rows = int(self.cu[-1]) + 2
        base = torch.randn(rows, vocab, generator=g) * spread
        self.logits = base.to(torch.bfloat16)
        self.draft = (base + torch.randn(rows, vocab, generator=g) * noise).to(torch.bfloat16) if draft else None
        self.parents, self.tokens = np.full(rows, -1, np.int32), np.zeros(rows, np.int32)
        likely = (self.draft if draft else self.logits).float()
        pick = torch.topk(likely + 0.8 * torch.randn(rows, vocab, generator=g), min(vocab, 8), 1).indices.numpy()
        for b, n in enumerate(sizes):
            kids = {}
            for i in range(1, n):
                p = int(rng.randint(max(0, i - fan), i))
                k = kids[p] = kids.get(p, -1) + 1
                self.parents[self.cu[b] + i] = p
                self.tokens[self.cu[b] + i] = pick[self.cu[b] + p, k % pick.shape[1]]
        self.uniforms = torch.rand(rows, generator=g).numpy()
        self.seeds = torch.randint(-2 ** 63, 2 ** 63 - 1, (rows,), generator=g).numpy()
        self.temps = np.array(temps if temps is not None else rng.choice([0.0, 0.6, 1.0, 1.3], len(sizes)), np.float32)
        self.vocab, self.sizes = vocab, sizes
        self.max_q = max(max(sizes), 1)

    def args(self):
        up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        return dict(logits=self.logits.cuda(), draft_logits=self.draft.cuda() if self.draft is not None else None,
                    tokens=up(self.tokens), parents=up(self.parents), uniforms=up(self.uniforms), seeds=up(self.seeds),
                    temperatures=up(self.temps), cu_q=up(self.cu))

    def outputs(self):
        b = len(self.sizes)
        i32 = dict(dtype=torch.int32, device="cuda")
        return dict(out_tokens=torch.full((b, self.max_q), 77, **i32), path=torch.full((b, self.max_q), 77, **i32),
                    counts=torch.full((b,), 77, **i32), accept_prob=torch.full((len(self.tokens),), 7.0, device="cuda"))

    def run(self, nvb, args=None, **kw):
        o = self.outputs()
        nvb.model.layer_verify(**(args or self.args()), **o, **kw)
        torch.cuda.synchronize()
        return o

    def reference(self):
        f = spec_ref.as64
        return spec_ref.verify(f(self.logits), f(self.draft) if self.draft is not None else None, self.tokens,
                               self.parents, self.uniforms.astype(np.float64), self.seeds, self.temps, self.cu,
                               self.max_q)


def same(case, o, ref=None):
    tokens, path, counts, prob, bound, margin, drawable = ref or case.reference()
    assert margin > 1e-5, "a borderline input"
    assert np.array_equal(o["counts"].cpu().numpy(), counts)
    assert np.array_equal(o["path"].cpu().numpy(), path)
    got, tokens = o["out_tokens"].cpu().numpy(), tokens.copy()
    for b, c in enumerate(counts):
        if c > 0 and got[b, c - 1] in drawable[b]:  # nearly always the one token of `tokens`
            tokens[b, c - 1] = got[b, c - 1]
    assert np.array_equal(got, tokens)
    a, n = o["accept_prob"].cpu().double().numpy(), case.cu[-1]
    assert (a[n:] == 7.0).all(), "rows behind the last sequence were written"
    off = np.abs(a - prob)[:n]
    assert (off <= bound[:n] + 2.0 ** -24).all(), float((off - bound[:n]).max())


VERIFY = [
    dict(sizes=[1], vocab=1000, fan=1), dict(sizes=[2], vocab=7, fan=1), dict(sizes=[5], vocab=1, fan=1),
    dict(sizes=[8, 3, 1, 20], vocab=1000, fan=1), dict(sizes=[8, 3, 1, 20], vocab=4099, fan=3),
    dict(sizes=[30, 30], vocab=513, fan=40), dict(sizes=[0, 6, 0, 4, 0], vocab=2048, fan=2),
    dict(sizes=[6] * 9, vocab=32003, fan=2), dict(sizes=[70], vocab=300, fan=6), dict(sizes=[5, 4], vocab=151936, fan=2),
]


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("spec", VERIFY)
def test_verify(nvb, spec, draft):
    case = Drafts(**spec, draft=draft, seed=len(spec["sizes"]) + spec["vocab"])
    same(case, case.run(nvb))


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 0.05, 1.0, 20.0])
def test_verify_temperatures(nvb, draft, temperature):
    case = Drafts([9, 12], 5000, 2, draft, [temperature] * 2, seed=40)
    same(case, case.run(nvb))


def test_verify_drafts_equal_to_the_target_are_accepted(nvb):
    case = Drafts([6, 6], 3001, 1, True, [1.0, 0.7], seed=41)
    case.draft = case.logits.clone()
    o = case.run(nvb)
    same(case, o)
    assert o["counts"].tolist() == [6, 6] and (o["accept_prob"][[1, 2, 7, 8]] == 1).all()


def test_verify_confident_draft_that_is_wrong(nvb):
    # the draft gives one token nearly everything: what is left of Q behind it is small numbers, not a difference
    case = Drafts([4, 4], 2000, 8, True, [1.0, 1.0], seed=42)
    case.parents[[1, 2, 3, 5, 6, 7]] = 0
    for b in (0, 4):
        case.draft[b, 5], case.tokens[b + 1] = 40.0, 5
        case.logits[b, 5] = -3.0
        case.tokens[b + 2:b + 4] = [9, 11]
        case.uniforms[b + 1:b + 4] = 0.999
    same(case, case.run(nvb))


def test_verify_the_same_token_twice_and_tokens_outside(nvb):
    for draft in (True, False):
        case = Drafts([5, 5], 900, 8, draft, [1.0, 0.0], seed=43)
        case.parents[[1, 2, 3, 4, 6, 7, 8, 9]] = 0
        case.tokens[1:5] = [30, 30, -1, 900]
        case.tokens[6:10] = [30, 30, -1, 900]
        case.uniforms[1:5] = 0.9999
        same(case, case.run(nvb))


@pytest.mark.parametrize("draft", [True, False])
def test_verify_masked_and_missing_logits(nvb, draft):
    # -inf and NaN have no probability, the lowest finite value next to none; all of a row may be gone
    case = Drafts([6, 6, 4], 1500, 2, draft, [1.0, 0.5, 0.0], seed=44)
    case.logits[:, ::3] = -math.inf
    case.logits[:, 1::7] = math.nan
    case.logits[:, 2::9] = torch.finfo(torch.bfloat16).min
    if draft:
        case.draft[:, ::5] = -math.inf
        case.draft[:, 1::11] = math.nan
    case.tokens[1], case.tokens[7] = 3, 1  # drafts that the target cannot give
    same(case, case.run(nvb))


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("value", [-math.inf, torch.finfo(torch.bfloat16).min, -1e4, 70.0])
def test_verify_long_stretches_of_masked_logits(nvb, draft, value):
    # whole parts of a row, the first tokens of others and a row's end hold one value, far from the rest (or three tokens
    # hold nearly all of it: e^-70 of the drafts is a normal FP32 number)
    case = Drafts([6, 5, 4], 40000, 3, draft, [1.0, 0.7 if value < 0 else 1.0, 0.0], seed=59)
    for x in (case.logits, case.draft) if draft else (case.logits,):
        if value < 0:
            x[:, :9000] = value
            x[:, 12288:15000] = value
            x[:, 36000:] = value
        else:
            x[:, 30000:30003] = value + torch.tensor([0.0, 2.0, -2.0])
    same(case, case.run(nvb))


def test_verify_rows_without_any_probability(nvb):
    case = Drafts([3, 3], 700, 1, True, [1.0, 0.0], seed=45)
    case.logits[:] = -math.inf
    o = case.run(nvb)
    assert o["counts"].tolist()[0] == 1 and o["out_tokens"][0, 0].item() == 0
    assert (o["accept_prob"][1:3] == 0).all()
    case.logits[:] = math.nan
    o = case.run(nvb)
    assert o["counts"].tolist() == [1, 1] and o["out_tokens"][:, 0].tolist() == [0, 0]


def test_verify_nodes_without_a_parent_are_never_reached(nvb):
    case = Drafts([6], 800, 1, True, [1.0], seed=46)
    case.parents[:6] = [-1, 0, -1, 3, 9, 1]
    o = case.run(nvb)
    same(case, o)
    assert (o["accept_prob"][2:5] == 0).all()


def test_verify_nothing_drafted_is_the_sampler(nvb):
    # one row per sequence: the token is layer_sample's, bit for bit, at every temperature
    vocab, rows = 20011, 40
    g = torch.Generator().manual_seed(47)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(torch.bfloat16).cuda()
    temps = (torch.rand(rows, generator=g) * 1.5).cuda()
    temps[::4] = 0
    seeds = torch.randint(-2 ** 63, 2 ** 63 - 1, (rows,), generator=g).cuda()
    want = torch.empty(rows, dtype=torch.int32, device="cuda")
    nvb.model.layer_sample(logits, temps, seeds, want)
    i32 = dict(dtype=torch.int32, device="cuda")
    out, path, counts = torch.empty(rows, 1, **i32), torch.empty(rows, 1, **i32), torch.empty(rows, **i32)
    nvb.model.layer_verify(logits, None, torch.zeros(rows, **i32), torch.full((rows,), -1, **i32),
                           torch.zeros(rows, device="cuda"), seeds, temps, torch.arange(rows + 1, **i32), out, path,
                           counts, torch.empty(rows, device="cuda"))
    assert torch.equal(out[:, 0], want) and (counts == 1).all() and (path == 0).all()


def test_verify_keeps_the_targets_distribution(nvb):
    # 40,000 sequences of one draft each, drawn from Q: the first emitted token is distributed as P. The counts of a
    # token of probability p are off by 5.5 standard deviations in one of 20 million.
    vocab, n = 12, 40000
    g = torch.Generator().manual_seed(48)
    target, draft = torch.randn(vocab, generator=g) * 1.5, torch.randn(vocab, generator=g) * 1.5
    target, draft = target.to(torch.bfloat16), draft.to(torch.bfloat16)
    p, q = torch.softmax(target.double(), 0), torch.softmax(draft.double(), 0)
    rows = 3 * n  # the root and two children without replacement
    both = torch.multinomial(q.float().expand(n, vocab), 2, generator=g).int()
    tokens = torch.cat([torch.zeros(n, 1, dtype=torch.int32), both], 1).reshape(-1)
    i32 = dict(dtype=torch.int32, device="cuda")
    out, path = torch.empty(n, 3, **i32), torch.empty(n, 3, **i32)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32).repeat(n)
    done = torch.zeros(vocab, dtype=torch.int64)
    for part in range(0, n, 10000):  # 10,000 sequences a call
        r = slice(3 * part, 3 * (part + 10000))
        m = 30000
        nvb.model.layer_verify(target.expand(m, vocab).contiguous().cuda(), draft.expand(m, vocab).contiguous().cuda(),
                               tokens[r].cuda(), parents[r].cuda(), torch.rand(m, generator=g).cuda(),
                               torch.randint(-2 ** 63, 2 ** 63 - 1, (m,), generator=g).cuda(),
                               torch.ones(10000, device="cuda"), torch.arange(0, m + 1, 3, **i32), out[:10000],
                               path[:10000], torch.empty(10000, **i32), torch.empty(m, device="cuda"))
        done += torch.bincount(out[:10000, 0].cpu().long(), minlength=vocab)
    spread = (n * p * (1 - p)).sqrt()
    assert ((done - n * p).abs() <= 5.5 * spread).all(), ((done - n * p) / spread).tolist()
    assert rows == tokens.numel()


def test_verify_captured_and_on_two_streams(nvb):
    cases = [Drafts([4, 8, 2], 3000, 2, True, seed=50), Drafts([8, 1, 5], 3000, 2, True, seed=51)]
    runs = []
    for case in cases:
        a, o, stream = case.args(), case.outputs(), torch.cuda.Stream()
        ws = torch.full((nvb.model.verify_workspace_bytes(len(case.tokens), len(case.sizes)),), 0xff, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        step = lambda a=a, o=o, s=stream, ws=ws: nvb.model.layer_verify(**a, **o, stream=s, workspace=ws)  # noqa: E731
        step()
        stream.synchronize()
        runs.append((nvb.capture(step, keep=[a, o, ws], stream=stream), a, o, stream, ws))
    for _ in range(3):
        for graph, a, o, stream, ws in runs:
            for t in o.values():
                t.fill_(7)
            ws.fill_(0xff)
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in runs:
            graph.replay(stream)
        torch.cuda.synchronize()
        for case, (_, _, o, _, _) in zip(cases, runs):
            same(case, o)


@pytest.mark.parametrize("what", ["verify", "sample"])
def test_a_captured_call_without_a_workspace_keeps_its_own(nvb, what):
    # what a replay writes is not memory that was given on since
    case, stream = Drafts([6, 9, 2], 40000, 2, True, seed=74), torch.cuda.Stream()
    a, o, out = case.args(), case.outputs(), torch.zeros(19, dtype=torch.int32, device="cuda")
    t = a["temperatures"].repeat_interleave(torch.tensor([6, 9, 4], device="cuda"))
    torch.cuda.synchronize()

    def call(out=out, o=o):
        if what == "verify":
            nvb.model.layer_verify(**a, **o, stream=stream)
        else:
            nvb.model.layer_sample(a["logits"], t, a["seeds"], out, stream=stream)

    with torch.cuda.stream(stream):
        want, want_out = case.outputs(), torch.zeros_like(out)
        call(want_out, want)  # leaves memory that the capture takes without asking the device for more
        stream.synchronize()
        graph = nvb.capture(call, keep=[a, o, out, t], stream=stream)
        held = [x for x in graph._keep if isinstance(x, torch.Tensor) and x is not out and x is not t]
        spans = [(x.data_ptr(), x.data_ptr() + x.nbytes) for x in held]
        assert spans
        size = max(x.nbytes for x in held)
        later = [torch.full((size,), 0x5a, dtype=torch.uint8, device="cuda") for _ in range(8)]
        for x in later:
            assert all(x.data_ptr() >= z or x.data_ptr() + size <= y for y, z in spans)
    for _ in range(2):
        for x in o.values():
            x.fill_(7)
        torch.cuda.synchronize()
        graph.replay(stream)
        torch.cuda.synchronize()
        assert all((x == 0x5a).all() for x in later)
        assert torch.equal(out, want_out) and (what == "sample" or all(torch.equal(o[n], want[n]) for n in o))


def test_verify_the_longest_chain(nvb):
    # 1,024 nodes whose drafts are all accepted: the draft's logits are the target's
    case = Drafts([1024, 5], 300, 1, True, [1.0, 0.0], seed=56, noise=0.0)
    o = case.run(nvb)
    same(case, o)
    assert o["counts"][0] == 1024 and o["path"][0].tolist() == list(range(1024))


def test_verify_the_widest_tree(nvb):
    # 1,023 children of one node, looked up: 290 tokens are rejected one after the other, and then again with nothing left
    case = Drafts([1024], 300, 1, False, [1.0], seed=57)
    case.parents[1:1024] = 0
    case.tokens[1:1024] = np.arange(1023) % 290
    case.uniforms[:] = 0.9999
    o = case.run(nvb)
    same(case, o)
    assert o["counts"][0] == 1 and o["out_tokens"][0, 0] >= 290


def test_verify_logits_past_32_bit_offsets(nvb):
    # 14,200 rows of 151,936 logits: the last tree's start past 2^31 elements. It gets what it gets alone.
    vocab, ones = 151936, 14200
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 10 GB for the logits")
    case = Drafts([6], vocab, 2, True, [0.8], seed=58)
    want, a = case.run(nvb), case.args()
    rows = ones + 6
    big = {}
    for name in ("logits", "draft_logits"):
        big[name] = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
        big[name][ones:] = a[name][:6]
    for name in ("tokens", "parents", "uniforms", "seeds"):
        big[name] = torch.cat([a[name].new_full((ones,), -1) if name == "parents" else a[name].new_zeros(ones), a[name][:6]])
    big["temperatures"] = torch.cat([torch.zeros(ones, device="cuda"), a["temperatures"]])
    big["cu_q"] = torch.cat([torch.arange(ones + 1, dtype=torch.int32, device="cuda"),
                             torch.tensor([rows], dtype=torch.int32, device="cuda")])
    i32 = dict(dtype=torch.int32, device="cuda")
    o = dict(out_tokens=torch.zeros(ones + 1, 6, **i32), path=torch.zeros(ones + 1, 6, **i32),
             counts=torch.zeros(ones + 1, **i32), accept_prob=torch.zeros(rows, device="cuda"))
    nvb.model.layer_verify(**big, **o)
    for name in ("out_tokens", "path", "counts"):
        assert torch.equal(o[name][-1], want[name][0]), name
    # the sums of a row are cut in other places: FP32 sums of 151,936 terms, in threads of a few hundred
    assert (o["accept_prob"][-6:] - want["accept_prob"][:6]).abs().max() <= 1e-5
    assert (o["counts"][:-1] == 1).all() and (o["out_tokens"][:-1, 0] == 0).all()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("temperature", [3e38, math.inf])
def test_verify_at_endless_temperatures(nvb, draft, temperature):
    # as at 1e30, where every finite logit has the same weight too, and logits of -inf none
    runs = []
    for t in (1e30, temperature):
        case = Drafts([7, 1, 4], 900, 3, draft, [t] * 3, seed=54)
        for x in (case.logits, case.draft) if draft else (case.logits,):
            x[:, ::3] = -math.inf
        runs.append(case.run(nvb))
    for name in runs[0]:
        assert torch.equal(runs[0][name], runs[1][name]), name
    assert (runs[1]["accept_prob"][1:7] > 0).any()
    last = runs[1]["out_tokens"].gather(1, (runs[1]["counts"] - 1).long()[:, None])
    assert (last % 3 != 0).all()


def test_verify_workspace_of_a_call_on_another_stream(nvb):
    # The workspace of a call without one is not given on to work of the current stream that may run before the call.
    case, stream = Drafts([8] * 4, 20000, 3, True, seed=55), torch.cuda.Stream()
    a, ref = case.args(), case.reference()
    size = nvb.model.verify_workspace_bytes(len(case.tokens), 4)
    for _ in range(4):
        o = case.outputs()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(20_000_000)
        nvb.model.layer_verify(**a, **o, stream=stream)
        for _ in range(50):
            torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        same(case, o, ref)


def test_verify_sequences_that_overlap_stay_in_bounds(nvb):
    # cu_q that falls: five sequences share eight rows, so that more nodes than rows have rejected children, and a row
    # is written by several. What comes out is not defined, but it names nodes, and nothing behind the workspace changes.
    case = Drafts([8], 500, 3, True, [1.0], seed=53)
    for parents in ([-1, 0, 0, 0, 1, 1, 4, 4], [-1, 0, 0, 2, 2, 0, 0, 6]):
        for cu in ([0, 8] * 5, [0, 8, 4, 8, 2, 8, 4, 8, 0, 8]):
            case.parents[:8] = parents
            case.uniforms[:] = 1.0
            a, batch = case.args(), 9
            a["cu_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
            a["temperatures"] = torch.ones(batch, device="cuda")
            i32 = dict(dtype=torch.int32, device="cuda")
            o = dict(out_tokens=torch.zeros(batch, 8, **i32), path=torch.zeros(batch, 8, **i32),
                     counts=torch.zeros(batch, **i32), accept_prob=torch.zeros(len(case.tokens), device="cuda"))
            size = nvb.model.verify_workspace_bytes(len(case.tokens), batch)
            ws = torch.full((size + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
            nvb.model.layer_verify(**a, **o, workspace=ws[:size])
            assert (ws[size:] == 0x5a).all()
            assert (o["counts"] >= 0).all() and (o["counts"] <= 8).all() and (o["counts"][1::2] == 0).all()
            assert (o["path"] >= -1).all() and (o["path"] < 8).all()


def test_verify_refuses(nvb):
    case = Drafts([4], 100, 1, True, seed=52)
    a, o = case.args(), case.outputs()
    for bad in (dict(logits=a["logits"].float()), dict(draft_logits=a["draft_logits"][:, :50]),
                dict(tokens=a["tokens"].long()), dict(seeds=a["seeds"].int()), dict(cu_q=a["cu_q"][:1]),
                dict(temperatures=a["temperatures"].cpu()), dict(path=o["path"][:, :2]), dict(counts=a["cu_q"][:1]),
                dict(out_tokens=o["path"]), dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                dict(logits=a["logits"].t().contiguous().t())):
        with pytest.raises((ValueError, nvb.model.ModelError)):
            nvb.model.layer_verify(**{**a, **o, **bad})


# -------------------------------------------------------- copies in the cache
def _caches(layers, blocks, block_size, kvh, dim, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(blocks, block_size, kvh, dim, generator=g).to(torch.bfloat16).cuda() for _ in range(2 * layers)]


@pytest.mark.parametrize("layers, block_size, kvh, dim", [(1, 256, 8, 128), (3, 256, 1, 128), (2, 16, 2, 64),
                                                          (2, 7, 3, 5), (70, 32, 1, 16), (1, 5, 1, 1)])
@pytest.mark.parametrize("partly", [True, False])
def test_copy_pages(nvb, layers, block_size, kvh, dim, partly):
    blocks = 9
    caches = _caches(layers, blocks, block_size, kvh, dim)
    want = [c.clone() for c in caches]
    src, dst = [3, 0, 3, 8, -1, 2, 9, 4, 6], [1, 5, 2, 7, 6, -1, 4, 9, 6]  # bad pages are skipped; 3 is copied twice
    rows = [1, block_size, 0, block_size // 2, 5, 5, 5, 5, 5]
    for c in want:
        for a, z, n in zip(src, dst, rows if partly else [block_size] * 9):
            if 0 <= a < blocks and 0 <= z < blocks:
                c[z, :n] = c[a, :n]
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    handle = nvb.CacheLayers(caches[:layers], caches[layers:])
    nvb.cache_copy_pages(handle, up(src), up(dst), up(rows) if partly else None)
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_copy_pages_of_unaligned_caches_and_row_counts_out_of_range(nvb):
    flat = torch.randn(2 * 4 * 8 * 2 * 8 + 1, device="cuda").to(torch.bfloat16)[1:]  # 2 bytes past a 16-byte border
    k, v = flat[:512].view(4, 8, 2, 8), flat[512:].view(4, 8, 2, 8)
    want_k, want_v = k.clone(), v.clone()
    for c in (want_k, want_v):
        c[1] = c[0]  # more rows than a page has: all of it; fewer than none: nothing
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    nvb.cache_copy_pages(nvb.CacheLayers([k], [v]), up([0, 2]), up([1, 3]), up([100, -4]))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


PATHS = [  # (nodes, context, path behind the root)
    [(4, 20, [1, 2, 3])], [(6, 250, [2, 4, 5])], [(8, 510, [1, 3, 7]), (1, 40, []), (5, 0, [4])],
    [(0, 100, None), (3, 255, [2])], [(300, 100, list(range(1, 300, 2)))], [(200, 3, list(range(2, 200)))],
]


@pytest.mark.parametrize("spec", PATHS)
@pytest.mark.parametrize("layers, block_size, kvh, dim", [(2, 256, 8, 128), (66, 256, 1, 16), (1, 7, 3, 5)])
def test_compact_paths(nvb, spec, layers, block_size, kvh, dim):
    lens = [c + n for n, c, _ in spec]
    pages = [max(1, (x + block_size - 1) // block_size) for x in lens]
    blocks = sum(pages)
    order, table, at = np.random.RandomState(1).permutation(blocks), np.full((len(spec), max(pages)), -1, np.int32), 0
    for b, m in enumerate(pages):
        table[b, :m] = order[at:at + m]
        at += m
    caches = _caches(layers, blocks, block_size, kvh, dim, 2)
    want = [c.clone() for c in caches]
    path = np.full((len(spec), max(max(n for n, _, _ in spec), 1)), -1, np.int32)
    counts = []
    for b, (n, ctx, moves) in enumerate(spec):
        counts.append(0 if moves is None else 1 + len(moves))
        if moves is not None:
            path[b, :1 + len(moves)] = [0] + moves
        slot = lambda x: (table[b, x // block_size], x % block_size)  # noqa: E731,B023
        for c, old in zip(want, caches):
            for d, node in enumerate(moves or [], 1):
                c[slot(ctx + d)] = old[slot(ctx + node)]
    up = lambda x: torch.from_numpy(np.array(x, np.int32)).cuda()  # noqa: E731
    new = torch.full((len(spec),), 99, dtype=torch.int32, device="cuda")
    nvb.cache_compact_paths(nvb.CacheLayers(caches[:layers], caches[layers:]),
                            up(np.concatenate([[0], np.cumsum([n for n, _, _ in spec])])), up(lens), up(table),
                            up(path), up(counts), new)
    assert new.tolist() == [c + k for (_, c, _), k in zip(spec, counts)]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_compact_paths_with_bad_pages_and_paths_stay_in_bounds(nvb):
    # nodes outside the tree, pages outside the cache, a length past the table: those moves are skipped
    caches = _caches(1, 3, 256, 2, 64, 3)
    want = [c.clone() for c in caches]
    for c, old in zip(want, caches):
        c[0, 12] = old[0, 14]
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    new = up([0, 0, 0])
    nvb.cache_compact_paths(nvb.CacheLayers(caches[:1], caches[1:]), up([0, 5, 10, 15]), up([15, 265, 600]),
                            up([[0, -1], [1, 7], [2, -1]]), up([[0, 9, 4, -1, 0]] * 2 + [[0, 1, 3, 4, -1]]),
                            up([5, 3, 4]), new)
    assert new.tolist() == [15, 263, 599]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_copies_past_32_bit_offsets(nvb):
    blocks = 8704
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 10 GB for the caches")
    caches = [torch.zeros(blocks, 256, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(1)
    for c in caches:
        c[-3:].normal_(generator=g)
    want = [c[-3:].clone() for c in caches]
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    handle, new = nvb.CacheLayers(caches[:1], caches[1:]), up([0])
    nvb.cache_copy_pages(handle, up([blocks - 1]), up([blocks - 3]))
    nvb.cache_compact_paths(handle, up([0, 6]), up([16]), up([[blocks - 2]]), up([[0, 3, 5]]), up([3]), new)
    for c, w in zip(caches, want):
        w[0] = w[2]
        w[1, 11], w[1, 12] = w[1, 13].clone(), w[1, 15].clone()
        assert torch.equal(c[-3:], w) and not c[0].any() and not c[1:4].any()


def test_cache_layers_refuse(nvb):
    k, v = _caches(1, 3, 256, 2, 64)
    for ks, vs in (([], []), ([k], []), ([k], [k]), ([k], [v.float()]), ([k], [v[:2]]), ([k], [v.cpu()]),
                   ([k.view(3, 256, 128)], [v.view(3, 256, 128)]), ([k, k[1:]], [v, v])):
        with pytest.raises(nvb.NvbError):
            nvb.CacheLayers(ks, vs)
    handle = nvb.CacheLayers([k], [v])
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    inside = k.view(torch.int32).view(-1)[:1]
    for bad in ((one, one.long()), (one.cpu(), one), (one, torch.zeros(2, dtype=torch.int32, device="cuda")),
                (one, inside)):
        with pytest.raises(nvb.NvbError):
            nvb.cache_copy_pages(handle, *bad)
    cu, table = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), one.view(1, 1)
    with pytest.raises(nvb.NvbError):
        nvb.cache_compact_paths(handle, cu, one, table, table.clone(), one.clone(), one)
    with pytest.raises(nvb.NvbError):
        nvb.cache_compact_paths(handle, cu, one, one, table.clone(), one.clone(), one.clone())


# ---------------------------------------------------------- a step of them all
@pytest.mark.parametrize("captured", [False, True])
def test_a_step_of_attention_verification_and_compaction(nvb, captured):
    """Two users' trees through attention, verification and compaction, all on
    the device and without a look at the results; the cache must then be what a
    chain of the accepted tokens alone would have left, so that attention of a
    chain over it equals attention over the tree's own nodes."""
    rng, qh, kvh, vocab, layers = np.random.RandomState(3), 8, 2, 503, 2
    case = Case([7, 5], [252, 90], qh, kvh, seed=60, spare_rows=0)
    host = __import__("importlib").import_module("nano_vllm_rs_b200.host")
    parents = [-1, 0, 0, 1, 1, 2, 3] + [-1, 0, 1, 1, 0]
    mask, depth = host.tree_mask(parents, case.cu)
    case.mask[:] = mask
    case.seens = [spec_ref.ancestors(parents[:7]), spec_ref.ancestors(parents[7:])]
    a = case.args()
    caches = [(a["k"].clone(), a["v"].clone()) for _ in range(layers)]
    handle = nvb.CacheLayers([k for k, _ in caches], [v for _, v in caches])
    drafts = Drafts([7, 5], vocab, 2, True, [1.0, 0.8], seed=61)
    d = drafts.args()
    for n in ("logits", "draft_logits", "tokens", "parents", "uniforms", "seeds"):
        d[n] = d[n][:12].contiguous()
    d["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
    drafts.parents[:12] = parents
    d["uniforms"][:] = torch.from_numpy(rng.rand(12).astype(np.float32) * 0.5).cuda()  # a few are accepted
    drafts.uniforms[:12] = d["uniforms"].cpu().numpy()
    o = {n: (t[:12] if n == "accept_prob" else t).contiguous() for n, t in drafts.outputs().items()}
    out, lse = torch.zeros_like(a["q"]), torch.zeros(case.rows, qh, device="cuda")
    new = torch.zeros(2, dtype=torch.int32, device="cuda")
    la, oa = nvb.tree_scratch(2, case.rows, qh, "cuda")
    ws = torch.empty(nvb.model.verify_workspace_bytes(12, 2), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()

    def step():
        for k, v in caches:
            nvb.paged_tree_fwd(**{**a, "k": k, "v": v}, out=out, lse=lse, num_splits=2, lse_accum=la, out_accum=oa,
                               stream=stream, **case.shape())
        nvb.model.layer_verify(**d, **o, stream=stream, workspace=ws)
        nvb.cache_compact_paths(handle, a["cu_q"], a["kv_lens"], a["block_table"], o["path"], o["counts"], new,
                                stream=stream)

    torch.cuda.synchronize()
    if captured:
        graph = nvb.capture(step, keep=[caches, out, lse, la, oa, ws, o, d, a, new], stream=stream)
        graph.replay(stream)
    else:
        step()
    torch.cuda.synchronize()
    close(case, out, lse, case.reference())
    drafts.cu = case.cu
    tokens, path, counts, _, _, margin, _ = spec_ref.verify(
        spec_ref.as64(d["logits"]), spec_ref.as64(d["draft_logits"]), drafts.tokens, drafts.parents,
        drafts.uniforms.astype(np.float64), drafts.seeds, drafts.temps, case.cu, drafts.max_q)
    assert margin > 1e-5 and counts.max() >= 2
    assert np.array_equal(o["out_tokens"].cpu().numpy(), tokens) and np.array_equal(o["counts"].cpu().numpy(), counts)
    ctx = [252, 90]
    assert new.tolist() == [c + n for c, n in zip(ctx, counts)]
    for k, v in caches:
        for old, kept in ((case.k, k), (case.v, v)):
            for b in range(2):
                for at in range(ctx[b] + counts[b]):
                    frm = at if at < ctx[b] else ctx[b] + path[b, at - ctx[b]]
                    assert torch.equal(kept[case.table[b, at // 256], at % 256].cpu(),
                                       old[case.table[b, frm // 256], frm % 256])
    # the accepted nodes as a chain over the compacted cache: the same attention
    rows = np.concatenate([case.cu[b] + path[b, :counts[b]] for b in range(2)])
    chain = dict(a, q=a["q"][torch.from_numpy(rows).cuda()].contiguous(), k=caches[0][0], v=caches[0][1],
                 cu_q=torch.tensor([0, counts[0], counts.sum()], dtype=torch.int32, device="cuda"), kv_lens=new,
                 tree_mask=torch.tensor([(2 << i) - 1 for n in counts for i in range(n)], device="cuda")[:, None])
    again = torch.zeros_like(chain["q"])
    nvb.paged_tree_fwd(**chain, out=again, **case.shape())
    picked = out[torch.from_numpy(rows).cuda()].float()
    assert (again.float() - picked).abs().max() <= 2 * BF16_HALF * 2 * picked.abs().max()
    assert depth.max() == 3


def test_the_models_caches_make_a_handle(nvb):
    m = nvb.model
    cfg = m.Qwen3Config(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4,
                        num_key_value_heads=2, vocab_size=512)
    model = m.Qwen3Model(cfg, m.ModelOptions(num_blocks=4, max_batch_tokens=64, max_sequences=2, max_model_len=512),
                         m.random_weights(cfg))
    handle = model.cache_layers()
    assert handle.layers == 3 and handle.shape == (4, 256, 2, 128)
    for layer in range(3):
        for c in model.kv_cache(layer):
            c.fill_(0)
            c[2] = layer + 1
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    nvb.cache_copy_pages(handle, up([2]), up([0]), up([100]))
    torch.cuda.synchronize()
    for layer in range(3):
        for c in model.kv_cache(layer):
            assert (c[0, :100] == layer + 1).all() and (c[0, 100:] == 0).all() and (c[1] == 0).all()
    del handle
    model.close()


# ------------------------------------------- sums of rows with far outliers
# Weights are taken in a unit up to 90 binary orders below the highest logit. Exponents of up to 90 are off by 90 * 2^-24
# steps of their product, 4e-6 of a weight and as much of a sum; log2(e) / T is off by 2^-23, 6e-6 over 72 orders; a
# thread's sum has up to 16 terms in a row and 20 joins behind it, 2e-6. Together less than the 3e-5 of spec_ref.verify.
def _padded(case, rows):
    """Arguments and outputs of `rows` rows, those behind the case's own without a sequence. (From 237 rows on, at
    148 SMs, a row of 151,936 tokens is read in 5 parts, below that in 32.)"""
    a, o = case.args(), case.outputs()
    more = rows - len(case.tokens)
    if more > 0:
        for name in ("logits", "draft_logits", "tokens", "parents", "uniforms", "seeds"):
            if a[name] is not None:
                a[name] = torch.cat([a[name], a[name].new_zeros(more, *a[name].shape[1:])])
        o["accept_prob"] = torch.full((rows,), 7.0, device="cuda")
    return a, o


def _same_with_rows(nvb, case, rows):
    # probabilities below 2^-126 are 0 (at the lowest temperatures many drafts' are; none lies at that border)
    exactly = spec_ref.softmax

    def softmax(l, temperature):
        p = exactly(l, temperature)
        return np.where(p < 2.0 ** -126, 0.0, p)

    with mock.patch.object(spec_ref, "softmax", softmax):
        ref = case.reference()
    # these inputs leave one token that may be drawn, whatever the roundings
    assert all(len(d) <= 1 for d in ref[-1])
    a, o = _padded(case, rows)
    nvb.model.layer_verify(**a, **o)
    n = len(case.tokens)
    assert (o["accept_prob"][n:] == 7.0).all()
    same(case, {**o, "accept_prob": o["accept_prob"][:n]}, ref)


@pytest.mark.parametrize("where", ["target", "draft"])
@pytest.mark.parametrize("temperature", [0.1, 0.25])
@pytest.mark.parametrize("rows", [0, 240])
def test_verify_leaders_behind_the_first_tokens_of_a_part(nvb, rows, temperature, where):
    # Two tokens share a row's probability, far above all others. T = 0.1: one among the first tokens of the row, the
    # other behind the first 2,048 of a part that begins 87.5 temperatures lower. T = 0.25: both 88.5 temperatures above
    # the first tokens of their parts, so that either part's sum in the unit of those is finite and the two together
    # are not. The drafted token is the second of them.
    vocab = 151936
    part = 8 * -(-(vocab // 8) // (5 if rows else 32))
    case = Drafts([2, 2, 2], vocab, 1, where == "draft", [temperature] * 3, seed=70)
    if temperature == 0.1:
        row = torch.randn(vocab, generator=torch.Generator().manual_seed(71)).clamp(-2, 2) * 4
        row[100], row[part + 7], row[part + 3000] = 24.75, 16.0, 24.75
        token = part + 3000
    else:
        row = torch.full((vocab,), -20.0)
        row[::part] = 0.0
        row[part + 3000] = row[2 * part + 4000] = 22.125
        token = 2 * part + 4000
    flat = torch.full((vocab,), -30.0)
    flat[token], flat[5] = 0.0, 1.4 * temperature  # 0.2 and 0.8
    for r in (0, 2, 4):
        (case.logits if where == "target" else case.draft)[r] = row
        if where == "draft":
            case.logits[r] = flat
        case.tokens[r + 1] = token
    case.uniforms[[1, 3, 5]] = [0.1, 0.75, 0.55]
    _, _, _, prob, _, _, _ = case.reference()
    assert abs(prob[1] - (0.5 if where == "target" else 0.4)) < 0.01
    _same_with_rows(nvb, case, rows)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows", [0, 240])
@pytest.mark.parametrize("temperature", [0.01, 0.02, 0.04, 0.15])
def test_verify_low_temperatures_of_long_rows(nvb, temperature, rows, draft):
    case = Drafts([2] * 24, 151936, 1, draft, [temperature] * 24, seed=72)
    # the drafts: the target's second highest, whose probability lies between 0 and 1/2
    top = case.logits.float().topk(2, 1).indices.numpy()
    case.tokens[1:48:2] = top[0:48:2, 1]
    _same_with_rows(nvb, case, rows)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows", [0, 240])
@pytest.mark.parametrize("low", [-70.0, -78.0, -85.0])
def test_verify_parts_that_begin_far_below_the_rest(nvb, low, rows, draft):
    vocab = 151936
    part = 8 * -(-(vocab // 8) // (5 if rows else 32))
    case = Drafts([2] * 12, vocab, 1, draft, [1.0] * 12, seed=73)
    for r in range(0, 24, 2):
        for x in (case.logits, case.draft) if draft else (case.logits,):
            for i in range(r % 3, -(-vocab // part), 3):
                x[r, i * part:i * part + 2048] = low
    # the drafts: likely tokens of those parts
    for r in range(0, 24, 2):
        at = (r % 3) * part + 2048
        case.tokens[r + 1] = at + int(case.logits[r, at:at + part - 2048].float().argmax())
    _same_with_rows(nvb, case, rows)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("value", [0.0, -0.0])
def test_verify_zeros_of_either_sign_are_equal_logits(nvb, draft, value):
    # T = 0, the highest logits are zeros: the lowest index among them, whatever their signs, as the sampler takes it;
    # for the test of a draft and for the next token, of nodes with and without children
    vocab = 20011
    case = Drafts([1, 2, 2, 3], vocab, 1, draft, [0.0] * 4, seed=75)
    rows, at = len(case.tokens), [17, 9000, 9001, 20010]
    case.logits[:] = -1.5
    for r in range(rows):
        case.logits[r, at[r % 3:]] = torch.tensor([value, -value, 0.0, -0.0][:len(at) - r % 3]).to(torch.bfloat16)
    case.parents[:8] = [-1, -1, 0, -1, 0, -1, 0, 1]
    case.tokens[:8] = [0, 0, at[1], 0, at[1], 0, at[2], at[1]]
    o = case.run(nvb)
    same(case, o)
    assert o["counts"].tolist() == [1, 2, 1, 2]
    want, seeds = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.from_numpy(case.seeds).cuda()
    nvb.model.layer_sample(case.logits.cuda(), torch.zeros(rows, device="cuda"), seeds, want)
    assert [want[i].item() for i in (0, 2, 3, 6)] == [o["out_tokens"][b, c - 1].item() for b, c in enumerate([1, 2, 1, 2])]


def test_verify_draws_what_wins_at_the_end_of_the_floats_range(nvb):
    # One CTA a sequence, chunks of 2,048 tokens. The first chunk's logits are 104 temperatures below zero. A token of
    # the second one scores 0.1; one of the third, 88.7 temperatures above the first chunk (e^88.7 is nearly the largest
    # float) with a noise of 15.5, scores 0.2 and is the one to draw. e^-104.1, by which the second's score outweighs
    # the first chunk's weights, is below every float.
    vocab, rows, seed, leader, token = 8192, 600, 1178, 3509, 5554  # both of the 183rd group of their chunks
    row = torch.full((vocab,), -3.0)
    row[:2048], row[leader], row[token] = -1.0, 0.00326, -151 / 1024
    row = row.to(torch.bfloat16)
    t = np.float32(1.0) / np.float32(104.0)
    score = spec_ref.as64(row) / np.float64(t) + spec_ref.gumbel(seed, vocab)
    assert np.argmax(score) == token and 0.05 < score[leader] < score[token] - 0.05 < 0.2
    i32 = dict(dtype=torch.int32, device="cuda")
    logits, seeds = row.expand(rows, vocab).contiguous().cuda(), torch.full((rows,), seed, device="cuda")
    temps = torch.full((rows,), float(t), device="cuda")
    out, path, counts = torch.zeros(rows, 1, **i32), torch.zeros(rows, 1, **i32), torch.zeros(rows, **i32)
    nvb.model.layer_verify(logits, None, torch.zeros(rows, **i32), torch.full((rows,), -1, **i32),
                           torch.zeros(rows, device="cuda"), seeds, temps, torch.arange(rows + 1, **i32), out, path,
                           counts, torch.empty(rows, device="cuda"))
    want = torch.empty(rows, **i32)
    nvb.model.layer_sample(logits, temps, seeds, want)
    assert (want == token).all() and torch.equal(out[:, 0], want)


# -------------------------------------- the drawn token, where `same` leaves it open
def _only(case, o, ref):
    f = spec_ref.as64
    sets = spec_ref.drawn_from(f(case.logits), f(case.draft) if case.draft is not None else None, case.tokens,
                               case.parents, case.seeds, case.temps, case.cu, ref[1], ref[2])
    for b, tokens in enumerate(sets):
        assert tokens is None or o["out_tokens"][b, ref[2][b] - 1].item() in tokens
    return [None if tokens is None else sorted(tokens) for tokens in sets]


def test_verify_the_widest_tree_draws_the_one_token(nvb):
    # 290 rejected looked-up drafts: what is left of P is divided 290 times, by the same sums for every token
    case = Drafts([1024], 300, 1, False, [1.0], seed=57)
    case.parents[1:1024] = 0
    case.tokens[1:1024] = np.arange(1023) % 290
    case.uniforms[:] = 0.9999
    o, ref = case.run(nvb), case.reference()
    assert _only(case, o, ref) == [[295]]


def test_verify_draws_among_the_tokens_that_rounding_leaves(nvb):
    # P and Q put all but 1e-28 on the same three tokens: their difference there is rounding, or another token is drawn
    case = Drafts([6, 5, 4], 40000, 3, True, [1.0, 1.0, 0.0], seed=59)
    for x in (case.logits, case.draft):
        x[:, 30000:30003] = 70.0 + torch.tensor([0.0, 2.0, -2.0])
    o, ref = case.run(nvb), case.reference()
    assert _only(case, o, ref)[0] == [12457, 30000, 30001, 30002]


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("spec", VERIFY)
def test_verify_draws_the_one_token(nvb, spec, draft):
    case = Drafts(**spec, draft=draft, seed=len(spec["sizes"]) + spec["vocab"])
    o, ref = case.run(nvb), case.reference()
    assert all(tokens is None or len(tokens) == 1 for tokens in _only(case, o, ref))


@pytest.mark.parametrize("where", ["target", "draft", "both", "lookup"])
@pytest.mark.parametrize("vocab", [3, 1500, 40001])
def test_verify_missing_logits_among_masked_ones(nvb, vocab, where):
    # NaN whose neighbours are all -inf (or lie outside the row): they are seen as missing there too, and what is left
    # after rejections is a number
    case = Drafts([5, 6, 4], vocab, 3, where != "lookup", [1.0, 4.0, 1.0], seed=77)
    masked = max(1, vocab - max(2, vocab // 3))
    for name, x in (("target", case.logits), ("draft", case.draft)):
        if name == where or where == "both" or (where == "lookup" and name == "target"):
            x[:, :masked] = -math.inf
            x[:, :masked:max(1, masked // 3)] = math.nan
    for b, n in enumerate(case.sizes):  # the drafts: the target's likely tokens, and one that is missing
        first = case.cu[b]
        case.parents[first + 1:first + n] = 0
        likely = masked + case.logits[first, masked:].float().argsort(descending=True).numpy()
        case.tokens[first + 1:first + n] = np.resize(likely[:n - 2], n - 1)
        case.tokens[first + 2] = 0
    case.uniforms[:] = 0.9999
    ref = case.reference()
    o = case.run(nvb)
    same(case, o, ref)
    _only(case, o, ref)
