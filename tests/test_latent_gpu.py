"""The latent-attention operators on the GPU against plain 64-bit forms.

Attention's tolerance, per element: the output is rounded to BF16 (half a step,
2^-8 of the value); each probability may be rounded to BF16 before the product
with the values (2^-8 of sum p |v|); the scores are FP32 sums of d products,
off by at most d steps of 2^-24 of sum |q k| (doubled: the tensor core's sums
truncate), which moves every probability by as much, relatively, and its sum
too. The sums over keys are FP32, one rounding for 16 keys (2^-23 of sum p |v|
each, truncated). FP32 exponentials and sums of the probabilities add 2^-16 at
most.

The store's tolerance: half a BF16 step, and for the latents the FP32 norm
(2^-20: a sum of 512 squares by halves, a square root and two products), for
rotated values two FP32 products and a sum of |a| and |z|.
"""
import math

import numpy as np
import pytest
import torch

import latent_ref as ref

pytestmark = pytest.mark.gpu

BF16_HALF = 2.0 ** -8
SCALE = 1.0 / math.sqrt(192)


def up(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def close(out, lse, want, rows, width, keys):
    o, s = ref.as64(out), ref.as64(lse)
    assert (o[rows:] == 7.0).all() and (s[rows:] == 7.0).all(), "rows behind the last sequence were written"
    o, s = o[:rows], s[:rows]
    ro, rs, weight, size = want
    score = 2 * width * 2.0 ** -24 * size
    sums = (keys / 16 + 1) * 2.0 ** -23 + 2.0 ** -16
    with np.errstate(invalid="ignore"):
        tol = BF16_HALF * np.abs(ro) + (BF16_HALF * (1 + BF16_HALF) + 2 * score[..., None] + sums) * weight
        fine = np.isfinite(ro)
        assert np.array_equal(np.isnan(o), np.isnan(ro))
        assert (np.abs(o - ro)[fine] <= tol[fine]).all(), float((np.abs(o - ro) / tol)[fine].max())
        fine = np.isfinite(rs)
        assert np.array_equal(np.isnan(s), np.isnan(rs))
        assert np.array_equal(s[~fine & ~np.isnan(rs)], rs[~fine & ~np.isnan(rs)])
        tol = score + 2.0 ** -16 + 2.0 ** -22 * np.abs(rs)
        assert (np.abs(s - rs)[fine] <= tol[fine]).all(), float((np.abs(s - rs) / tol)[fine].max())


# ------------------------------------------------------------ absorbed form
class Absorbed:
    def __init__(self, queries, lens, heads, page=256, seed=0, spare_rows=3, spare_pages=2, scratch_sms=None):
        rng, g = np.random.RandomState(seed), torch.Generator().manual_seed(seed)
        self.queries, self.lens, self.heads, self.page = list(queries), list(lens), heads, page
        pages = [(max(x, 0) + page - 1) // page for x in lens]
        self.blocks, self.stride = sum(pages) + spare_pages, max(max(pages), 1)
        order, at = rng.permutation(self.blocks), 0
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        for b, m in enumerate(pages):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.cu = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
        self.rows = int(self.cu[-1]) + spare_rows
        self.q = torch.randn(self.rows, heads, 576, generator=g).to(torch.bfloat16)
        self.cache = torch.randn(self.blocks, page, 576, generator=g).to(torch.bfloat16)
        # what lies behind a sequence, and in pages that nobody has, is not a number
        used = np.zeros(self.blocks * page, bool)
        for b, length in enumerate(lens):
            j = np.arange(max(length, 0))
            used[self.table[b, j // page] * page + j % page] = True
        self.cache.view(-1, 576)[torch.from_numpy(~used)] = math.nan
        self.sms = scratch_sms

    def slot(self, b, j):
        return int(self.table[b, j // self.page]) * self.page + j % self.page

    def args(self):
        return dict(q=self.q.cuda(), cache=self.cache.cuda(), cu_q=up(self.cu),
                    kv_lens=up(np.array(self.lens, np.int32)), block_table=up(self.table))

    def scratch(self, nvb):
        s = nvb.latent_scratch("cuda")
        if self.sms:
            s = s[:nvb.library().nvb_latent_scratch_floats(self.sms)]
        return s.fill_(math.nan)  # nothing may be taken from what it held before

    def run(self, nvb, args=None, stream=None, scratch=None, max_q=None):
        out = torch.full((self.rows, self.heads, 512), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((self.rows, self.heads), 7.0, device="cuda")
        scratch = self.scratch(nvb) if scratch is None else scratch
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        nvb.paged_latent_fwd(**(args or self.args()), out=out, lse=lse, max_q=max_q or max(max(self.queries), 1),
                             scale=SCALE, scratch=scratch, stream=stream)
        torch.cuda.synchronize()
        assert nvb.device_error() == 0
        return out, lse

    def check(self, out, lse):
        want = ref.absorbed(ref.as64(self.q), ref.as64(self.cache), self.cu, self.lens, self.table, SCALE)
        close(out, lse, want, int(self.cu[-1]), 576, max(max(self.lens), 1))

    def go(self, nvb, **kw):
        out, lse = self.run(nvb, **kw)
        self.check(out, lse)
        return out, lse


@pytest.mark.parametrize("queries, lens", [
    ([1], [1]), ([1], [2]), ([1], [63]), ([1], [64]), ([1], [65]), ([1], [127]), ([1], [129]), ([1], [500]),
    ([2], [2]), ([2], [65]), ([3], [300]), ([5], [64]), ([5], [67]), ([9], [1000]), ([64], [64]), ([65], [190]),
    ([1, 1, 1, 1], [1, 700, 64, 257]), ([4, 1, 9, 2], [4, 700, 138, 66])])
def test_absorbed(nvb, queries, lens):
    Absorbed(queries, lens, 16, seed=sum(lens)).go(nvb)


@pytest.mark.parametrize("heads", [1, 5, 8, 15, 17, 20, 33, 48, 63, 64, 65, 96, 128, 130, 256])
@pytest.mark.parametrize("queries", [1, 3])
def test_absorbed_head_counts(nvb, heads, queries):
    Absorbed([queries, queries], [130, 321], heads, seed=heads).go(nvb)


@pytest.mark.parametrize("page", [64, 128, 192, 256, 1024])
def test_absorbed_page_sizes(nvb, page):
    Absorbed([1, 2, 1], [1500, 63, 700], 16, page, seed=page).go(nvb)


def test_absorbed_queries_that_see_no_key(nvb):
    # more queries than keys, sequences without keys, without queries, with lengths that cannot be
    case = Absorbed([5, 2, 0, 1, 3, 1, 70], [2, 0, 100, 1, 200, 65, 64], 16, seed=1)
    case.go(nvb)
    args = case.args()
    case.lens[4] = -3
    case.lens[5] = case.stride * case.page + 1
    args["kv_lens"] = up(np.array(case.lens, np.int32))
    case.check(*case.run(nvb, args=args))


def test_absorbed_bad_pages_mask_their_tokens(nvb):
    case = Absorbed([1, 2, 1], [900, 1025, 256], 20, seed=2)
    case.table[0, 1], case.table[1, 4], case.table[2, 0] = -1, case.blocks, 2 ** 31 - 1
    case.go(nvb)


def test_absorbed_lone_long_sequences(nvb):
    Absorbed([1], [20000], 16, seed=3).go(nvb)
    Absorbed([3], [9001], 40, 64, seed=4).go(nvb)
    Absorbed([1], [6000], 128, 128, seed=5).go(nvb)


@pytest.mark.parametrize("seed", range(6))
def test_absorbed_ragged_batches(nvb, seed):
    rng = np.random.RandomState(seed)
    batch = [200, 30, 7, 64, 3, 500][seed]
    lens = [int(math.exp(rng.uniform(0, math.log([300, 1500, 4000, 600, 6000, 130][seed])))) for _ in range(batch)]
    queries = [int(rng.randint(0, 5)) for _ in lens]
    queries[-1] = max(queries[-1], 1)
    Absorbed(queries, lens, [16, 32, 64, 4, 128, 8][seed], [256, 64, 128, 64, 256, 64][seed], seed=seed).go(nvb)


@pytest.mark.parametrize("heads, queries", [(128, [1, 2, 1]), (96, [3, 1, 2]), (256, [1, 1, 2])])
def test_absorbed_row_tiles_that_read_their_keys_together(nvb, heads, queries):
    # more tiles than L2 is trusted with, sequences of different numbers of row tiles
    Absorbed(queries, [30000, 12001, 20000], heads, 64, seed=heads).go(nvb)


def test_absorbed_context_of_millions(nvb):
    # the pages of 1024 keys over and over: each key's probability is shared by its copies
    times = 4200
    case = Absorbed([1], [1024], 16, 256, seed=16)
    args = case.args()
    args["kv_lens"] = up(np.array([1024 * times], np.int32))
    args["block_table"] = args["block_table"].repeat(1, times)
    out, lse = case.run(nvb, args=args)
    want = ref.absorbed(ref.as64(case.q), ref.as64(case.cache), case.cu, case.lens, case.table, SCALE)
    want[1] += math.log(times)
    close(out, lse, want, 1, 576, 1024 * times / 148)


@pytest.mark.parametrize("sms", [1, 2, 5, 37])
def test_absorbed_with_less_scratch(nvb, sms):
    Absorbed([1, 2, 1, 1], [700, 1300, 3, 64], 48, seed=sms, scratch_sms=sms).go(nvb)


@pytest.mark.parametrize("max_q", [1, 2, 40])
def test_absorbed_max_q_only_guides(nvb, max_q):
    Absorbed([3, 1, 7], [700, 1300, 64], 32, seed=7).go(nvb, max_q=max_q)


def test_absorbed_largest_bounds_of_a_call(nvb):
    # the most sequences, heads and max_q and a table of a million keys: their product passes 64 bits
    case = Absorbed([2], [700], 256, seed=17)
    batch, page, mine = 65535, 1 << 20, 40000
    args = case.args()
    cache = torch.zeros(1, page, 576, dtype=torch.bfloat16, device="cuda")
    for j in range(0, 700, case.page):
        at, n = case.slot(0, j), min(case.page, 700 - j)
        cache[0, j:j + n] = case.cache.view(-1, 576)[at:at + n].cuda()
    cu, lens = torch.zeros(batch + 1, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32)
    cu[mine + 1:], lens[mine] = 2, 700
    table = torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
    args.update(cache=cache, cu_q=cu.cuda(), kv_lens=lens.cuda(), block_table=table)
    case.check(*case.run(nvb, args=args, max_q=2 ** 31 - 1))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_absorbed_keys_that_a_query_does_not_see(nvb, value):
    # the last two drafts' rows are not finite: the first queries' results do not change
    case = Absorbed([4, 1], [131, 90], 16, seed=8)
    clean, clean_lse = case.go(nvb)
    for j, at in ((129, 3), (130, 575), (130, 100)):
        case.cache.view(-1, 576)[case.slot(0, j), at] = value
    out, lse = case.run(nvb)
    assert torch.equal(out[:2], clean[:2]) and torch.equal(lse[:2], clean_lse[:2])
    assert torch.equal(out[4:5], clean[4:5]) and torch.equal(lse[4:5], clean_lse[4:5])
    want = ref.absorbed(ref.as64(case.q), ref.as64(case.cache), case.cu, case.lens, case.table, SCALE)
    bad = np.isnan(want[1][:4])  # LSE of queries that see them
    if math.isnan(value):
        assert bad[2:].all()
    assert np.array_equal(np.isnan(ref.as64(lse)[:4]), bad)
    assert np.isnan(ref.as64(out)[:4][bad]).all()


def test_absorbed_scores_far_apart(nvb):
    # probabilities from 1 down to 0, maxima that rise from tile to tile by more than 2^8
    case = Absorbed([2, 1], [700, 321], 16, seed=9)
    steps = torch.linspace(0.2, 6.0, case.cache.shape[1])[None, :, None]
    case.cache = (case.cache.float() * steps).to(torch.bfloat16)
    case.q = (case.q.float() * 3).to(torch.bfloat16)
    case.go(nvb)


def test_absorbed_equal_in_every_run(nvb):
    case = Absorbed([1, 2, 1, 1, 1], [3000, 1300, 3, 640, 5000], 32, seed=10)
    first = case.go(nvb)
    for _ in range(5):
        again = case.run(nvb)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_absorbed_without_lse_on_another_stream(nvb):
    case = Absorbed([1, 2], [700, 1300], 16, seed=11)
    want = case.go(nvb)
    stream = torch.cuda.Stream()
    got = case.run(nvb, stream=stream)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    out = torch.zeros_like(want[0])
    nvb.paged_latent_fwd(**case.args(), out=out, max_q=2, scale=SCALE, scratch=nvb.latent_scratch("cuda"))
    torch.cuda.synchronize()
    assert torch.equal(out[:3], want[0][:3])


def test_absorbed_captured_with_lengths_that_change(nvb):
    case = Absorbed([1, 1, 1], [900, 700, 64], 16, seed=12)
    args, scratch = case.args(), nvb.latent_scratch("cuda")
    out = torch.zeros(case.rows, 16, 512, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(case.rows, 16, device="cuda")

    def step():
        nvb.paged_latent_fwd(**args, out=out, lse=lse, max_q=1, scale=SCALE, scratch=scratch)

    step()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = nvb.capture(step, keep=[out, lse, scratch, *args.values()], stream=side)
        for lens in ([900, 700, 64], [1, 650, 63], [513, 2, 1]):
            args["kv_lens"].copy_(up(np.array(lens, np.int32)))
            out.fill_(7.0)
            lse.fill_(7.0)
            graph.replay(stream=side)
            side.synchronize()
            case.lens = lens
            case.check(out, lse)
    graph.close()


def test_absorbed_calls_that_overlap_with_scratch_of_their_own(nvb):
    cases = [Absorbed([1] * 20, [400 + 90 * i for i in range(20)], 32, seed=s) for s in (13, 14)]
    want = [c.go(nvb) for c in cases]
    args, streams = [c.args() for c in cases], [torch.cuda.Stream() for _ in cases]
    scratch = [nvb.latent_scratch("cuda") for _ in cases]
    outs = [torch.zeros_like(w[0]) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for a, s, x, o in zip(args, streams, scratch, outs):
            nvb.paged_latent_fwd(**a, out=o, max_q=1, scale=SCALE, scratch=x, stream=s)
    torch.cuda.synchronize()
    for o, w, c in zip(outs, want, cases):
        assert torch.equal(o[:c.cu[-1]], w[0][:c.cu[-1]])


def test_absorbed_cache_past_32_bit_offsets(nvb):
    # 2^31 elements are 3.7 million rows; the last pages of a cache of 4.2 million
    case = Absorbed([1, 1], [130, 200], 16, seed=15)
    args = case.args()
    blocks = 16500
    cache = torch.zeros(blocks, 256, 576, dtype=torch.bfloat16, device="cuda")
    cache[blocks - case.blocks:] = args["cache"]
    args["cache"] = cache
    table = args["block_table"]
    args["block_table"] = torch.where(table >= 0, table + (blocks - case.blocks), table)
    case.check(*case.run(nvb, args=args))


# ------------------------------------------------------------ expanded form
class Expanded:
    def __init__(self, queries, keys, heads, seed=0, spare=3, std=1.5):
        g = torch.Generator().manual_seed(seed)
        self.queries, self.keys, self.heads = list(queries), list(keys), heads
        self.cu_q = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
        self.cu_k = np.concatenate([[0], np.cumsum(keys)]).astype(np.int32)
        self.rows, self.total_k = int(self.cu_q[-1]) + spare, int(self.cu_k[-1]) + spare
        self.q = (torch.randn(self.rows, heads, 192, generator=g) * std).to(torch.bfloat16)
        self.kv = torch.randn(self.total_k, heads, 256, generator=g).to(torch.bfloat16)
        self.rope = torch.randn(self.total_k, 64, generator=g).to(torch.bfloat16)
        self.kv[self.cu_k[-1]:] = math.nan  # what lies behind the last sequence is not a number
        self.rope[self.cu_k[-1]:] = math.nan

    def args(self):
        return dict(q=self.q.cuda(), kv=self.kv.cuda(), k_rope=self.rope.cuda(), cu_q=up(self.cu_q), cu_k=up(self.cu_k))

    def run(self, nvb, args=None, stream=None, max_q=None):
        out = torch.full((self.rows, self.heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((self.rows, self.heads), 7.0, device="cuda")
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        nvb.latent_prefill_fwd(**(args or self.args()), out=out, lse=lse, max_q=max_q or max(max(self.queries), 1),
                               scale=SCALE, stream=stream)
        torch.cuda.synchronize()
        assert nvb.device_error() == 0
        return out, lse

    def check(self, out, lse):
        want = ref.expanded(ref.as64(self.q), ref.as64(self.kv), ref.as64(self.rope), self.cu_q, self.cu_k, SCALE)
        close(out, lse, want, int(self.cu_q[-1]), 192, max(max(self.keys), 1))

    def go(self, nvb, **kw):
        out, lse = self.run(nvb, **kw)
        self.check(out, lse)
        return out, lse


@pytest.mark.parametrize("queries, keys", [
    ([1], [1]), ([1], [300]), ([2], [2]), ([63], [63]), ([64], [64]), ([65], [65]), ([127], [127]), ([128], [128]),
    ([129], [129]), ([255], [256]), ([256], [256]), ([257], [257]), ([300], [300]), ([5], [133]), ([130], [700]),
    ([513], [515]), ([128], [1000]), ([1, 7, 200, 64], [1, 9, 200, 500])])
def test_expanded(nvb, queries, keys):
    Expanded(queries, keys, 2, seed=sum(keys)).go(nvb)


@pytest.mark.parametrize("heads", [1, 3, 16, 40, 256])
def test_expanded_head_counts(nvb, heads):
    Expanded([40, 7], [70, 7], heads, seed=heads).go(nvb)


def test_expanded_queries_that_see_no_key(nvb):
    case = Expanded([5, 2, 0, 3, 200, 140], [2, 0, 100, 3, 60, 1], 4, seed=1)
    case.go(nvb)
    # keys outside the tensor: the sequence's rows are 0
    args = case.args()
    args["cu_k"][-1] = case.total_k + 1
    out, lse = case.run(nvb, args=args)
    last = slice(int(case.cu_q[-2]), int(case.cu_q[-1]))
    assert (out[last] == 0).all() and (lse[last] == -math.inf).all()


@pytest.mark.parametrize("seed", range(5))
def test_expanded_ragged_batches(nvb, seed):
    rng = np.random.RandomState(seed)
    batch = [40, 9, 3, 17, 150][seed]
    queries = [int(math.exp(rng.uniform(0, math.log([200, 400, 700, 150, 30][seed])))) for _ in range(batch)]
    keys = [n + int(rng.choice([0, 0, 1, 100, 300])) for n in queries]
    queries[1] = 0
    Expanded(queries, keys, [2, 3, 2, 5, 1][seed], seed=seed).go(nvb)


@pytest.mark.parametrize("queries, keys, heads", [
    ([600], [600], 64), ([130, 300, 257, 1, 255], [130, 420, 257, 600, 256], 40), ([129] * 12, [129] * 12, 13),
    ([300, 5, 200, 140], [260, 5, 10, 1], 50), ([400, 270], [1100, 399], 52)])
def test_expanded_pairs_of_query_tiles(nvb, queries, keys, heads):
    # enough items for all SMs: two tiles each, the second one whole, in part or empty, with fewer keys than queries
    Expanded(queries, keys, heads, seed=heads).go(nvb)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_expanded_pairs_keys_that_a_query_does_not_see(nvb, value):
    case = Expanded([500, 330], [500, 400], 50, seed=12)
    clean, clean_lse = case.go(nvb)
    for key in (3, 130, 300, 499):
        case.kv[key, :, 128 + key % 128] = value
    out, lse = case.run(nvb)
    assert torch.equal(lse, clean_lse) and torch.equal(out[500:], clean[500:])
    want = torch.zeros(500, 128, dtype=torch.bool, device="cuda")
    for key in (3, 130, 300, 499):
        want[key:, key % 128] = True
    bad = torch.isnan(out[:500]) if math.isnan(value) else out[:500] == value
    assert torch.equal(bad, want[:, None].expand(500, 50, 128))
    assert torch.equal(torch.where(bad, 0, out[:500]), torch.where(bad, 0, clean[:500]))


def test_expanded_leaves_rows_past_max_q(nvb):
    case = Expanded([300, 40], [300, 50], 2, seed=3)
    want = case.go(nvb)
    out, lse = case.run(nvb, max_q=129)
    kept = [r for r in range(340) if not 129 <= r < 300]
    assert torch.equal(out[kept], want[0][kept]) and torch.equal(lse[kept], want[1][kept])
    assert (out[129:300] == 7.0).all() and (lse[129:300] == 7.0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_expanded_keys_that_a_query_does_not_see(nvb, value):
    case = Expanded([150, 70], [150, 200], 3, seed=4)
    clean, clean_lse = case.go(nvb)
    case.kv[100, 1, 200] = value  # a value: seen from query 100 on
    case.kv[149, 2, 5] = value    # a key
    case.rope[140] = value        # a key of all heads
    out, lse = case.run(nvb)
    assert torch.equal(out[:100], clean[:100]) and torch.equal(lse[:100], clean_lse[:100])
    assert torch.equal(out[150:220], clean[150:220]) and torch.equal(lse[150:220], clean_lse[150:220])
    assert torch.equal(out[100:140, [0, 2]], clean[100:140, [0, 2]])
    assert torch.equal(lse[:140], clean_lse[:140])
    want = ref.expanded(ref.as64(case.q), ref.as64(case.kv), ref.as64(case.rope), case.cu_q, case.cu_k, SCALE)
    got = ref.as64(out)[100:140, 1]
    spot = want[0][100:140, 1]
    assert np.array_equal(np.isnan(got), np.isnan(spot)) and np.array_equal(np.isinf(got), np.isinf(spot))
    if not math.isnan(value):
        assert (got[:, 72] == value).all()
    assert np.array_equal(np.isnan(ref.as64(lse)[140:150]), np.isnan(want[1][140:150]))


def test_expanded_values_seen_in_full_tiles_that_are_not_finite(nvb):
    # every query of the second tile sees the key
    case = Expanded([300], [300], 1, seed=5)
    case.kv[17, 0, 140] = math.inf
    out, lse = case.run(nvb)
    want = ref.expanded(ref.as64(case.q), ref.as64(case.kv), ref.as64(case.rope), case.cu_q, case.cu_k, SCALE)
    got = ref.as64(out)[:300, 0]
    assert np.array_equal(np.isinf(got), np.isinf(want[0][:, 0])) and not np.isnan(got).any()


def test_expanded_scores_far_apart(nvb):
    case = Expanded([300, 20], [300, 320], 2, seed=6, std=6.0)
    case.kv = (case.kv.float() * torch.linspace(0.2, 4.0, case.total_k)[:, None, None]).to(torch.bfloat16)
    case.go(nvb)


def test_expanded_rope_rows_of_longer_rows_and_other_streams(nvb):
    case = Expanded([200, 33], [200, 90], 4, seed=7)
    want = case.go(nvb)
    args = case.args()
    wide = torch.zeros(case.total_k, 576, dtype=torch.bfloat16, device="cuda")
    wide[:, 512:] = args["k_rope"]
    args["k_rope"] = wide[:, 512:]
    got = case.run(nvb, args=args, stream=torch.cuda.Stream())
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_expanded_equal_in_every_run_and_captured(nvb):
    case = Expanded([400, 33, 128, 260], [400, 90, 500, 260], 8, seed=8)
    want = case.go(nvb)
    args = case.args()
    out, lse = torch.full_like(want[0], 7.0), torch.full_like(want[1], 7.0)

    def step():
        nvb.latent_prefill_fwd(**args, out=out, lse=lse, max_q=400, scale=SCALE)

    step()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = nvb.capture(step, keep=[out, lse, *args.values()], stream=side)
        for _ in range(5):
            out.fill_(7.0)
            lse.fill_(7.0)
            graph.replay(stream=side)
            side.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    graph.close()


def test_expanded_calls_that_overlap(nvb):
    cases = [Expanded([300, 20, 128], [300, 320, 140], 6, seed=s) for s in (9, 10)]
    want = [c.go(nvb) for c in cases]
    args, streams = [c.args() for c in cases], [torch.cuda.Stream() for _ in cases]
    outs = [torch.full_like(w[0], 7.0) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for a, s, o in zip(args, streams, outs):
            nvb.latent_prefill_fwd(**a, out=o, max_q=300, scale=SCALE, stream=s)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w[0])


def test_expanded_keys_past_32_bit_offsets(nvb):
    # 64 heads x 256 values: 2^31 elements are 131,072 keys
    heads, first = 64, 131072
    case = Expanded([70], [70], heads, seed=11, spare=0)
    args = case.args()
    kv = torch.zeros(first + 70, heads, 256, dtype=torch.bfloat16, device="cuda")
    kv[first:] = args["kv"]
    rope = torch.zeros(first + 70, 64, dtype=torch.bfloat16, device="cuda")
    rope[first:] = args["k_rope"]
    args.update(kv=kv, k_rope=rope, cu_k=up(np.array([first, first + 70], np.int32)))
    case.check(*case.run(nvb, args=args))


# ------------------------------------------------------------ store, gather
def table_of(nvb, positions=512):
    return up(nvb.host.rope_table(positions, 64, 10000.0, scaling="linear", factor=2.0))


def check_rotated(got, x, table, positions, interleaved):
    t = ref.as64(table)
    inside = (positions >= 0) & (positions < len(t))
    t = np.where(inside[:, None], t[np.clip(positions, 0, len(t) - 1)], np.concatenate([np.ones(32), np.zeros(32)]))
    cos, sin = t[:, :32], t[:, 32:]
    if x.ndim == 3:
        cos, sin = cos[:, None], sin[:, None]
    want = ref.rotate(x, cos, sin, interleaved)
    size = ref.rotate(np.abs(x), np.abs(cos), -np.abs(sin), interleaved)
    size = np.maximum(size, ref.rotate(np.abs(x), np.abs(cos), np.abs(sin), interleaved))
    assert (np.abs(got - want) <= BF16_HALF * np.abs(want) + 2.0 ** -22 * np.abs(size)).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows, heads", [(1, 1), (1, 16), (3, 5), (33, 8), (70, 9), (257, 20)])
def test_store(nvb, rows, heads, interleaved):
    rng, g = np.random.RandomState(rows), torch.Generator().manual_seed(rows)
    blocks, page = rows // 64 + 3, 64
    table = table_of(nvb)
    fused = (torch.randn(rows, 640, generator=g) * 2).to(torch.bfloat16).cuda()
    kv = fused[:, 64:]  # a slice of a longer projection
    weight = (1 + 0.2 * torch.randn(512, generator=g)).to(torch.bfloat16).cuda()
    q = torch.randn(rows, heads, 192, generator=g).to(torch.bfloat16).cuda()
    q_out = torch.randn(rows, heads, 576, generator=g).to(torch.bfloat16).cuda()
    cache = torch.randn(blocks, page, 576, generator=g).to(torch.bfloat16).cuda()
    positions = rng.randint(-2, 515, rows).astype(np.int32)
    slots = rng.permutation(blocks * page)[:rows].astype(np.int32)
    if rows > 2:
        slots[0], slots[1] = -1, blocks * page  # skipped
    before, q_before = ref.as64(cache).reshape(-1, 576), ref.as64(q_out)
    nvb.latent_store(kv, weight, up(positions), up(slots), cache, q=q[..., 128:], q_out=q_out[..., 512:], eps=1e-5,
                     rope_table=table, interleaved=interleaved)
    torch.cuda.synchronize()
    after, x = ref.as64(cache).reshape(-1, 576), ref.as64(kv)
    written = (slots >= 0) & (slots < blocks * page)
    rest = np.setdiff1d(np.arange(blocks * page), slots[written])
    assert np.array_equal(after[rest], before[rest])
    want = ref.normalise(x[written, :512], ref.as64(weight), 1e-5)
    got = after[slots[written]]
    assert (np.abs(got[:, :512] - want) <= (BF16_HALF + 2.0 ** -20) * np.abs(want)).all()
    check_rotated(got[:, 512:], x[written, 512:], table, positions[written], interleaved)
    turned = ref.as64(q_out)
    assert np.array_equal(turned[..., :512], q_before[..., :512])
    check_rotated(turned[..., 512:], ref.as64(q)[..., 128:], table, positions, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_store_in_place_queries_only_and_latents_only(nvb, interleaved):
    g, table = torch.Generator().manual_seed(1), table_of(nvb)
    q = torch.randn(40, 7, 192, generator=g).to(torch.bfloat16).cuda()
    positions = up(np.arange(40, dtype=np.int32) * 3)
    apart = torch.zeros(7, 40, 64, dtype=torch.bfloat16, device="cuda")  # heads first
    nvb.latent_store(None, None, positions, None, None, q=q[..., 128:], q_out=apart.transpose(0, 1), rope_table=table,
                     interleaved=interleaved)
    before = ref.as64(q)
    nvb.latent_store(None, None, positions, None, None, q=q[..., 128:], rope_table=table, interleaved=interleaved)
    torch.cuda.synchronize()
    assert torch.equal(q[..., 128:], apart.transpose(0, 1))
    assert np.array_equal(ref.as64(q)[..., :128], before[..., :128])
    check_rotated(ref.as64(q)[..., 128:], before[..., 128:], table, np.arange(40) * 3, interleaved)
    kv = torch.randn(1, 576, generator=g).to(torch.bfloat16).cuda()
    weight = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(2, 64, 576, dtype=torch.bfloat16, device="cuda")
    nvb.latent_store(kv, weight, positions[:1], up(np.array([65], np.int32)), cache, rope_table=table,
                     interleaved=interleaved)
    torch.cuda.synchronize()
    assert (cache[1, 1] != 0).any() and not (cache[0] != 0).any()


@pytest.mark.parametrize("kv_first", [False, True])
def test_store_of_one_projection(nvb, kv_first):
    # queries and latents are slices of the same rows, the queries turned in place
    g, table = torch.Generator().manual_seed(3), table_of(nvb)
    x = torch.randn(37, 5 * 192 + 576, generator=g).to(torch.bfloat16).cuda()
    kv, q = (x[:, :576], x[:, 576:]) if kv_first else (x[:, 5 * 192:], x[:, :5 * 192])
    q, before = q.view(37, 5, 192), ref.as64(x)
    turned = torch.zeros(37, 5, 64, dtype=torch.bfloat16, device="cuda")
    caches = torch.zeros(2, 1, 64, 576, dtype=torch.bfloat16, device="cuda")
    weight, positions = torch.ones(512, dtype=torch.bfloat16, device="cuda"), up(np.arange(37, dtype=np.int32) * 5)
    slots = up(np.arange(37, dtype=np.int32))
    nvb.latent_store(kv.clone(), weight, positions, slots, caches[0], q=q[..., 128:].clone(), q_out=turned, rope_table=table)
    nvb.latent_store(kv, weight, positions, slots, caches[1], q=q[..., 128:], rope_table=table)
    torch.cuda.synchronize()
    assert torch.equal(caches[0], caches[1]) and torch.equal(q[..., 128:], turned)
    want = torch.from_numpy(before).to(torch.bfloat16).cuda()
    parts = want[:, 576:] if kv_first else want[:, :5 * 192]
    parts.view(37, 5, 192)[..., 128:] = turned
    assert torch.equal(x, want)


def test_store_strides_of_single_rows_and_heads(nvb):
    g, table = torch.Generator().manual_seed(2), table_of(nvb)
    x = torch.randn(3, 5, 64, generator=g).to(torch.bfloat16).cuda()
    positions = up(np.array([7, 8, 9], np.int32))
    for part, at in ((x[:1], positions[:1]), (x[:, :1], positions), (x[1:2, 2:3], positions[1:2])):
        odd = part.as_strided(part.shape, (part.stride(0) if part.shape[0] > 1 else 3,
                                           part.stride(1) if part.shape[1] > 1 else 1, 1), part.storage_offset())
        out = torch.zeros(part.shape, dtype=torch.bfloat16, device="cuda")
        nvb.latent_store(None, None, at, None, None, q=odd, q_out=out, rope_table=table)
        torch.cuda.synchronize()
        check_rotated(ref.as64(out), ref.as64(part), table, at.cpu().numpy(), False)


def test_store_values_at_the_ends_of_the_range(nvb):
    # zero rows (eps alone under the root), large and tiny ones; infinities and NaN stay in their row
    table = table_of(nvb)
    kv = torch.zeros(5, 576, dtype=torch.bfloat16, device="cuda")
    kv[1] = 1e18
    kv[2] = 1e-30
    kv[3] = math.nan
    weight = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(1, 64, 576, dtype=torch.bfloat16, device="cuda")
    nvb.latent_store(kv, weight, up(np.zeros(5, np.int32)), up(np.arange(5, dtype=np.int32)), cache, rope_table=table)
    torch.cuda.synchronize()
    got = ref.as64(cache)[0]
    assert (got[0] == 0).all() and (got[1, :512] == 1).all() and np.isfinite(got[2]).all()
    assert np.isnan(got[3]).all() and (got[4:] == 0).all()


@pytest.mark.parametrize("lens, page", [([1], 64), ([64], 64), ([0, 65, 1], 64), ([300, 0, 0, 7, 1000], 256),
                                        ([5] * 40, 64), ([9, 130, 77], 48)])
def test_gather(nvb, lens, page):
    rng, g = np.random.RandomState(len(lens)), torch.Generator().manual_seed(page)
    pages = [(x + page - 1) // page for x in lens]
    blocks = sum(pages) + 2
    order, at = rng.permutation(blocks), 0
    table = np.full((len(lens), max(max(pages), 1)), -1, np.int32)
    for b, m in enumerate(pages):
        table[b, :m] = order[at:at + m]
        at += m
    cache = torch.randn(blocks, page, 576, generator=g).to(torch.bfloat16).cuda()
    if len(lens) > 2 and pages[-1]:
        table[-1, 0] = blocks  # a page that the cache does not have
    cu = np.concatenate([[2], 2 + np.cumsum(lens)]).astype(np.int32)  # two rows before the first sequence
    total = int(cu[-1]) + 3
    latent = torch.full((total, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    rope = torch.full((total, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    wide = torch.full((total, 640), 7.0, dtype=torch.bfloat16, device="cuda")
    nvb.latent_gather(cache, up(table), up(cu), latent, rope)
    nvb.latent_gather(cache, up(table), up(cu), wide[:, :512], wide[:, 512:576])
    torch.cuda.synchronize()
    want, flat = np.full((total, 576), 7.0), ref.as64(cache).reshape(-1, 576)
    for b, n in enumerate(lens):
        for j in range(n):
            p = table[b, j // page]
            want[cu[b] + j] = flat[p * page + j % page] if 0 <= p < blocks else 0.0
    assert np.array_equal(ref.as64(latent), want[:, :512]) and np.array_equal(ref.as64(rope), want[:, 512:])
    assert np.array_equal(ref.as64(wide)[:, :576], want) and (wide[:, 576:] == 7.0).all()


def test_gather_past_32_bit_offsets(nvb):
    blocks = 16500
    cache = torch.zeros(blocks, 256, 576, dtype=torch.bfloat16, device="cuda")
    cache[-1] = torch.randn(256, 576, device="cuda").to(torch.bfloat16)
    latent = torch.zeros(300, 512, dtype=torch.bfloat16, device="cuda")
    rope = torch.zeros(300, 64, dtype=torch.bfloat16, device="cuda")
    nvb.latent_gather(cache, up(np.array([[blocks - 1, 0]], np.int32)), up(np.array([0, 300], np.int32)), latent, rope)
    torch.cuda.synchronize()
    assert torch.equal(latent[:256], cache[-1, :, :512]) and torch.equal(rope[:256], cache[-1, :, 512:])
    assert not latent[256:].any()


# --------------------------------------------------------------- together
def test_a_prompt_in_chunks_and_decode_steps_through_all_operators(nvb):
    """Two prompts in two chunks by the expanded form, then decode steps by the absorbed form, against 64-bit
    attention of the same layer over the values that the cache holds."""
    heads, page, g = 8, 64, torch.Generator().manual_seed(3)
    lens = [150, 90]
    table = np.array([[3, 0, 5, 7], [1, 4, 2, 6]], np.int32)
    total = 200

    def values(std, *shape):
        return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16).cuda()

    kv_in, q_in = values(2.0, 2, total, 576), values(1.0, 2, total, heads, 192)
    weight = (1 + 0.1 * torch.randn(512, generator=g)).to(torch.bfloat16).cuda()
    w_k, w_v = values(512 ** -0.5, heads, 128, 512), values(512 ** -0.5, heads, 128, 512)
    w_kv = torch.cat([w_k, w_v], 1)  # [heads, 256, 512]
    cache = torch.zeros(8, page, 576, dtype=torch.bfloat16, device="cuda")
    rope_table, scratch = table_of(nvb), nvb.latent_scratch("cuda")
    results = [[], []]
    done = [0, 0]

    def slots(b, lo, hi):
        j = np.arange(lo, hi)
        return table[b, j // page] * page + j % page

    def step(counts, absorbed):
        spans = [(d, d + c) for d, c in zip(done, counts)]
        pick = lambda x: torch.cat([x[b, lo:hi] for b, (lo, hi) in enumerate(spans)])  # noqa: E731
        q = pick(q_in).contiguous()
        rows = q.shape[0]
        positions = np.concatenate([np.arange(lo, hi) for lo, hi in spans]).astype(np.int32)
        where = np.concatenate([slots(b, lo, hi) for b, (lo, hi) in enumerate(spans)]).astype(np.int32)
        cu_q = up(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        kv_lens = np.array([hi for _, hi in spans], np.int32)
        wide = torch.zeros(rows, heads, 576, dtype=torch.bfloat16, device="cuda")
        q_out = wide[..., 512:] if absorbed else q[..., 128:]
        nvb.latent_store(pick(kv_in), weight, up(positions), up(where), cache, q=q[..., 128:], q_out=q_out,
                         rope_table=rope_table, interleaved=True)
        if absorbed:
            wide[..., :512] = torch.einsum("rhd,hdc->rhc", q[..., :128], w_k)
            mid = torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device="cuda")
            nvb.paged_latent_fwd(wide, cache, mid, cu_q, up(kv_lens), up(table), max_q=max(counts), scale=SCALE,
                                 scratch=scratch)
            out = torch.einsum("rhc,hdc->rhd", mid, w_v)
        else:
            cu_k = up(np.concatenate([[0], np.cumsum(kv_lens)]).astype(np.int32))
            keys = int(kv_lens.sum())
            latent = torch.empty(keys, 512, dtype=torch.bfloat16, device="cuda")
            rope = torch.empty(keys, 64, dtype=torch.bfloat16, device="cuda")
            nvb.latent_gather(cache, up(table), cu_k, latent, rope)
            kv = (latent @ w_kv.reshape(-1, 512).T).view(keys, heads, 256)
            out = torch.empty(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
            nvb.latent_prefill_fwd(q, kv, rope, out, cu_q, cu_k, max_q=max(counts), scale=SCALE)
        at = 0
        for b, (lo, hi) in enumerate(spans):
            results[b].append(out[at:at + hi - lo])
            at += hi - lo
            done[b] = hi

    step([70, 90], False)
    step([80, 1], False)
    for counts in ([1, 1], [1, 1], [3, 2], [1, 4]):
        step(counts, True)
    torch.cuda.synchronize()
    assert nvb.device_error() == 0
    t = ref.as64(rope_table)
    for b in range(2):
        n = done[b]
        rows = ref.as64(cache).reshape(-1, 576)[slots(b, 0, n)]
        x = ref.as64(kv_in[b, :n])
        want = ref.normalise(x[:, :512], ref.as64(weight), 1e-6)
        assert (np.abs(rows[:, :512] - want) <= (BF16_HALF + 2.0 ** -20) * np.abs(want)).all()
        q = ref.as64(q_in[b, :n])
        q_rope = ref.rotate(q[..., 128:], t[:n, None, :32], t[:n, None, 32:], True)
        k = np.einsum("mc,hdc->mhd", rows[:, :512], ref.as64(w_k))
        v = np.einsum("mc,hdc->mhd", rows[:, :512], ref.as64(w_v))
        s = (np.einsum("nhd,mhd->nhm", q[..., :128], k) + np.einsum("nhd,md->nhm", q_rope, rows[:, 512:])) * SCALE
        s = np.where(np.arange(n)[None, None, :] <= np.arange(n)[:, None, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want = np.einsum("nhm,mhd->nhd", p, v)
        got = ref.as64(torch.cat(results[b]))
        # BF16 queries, keys or absorbed queries, values, probabilities and sums between the steps: each of scores is
        # off by up to three half steps of sum |q k| and moves its probability by as much
        size = (np.einsum("nhd,mhd->nhm", np.abs(q[..., :128]), np.abs(k)) +
                np.einsum("nhd,md->nhm", np.abs(q_rope), np.abs(rows[:, 512:]))) * SCALE
        moved = 2 * 3 * BF16_HALF * np.max(np.where(np.isfinite(s), size, 0), -1)
        mass = np.einsum("nhm,mhd->nhd", p, np.einsum("mc,hdc->mhd", np.abs(rows[:, :512]), np.abs(ref.as64(w_v))))
        tol = (moved[..., None] + 4 * BF16_HALF) * mass
        assert (np.abs(got - want) <= tol).all()
        assert np.abs(got - want).mean() <= 0.05 * np.abs(want).mean()
