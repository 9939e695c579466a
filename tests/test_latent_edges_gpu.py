"""Values at the ends of their range in the latent-attention operators, on the
GPU: what a query does not see has no part in its result, what it sees counts
alike wherever it lies in a tile. Forms and tolerances of test_latent_gpu.py."""
import math

import numpy as np
import pytest
import torch

import latent_ref as ref
from test_latent_gpu import BF16_HALF, SCALE, Absorbed, Expanded, table_of, up

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ expanded form
@pytest.mark.parametrize("value", [3.3e38, -3.3e38, 1e36])
@pytest.mark.parametrize("queries, keys, heads", [([300, 140], [300, 200], 2), ([500, 330], [500, 400], 50)])
def test_expanded_large_values_that_a_query_does_not_see(nvb, queries, keys, heads, value):
    # from one key of a tile on, at each place of 16, in tiles at the causal border of lone tiles and of pairs
    case = Expanded(queries, keys, heads, seed=21)
    clean, clean_lse = case.go(nvb)
    for seq, first in ((0, 100), (1, keys[1] - 33)):
        case.kv[case.cu_k[seq] + first:case.cu_k[seq + 1], :, 128:] = value
    out, lse = case.run(nvb)
    assert torch.equal(lse, clean_lse)
    for seq, first in ((0, 100), (1, keys[1] - 33)):
        rows = slice(int(case.cu_q[seq]), int(case.cu_q[seq]) + first - (keys[seq] - queries[seq]))
        assert torch.equal(out[rows], clean[rows])


def test_expanded_large_values_of_keys_that_weigh_nothing(nvb):
    # seen, with probabilities of 2^-150 and less: all 400 of them together add less than 2^-13
    case = Expanded([200], [400], 2, seed=22)
    case.q[:, :, 0], case.kv[:, :, 0] = 16.0, 0.0
    keys = torch.arange(400)
    far = (keys % 23 == 5) | (keys % 16 >= 14)
    case.kv[:400][far, :, 0] = -256.0  # -295 in the exponent of e
    case.kv[:400][far, :, 128:] = 0.0
    clean, clean_lse = case.go(nvb)
    case.kv[:400][far, :, 128:] = 3.3e38
    out, lse = case.run(nvb)
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


# ------------------------------------------------------------ absorbed form
def same_where_not_finite(case, out, lse):
    want = ref.absorbed(ref.as64(case.q), ref.as64(case.cache), case.cu, case.lens, case.table, SCALE)
    rows = int(case.cu[-1])
    o, s = ref.as64(out)[:rows], ref.as64(lse)[:rows]
    assert np.array_equal(np.isnan(o), np.isnan(want[0])) and np.array_equal(np.isnan(s), np.isnan(want[1]))
    assert np.isfinite(o[~np.isnan(o)]).all()
    return want


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("queries, lens, heads, places", [
    ([4, 1], [131, 90], 16, ((129, 3), (130, 100), (130, 511))),  # in the last tile, two keys of it seen in part
    ([4, 1], [131, 90], 16, ((3, 3), (70, 200))),                 # in tiles that all rows see whole
    ([5, 1], [131, 90], 33, ((126, 5), (127, 6), (128, 7))),      # row tiles of two queries, at a tile's end
    ([70], [190], 1, ((125, 0), (130, 256), (189, 300))),         # a row tile over two tiles of keys
    ([3, 1], [9000, 700], 8, ((8998, 130), (8999, 131), (10, 7))),  # joined from parts
    ([2, 2], [3000, 2900], 130, ((2998, 1), (2999, 2)))])         # several row tiles, joined
def test_absorbed_not_finite_in_seen_keys(nvb, queries, lens, heads, places, value):
    # scores of either infinity or NaN: an infinite score makes the sums NaN, or has probability 0 and 0 * inf its element
    case = Absorbed(queries, lens, heads, 64, seed=23)
    for j, at in places:
        case.cache.view(-1, 576)[case.slot(0, j), at] = value
    want = same_where_not_finite(case, *case.run(nvb))
    if math.isinf(value):  # both kinds are there
        assert (np.isnan(want[0]).any(-1) & ~np.isnan(want[1])).any() and np.isnan(want[1]).any()


@pytest.mark.parametrize("parts", [2, 40])
def test_absorbed_nan_score_in_a_part_that_weighs_nothing(nvb, parts):
    # all other keys of the part are 2^-400 of those of the others
    case = Absorbed([1], [64 * parts * 4], 8, 64, seed=24)
    flat, first = case.cache.view(-1, 576), [case.slot(0, j) for j in range(64 * 4)]
    case.q[:, :, 0], case.cache[..., 0] = 16.0, 0.0
    flat[first, 0] = -256.0
    clean = case.run(nvb)
    flat[case.slot(0, 77), 575] = math.nan
    out, lse = case.run(nvb)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isfinite(clean[0]).all() and torch.isfinite(clean[1]).all()


# ------------------------------------------------------------ store, gather
def stored(nvb, kv, weight, eps):
    rows = kv.shape[0]
    cache = torch.full((rows // 64 + 1, 64, 576), 7.0, dtype=torch.bfloat16, device="cuda")
    nvb.latent_store(kv.cuda(), weight.cuda(), up(np.zeros(rows, np.int32)), up(np.arange(rows, dtype=np.int32)), cache,
                     eps=eps, rope_table=table_of(nvb))
    torch.cuda.synchronize()
    got = ref.as64(cache).reshape(-1, 576)
    assert (got[rows:] == 7.0).all()
    return got[:rows]


def near(got, want):
    # half a BF16 step (2^-134 below the normal numbers), the FP32 norm as in test_latent_gpu.py
    assert (np.abs(got - want) <= (BF16_HALF + 2.0 ** -20) * np.abs(want) + 2.0 ** -134).all()


@pytest.mark.parametrize("eps", [1e30, 1e38, 3.4e38])
def test_store_eps_beside_large_values(nvb, eps):
    g = torch.Generator().manual_seed(32)
    kv, weight = torch.randn(6, 576, generator=g), torch.ones(512, dtype=torch.bfloat16)
    kv[1:] *= 2.0 ** torch.tensor([50.0, 60.0, 62.0, 64.0, 100.0])[:, None]
    kv = kv.to(torch.bfloat16)
    near(stored(nvb, kv, weight, eps)[:, :512], ref.normalise(ref.as64(kv)[:, :512], 1.0, float(np.float32(eps))))


def test_store_rows_of_large_and_ordinary_values(nvb):
    # the sum of squares just below and above the largest float, huge values among ordinary ones, tiny rows
    g = torch.Generator().manual_seed(31)
    kv = torch.randn(40, 576, generator=g)
    weight = (1 + 0.2 * torch.randn(512, generator=g)).to(torch.bfloat16)
    for r in range(8):
        kv[r, :512] *= 2.0 ** (55 + r)   # 512 of them: squares that sum to 2^(119 + 2 r)
    kv[8:16, 5] = 2.0 ** torch.arange(60, 68).float()
    kv[16, 17], kv[17, 511], kv[18, 0] = 2.0 ** 100, -2.0 ** 120, 3e38
    kv[19, :512] = 3e38
    kv[20, :256] *= 2.0 ** 64
    kv[21, :512] = 1e-30
    kv[22, :512] *= 1e-20
    kv = kv.to(torch.bfloat16)
    want = ref.normalise(ref.as64(kv)[:, :512], ref.as64(weight), 1e-6)
    got = stored(nvb, kv, weight, 1e-6)
    near(got[:, :512], want)
    assert (got[21, :512] != 0).all()


def test_store_infinities_stay_in_their_row(nvb):
    g = torch.Generator().manual_seed(33)
    kv, weight = torch.randn(6, 576, generator=g).to(torch.bfloat16), torch.ones(512, dtype=torch.bfloat16)
    kv[1, 7], kv[3, 500], kv[4, 575] = math.inf, -math.inf, math.inf
    got = stored(nvb, kv, weight, 1e-6)
    x = ref.as64(kv)
    for r in (0, 2, 4, 5):
        near(got[r, :512], ref.normalise(x[r, :512], 1.0, 1e-6))
    for r, at in ((1, 7), (3, 500)):  # inf / inf, and finite / inf
        assert np.isnan(got[r, at]) and (np.delete(got[r, :512], at) == 0).all()
    assert np.array_equal(np.isfinite(got[:, 512:]).all(1), [True, True, True, True, False, True])
    assert np.isfinite(got[4, 512:543]).all()  # the pairs beside the infinity's


@pytest.mark.parametrize("rows", [1, 33])
def test_store_latents_alone(nvb, rows):
    g = torch.Generator().manual_seed(34)
    kv, weight = torch.randn(rows, 576, generator=g).to(torch.bfloat16), (torch.randn(512, generator=g)).to(torch.bfloat16)
    got = stored(nvb, kv, weight, 1e-5)
    near(got[:, :512], ref.normalise(ref.as64(kv)[:, :512], ref.as64(weight), 1e-5))
    assert np.array_equal(got[:, 512:], ref.as64(kv)[:, 512:])  # position 0


@pytest.mark.parametrize("first", [-2 ** 31, -2 ** 31 + 3, -2 ** 30, -2])
@pytest.mark.parametrize("page", [1, 64])
def test_gather_offsets_below_zero(nvb, first, page):
    # the first sequence's rows are keys from -first on: behind its page table, as far as they are
    cache = torch.randn(6, page, 576, device="cuda").to(torch.bfloat16)
    table = np.array([[5, 0, 2], [1, 3, 4]], np.int32)
    cu = np.array([first, 4, 4 + page], np.int32)
    latent = torch.full((5 + page, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    rope = torch.full((5 + page, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    nvb.latent_gather(cache, up(table), up(cu), latent, rope)
    torch.cuda.synchronize()
    want, flat = np.full((5 + page, 576), 7.0), ref.as64(cache).reshape(-1, 576)
    for row in range(4 + page):
        b, key = (0, row - first) if row < 4 else (1, row - 4)
        want[row] = flat[table[b, key // page] * page + key % page] if key < 3 * page else 0.0
    assert np.array_equal(np.concatenate([ref.as64(latent), ref.as64(rope)], 1), want)
