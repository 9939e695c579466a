"""Values at the ends of their range in the latent-attention operators, on the
GPU: what a query does not see has no part in its result, what it sees counts
alike wherever it lies in a tile. Forms and tolerances of test_latent_gpu.py."""
import pytest
import torch

from test_latent_gpu import Expanded

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
    # seen, with probabilities of 2^-150 and less: less than 2^-22 of the largest value for all 400 together
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
