"""The sequence operators on a GPU at their edges: what lanes without a row, hidden places, infinities, very low scores, high biases and cut sequences
leave in the results of the others; against float64 within the oracle's bounds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from bigc_hip import sequence
from oracle import sequence_oracle as O
from test_hip_sequence import DEV, TYPES, Case, eps_of, near, table, tiny_of


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("times", [1, 128])
def test_capped_scores_of_hidden_nan(t, what, times):
    """a capped score of a hidden place is NaN, and so is its slope: neither takes part (one pair of sequences: blocks of 32 rows; 128: of 128)"""
    doc = torch.tensor([0] * 30 + [-1] * 5 + [1] * 60 + [-1] * 5)
    k_doc = torch.cat([doc, torch.tensor([2] * 90)] * times + [torch.zeros(3, dtype=torch.int64)]).to(torch.int32)
    q_doc = torch.cat([doc, torch.tensor([2] * 40)] * times + [torch.zeros(3, dtype=torch.int64)]).to(torch.int32)
    c = Case(t, [(100, 100), (40, 90)] * times, heads=(4, 4), hd=32, q_doc=q_doc, k_doc=k_doc, causal=True, window=(50, -1), softcap=4.0,
             rel_table=table(8, 4), rel_map=sequence.rel_bucket_map(8, 20))
    for s in range(times):
        for x, at in ((c.q, 140 * s), (c.go, 140 * s), (c.k, 190 * s), (c.v, 190 * s)):
            x[at + 30:at + 35] = what
            x[at + 95:at + 100] = what
    got = c.check()
    for n, rows in (("o", 140 * times), ("dq", 140 * times), ("dk", 190 * times), ("dv", 190 * times), ("d_rel_table", 8)):
        assert torch.isfinite(got[n][:rows]).all(), n


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n", [2, 33, 100])
@pytest.mark.parametrize("times", [1, 128])
def test_rows_whose_scores_are_all_far_below_zero(t, n, times):
    """softmax does not care for an offset that all scores share; nor do the gradients of the last keys, beside which there are lanes without a key"""
    c = Case(t, [(n, n)] * times, heads=(4, 4), hd=32, qk=0.5)
    a = (40 / 32 ** 0.5) ** 0.5                                             # a^2 hd / sqrt(hd) = 40
    c.q = (c.q.float() + a).to(c.t)
    c.k = (c.k.float() - a).to(c.t)
    c.check()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n", [2, 33, 100])
@pytest.mark.parametrize("value", [100.0, -100.0])
@pytest.mark.parametrize("times", [1, 64])
def test_biases_beyond_the_exponents_range(t, n, value, times):
    """2^(100 log2 e) is no f32: lanes without a row, whose scores have no maximum taken off, leave nothing in the table's gradient"""
    Case(t, [(n, n), (n, 2 * n)] * times, heads=(4, 4), hd=32, rel_table=value + table(8, 4), rel_map=sequence.rel_bucket_map(8, 20)).check()
