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


def even_spread(c, n):
    """gradients of one sequence of n rows whose every row spreads evenly, P = 1 / n, and the bounds of their errors: P and dS take the half type's rounding r, delta that of an
    o from P in two parts (2 r^2), and the sums in f32 at most 2 (hd + n + 16) steps of 2^-24 of the absolute values they add"""
    q, k, v, go = (x[:n, 0].double() for x in (c.q, c.k, c.v, c.go))
    r, u = eps_of(c.t) / 2, 2.0 ** -24
    scale, e = c.hd ** -0.5, 2 * (c.hd + n + 16) * u
    o = v.mean(0, keepdim=True)
    ds = (go @ v.t() - go @ o.t()) / n
    reach = (go.abs() @ v.abs().t() + (go.abs() @ v.abs().mean(0, keepdim=True).t())) / n
    es = reach * (e + 2 * r * r) + r * ds.abs()
    want = dict(dq=scale * ds @ k, dk=scale * ds.t() @ q, dv=(go.sum(0, keepdim=True) / n).expand(n, -1))
    tol = dict(dq=scale * es @ k.abs(), dk=scale * es.t() @ q.abs(), dv=((r + e) * go.abs().sum(0, keepdim=True) / n).expand(n, -1))
    return {name: (w, tol[name] + (r + u) * (w.abs() + tol[name])) for name, w in want.items()}


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("value", [-1e5, -1e7, -1e8, -1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("n", [4, 70])
def test_gradients_of_rows_with_one_very_low_bias(t, value, n):
    """Every visible key of every row has the same very low bias.  From -1e9 on no f32 holds bias + score, and the row spreads evenly; at the others the scores' rest in f32 is
    given its place in the bound by leaving the scores out (scale 0 where they would still count)."""
    lost = value <= -1e9
    c = Case(t, [(n, n)], heads=(1, 1), hd=64, rel_table=torch.full((4, 1), value), rel_map=sequence.rel_bucket_map(4, 2 * n), **({} if lost else dict(scale=0.0)))
    got = c.run()
    want = even_spread(c, n)
    near("o", got["o"][:n, 0], c.v[:n, 0].double().mean(0, keepdim=True).expand(n, -1), 2 * (eps_of(c.t) + 2.0 ** -20) * c.v[:n, 0].double().abs().mean(0))
    for name in ("dq", "dk", "dv"):
        w, tol = want[name]
        if not lost and name != "dv":
            w, tol = torch.zeros_like(w), torch.zeros_like(tol)
        near(name, got[name][:n, 0], w, tol, tiny_of(c.t))
    # a row's dS adds up to nothing, its error to that of the bound above: (e + 2 r^2) times sum |d_o| (|v| + |o|)
    most = (2 * (64 + n + 16) * 2.0 ** -24 + eps_of(c.t) ** 2 / 2) * 2 * float((c.go[:n].double().abs().sum((1, 2)) * c.v[:n].double().abs().max()).sum())
    assert float(got["d_rel_table"].double().sum().abs()) <= most


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min])
def test_gradients_with_buckets_of_the_lowest_value(t, value):
    tab = table(8, 2)
    tab[3] = value
    tab[0] = value
    Case(t, [(60, 60), (1, 1), (5, 90)], rel_table=tab, rel_map=sequence.rel_bucket_map(8, 20)).check()
    c = Case(t, [(70, 70)], rel_table=torch.full((8, 2), value), rel_map=sequence.rel_bucket_map(8, 20))
    got = c.run()
    if value == float("-inf"):
        assert all((got[n] == 0).all() for n in ("dq", "dk", "dv", "d_rel_table"))


CLEAN = {}


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("what", [float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["q", "k", "v", "go"])
@pytest.mark.parametrize("times", [1, 160])
def test_a_document_with_infinities_leaves_the_others_alone(t, what, where, times):
    """a document of Inf that shares blocks, waves and tiles with one that ends long behind it, and one before (160 times the same sequence: blocks of 128 rows)"""
    n = 600
    doc = torch.tensor([0] * 70 + [1] * 50 + [2] * 480 + [0] * 3, dtype=torch.int32)
    c = Case(t, [(n, n)], hd=32, q_doc=doc, k_doc=doc)
    if t not in CLEAN:
        CLEAN[t] = c.want()
    want = CLEAN[t]
    getattr(c, where)[70:120, :, 3] = what                               # (one column: dS is Inf then, not NaN)
    q, k, v, go = (x[:n].repeat(times, 1, 1).to(DEV) for x in (c.q, c.k, c.v, c.go))
    docs = doc[:n].repeat(times).to(DEV)
    off = n * torch.arange(times + 1, dtype=torch.int32, device=DEV)
    o, saved = sequence.attend(q, k, v, off, off, n, n, q_doc=docs, k_doc=docs, save=True)
    keep = torch.cat([torch.arange(70), torch.arange(120, n)])
    for name, g in zip(("o", "dq", "dk", "dv"), (o,) + sequence.attend_bwd(saved, go)[:3]):
        for s in range(0, times, 53):
            near(name, g[n * s:n * (s + 1)][keep.to(DEV)], want[name][keep], want["tol_" + name][keep], tiny_of(c.t))


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("nq", [1, 40, 300])
def test_a_score_of_minus_infinity_takes_no_weight(t, nq):
    """a seen key with -Inf in a column where every query holds 1: the score is -Inf whatever the other bits of 1 are, in rows few or many"""
    c = Case(t, [(nq, 300)], heads=(2, 2), hd=32)
    c.q[..., 5] = 1.0
    c.k[20, :, 5] = float("-inf")
    got = c.run()
    doc = torch.zeros(303, dtype=torch.int32)
    doc[20] = -1                                                            # the same key behind a mask
    c.kw.update(q_doc=torch.zeros(nq + 3, dtype=torch.int32), k_doc=doc)
    want = c.want()
    for name in ("o", "lse", "dq", "dk", "dv"):
        n = nq if name in ("o", "lse", "dq") else 300
        near(name, got[name][:n], want[name][:n], want["tol_" + name][:n], tiny_of(c.t))


@pytest.mark.parametrize("t", sorted(TYPES))
def test_rows_behind_a_cut_are_zero(t, monkeypatch):
    """sequences longer than max_q and max_k are cut to them; what lies behind the cut is a row outside every sequence"""
    c = Case(t, [(5, 5), (90, 90), (0, 7), (70, 20)], heads=(4, 2), hd=40)
    (q, k, v, go), _ = c.args(DEV)
    off = c.q_off.to(DEV), c.k_off.to(DEV)
    for max_q, max_k in ((64, 16), (0, 16), (64, 0), (3, 90)):
        monkeypatch.setattr(torch.Tensor, "new_empty", lambda self, shape, dtype=None: self.new_full(shape, 99, dtype=dtype or self.dtype))
        o, saved = sequence.attend(q, k, v, *off, max_q, max_k, save=True)
        got = dict(zip(("dq", "dk", "dv"), sequence.attend_bwd(saved, go)), o=o)
        kept = torch.full(q.shape, 7.0, dtype=c.t, device=DEV)
        sequence.attend(q, k, v, *off, max_q, max_k, out=kept, save=True)      # (as above: without, half types keep fewer bits of P)
        monkeypatch.undo()
        for name, offs, longest in (("o", c.q_off, max_q), ("dq", c.q_off, max_q), ("dk", c.k_off, max_k), ("dv", c.k_off, max_k)):
            own = torch.zeros(got[name].shape[0], dtype=torch.bool)
            for a, b in zip(offs[:-1].tolist(), offs[1:].tolist()):
                own[a:min(b, a + longest)] = True
            assert (got[name].cpu()[~own] == 0).all(), name
            assert (got[name].cpu()[own] != 99).all(), name
            if name == "o":
                assert (kept.cpu()[~own] == 7).all() and torch.equal(kept.cpu()[own], got["o"].cpu()[own])


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("cap", [64.0, 65.0, 1e3, 1e4, 1e6, 1e20, 1e37])
def test_caps_far_above_the_scores(t, cap):
    """a cap that hardly bends a score leaves it with all its bits"""
    Case(t, [(70, 70), (1, 200), (40, 90)], softcap=cap, causal=True, rel_table=table(8, 2), rel_map=sequence.rel_bucket_map(8, 30)).check()
    Case(t, [(1, 300), (1, 7)], softcap=cap, causal=True).check(train=False)


def test_many_short_caches_beside_room_for_long_ones():
    """one token for each of 256 streams with 64 heads over one key head, where max_k is that of a cache of 131072 rows"""
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(1, 40, (256,), generator=g)
    k_off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)
    q_off = torch.arange(257, dtype=torch.int32)
    q, k, v = (torch.randn(n, h, 32, generator=g).to(torch.bfloat16) for n, h in ((256, 64), (int(lens.sum()), 1), (int(lens.sum()), 1)))
    o = sequence.attend(q.to(DEV), k.to(DEV), v.to(DEV), q_off.to(DEV), k_off.to(DEV), 1, 131072, causal=True)
    want = O.attention(q[:8], k, v, q_off[:9], k_off[:9], causal=True, half_eps=eps_of(torch.bfloat16))
    near("o", o[:8], want["o"], want["tol_o"])
    want = O.attention(q[248:], k, v, q_off[:9], k_off[248:], causal=True, half_eps=eps_of(torch.bfloat16))
    near("o", o[248:], want["o"], want["tol_o"])


@pytest.mark.parametrize("value", [-1e8, -3e7, 1e8])
def test_a_large_common_bias_takes_no_second_pass(value):
    """f16: a bias of 1e8 on every distance costs no more than none (the pass over non-finite results took 6.2 times as long here)"""
    n, h = 2048, 8
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(n, h, 64, generator=g).to(torch.float16).to(DEV) for _ in range(3))
    off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    bucket = sequence.rel_bucket_map(4, 8).to(DEV)

    def fastest(bias):
        table, times = torch.full((4, h), bias, device=DEV), []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            sequence.attend(q, k, v, off, off, n, n, rel_table=table, rel_map=bucket)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert fastest(value) < 3 * fastest(0.0)
