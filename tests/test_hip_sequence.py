"""GPU parity of the sequence operators (bigc_hip/sequence.py) against their float64 statements (oracle/sequence_oracle.py), element by element
within bounds that the oracle derives from the types' rounding steps."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from bigc_hip import _lib, sequence
from oracle import sequence_oracle as O

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def eps_of(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps


def tiny_of(t):
    """what a result of f16 may be off below its normal range: half the step of its subnormals"""
    return 2.0 ** -25 if t == torch.float16 else 0.0


def near(name, got, want, tol, tiny=0.0):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    inf = torch.isinf(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name + ": NaN"
    assert torch.equal(got[inf], want[inf]), name + ": infinities"
    off = (got - want).abs()
    off[inf | torch.isnan(want)] = 0
    bad = off > tol + tiny + 1e-30
    assert not bad.any(), "%s: %d of %d elements off, worst %.3g where %.3g is allowed (value %.3g)" % (
        name, int(bad.sum()), bad.numel(), float(off[bad].max()), float((tol + tiny).expand_as(off)[bad][off[bad].argmax()]), float(want[bad][off[bad].argmax()]))


class Case(object):
    """ragged inputs on the CPU and their device copies"""

    def __init__(self, t, lens, heads=(2, 2), hd=64, seed=0, qk=1.5, tail=3, pad_cols=0, **kw):
        g = torch.Generator().manual_seed(seed + 17 * len(lens) + hd)
        self.t, self.kw = TYPES[t], {k: v for k, v in kw.items() if v is not None}
        nq, nk = sum(a for a, _ in lens) + tail, sum(b for _, b in lens) + tail          # `tail` rows behind the last sequence
        h, hk = heads
        self.q_off = torch.tensor(np.cumsum([0] + [a for a, _ in lens]), dtype=torch.int32)
        self.k_off = torch.tensor(np.cumsum([0] + [b for _, b in lens]), dtype=torch.int32)
        self.max_q, self.max_k = max([a for a, _ in lens] + [0]), max([b for _, b in lens] + [0])

        def make(n, heads, s):
            return (torch.randn(n, heads, hd + pad_cols, generator=g) * s).to(self.t)

        self.q, self.k, self.v, self.go = make(nq, h, qk), make(nk, hk, qk), make(nk, hk, 1.0), make(nq, h, 1.0)
        self.hd = hd

    def args(self, dev):
        kw = {k: (v.to(dev) if isinstance(v, torch.Tensor) else v) for k, v in self.kw.items()}
        cut = [x.to(dev)[..., :self.hd] for x in (self.q, self.k, self.v, self.go)]
        return cut, kw

    def want(self, train=True):
        (q, k, v, go), kw = self.args("cpu")
        return O.attention(q, k, v, self.q_off, self.k_off, d_o=go if train else None, half_eps=eps_of(self.t), **kw)

    def run(self, train=True, dev=DEV):
        (q, k, v, go), kw = self.args(dev)
        o, saved = sequence.attend(q, k, v, self.q_off.to(dev), self.k_off.to(dev), self.max_q, self.max_k, save=True, **kw)
        got = dict(o=o, lse=saved.lse)
        if train:
            got.update(zip(("dq", "dk", "dv", "d_rel_table"), sequence.attend_bwd(saved, go)))
        torch.cuda.synchronize()
        return got

    def check(self, train=True):
        got, want = self.run(train), self.want(train)
        nq = int(self.q_off[-1])
        for name in ("o", "lse", "dq", "dk", "dv", "d_rel_table"):
            if name in want:
                g, w, t = got[name], want[name], want["tol_" + name]
                if name in ("o", "lse"):
                    g, w, t = g[:nq], w[:nq], t[:nq]
                near(name, g, w, t, tiny_of(self.t) if g.dtype == torch.float16 else 0.0)
        return got


RAGGED = [(1, 1), (3, 3), (64, 64), (0, 5), (65, 130), (7, 0), (33, 257), (129, 129)]


def table(n, h, seed=3):
    return torch.randn(n, h, generator=torch.Generator().manual_seed(seed))


VARIANTS = {
    "plain": {},
    "causal": dict(causal=True),
    "cap": dict(softcap=4.0, causal=True),
    "slopes": dict(slopes=torch.tensor([0.25, 0.01])),
    "window": dict(window=(40, 9)),
    "window_causal": dict(causal=True, window=(31, -1)),
    "window_0": dict(window=(0, 0)),
    "prefix": dict(causal=True, window=(20, -1), prefix_len=torch.tensor([0, 2, 70, 1, 100, 0, 5, 64], dtype=torch.int32)),
    "buckets": dict(rel_table=table(32, 2), rel_map=sequence.rel_bucket_map(32, 100)),
    "buckets_causal_cap": dict(rel_table=table(9, 2), rel_map=sequence.rel_bucket_map(9, 64, two_sided=False), causal=True, softcap=8.0),
    "bucket_one": dict(rel_table=table(1, 2), rel_map=torch.zeros(1, dtype=torch.int32)),
    "everything": dict(softcap=6.0, causal=True, window=(50, -1), slopes=torch.tensor([0.1, 0.5]), rel_table=table(8, 2), rel_map=sequence.rel_bucket_map(8, 20),
                       prefix_len=torch.tensor([1, 0, 3, 2, 90, 0, 40, 11], dtype=torch.int32)),
}


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("name", sorted(VARIANTS))
def test_attention_variants(t, name):
    Case(t, RAGGED, **VARIANTS[name]).check()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("heads,hd", [((1, 1), 8), ((3, 1), 24), ((6, 2), 32), ((4, 4), 72), ((8, 2), 96), ((5, 5), 112), ((8, 1), 128), ((16, 4), 128)])
def test_attention_heads(t, heads, hd):
    Case(t, [(70, 70), (1, 100), (5, 37)], heads=heads, hd=hd, causal=True, slopes=torch.linspace(0.0, 0.3, heads[0]),
         rel_table=table(6, heads[0]), rel_map=sequence.rel_bucket_map(6, 30)).check()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("group", [1, 4, 7, 40])
def test_attention_one_token(t, group):
    """single queries over caches of any length, split over the keys"""
    Case(t, [(1, n) for n in (1, 2, 31, 32, 33, 1000, 0, 4097)], heads=(2 * group, 2), hd=64, causal=True, softcap=20.0).check(train=False)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_attention_chunk_behind_a_long_cache(t):
    Case(t, [(40, 3001), (3, 700), (100, 120)], heads=(6, 2), hd=128, causal=True, window=(900, -1),
         prefix_len=torch.tensor([70, 0, 4], dtype=torch.int32)).check(train=False)


def documents(lens, seed, interleaved):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n, _ in lens:
        if interleaved:
            d = torch.randint(-1, 4, (n,), generator=g)
        else:
            d = torch.sort(torch.randint(0, 5, (n,), generator=g)).values
            d[n - n // 7:] = -1
        out.append(d)
    return torch.cat(out + [torch.zeros(3, dtype=torch.int64)]).to(torch.int32)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_documents(t, interleaved, causal):
    lens = [(300, 300), (1, 1), (77, 77), (130, 130)]
    doc = documents(lens, 5, interleaved)
    Case(t, lens, causal=causal, q_doc=doc, k_doc=doc, prefix_len=torch.tensor([9, 0, 0, 30], dtype=torch.int32)).check()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_what_a_hidden_place_holds_takes_no_part(t, what):
    """padding rows, keys behind the queries' reach and the rows behind the last sequence hold NaN or Inf"""
    lens = [(100, 100), (40, 90)]
    doc = torch.cat([torch.tensor([0] * 30 + [-1] * 5 + [1] * 60 + [-1] * 5), torch.tensor([2] * 90), torch.zeros(3, dtype=torch.int64)]).to(torch.int32)
    q_doc = torch.cat([doc[:100], doc[150:190], doc[-3:]])
    c = Case(t, lens, q_doc=q_doc, k_doc=doc, causal=True, window=(50, -1))
    for x in (c.q, c.go):
        x[30:35] = what
        x[95:100] = what
        x[140:] = what
    for x in (c.k, c.v):
        x[30:35] = what
        x[95:100] = what
        x[190:] = what
    assert bool(O.seen_matrix(40, 90, True, (50, -1))[0][:, 0].any()) is True
    want = c.want()
    assert all(torch.isfinite(want[n]).all() for n in ("dq", "dk", "dv"))
    got = c.check()
    for n in ("dq", "dk", "dv"):
        assert torch.isfinite(got[n]).all(), n


@pytest.mark.parametrize("t", sorted(TYPES))
def test_a_document_with_nan_leaves_the_others_alone(t):
    """values, keys, queries and gradients of one document are NaN: the other documents' results are what they were"""
    lens = [(200, 200)]
    doc = torch.tensor([0] * 70 + [1] * 50 + [2] * 80 + [0] * 3, dtype=torch.int32)
    clean, bad = (Case(t, lens, q_doc=doc, k_doc=doc) for _ in range(2))
    for x in (bad.q, bad.k, bad.v, bad.go):
        x[70:120] = float("nan")
    a, b = clean.run(), bad.run()
    want = clean.want()
    for n in ("o", "dq", "dk", "dv"):
        keep = torch.cat([torch.arange(70), torch.arange(120, 200)])
        near(n, b[n].cpu()[keep], want[n][keep], want["tol_" + n][keep], tiny_of(TYPES[t]))
        assert torch.isnan(b[n].cpu()[70:120]).all(), n
        assert torch.isfinite(a[n]).all()


@pytest.mark.parametrize("t", sorted(TYPES))
def test_a_seen_value_that_is_infinite_arrives(t):
    c = Case(t, [(40, 40)], causal=True)
    c.v[20, 1, 5] = float("inf")
    c.v[25, 0, 3] = float("nan")
    got = c.run(train=False)["o"].cpu()
    assert torch.isfinite(got[:20]).all()
    assert torch.isinf(got[20:40, 1, 5]).all() and (got[20:40, 1, 5] > 0).all()
    assert torch.isnan(got[25:40, 0, 3]).all()
    rest = got[:40].clone()
    rest[20:, 1, 5] = 0
    rest[25:, 0, 3] = 0
    assert torch.isfinite(rest).all()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min])
def test_bias_of_the_lowest_value(t, value):
    """a bucket of -inf hides its distances; one of the lowest finite value leaves a row that has nothing else evenly spread"""
    tab = table(8, 2)
    tab[3] = value
    tab[0] = value
    m = sequence.rel_bucket_map(8, 20)
    Case(t, [(60, 60), (1, 1), (5, 90)], rel_table=tab, rel_map=m).check(train=False)
    c = Case(t, [(6, 6)], rel_table=torch.full((8, 2), value), rel_map=m)
    got = c.run(train=False)["o"].cpu()[:6].double()
    if value == float("-inf"):
        assert (got == 0).all()
    else:
        mean = c.v[:6].double().mean(0)
        assert float((got - mean).abs().max()) < 4 * max(eps_of(TYPES[t]), 2.0 ** -20) * float(c.v[:6].double().abs().max())


@pytest.mark.parametrize("t", sorted(TYPES))
def test_large_and_small_magnitudes(t):
    """sharp rows (scores of some hundreds), values and gradients far from 1"""
    big = {"f32": 1e18, "bf16": 1e18, "f16": 64.0}[t]
    small = {"f32": 1e-18, "bf16": 1e-18, "f16": 0.125}[t]
    for scale_v, scale_g in ((big, small), (small, big)):
        c = Case(t, [(90, 90), (3, 70)], qk=6.0)
        c.v = (c.v.float() * scale_v).to(c.t)
        c.go = (c.go.float() * scale_g).to(c.t)
        c.check()


def test_rows_outside_every_sequence_stay_as_they_were():
    c = Case("bf16", [(5, 9), (20, 20)], tail=70)
    (q, k, v, go), kw = c.args(DEV)
    out = torch.full(q.shape, 7.0, dtype=c.t, device=DEV)
    got = sequence.attend(q, k, v, c.q_off.to(DEV), c.k_off.to(DEV), c.max_q, c.max_k, out=out)
    assert got is out and (out[25:] == 7).all() and not (out[:25] == 7).all()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strides(t):
    """rows and heads inside wider tensors, heads outside rows, and outputs of another layout"""
    c = Case(t, [(50, 80), (3, 3)], heads=(4, 2), hd=40, pad_cols=8, causal=True)
    c.check()
    (q, k, v, go), kw = c.args(DEV)
    off = (c.q_off.to(DEV), c.k_off.to(DEV), c.max_q, c.max_k)
    base = sequence.attend(q, k, v, *off, **kw)
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    out = torch.zeros(4, q.shape[0], 40, dtype=c.t, device=DEV).transpose(0, 1)
    sequence.attend(*by_head, *off, out=out, **kw)
    assert torch.equal(out, base)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_repeats_bit_for_bit(t):
    c = Case(t, [(300, 300), (90, 400)], heads=(4, 2), tail=0, causal=True, rel_table=table(16, 4), rel_map=sequence.rel_bucket_map(16, 90))
    a = c.run()
    for _ in range(3):
        b = c.run()
        for n in a:
            assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-3])
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_scales(t, scale, cap):
    """scores that fall with the product, and that do not depend on it, with and without masks and biases"""
    Case(t, [(70, 70), (1, 200), (40, 90)], scale=scale, softcap=cap, causal=True).check()
    Case(t, [(70, 70), (1, 200)], scale=scale, softcap=cap, rel_table=table(8, 2), rel_map=sequence.rel_bucket_map(8, 30)).check()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("radius", [0, 1, 700, 1023])
def test_bias_radius(t, radius):
    """biases of one distance up to a thousand, in sequences shorter and longer than that"""
    m = torch.randint(0, 5, (2 * radius + 1,), generator=torch.Generator().manual_seed(radius)).to(torch.int32)
    Case(t, [(300, 300), (60, 900)], hd=32, rel_table=table(5, 2), rel_map=m, causal=True).check()


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_bias_radius_at_its_limit(t):
    m = torch.randint(0, 5, (4095,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    for hd in (64, 128):
        Case(t, [(100, 100), (3, 700)], hd=hd, heads=(4, 2), rel_table=table(5, 4), rel_map=m).check()


def test_a_wide_bias_gradient_of_wide_f32_heads_is_refused():
    c = Case("f32", [(100, 100)], hd=128, rel_table=table(5, 2), rel_map=torch.zeros(4095, dtype=torch.int32))
    c.check(train=False)
    with pytest.raises(AssertionError, match="1023"):
        c.run()


@pytest.mark.parametrize("t", sorted(TYPES))
def test_many_blocks_and_few(t):
    """enough rows for whole blocks of 128, and the same sequences among fewer"""
    one = [(260, 260), (130, 200)]
    Case(t, one * 30, heads=(10, 5), hd=32, causal=True, softcap=9.0).check()
    Case(t, one, heads=(10, 5), hd=32, causal=True, softcap=9.0).check()


def test_a_short_sequence_in_a_large_buffer():
    """the workspace of a call goes by its sequences, not by the buffer they lie in"""
    rows = 400000
    g = torch.Generator().manual_seed(3)
    q = torch.zeros(rows, 2, 64, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.randn(5000, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    q[7] = torch.randn(2, 64, generator=g).to(torch.bfloat16).to(DEV)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    off = torch.tensor([7, 8], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    sequence.attend(q, k.to(DEV), v.to(DEV), off, torch.tensor([0, 5000], dtype=torch.int32, device=DEV), 1, 5000, out=out)
    assert torch.cuda.max_memory_allocated() - before < q.numel() * 2 + 20e6
    want = O.attention(q[7:8].cpu(), k, v, [0, 1], [0, 5000], half_eps=eps_of(torch.bfloat16))
    near("o", out[7:8], want["o"], want["tol_o"])


def test_one_row_of_any_row_stride():
    x = torch.randn(3 * 128 + 5, device=DEV)
    q = x[:128].as_strided((1, 2, 64), (131, 64, 1))
    off = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    # one key: o = (p v) (1 / p) with p = 2^r and r what fma(s, c, -m) leaves of m's rounding: three roundings of half a step, 2^-24 of the value each
    assert ((sequence.attend(q, q, q, off, off, 1, 1) - q).abs() <= 3.01 * 2.0 ** -24 * q.abs()).all()


@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("t", sorted(TYPES))
def test_the_tables_gradient_has_no_errors_of_one_sign(t, hd):
    """Over a whole row dS sums to nothing, so that the far bucket's gradient is a small difference of large sums: an error of every dP to one side, however small, adds
    up over rows and keys.  o takes one rounding (2^-25 at most, at random) for each of its 63 tiles and dP a few: sqrt(63) 2^-25 < 2^-22 each of |d_o| |o| in a
    row's sum, 2^-21 together, and rows add up as the root of their squares; what the near buckets have of their own is f32 rounding, 2^-21 of the table."""
    n, h = 2000, 4
    g = torch.Generator().manual_seed(hd)
    q, k, v, go = [torch.randn(n, h, hd, generator=g).to(TYPES[t]).to(DEV) for _ in range(4)]
    table = (0.5 * torch.randn(16, h, generator=g)).to(DEV)
    bucket = sequence.rel_bucket_map(16, 64).to(DEV)
    off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    _, saved = sequence.attend(q, k, v, off, off, n, n, rel_table=table, rel_map=bucket, save=True)
    got = sequence.attend_bwd(saved, go)[3].double()
    q, k, v, go = [x.double().transpose(0, 1).contiguous() for x in (q, k, v, go)]
    place = torch.arange(n, device=DEV)
    at = bucket.long()[(place[None] - place[:, None]).clamp(-64, 64) + 64]
    p = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) * hd ** -0.5 + table.double().T[:, at], -1)
    dp = torch.bmm(go, v.transpose(1, 2).contiguous())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    want = torch.stack([torch.zeros(16, dtype=torch.float64, device=DEV).index_add_(0, at.flatten(), x.flatten()) for x in ds], 1)
    rows = (go.norm(dim=-1) * torch.bmm(p, v).norm(dim=-1)).norm()
    assert (got - want).norm() <= 2.0 ** -21 * (rows + want.norm())


def test_two_streams_at_once():
    cases = [Case("bf16", [(300, 300), (1, 4000)], heads=(4, 2), seed=s, causal=True) for s in (1, 2)]
    want = [c.run() for c in cases]
    ins = [(c.args(DEV)[0], c.q_off.to(DEV), c.k_off.to(DEV)) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(8):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                (q, k, v, go), qo, ko = ins[i]
                o, saved = sequence.attend(q, k, v, qo, ko, c.max_q, c.max_k, save=True, causal=True)
                got[i].append((o,) + sequence.attend_bwd(saved, go)[:3])
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, n in zip(g, ("o", "dq", "dk", "dv")):
                assert torch.equal(a, want[i][n])


def test_offsets_beyond_32_bits():
    """a cache whose rows lie more than 2^32 elements apart"""
    ld = 1 << 17
    rows = (1 << 15) + 200
    g = torch.Generator().manual_seed(1)
    kv = torch.empty(rows, ld, dtype=torch.bfloat16, device=DEV)
    k, v = kv[:, 64:192].view(rows, 2, 64), kv[:, 1024:1152].view(rows, 2, 64)
    a, b = rows - 150, rows
    kv[a:b, :2048] = torch.randn(b - a, 2048, generator=g).to(torch.bfloat16).to(DEV)
    q = torch.randn(3, 2, 64, generator=g).to(torch.bfloat16)
    o = sequence.attend(q.to(DEV), k, v, torch.tensor([0, 3], dtype=torch.int32, device=DEV), torch.tensor([a, b], dtype=torch.int32, device=DEV), 3, b - a, causal=True)
    want = O.attention(q, k[a:b].cpu(), v[a:b].cpu(), [0, 3], [0, b - a], causal=True, half_eps=eps_of(torch.bfloat16))
    near("o", o, want["o"], want["tol_o"])


def test_nothing_to_do():
    z = torch.zeros(0, 2, 64, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert sequence.attend(z, z, z, one, one, 0, 0).shape == (0, 2, 64)
    off = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    none = torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    q = torch.ones(4, 2, 64, device=DEV)
    o, saved = sequence.attend(q, z, z, off, none, 4, 0, save=True)
    assert (o == 0).all() and torch.isinf(saved.lse).all()
    dq, dk, dv, _ = sequence.attend_bwd(saved, q)
    assert (dq == 0).all() and dk.shape[0] == 0
    tab = torch.ones(8, 2, device=DEV)
    o, saved = sequence.attend(z, q, q, none, off, 0, 4, rel_table=tab, rel_map=sequence.rel_bucket_map(8, 20).to(DEV), save=True)
    dq, dk, dv, dt = sequence.attend_bwd(saved, z)
    assert (dk == 0).all() and (dv == 0).all() and (dt == 0).all()


# ---- norm and rotation -------------------------------------------------------------------------------------------------------------------

def norm_case(t, rows, heads, hd, n_freq, far, seed=0, weights=True):
    g = torch.Generator().manual_seed(seed + rows + hd)
    t = TYPES[t]
    h, hk = heads
    qkv = (torch.randn(rows, (h + 2 * hk) * hd, generator=g) * 1.5).to(t)
    pos = torch.randint(0, far + 1, (rows,), generator=g).to(torch.int32)
    inv = 10000.0 ** (-torch.arange(n_freq, dtype=torch.float64) / max(1, n_freq)) if n_freq else None
    w = [1 + 0.2 * torch.randn(hd, generator=g) if weights else None for _ in range(2)]
    go = [torch.randn(rows, n, hd, generator=g).to(t) for n in (h, hk)]
    return qkv, pos, inv, w, go


def norm_tol(x, w, y, half_eps):
    """f32 arithmetic on a head: the norm to (hd + 16) u, the rotation's two products of turned columns to 8 u, then the rounding"""
    u = 2.0 ** -24
    n = x.double().abs() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6) * (1.0 if w is None else w.double().abs())
    return ((x.shape[-1] + 16) * u + 8 * u) * n.amax(-1, keepdim=True) * 2 + (half_eps / 2 + u) * y.abs()


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("rows,heads,hd,n_freq,interleaved,far", [
    (1, (8, 2), 128, 64, False, 131071), (37, (4, 4), 64, 16, False, 500), (5, (3, 1), 24, 12, True, 2 ** 31 - 1), (700, (8, 8), 64, 32, True, 5000),
    (33, (2, 1), 256, 128, False, 4096), (3, (40, 0), 8, 4, False, 10), (65, (1, 1), 96, 0, False, 0), (2049, (6, 2), 128, 64, True, 1 << 20), (9, (2, 2), 40, 5, False, 99)])
def test_head_norm_rope(t, rows, heads, hd, n_freq, interleaved, far):
    qkv, pos, inv, w, go = norm_case(t, rows, heads, hd, n_freq, far)
    h, hk = heads
    cut = lambda x: (x[:, :h * hd].view(rows, h, hd), x[:, h * hd:(h + hk) * hd].view(rows, hk, hd))  # noqa: E731
    if hd * (h + 2 * hk) * qkv.element_size() % 16:
        pytest.skip("rows of whole 16 bytes only")
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    q, k = cut(dev(qkv))
    extra = (dev(w[0]), dev(w[1]), dev(pos), dev(inv))
    got = sequence.head_norm_rope(q, k, *extra, interleaved=interleaved)
    grads = sequence.head_norm_rope_bwd(dev(go[0]), dev(go[1]), q, k, *extra, interleaved=interleaved)
    e, u = eps_of(TYPES[t]), 2.0 ** -24
    for i, (x, name) in enumerate(zip(cut(qkv), "qk")):
        if x.shape[1] == 0:
            continue
        xd, wd = x.double().requires_grad_(), w[i].double().requires_grad_()
        y = O.norm_rope(xd, wd, pos, inv, interleaved=interleaved)
        near(name, got[i], y.detach(), norm_tol(x, w[i], y.detach(), e), tiny_of(TYPES[t]))
        dx, dw = torch.autograd.grad(y, (xd, wd), go[i].double())
        G = go[i].double().abs().amax(-1, keepdim=True) * 1.5
        r = 1 / torch.sqrt((xd.detach() ** 2).mean(-1, keepdim=True) + 1e-6)
        hat = xd.detach().abs() * r
        c = (3 * hd + 64) * u
        near("d" + name, grads[i], dx, c * r * G * w[i].abs().max().double() * (1 + hat * hat.mean(-1, keepdim=True)) + (e / 2 + u) * dx.abs(), tiny_of(TYPES[t]))
        near("dw" + name, grads[2 + i], dw, (c + 64 * u + math.sqrt(rows) * u) * (G * hat).sum((0, 1)))


@pytest.mark.parametrize("t", sorted(TYPES))
def test_head_norm_rope_in_place_and_without_weights(t):
    qkv, pos, inv, w, go = norm_case(t, 50, (4, 2), 64, 32, 900, weights=False)
    q, k = qkv[:, :256].view(50, 4, 64), qkv[:, 256:384].view(50, 2, 64)
    d = qkv.to(DEV)
    qd, kd = d[:, :256].view(50, 4, 64), d[:, 256:384].view(50, 2, 64)
    want = sequence.head_norm_rope(qd, kd, None, None, pos.to(DEV), inv.to(DEV))
    near("q", want[0], O.norm_rope(q.double(), None, pos, inv), norm_tol(q, None, O.norm_rope(q.double(), None, pos, inv), eps_of(TYPES[t])), tiny_of(TYPES[t]))
    g = sequence.head_norm_rope_bwd(go[0].to(DEV), go[1].to(DEV), qd, kd, None, None, pos.to(DEV), inv.to(DEV))
    assert g[2] is None and g[3] is None
    sequence.head_norm_rope(qd, kd, None, None, pos.to(DEV), inv.to(DEV), out=(qd, kd))
    assert torch.equal(qd, want[0]) and torch.equal(kd, want[1])
    assert torch.equal(d[:, 384:].cpu(), qkv[:, 384:])


def test_head_norm_rope_rows_of_zeros_and_no_rows():
    inv = torch.ones(32, dtype=torch.float64, device=DEV)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    w = torch.ones(64, device=DEV)
    z = torch.zeros(4, 2, 64, device=DEV)
    q, k = sequence.head_norm_rope(z, z, w, w, pos, inv)
    assert (q == 0).all() and (k == 0).all()
    dq, dk, dwq, dwk = sequence.head_norm_rope_bwd(torch.ones_like(z), torch.ones_like(z), z, z, w, w, pos, inv)
    assert torch.isfinite(dq).all() and (dwq == 0).all()
    none = torch.zeros(0, 2, 64, device=DEV)
    q, k = sequence.head_norm_rope(none, none, w, w, pos[:0], inv)
    assert q.shape == (0, 2, 64)
    dq, dk, dwq, dwk = sequence.head_norm_rope_bwd(none, none, none, none, w, w, pos[:0], inv)
    assert (dwq == 0).all() and (dwk == 0).all()


# ---- together, streams and graphs --------------------------------------------------------------------------------------------------------

def layer(x, w, lens, extra, kw, go=None):
    """in-projection -> norm and rotation -> attention (-> gradients back to x and every parameter), as a model's layer would run them"""
    off, n, h, hk, hd, max_len = lens
    qkv = x @ w["in"].t()
    q, k, v = qkv[:, :h * hd].view(n, h, hd), qkv[:, h * hd:(h + hk) * hd].view(n, hk, hd), qkv[:, (h + hk) * hd:].view(n, hk, hd)
    qr, kr = sequence.head_norm_rope(q, k, w["q"], w["k"], *extra)
    o, saved = sequence.attend(qr, kr, v, off, off, max_len, max_len, rel_table=w["table"], save=True, **kw)
    if go is None:
        return o
    dq, dk, dv, dt = sequence.attend_bwd(saved, go)
    dq, dk, dwq, dwk = sequence.head_norm_rope_bwd(dq, dk, q, k, w["q"], w["k"], *extra)
    dqkv = torch.cat([dq.flatten(1), dk.flatten(1), dv.flatten(1)], 1)
    return o, dqkv @ w["in"], dqkv.t() @ x, dwq, dwk, dt


def test_a_layer_together_against_float64():
    g = torch.Generator().manual_seed(4)
    lens, h, hk, hd, d = [70, 1, 33], 4, 2, 32, 48
    n, off = sum(lens), torch.tensor([0, 70, 71, 104], dtype=torch.int32)
    x = torch.randn(n, d, generator=g)
    w = {"in": torch.randn((h + 2 * hk) * hd, d, generator=g) / d ** 0.5, "q": 1 + 0.1 * torch.randn(hd, generator=g), "k": 1 + 0.1 * torch.randn(hd, generator=g),
         "table": table(16, h)}
    m = sequence.rel_bucket_map(16, 40, two_sided=False)
    pos, inv = torch.cat([torch.arange(l) for l in lens]).to(torch.int32), 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    go = torch.randn(n, h, hd, generator=g)
    D = lambda t: t.to(DEV)  # noqa: E731
    got = layer(D(x), {k: D(v) for k, v in w.items()}, (D(off), n, h, hk, hd, 70), (D(pos), D(inv)), dict(rel_map=D(m), causal=True, softcap=10.0), D(go))
    p = {k: v.double().requires_grad_() for k, v in w.items()}
    xd = x.double().requires_grad_()
    qkv = xd @ p["in"].t()
    q = O.norm_rope(qkv[:, :h * hd].view(n, h, hd), p["q"], pos, inv)
    k = O.norm_rope(qkv[:, h * hd:(h + hk) * hd].view(n, hk, hd), p["k"], pos, inv)
    v = qkv[:, (h + hk) * hd:].view(n, hk, hd)
    outs = []
    for a, b in zip(off[:-1].tolist(), off[1:].tolist()):
        seen, dist = O.seen_matrix(b - a, b - a, True)
        for i in range(h):
            s = 10 * torch.tanh(q[a:b, i] @ k[a:b, i // 2].t() * hd ** -0.5 / 10) + p["table"][:, i][m.long()][dist.clamp(-40, 40) + 40]
            outs.append((a, b, i, torch.softmax(s.masked_fill(~seen, float("-inf")), 1) @ v[a:b, i // 2]))
    o = torch.zeros(n, h, hd, dtype=torch.float64)
    for a, b, i, y in outs:
        o = o + torch.nn.functional.pad(y, (0, 0, a, n - b)).unsqueeze(1) * torch.nn.functional.one_hot(torch.tensor(i), h)[None, :, None]
    want = [o] + list(torch.autograd.grad(o, (xd, p["in"], p["q"], p["k"], p["table"]), go.double()))
    for name, y, z in zip(("o", "dx", "din", "dwq", "dwk", "dtable"), got, want):
        # three operators of f32 after one another, sums of at most a few hundred terms each: a few hundred steps of 2^-24 of the largest value
        assert float((y.double().cpu() - z.detach()).abs().max()) < 1000 * 2.0 ** -24 * float(z.detach().abs().max()), name


@pytest.mark.parametrize("t", sorted(TYPES))
def test_captured_and_replayed(t):
    """one graph of forward and backward, replayed on changed inputs between eager calls; two graphs in turn"""
    mk = lambda seed: Case(t, [(40, 40), (1, 300), (130, 200)], heads=(4, 2), seed=seed, causal=True, rel_table=table(16, 4), rel_map=sequence.rel_bucket_map(16, 50))  # noqa: E731
    graphs = []
    for seed in (1, 2):
        c = mk(seed)
        (q, k, v, go), kw = c.args(DEV)
        q, k, v, go = (x.clone() for x in (q, k, v, go))
        off = (c.q_off.to(DEV), c.k_off.to(DEV))

        def step(q=q, k=k, v=v, go=go, off=off, kw=kw, c=c):
            o, saved = sequence.attend(q, k, v, *off, c.max_q, c.max_k, save=True, **kw)
            return (o,) + sequence.attend_bwd(saved, go)

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step, (q, k, v, go)))
    for rep in range(4):
        for graph, out, step, ins in graphs:
            for x in ins:
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(rep)).to(x.dtype))
            graph.replay()
            torch.cuda.synchronize()
            want = step()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_on_a_stream_of_its_own():
    c = Case("bf16", [(200, 200), (30, 500)], heads=(4, 2), causal=True)
    want = c.run()
    (q, k, v, go), kw = c.args(DEV)
    off = (c.q_off.to(DEV), c.k_off.to(DEV))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = []
        for _ in range(5):
            o, saved = sequence.attend(q, k, v, *off, c.max_q, c.max_k, save=True, **kw)
            got.append((o,) + sequence.attend_bwd(saved, go)[:3])
    s.synchronize()
    for g in got:
        for a, n in zip(g, ("o", "dq", "dk", "dv")):
            assert torch.equal(a, want[n])


def test_gradients_against_differences():
    """f32: the directional derivative of sum(o * go) along a random direction"""
    c = Case("f32", [(30, 45)], heads=(2, 1), hd=16, causal=True, softcap=5.0, rel_table=table(8, 2), rel_map=sequence.rel_bucket_map(8, 20), qk=1.0)
    got = c.run()
    g = torch.Generator().manual_seed(9)

    def value(q, k, v, tab):
        kw = dict(c.kw, rel_table=tab)
        o = O.attention(q, k, v, c.q_off, c.k_off, **kw)["o"]
        return float((o[:30] * c.go[:30].double()).sum())

    base = [x.double() for x in (c.q, c.k, c.v, c.kw["rel_table"])]
    for i, name in enumerate(("dq", "dk", "dv", "d_rel_table")):
        step = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = ([x + (h * step if j == i else 0) for j, x in enumerate(base)] for h in (h, -h))
        slope = (value(*up) - value(*down)) / (2 * h)
        mine = float((got[name].double().cpu() * step).sum())
        # the quotient's own error is of the order h^2; the gradients are f32 sums
        assert abs(slope - mine) < 1e-4 * float((got[name].double().cpu().abs() * step.abs()).sum()), name
