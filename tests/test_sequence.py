"""The sequence operators without a GPU: refusals of the C entry points and of the tensor functions, and the bucket map."""
import ctypes
import math

import pytest
import torch

from bigc_hip import _lib, sequence
from bigc_hip._lib import bigc_head_norm, bigc_seq_attn


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


FAKE = 1 << 20        # an address of whole 16 bytes that nothing reads: every call below is refused, or has nothing to do


def attn(**kw):
    a = bigc_seq_attn()
    a.dtype, a.n_seq, a.n_head, a.n_kv_head, a.head_dim, a.max_q, a.max_k = 2, 1, 4, 2, 64, 8, 8
    a.window_left = a.window_right = -1
    a.scale, a.n_q, a.n_k = 0.125, 8, 8
    a.q_off = a.k_off = FAKE
    for n in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        setattr(a, n, FAKE)
        setattr(a, {"d_o": "lddo"}.get(n, "ld" + n), 256)
        setattr(a, {"d_o": "hsdo"}.get(n, "hs" + n), 64)
    a.stats = FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD = [dict(dtype=3), dict(dtype=-1), dict(n_seq=-1), dict(n_head=0), dict(n_head=5), dict(n_kv_head=0), dict(head_dim=0), dict(head_dim=12), dict(head_dim=136),
       dict(n_q=-1), dict(n_k=1 << 31), dict(max_q=-1), dict(max_k=-3), dict(q_off=None), dict(k_off=None), dict(window_left=-2), dict(window_right=-5),
       dict(scale=math.inf), dict(scale=math.nan), dict(softcap=-1.0), dict(softcap=math.nan), dict(q_doc=FAKE), dict(k_doc=FAKE), dict(rel_table=FAKE),
       dict(rel_map=FAKE), dict(rel_table=FAKE, rel_map=FAKE, n_bucket=0, bias_radius=3), dict(rel_table=FAKE, rel_map=FAKE, n_bucket=4, bias_radius=2048),
       dict(rel_table=FAKE, rel_map=FAKE, n_bucket=4, bias_radius=-1), dict(n_seq=1 << 20, max_q=1 << 12), dict(n_seq=1 << 20, max_k=1 << 12)]
BAD_ROWS = [dict(q=None), dict(k=None), dict(v=FAKE + 8), dict(o=FAKE + 2), dict(ldq=260), dict(hsq=4), dict(ldk=-256), dict(hsv=-64)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_attention_refuses(lib, kw):
    a = attn(**kw)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1 and lib.bigc_last_error()
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1
    assert lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0) == 0
    with pytest.raises(AssertionError):
        _lib.check(lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 40))


@pytest.mark.parametrize("kw", BAD_ROWS, ids=str)
def test_attention_refuses_rows(lib, kw):
    a = attn(**kw)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1


@pytest.mark.parametrize("kw", [dict(d_o=None), dict(dq=FAKE + 4), dict(lddk=3), dict(hsdv=1), dict(stats=None), dict(stats=FAKE + 4), dict(d_rel_table=FAKE)], ids=str)
def test_attention_backward_refuses(lib, kw):
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(attn(**kw)), FAKE, 1 << 40) == -1


def test_attention_refuses_a_small_workspace(lib):
    a = attn()
    need = lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 1)
    assert need > 0
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, need - 1) == -4
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), None, need) == -4
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE + 4, need) == -4
    assert lib.bigc_seq_attn_fwd(None, None, None, 0) == -1
    assert lib.bigc_seq_attn_bwd(None, None, None, 0) == -1


def test_attention_of_nothing_is_done(lib):
    a = attn(n_seq=0, n_q=0, n_k=0, max_q=0, max_k=0, q=None, k=None, v=None, o=None, q_off=None, k_off=None)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), None, 0) == 0


def norm(**kw):
    a = bigc_head_norm()
    a.dtype, a.n_q_head, a.n_k_head, a.head_dim, a.n_freq, a.eps, a.n_rows = 1, 4, 2, 64, 32, 1e-6, 8
    a.pos = a.inv_freq = FAKE
    for n, ld, hs in (("q", "ldq", "hsq"), ("k", "ldk", "hsk"), ("q_out", "ldqo", "hsqo"), ("k_out", "ldko", "hsko"), ("dq_out", "lddqo", "hsdqo"),
                      ("dk_out", "lddko", "hsdko"), ("dq", "lddq", "hsdq"), ("dk", "lddk", "hsdk")):
        setattr(a, n, FAKE)
        setattr(a, ld, 256)
        setattr(a, hs, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(dtype=7), dict(n_q_head=-1), dict(n_q_head=0, n_k_head=0), dict(head_dim=20), dict(head_dim=264), dict(n_rows=-1), dict(n_rows=1 << 31),
                                dict(n_freq=33), dict(n_freq=-1), dict(pos=None), dict(inv_freq=None), dict(eps=-1.0), dict(eps=math.nan), dict(q=None), dict(k=FAKE + 1),
                                dict(ldq=12), dict(hsk=2), dict(ldk=-8)], ids=str)
def test_head_norm_refuses(lib, kw):
    assert lib.bigc_head_norm_rope_fwd(None, ctypes.byref(norm(**kw))) == -1 and lib.bigc_last_error()
    assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(norm(**kw)), FAKE, 1 << 40) == -1


def test_head_norm_refuses_outputs_and_workspace(lib):
    assert lib.bigc_head_norm_rope_fwd(None, ctypes.byref(norm(q_out=FAKE + 4))) == -1
    assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(norm(dq=None)), FAKE, 1 << 40) == -1
    need = lib.bigc_head_norm_rope_workspace_bytes(ctypes.byref(norm()))
    assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(norm()), FAKE, need - 1) == -4
    assert lib.bigc_head_norm_rope_fwd(None, None) == -1
    assert lib.bigc_head_norm_rope_fwd(None, ctypes.byref(norm(n_rows=0, q=None, k=None, pos=None))) == 0


def test_tensor_functions_refuse():
    off = torch.tensor([0, 4], dtype=torch.int32)
    q = torch.zeros(4, 2, 64)
    refused = [
        dict(q=q.double()), dict(q=q[0]), dict(k=torch.zeros(4, 2, 32)), dict(v=torch.zeros(4, 1, 64)), dict(k=q.half()), dict(q_off=off.long()),
        dict(q=torch.zeros(4, 2, 128)[..., ::2]), dict(slopes=torch.zeros(3)), dict(rel_table=torch.zeros(4, 2)), dict(rel_map=torch.zeros(3, dtype=torch.int32)),
        dict(rel_table=torch.zeros(4, 2), rel_map=torch.zeros(4, dtype=torch.int32)), dict(prefix_len=torch.zeros(2, dtype=torch.int32)), dict(q_doc=off),
        dict(rel_table=torch.zeros(4, 3), rel_map=torch.zeros(3, dtype=torch.int32)), {}]
    for kw in refused:
        a = dict(dict(q=q, k=q, v=q, q_off=off, k_off=off, max_q=4, max_k=4), **kw)
        with pytest.raises(AssertionError):
            sequence.attend(**a)
    w, pos, inv = torch.ones(64), torch.zeros(4, dtype=torch.int32), torch.ones(32, dtype=torch.float64)
    for kw in (dict(wq=torch.ones(32)), dict(pos=pos.long()), dict(inv_freq=inv.float()), dict(k=q.half()), dict(pos=None), {}):
        a = dict(dict(q=q, k=q, wq=w, wk=w, pos=pos, inv_freq=inv), **kw)
        with pytest.raises(AssertionError):
            sequence.head_norm_rope(**a)


@pytest.mark.parametrize("n,m,two", [(32, 128, True), (16, 64, True), (8, 20, True), (9, 64, False), (64, 300, False), (4, 2, True), (32, 129, False)])
def test_bucket_map(n, m, two):
    got = sequence.rel_bucket_map(n, m, two, radius=m + 5).tolist()
    side = n // 2 if two else n
    e = side // 2
    for i, d in enumerate(range(-m - 5, m + 6)):
        k = abs(d) if two else max(-d, 0)
        if k < e:
            b = k
        else:                                    # a border hit exactly is moved by rounding: 1e-9 is far below the next whole number's distance
            b = min(side - 1, e + int(math.floor(math.log(k / e) / math.log(m / e) * (side - e) + 1e-9)))
        assert got[i] == b + (side if two and d > 0 else 0), d
    assert max(got) < n and sequence.rel_bucket_map(n, m, two).shape[0] == 2 * m + 1


def test_bucket_map_refuses():
    for a in ((2, 20, True), (9, 20, True), (32, 8, True), (8, 20, True, -1)):
        with pytest.raises(AssertionError):
            sequence.rel_bucket_map(*a)
