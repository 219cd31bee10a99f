"""The sequence operators without a GPU: the ends of what their C entry points and tensor functions take."""
import ctypes

import pytest
import torch

from bigc_hip import sequence
from test_sequence import FAKE, attn, lib, norm  # noqa: F401


@pytest.mark.parametrize("softcap", [1e-45, 1e-39])
def test_a_cap_whose_reciprocal_is_no_number_is_refused(lib, softcap):
    a = attn(softcap=softcap)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 1 << 40) == -1


def test_many_streams_over_long_caches_are_taken(lib):
    """what counts is the launch's blocks, not sequences x longest cache x heads: one token for each of 256 streams, the longest cache of 131072 rows, 64 heads"""
    a = attn(n_seq=256, n_head=64, n_kv_head=1, max_q=1, max_k=131072, n_q=256, n_k=1 << 20, ldq=4096, ldo=4096)
    need = lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0)
    assert need > 0
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, need - 1) == -4


def test_more_blocks_than_a_launch_holds_are_refused(lib):
    for kw in (dict(n_seq=1 << 22, n_head=4, n_kv_head=4), dict(n_seq=1 << 14, max_q=1 << 17, n_q=1 << 20), dict(n_seq=1 << 23, n_head=2, n_kv_head=2)):
        a = attn(**kw)
        assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 60) == -1, kw
        assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 1 << 60) == -1, kw
        assert lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0) == lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 1) == 0, kw


def test_the_stride_of_a_single_row_is_not_read(lib):
    a = attn(n_q=1, n_k=1, max_q=1, max_k=1, **{n: -4 for n in ("ldq", "ldk", "ldv", "ldo")})
    a.ldq = 1 << 40
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 0) == -4
    n = norm(n_rows=1, ldq=-4, lddqo=-8)
    assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(n), FAKE, 0) == -4


@pytest.mark.parametrize("kw", [dict(max_k=2 ** 31 - 10), dict(max_q=2 ** 31 - 10, max_k=1), dict(max_q=2 ** 30, max_k=2 ** 30)], ids=str)
def test_places_that_int32_cannot_count_are_refused(lib, kw):
    a = attn(n_head=1, n_kv_head=1, **kw)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(a), FAKE, 1 << 60) == -1
    assert lib.bigc_seq_attn_bwd(None, ctypes.byref(a), FAKE, 1 << 60) == -1
    assert lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0) == 0


def test_a_cache_of_almost_all_places_is_split(lib):
    n = 2 ** 31 - 2 ** 20 - 8
    a = attn(n_head=2, n_kv_head=2, max_q=1, n_q=1, max_k=n, n_k=n)
    one = 2 * (64 + 2) * 4                                                 # a chunk's sums and statistics, two heads
    assert lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0) > 100 * one


STRIDES = [(0, 64), (8, 64), (256, 0), (256, 32), (64, 64), (128, 64), (64, 128), (192, 128), (320, 192), (256, 64), (64, 512), (72, 1024), (512, 64), (384, 64), (520, 136)]


@pytest.mark.parametrize("strides", STRIDES, ids=str)
def test_outputs_that_overlap_themselves_are_refused(lib, strides):
    """rows or heads that share a place would be written by two blocks at once; any other layout is taken (such a call ends at its workspace of no bytes)"""
    ld, hs = strides

    def due(heads):                                                        # 8 rows of 64 columns
        return -1 if any(abs(r * ld - h * hs) < 64 for h in range(heads) for r in range(-7, 8) if (r, h) != (0, 0)) else -4

    split = dict(n_q=8, max_q=1, n_seq=1, n_k=1 << 20, max_k=1 << 20)      # (a forward that needs a workspace)
    assert lib.bigc_seq_attn_fwd(None, ctypes.byref(attn(ldo=ld, hso=hs, **split)), FAKE, 0) == due(4)
    for n, heads in (("q", 4), ("k", 2), ("v", 2)):
        assert lib.bigc_seq_attn_bwd(None, ctypes.byref(attn(**{"ldd" + n: ld, "hsd" + n: hs})), FAKE, 0) == due(heads), n
    for n, heads in (("q", 4), ("k", 2)):
        a = norm(**{"d" + n: FAKE << 1, "ldd" + n: ld, "hsd" + n: hs})
        assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(a), FAKE, 0) == due(heads), n
        if due(heads) == -1:
            a = norm(**{n + "_out": FAKE << 1, "ld" + n + "o": ld, "hs" + n + "o": hs})
            assert lib.bigc_head_norm_rope_fwd(None, ctypes.byref(a)) == -1


def test_in_place_with_other_strides_is_refused(lib):
    assert lib.bigc_head_norm_rope_fwd(None, ctypes.byref(norm(ldqo=320))) == -1
    assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(norm(lddk=512)), FAKE, 0) == -1


def test_tensor_functions_refuse_what_the_structure_cannot_hold():
    """(the message names the argument: on a machine without a GPU every call ends in an AssertionError, for its device)"""
    off = torch.tensor([0, 4], dtype=torch.int32)
    q = torch.zeros(4, 2, 64)
    base = dict(q=q, k=q, v=q, q_off=off, k_off=off, max_q=4, max_k=4)
    for name, kw in (("max_q", dict(max_q=(1 << 32) + 4)), ("max_k", dict(max_k=1 << 31)), ("max_k", dict(max_k=4.0)), ("max_q", dict(max_q=None)), ("window", dict(window=((1 << 32) - 1, -1))),
                     ("window", dict(window=(2, 1 << 33))), ("window", dict(window=3)), ("window", dict(window=(1, 2, 3))), ("q_off", dict(q_off=None)), ("k_off", dict(k_off=[0, 4])),
                     ("q_off", dict(q_off=torch.tensor(4, dtype=torch.int32))), ("q_off", dict(q_off=off[:0])), ("softcap", dict(softcap="no")), ("scale", dict(scale=[1.0, 2.0])),
                     ("rel_table", dict(rel_table=[[0.0]], rel_map=off)), ("rel_map", dict(rel_table=torch.zeros(3, 2), rel_map=off[0])), ("a GPU", {})):
        with pytest.raises(AssertionError, match=name):
            sequence.attend(**dict(base, **kw))
    w, pos, inv = torch.ones(64), torch.zeros(4, dtype=torch.int32), torch.ones(32, dtype=torch.float64)
    for name, kw in (("inv_freq", dict(inv_freq=inv[0])), ("inv_freq", dict(inv_freq=[1.0])), ("eps", dict(eps=None)), ("out", dict(out=q)), ("out", dict(out=(q,))), ("a GPU", {})):
        with pytest.raises(AssertionError, match=name):
            sequence.head_norm_rope(**dict(dict(q=q, k=q, wq=w, wk=w, pos=pos, inv_freq=inv), **kw))


def test_head_norm_goes_by_what_a_launch_holds(lib):
    a = norm(n_rows=1 << 28, n_q_head=4, n_k_head=4, head_dim=8, n_freq=4, ldq=32)
    assert lib.bigc_head_norm_rope_bwd(None, ctypes.byref(a), FAKE, 0) == -4       # (its blocks take rows in turn)
    a = norm(n_rows=(1 << 31) - 1, n_q_head=1, n_k_head=0, head_dim=8, n_freq=4)
    assert lib.bigc_head_norm_rope_fwd(None, ctypes.byref(a)) == -1
    assert b"launch" in lib.bigc_last_error()
