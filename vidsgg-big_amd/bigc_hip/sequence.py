"""Sequence operators on torch tensors: attention over ordered ragged rows (capped scores, distance biases, a learned bias by buckets, causal /
window / prefix / document masks, shared key heads) with its backward, and the norm of every query and key head with its position rotation.

Thin checks and allocations around ``bigc_seq_attn_*`` and ``bigc_head_norm_rope_*`` of ``include/bigc_hip.h``, which holds the formulas.  A
call works on its tensors' device, on that device's current stream; nothing is kept between calls, nothing waits for the GPU, and every call
may be captured into a graph (outputs and workspaces are torch allocations of the call).  Wrong shapes, types, devices or alignments raise
``AssertionError`` before anything runs.  The gradients are calls of their own (no autograd node): a ``torch.autograd.Function`` of a model
calls them from its ``backward``, as the training steps of this package do with theirs.
"""
import ctypes

import torch

from . import _lib
from ._lib import bigc_head_norm, bigc_seq_attn

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def rel_bucket_map(n_bucket, max_distance, two_sided=True, radius=None):
    """int32 (2 * radius + 1): the bucket of every distance key - query in [-radius, radius] (radius: max_distance unless given).  Each side has
    n_bucket / 2 buckets (two_sided; else all n_bucket lie behind the query and keys ahead share bucket 0); half of a side's buckets hold one
    distance each, the others grow with the logarithm up to max_distance, from where on the last one holds everything.  The borders are decided
    in whole numbers: log(n / e) / log(m / e) * c >= t exactly when n^c >= m^t e^(c - t)."""
    side = n_bucket // 2 if two_sided else n_bucket
    e = side // 2
    c = side - e
    assert side >= 2 and (not two_sided or n_bucket % 2 == 0), "rel_bucket_map: %d buckets" % n_bucket
    assert max_distance > e, "rel_bucket_map: max_distance %d has to be beyond the %d distances with a bucket of their own" % (max_distance, e)
    radius = max_distance if radius is None else radius
    assert radius >= 0, "rel_bucket_map: radius %d" % radius
    first = [next(n for n in range(e, max_distance + 1) if n ** c >= max_distance ** t * e ** (c - t)) for t in range(c)]
    out = []
    for d in range(-radius, radius + 1):
        n = abs(d) if two_sided else max(-d, 0)
        b = n if n < e else e - 1 + sum(n >= f for f in first)
        out.append(b + (side if two_sided and d > 0 else 0))
    return torch.tensor(out, dtype=torch.int32)


def _rows(name, t, like, shape):
    """(address, row stride, head stride) of a (rows, heads, columns) tensor whose columns lie side by side"""
    assert isinstance(t, torch.Tensor) and t.dim() == 3, "%s: a (rows, heads, columns) tensor" % name
    assert t.dtype == like.dtype and t.device == like.device, "%s: %s on %s next to %s on %s" % (name, t.dtype, t.device, like.dtype, like.device)
    assert tuple(t.shape) == tuple(shape), "%s: shape %s, not %s" % (name, tuple(t.shape), tuple(shape))
    s = t.stride()
    assert s[2] == 1 or t.shape[2] == 1, "%s: the columns of a head have to lie side by side (strides %s)" % (name, s)
    return t.data_ptr(), s[0], s[1]


def _vector(name, t, dtype, shape, device):
    if t is None:
        return None
    assert isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == device, "%s: a %s tensor on %s" % (name, dtype, device)
    assert tuple(t.shape) == tuple(shape) and t.is_contiguous(), "%s: contiguous, of shape %s (not %s)" % (name, tuple(shape), tuple(t.shape))
    return t.data_ptr()


class _On(object):
    """the device's current stream; the device is current inside (a launch goes to the current device)"""

    def __init__(self, device):
        assert device.type == "cuda", "the operators run on a GPU (tensors are on %s)" % device
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None
        self.device = device

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _workspace(lib, nbytes, device):
    return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None


class SavedAttention(object):
    """What ``attend(..., save=True)`` keeps for ``attend_bwd``: the arguments, the output (before its rounding too, for f16 / bf16) and the
    rows' log-sum-exp.  The tensors must not change in between."""

    def __init__(self, args, tensors, o, lse, o32):
        self.args, self.tensors, self.o, self.lse, self.o32 = args, tensors, o, lse, o32


def attend(q, k, v, q_off, k_off, max_q, max_k, scale=None, softcap=0.0, slopes=None, rel_table=None, rel_map=None, causal=False, window=(-1, -1),
           prefix_len=None, q_doc=None, k_doc=None, out=None, save=False):
    """Attention of the rows of ``q`` (n_q, n_head, head_dim) over those of ``k``, ``v`` (n_k, n_kv_head, head_dim), f32, f16 or bf16, any row and
    head strides of whole 16 bytes.  Sequence s owns rows q_off[s]:q_off[s + 1] and k_off[s]:k_off[s + 1] (int32, on the device) of at most
    max_q and max_k rows; its queries are its last rows (one query per sequence: a decoding step).  scale: 1 / sqrt(head_dim) unless given;
    softcap: scores become softcap * tanh(score / softcap); slopes (n_head) f32: minus slope times distance; rel_table (n_bucket, n_head) f32 and
    rel_map (2 R + 1) int32: the bias of a distance clipped to [-R, R] (``rel_bucket_map``); causal; window (left, right): keys at most so far
    behind / ahead, -1 for no limit; prefix_len (n_seq) int32: the first keys of a sequence are seen by all its rows; q_doc, k_doc (n_q), (n_k)
    int32: rows see keys of their own document, a negative number is padding.  A row that sees nothing gives 0.
    -> o (n_q, n_head, head_dim), or (o, SavedAttention) with ``save``; rows outside every sequence are not written (0 unless ``out`` is given)."""
    lib = _lib.load()
    assert isinstance(q, torch.Tensor) and q.dim() == 3 and q.dtype in _DTYPES, "q: a (rows, heads, columns) tensor of f32, f16 or bf16"
    n_q, n_head, hd = q.shape
    assert isinstance(k, torch.Tensor) and k.dim() == 3, "k: a (rows, heads, columns) tensor"
    n_k, n_kv = k.shape[0], k.shape[1]
    dev, n_seq = q.device, q_off.shape[0] - 1
    a = bigc_seq_attn()
    a.dtype, a.n_seq, a.n_head, a.n_kv_head, a.head_dim, a.max_q, a.max_k = _DTYPES[q.dtype], n_seq, n_head, n_kv, hd, max_q, max_k
    a.causal, (a.window_left, a.window_right) = bool(causal), window
    a.scale, a.softcap = hd ** -0.5 if scale is None else scale, softcap
    a.n_q, a.n_k = n_q, n_k
    a.q, a.ldq, a.hsq = _rows("q", q, q, (n_q, n_head, hd))
    a.k, a.ldk, a.hsk = _rows("k", k, q, (n_k, n_kv, hd))
    a.v, a.ldv, a.hsv = _rows("v", v, q, (n_k, n_kv, hd))
    a.q_off = _vector("q_off", q_off, torch.int32, (n_seq + 1,), dev)
    a.k_off = _vector("k_off", k_off, torch.int32, (n_seq + 1,), dev)
    a.slopes = _vector("slopes", slopes, torch.float32, (n_head,), dev)
    if rel_table is not None or rel_map is not None:
        assert rel_table is not None and rel_map is not None, "rel_table and rel_map come together"
        assert rel_table.dim() == 2 and rel_map.dim() == 1 and rel_map.shape[0] % 2 == 1, "rel_table (n_bucket, n_head), rel_map (2 R + 1)"
        a.bias_radius, a.n_bucket = rel_map.shape[0] // 2, rel_table.shape[0]
        a.rel_table = _vector("rel_table", rel_table, torch.float32, (a.n_bucket, n_head), dev)
        a.rel_map = _vector("rel_map", rel_map, torch.int32, (rel_map.shape[0],), dev)
    a.prefix_len = _vector("prefix_len", prefix_len, torch.int32, (n_seq,), dev)
    a.q_doc = _vector("q_doc", q_doc, torch.int32, (n_q,), dev)
    a.k_doc = _vector("k_doc", k_doc, torch.int32, (n_k,), dev)
    assert (q_doc is None) == (k_doc is None), "q_doc and k_doc come together"
    with _On(dev) as stream:
        need = lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0)
        o = torch.zeros((n_q, n_head, hd), dtype=q.dtype, device=dev) if out is None else out
        a.o, a.ldo, a.hso = _rows("out", o, q, (n_q, n_head, hd))
        lse = o32 = None
        if save:
            lse = torch.empty((n_q, n_head), dtype=torch.float32, device=dev)
            a.lse = lse.data_ptr()
            if q.dtype != torch.float32:
                o32 = torch.empty((n_q, n_head, hd), dtype=torch.float32, device=dev)
                a.o32 = o32.data_ptr()
        ws = _workspace(lib, need, dev)
        _lib.check(lib.bigc_seq_attn_fwd(stream, ctypes.byref(a), _lib.ptr(ws), need))
    if not save:
        return o
    return o, SavedAttention(a, (q, k, v, q_off, k_off, slopes, rel_table, rel_map, prefix_len, q_doc, k_doc), o, lse, o32)


def attend_bwd(saved, d_o):
    """Gradients of ``attend`` for the output's gradient ``d_o`` -> (dq, dk, dv, d_rel_table or None); dk, dv summed over the query heads of a key
    head.  Rows outside every sequence get 0.  Repeats bit for bit."""
    lib = _lib.load()
    q, k, v = saved.tensors[:3]
    rel_table = saved.tensors[6]
    a = bigc_seq_attn()
    ctypes.memmove(ctypes.byref(a), ctypes.byref(saved.args), ctypes.sizeof(a))
    a.d_o, a.lddo, a.hsdo = _rows("d_o", d_o, q, q.shape)
    with _On(q.device) as stream:
        dq, dk, dv = (torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        for name, t in (("q", dq), ("k", dk), ("v", dv)):
            setattr(a, "d" + name, t.data_ptr())
            setattr(a, "ldd" + name, t.stride(0))
            setattr(a, "hsd" + name, t.stride(1))
        dt = None
        if rel_table is not None:
            dt = torch.empty_like(rel_table)
            a.d_rel_table = dt.data_ptr()
        need = lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 1)
        ws = _workspace(lib, need, q.device)
        _lib.check(lib.bigc_seq_attn_bwd(stream, ctypes.byref(a), _lib.ptr(ws), need))
    return dq, dk, dv, dt


def _norm_args(q, k, wq, wk, pos, inv_freq, eps, interleaved):
    assert isinstance(q, torch.Tensor) and q.dim() == 3 and q.dtype in _DTYPES, "q: a (rows, heads, columns) tensor of f32, f16 or bf16"
    n, h, hd = q.shape
    assert isinstance(k, torch.Tensor) and k.dim() == 3, "k: a (rows, heads, columns) tensor"
    a, dev = bigc_head_norm(), q.device
    a.dtype, a.n_q_head, a.n_k_head, a.head_dim, a.n_rows = _DTYPES[q.dtype], h, k.shape[1], hd, n
    a.interleaved, a.eps = bool(interleaved), eps
    a.q, a.ldq, a.hsq = _rows("q", q, q, (n, h, hd))
    a.k, a.ldk, a.hsk = _rows("k", k, q, (n, k.shape[1], hd))
    a.wq = _vector("wq", wq, torch.float32, (hd,), dev)
    a.wk = _vector("wk", wk, torch.float32, (hd,), dev)
    if inv_freq is not None:
        a.n_freq = inv_freq.shape[0]
        a.inv_freq = _vector("inv_freq", inv_freq, torch.float64, (inv_freq.shape[0],), dev)
        a.pos = _vector("pos", pos, torch.int32, (n,), dev)
    return a


def head_norm_rope(q, k, wq, wk, pos, inv_freq, eps=1e-6, interleaved=False, out=None):
    """RMS norm of every head of ``q`` (rows, n_head, head_dim) and ``k`` (rows, n_kv_head, head_dim) times ``wq`` / ``wk`` (head_dim) f32 (None:
    1), then the rotation of the first 2 * len(inv_freq) columns by pos[row] * inv_freq (int32 (rows), f64; inv_freq None: no rotation).  q and k may be
    slices of one projection's output (16-byte strides); ``out``: a pair of tensors, which may be (q, k) themselves.  -> (q', k')"""
    lib = _lib.load()
    a = _norm_args(q, k, wq, wk, pos, inv_freq, eps, interleaved)
    with _On(q.device) as stream:
        qo, ko = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)) if out is None else out
        a.q_out, a.ldqo, a.hsqo = _rows("out[0]", qo, q, q.shape)
        a.k_out, a.ldko, a.hsko = _rows("out[1]", ko, q, k.shape)
        _lib.check(lib.bigc_head_norm_rope_fwd(stream, ctypes.byref(a)))
    return qo, ko


def head_norm_rope_bwd(d_q, d_k, q, k, wq, wk, pos, inv_freq, eps=1e-6, interleaved=False):
    """Gradients of ``head_norm_rope`` for those of its outputs, from its inputs as they were -> (dq, dk, dwq, dwk); a weight that is None gets None."""
    lib = _lib.load()
    a = _norm_args(q, k, wq, wk, pos, inv_freq, eps, interleaved)
    a.dq_out, a.lddqo, a.hsdqo = _rows("d_q", d_q, q, q.shape)
    a.dk_out, a.lddko, a.hsdko = _rows("d_k", d_k, q, k.shape)
    with _On(q.device) as stream:
        dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        a.dq, a.lddq, a.hsdq = dq.data_ptr(), dq.stride(0), dq.stride(1)
        a.dk, a.lddk, a.hsdk = dk.data_ptr(), dk.stride(0), dk.stride(1)
        dwq, dwk = (None if w is None else torch.empty_like(w) for w in (wq, wk))
        a.dwq, a.dwk = _lib.ptr(dwq), _lib.ptr(dwk)
        need = lib.bigc_head_norm_rope_workspace_bytes(ctypes.byref(a))
        ws = _workspace(lib, need, q.device)
        _lib.check(lib.bigc_head_norm_rope_bwd(stream, ctypes.byref(a), _lib.ptr(ws), need))
    return dq, dk, dwq, dwk
