"""Sequence operators on torch tensors: attention over ordered ragged rows (capped scores, distance biases, a learned bias by buckets, causal /
window / prefix / document masks, shared key heads) with its backward, and the norm of every query and key head with its position rotation.

Thin checks and allocations around ``bigc_seq_attn_*`` and ``bigc_head_norm_rope_*`` of ``include/bigc_hip.h``, which holds the formulas.  A
call works on its tensors' device, on that device's current stream; nothing is kept between calls, nothing waits for the GPU, and every call
may be captured into a graph (outputs and workspaces are torch allocations of the call).  Wrong shapes, types, devices or alignments raise
``AssertionError`` before anything runs.  The gradients are calls of their own (no autograd node): a ``torch.autograd.Function`` of a model
calls them from its ``backward``, as the training steps of this package do with theirs.
"""
import ctypes
import math
import operator

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


def _rows(name, t, dtype, device, shape):
    """(address, row stride, head stride) of a (rows, heads, columns) tensor whose columns lie side by side"""
    assert isinstance(t, torch.Tensor), "%s: a tensor" % name
    assert t.dtype is dtype and t.device == device, "%s: %s on %s next to %s on %s" % (name, t.dtype, t.device, dtype, device)
    assert t.shape == shape, "%s: shape %s, not %s" % (name, tuple(t.shape), tuple(shape))
    s = t.stride()
    assert s[2] == 1 or shape[2] == 1, "%s: the columns of a head have to lie side by side (strides %s)" % (name, s)
    return t.data_ptr(), s[0], s[1]


def _vector(name, t, dtype, shape, device):
    if t is None:
        return None
    assert isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device, "%s: a %s tensor on %s" % (name, dtype, device)
    assert t.shape == shape and t.is_contiguous(), "%s: contiguous, of shape %s (not %s)" % (name, tuple(shape), tuple(t.shape))
    return t.data_ptr()


def _heads(name, t):
    assert isinstance(t, torch.Tensor) and t.dim() == 3 and t.dtype in _DTYPES, "%s: a (rows, heads, columns) tensor of f32, f16 or bf16" % name
    return t.shape


def _whole(name, x):
    """x as an int32 of the C structure (ctypes would take any whole number modulo 2^32)"""
    try:
        n = operator.index(x)
    except TypeError:
        n = None
    assert n is not None and -1 << 31 <= n < 1 << 31, "%s: %r is no int32" % (name, x)
    return n


def _number(name, x):
    """x as a float of the C structure"""
    try:
        return float(x)
    except (TypeError, ValueError):
        raise AssertionError("%s: %r is no number" % (name, x))


def _on(device):
    """A guard that makes the tensors' device the current one (a launch goes to the current device), or None where it is"""
    assert device.type == "cuda", "the operators run on a GPU (tensors are on %s)" % device
    return None if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)            # torch.cuda.current_stream(device).cuda_stream, without the objects


class SavedAttention(object):
    """What ``attend(..., save=True)`` keeps for ``attend_bwd``: the arguments, the output (with more bits too, for f16 / bf16)
    and the rows' softmax statistics.  The tensors must not change in between."""

    def __init__(self, args, tensors, o, stats, o32):
        self.args, self.tensors, self.o, self.stats, self.o32 = args, tensors, o, stats, o32

    @property
    def lse(self):
        """(n_q, n_head) f32: log of the sum of exp of a row's scores, -inf where it sees nothing (rows outside every sequence: undefined)"""
        m, l = self.stats.unbind(-1)
        lowest = torch.finfo(torch.float32).min                          # stands for every score from there up to times ln 2
        return torch.where(l == 0, torch.full_like(m, float("-inf")), torch.where(m == lowest, m, m * math.log(2.0) + torch.log(l)))


def attend(q, k, v, q_off, k_off, max_q, max_k, scale=None, softcap=0.0, slopes=None, rel_table=None, rel_map=None, causal=False, window=(-1, -1),
           prefix_len=None, q_doc=None, k_doc=None, out=None, save=False):
    """Attention of the rows of ``q`` (n_q, n_head, head_dim) over those of ``k``, ``v`` (n_k, n_kv_head, head_dim), f32, f16 or bf16, any row and
    head strides of whole 16 bytes.  Sequence s owns rows q_off[s]:q_off[s + 1] and k_off[s]:k_off[s + 1] (int32, on the device) of at most
    max_q and max_k rows (a longer one is cut to its first); its queries are its last rows (one query per sequence: a decoding step).  scale: 1 / sqrt(head_dim) unless given;
    softcap: scores become softcap * tanh(score / softcap); slopes (n_head) f32: minus slope times distance; rel_table (n_bucket, n_head) f32 and
    rel_map (2 R + 1) int32: the bias of a distance clipped to [-R, R] (``rel_bucket_map``; R at most 2047, 1023 for the gradient of f32 heads over 64 columns); causal; window (left, right): keys at most so far
    behind / ahead, -1 for no limit; prefix_len (n_seq) int32: the first keys of a sequence are seen by all its rows; q_doc, k_doc (n_q), (n_k)
    int32: rows see keys of their own document, a negative number is padding.  A row that sees nothing gives 0.
    -> o (n_q, n_head, head_dim), or (o, SavedAttention) with ``save``; rows outside every sequence are not written (0 unless ``out`` is given)."""
    shape = _heads("q", q)
    dtype, dev, hd = q.dtype, q.device, shape[2]
    max_q, max_k, scale, softcap = _whole("max_q", max_q), _whole("max_k", max_k), _number("scale", max(1, hd) ** -0.5 if scale is None else scale), _number("softcap", softcap)
    assert isinstance(window, (tuple, list)) and len(window) == 2, "window: (left, right)"
    left, right = _whole("window", window[0]), _whole("window", window[1])
    assert isinstance(q_off, torch.Tensor) and isinstance(k_off, torch.Tensor) and q_off.dim() == 1 and q_off.shape[0] > 0, "q_off, k_off: int32 tensors (n_seq + 1)"
    for name, t, dim in (("rel_table", rel_table, 2), ("rel_map", rel_map, 1)):
        assert t is None or (isinstance(t, torch.Tensor) and t.dim() == dim), "%s: a tensor of %d dimensions" % (name, dim)
    guard = _on(dev)
    if guard is not None:
        with guard:
            return attend(q, k, v, q_off, k_off, max_q, max_k, scale, softcap, slopes, rel_table, rel_map, causal, window, prefix_len, q_doc, k_doc, out, save)
    lib = _lib.load()
    kshape = (_heads("k", k)[0], k.shape[1], hd)
    n_q, n_head, n_seq = shape[0], shape[1], q_off.shape[0] - 1
    assert (q_doc is None) == (k_doc is None), "q_doc and k_doc come together"
    n_bucket = radius = 0
    if rel_table is not None or rel_map is not None:
        assert rel_table is not None and rel_map is not None, "rel_table and rel_map come together"
        assert rel_map.shape[0] % 2 == 1, "rel_table (n_bucket, n_head), rel_map (2 R + 1)"
        n_bucket, radius = rel_table.shape[0], rel_map.shape[0] // 2
    i32, f32 = torch.int32, torch.float32
    o = q.new_empty(shape) if out is None else out
    stats = o32 = None
    if save:
        stats = q.new_empty((n_q, n_head, 2), dtype=f32)
        if dtype is not f32:                                             # see o32 in bigc_hip.h
            o32 = q.new_empty(shape, dtype=f32)
    a = bigc_seq_attn(                                                   # the fields in the structure's order
        _DTYPES[dtype], n_seq, n_head, kshape[1], hd, max_q, max_k, 1 if causal else 0, left, right, 1 if out is None else 0, radius, n_bucket,
        scale, softcap, n_q, kshape[0],
        _vector("q_off", q_off, i32, (n_seq + 1,), dev), _vector("k_off", k_off, i32, (n_seq + 1,), dev), _vector("slopes", slopes, f32, (n_head,), dev),
        _vector("rel_table", rel_table, f32, (n_bucket, n_head), dev), _vector("rel_map", rel_map, i32, (2 * radius + 1,), dev),
        _vector("prefix_len", prefix_len, i32, (n_seq,), dev), _vector("q_doc", q_doc, i32, (n_q,), dev), _vector("k_doc", k_doc, i32, (kshape[0],), dev),
        *_rows("q", q, dtype, dev, shape), *_rows("k", k, dtype, dev, kshape), *_rows("v", v, dtype, dev, kshape), *_rows("out", o, dtype, dev, shape),
        _lib.ptr(stats), _lib.ptr(o32))
    need = lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 0)
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    _lib.check(lib.bigc_seq_attn_fwd(_stream(dev), ctypes.byref(a), _lib.ptr(ws), need))
    if not save:
        return o
    return o, SavedAttention(a, (q, k, v, q_off, k_off, slopes, rel_table, rel_map, prefix_len, q_doc, k_doc), o, stats, o32)


def attend_bwd(saved, d_o):
    """Gradients of ``attend`` for the output's gradient ``d_o`` -> (dq, dk, dv, d_rel_table or None); dk, dv summed over the query heads of a key
    head.  Rows outside every sequence get 0.  Repeats bit for bit."""
    q, k, v = saved.tensors[:3]
    guard = _on(q.device)
    if guard is not None:
        with guard:
            return attend_bwd(saved, d_o)
    lib = _lib.load()
    a = bigc_seq_attn()
    ctypes.memmove(ctypes.byref(a), ctypes.byref(saved.args), ctypes.sizeof(a))
    a.d_o, a.lddo, a.hsdo = _rows("d_o", d_o, q.dtype, q.device, q.shape)
    a.zero_rest = 1
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    a.dq, a.lddq, a.hsdq = _rows("dq", dq, q.dtype, q.device, q.shape)
    a.dk, a.lddk, a.hsdk = _rows("dk", dk, q.dtype, q.device, k.shape)
    a.dv, a.lddv, a.hsdv = _rows("dv", dv, q.dtype, q.device, v.shape)
    dt = None
    if saved.tensors[6] is not None:
        dt = torch.empty_like(saved.tensors[6])
        a.d_rel_table = dt.data_ptr()
    need = lib.bigc_seq_attn_workspace_bytes(ctypes.byref(a), 1)
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    _lib.check(lib.bigc_seq_attn_bwd(_stream(q.device), ctypes.byref(a), _lib.ptr(ws), need))
    return dq, dk, dv, dt


def _norm_args(q, k, wq, wk, pos, inv_freq, eps, interleaved):
    shape, kshape = _heads("q", q), _heads("k", k)
    dtype, dev, n, hd = q.dtype, q.device, shape[0], shape[2]
    assert inv_freq is None or (isinstance(inv_freq, torch.Tensor) and inv_freq.dim() == 1), "inv_freq: a float64 tensor (n_freq)"
    n_freq = 0 if inv_freq is None else inv_freq.shape[0]
    assert inv_freq is None or pos is not None, "inv_freq without pos"
    f32 = torch.float32
    return bigc_head_norm(                                               # the fields in the structure's order
        _DTYPES[dtype], shape[1], kshape[1], hd, n_freq, 1 if interleaved else 0, _number("eps", eps), n, _vector("pos", pos, torch.int32, (n,), dev),
        _vector("inv_freq", inv_freq, torch.float64, (n_freq,), dev), _vector("wq", wq, f32, (hd,), dev), _vector("wk", wk, f32, (hd,), dev),
        *_rows("q", q, dtype, dev, shape), *_rows("k", k, dtype, dev, (n, kshape[1], hd)))


def head_norm_rope(q, k, wq, wk, pos, inv_freq, eps=1e-6, interleaved=False, out=None):
    """RMS norm of every head of ``q`` (rows, n_head, head_dim) and ``k`` (rows, n_kv_head, head_dim) times ``wq`` / ``wk`` (head_dim) f32 (None:
    1), then the rotation of the first 2 * len(inv_freq) columns by pos[row] * inv_freq (int32 (rows), f64; inv_freq None: no rotation).  q and k may be
    slices of one projection's output (16-byte strides); ``out``: a pair of tensors, which may be (q, k) themselves.  -> (q', k')"""
    a = _norm_args(q, k, wq, wk, pos, inv_freq, eps, interleaved)
    dtype, dev = q.dtype, q.device
    assert out is None or (isinstance(out, (tuple, list)) and len(out) == 2), "out: a pair of tensors"
    guard = _on(dev)
    if guard is not None:
        with guard:
            return head_norm_rope(q, k, wq, wk, pos, inv_freq, eps, interleaved, out)
    qo, ko = (q.new_empty(q.shape), k.new_empty(k.shape)) if out is None else out
    a.q_out, a.ldqo, a.hsqo = _rows("out[0]", qo, dtype, dev, q.shape)
    a.k_out, a.ldko, a.hsko = _rows("out[1]", ko, dtype, dev, k.shape)
    _lib.check(_lib.load().bigc_head_norm_rope_fwd(_stream(dev), ctypes.byref(a)))
    return qo, ko


def head_norm_rope_bwd(d_q, d_k, q, k, wq, wk, pos, inv_freq, eps=1e-6, interleaved=False):
    """Gradients of ``head_norm_rope`` for those of its outputs, from its inputs as they were -> (dq, dk, dwq, dwk); a weight that is None gets None."""
    a = _norm_args(q, k, wq, wk, pos, inv_freq, eps, interleaved)
    dtype, dev = q.dtype, q.device
    guard = _on(dev)
    if guard is not None:
        with guard:
            return head_norm_rope_bwd(d_q, d_k, q, k, wq, wk, pos, inv_freq, eps, interleaved)
    lib = _lib.load()
    a.dq_out, a.lddqo, a.hsdqo = _rows("d_q", d_q, dtype, dev, q.shape)
    a.dk_out, a.lddko, a.hsdko = _rows("d_k", d_k, dtype, dev, k.shape)
    dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
    a.dq, a.lddq, a.hsdq = _rows("dq", dq, dtype, dev, q.shape)
    a.dk, a.lddk, a.hsdk = _rows("dk", dk, dtype, dev, k.shape)
    dwq, dwk = (None if w is None else torch.empty_like(w) for w in (wq, wk))
    a.dwq, a.dwk = _lib.ptr(dwq), _lib.ptr(dwk)
    need = lib.bigc_head_norm_rope_workspace_bytes(ctypes.byref(a))
    ws = q.new_empty((need,), dtype=torch.uint8)
    _lib.check(lib.bigc_head_norm_rope_bwd(_stream(dev), ctypes.byref(a), _lib.ptr(ws), need))
    return dq, dk, dwq, dwk
