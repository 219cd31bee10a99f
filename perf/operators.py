"""Work cases of the sequence operators (``vidsgg-big_amd/bigc_hip/sequence.py``): ragged attention with capped scores, distance biases and
masks, the same with a learned position bias by buckets, and the norm of every query and key head with its position rotation.

``run`` computes a case either by elementary torch operations (``own`` false) or by the library's operators (``own`` true); ``exact``
evaluates the operators' definitions in 64 bits."""
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

ATTENTION = dict(op="attention", type="bf16", train=False, n_seq=1, q_max=0, k_min=1, k_max=1, heads=8, kv_heads=8, hd=64, cap=0.0, slopes=False,
                 buckets=0, max_dist=0, two_sided=True, causal=False, window=-1, prefix=False, docs=False, lens=1)
NORM = dict(op="norm", type="bf16", train=False, rows=1, heads=8, kv_heads=8, hd=64, rot=64, interleaved=False, far=0, lens=1)


def listed():
    a, n = ATTENTION, NORM
    return [
        # the tracklets of 64 videos, encoded in one call (8 heads of 64 in f32, as the models' encoder has them), nearer tracklets preferred
        dict(a, name="encode_videos_f32", type="f32", n_seq=64, k_min=16, k_max=180, slopes=True, lens=11),
        # one token of one short stream: nothing but latency
        dict(a, name="one_token_f16", type="f16", q_max=1, k_min=257, k_max=257, cap=30.0, causal=True, lens=12),
        # a serving step: one new token for each of 48 streams, whose caches hold from a few rows to long ones
        dict(a, name="tokens_48_bf16", n_seq=48, q_max=1, k_max=16384, heads=32, kv_heads=8, hd=128, cap=50.0, causal=True, lens=13),
        # a few chunks of new tokens behind long caches, with a sliding window and a prefix that every token sees
        dict(a, name="chunks_bf16", n_seq=4, q_max=500, k_min=1000, k_max=8000, heads=32, kv_heads=4, hd=128, causal=True, window=4095, prefix=True, lens=14),
        # one long prompt: the largest product
        dict(a, name="prompt_8k_bf16", k_min=8192, k_max=8192, heads=32, kv_heads=8, hd=128, cap=50.0, causal=True, lens=15),
        # a training step on two packed rows of documents with padding at their ends
        dict(a, name="packed_train_f16", type="f16", train=True, n_seq=2, k_min=4096, k_max=4096, heads=12, kv_heads=4, causal=True, docs=True, lens=16),
        # a training step's attention over the clips of the 8 videos of a batch, f32, position bias by buckets in both directions
        dict(a, name="clips_bucket_train_f32", type="f32", train=True, n_seq=8, k_min=100, k_max=512, buckets=32, max_dist=128, lens=17),
        # the same of a larger encoder on longer sequences
        dict(a, name="bucket_train_bf16", train=True, n_seq=4, k_min=1400, k_max=2048, heads=16, kv_heads=16, buckets=32, max_dist=128, lens=18),
        # queries and keys of one decoding step of 8 streams: latency
        dict(n, name="norm_tokens_bf16", rows=8, heads=32, kv_heads=8, hd=128, rot=128, far=131071, lens=19),
        # those of a long prompt, pairs side by side
        dict(n, name="norm_prompt_f16", type="f16", rows=16384, heads=32, kv_heads=8, hd=128, rot=128, interleaved=True, lens=20),
        # those of the clips of a small training batch, f32, the rotation on half of the columns
        dict(n, name="norm_clips_train_f32", type="f32", train=True, rows=1801, rot=32, lens=21),
        # those of a training batch of long sequences
        dict(n, name="norm_train_bf16", train=True, rows=8192, heads=24, kv_heads=8, hd=128, rot=128, lens=22),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["one", "chunk", "forward", "train", "bucket", "bucket", "norm", "norm", "norm_train"])
    t = rng.choice(["f32", "f16", "bf16", "bf16"])
    hd = rng.choice([32, 64, 64, 96, 128, 128])
    lens = rng.randrange(1, 1 << 30)
    kv = rng.choice([1, 2, 4, 8])
    if kind in ("norm", "norm_train"):
        heads = kv * rng.choice([1, 2, 4])
        c = dict(NORM, type=t, train=kind == "norm_train", rows=_log(rng, 1, 8192), heads=heads, kv_heads=kv, hd=hd, rot=rng.choice([hd, hd // 2]),
                 interleaved=rng.random() < 0.5, far=rng.choice([0, 0, 200000]), lens=lens)
        return c
    g = rng.choice([1, 1, 2, 3, 4, 8]) if kv < 8 else rng.choice([1, 2, 4])
    c = dict(ATTENTION, type=t, heads=kv * g, kv_heads=kv, hd=hd, causal=rng.random() < 0.6, lens=lens)
    if kind == "one":
        c.update(n_seq=_log(rng, 1, 48), q_max=1, k_max=_log(rng, 1, 16384), causal=True, cap=rng.choice([0.0, 30.0, 50.0]), slopes=rng.random() < 0.4)
    elif kind == "chunk":
        c.update(n_seq=_log(rng, 1, 8), q_max=_log(rng, 2, 500), k_max=_log(rng, 20, 8000), causal=True, window=rng.choice([-1, 255, 1023, 4095]),
                 prefix=rng.random() < 0.4, cap=rng.choice([0.0, 30.0]))
    elif kind == "forward":
        n = _log(rng, 8, 4000)
        c.update(n_seq=max(1, min(64, _log(rng, 1, 64), 8000 // n)), k_min=max(1, n // rng.choice([1, 3, 10])), k_max=n, cap=rng.choice([0.0, 0.0, 50.0]),
                 slopes=rng.random() < 0.4, docs=rng.random() < 0.3)
    else:
        n = _log(rng, 16, 2000)
        c.update(train=True, n_seq=max(1, min(16, _log(rng, 1, 16), 5000 // n)), k_min=max(1, n // rng.choice([1, 3])), k_max=n,
                 cap=rng.choice([0.0, 0.0, 30.0]))
        if kind == "bucket":
            c.update(buckets=rng.choice([16, 32, 64]), max_dist=rng.choice([64, 128, 300]), two_sided=not c["causal"])
        else:
            c.update(slopes=rng.random() < 0.3, docs=rng.random() < 0.5, prefix=rng.random() < 0.3, window=rng.choice([-1, -1, 100]))
    return c


# ---- the lengths, documents and prefixes of a case (its own, not the seed's) ------------------------------------------------------------

def _plan(case):
    r = random.Random(case["lens"])
    k = [case["k_max"]] + [r.randint(case["k_min"], case["k_max"]) for _ in range(case["n_seq"] - 1)]
    if case["docs"]:                                             # packed rows: all of one length
        k = [case["k_max"]] * case["n_seq"]
    q = list(k) if not case["q_max"] else [min(n, case["q_max"] if case["q_max"] == 1 or i == 0 else r.randint(1, case["q_max"])) for i, n in enumerate(k)]
    prefix = [r.randint(0, max(1, n // 4)) for n in k] if case["prefix"] else [0] * len(k)
    ids = []
    for n in k:
        row, d = [], 0
        end = n - r.randint(0, n // 16)
        while len(row) < end:
            row += [d] * min(end - len(row), r.randint(1, max(2, n // 4)))
            d += 1
        ids.append(row + [-1] * (n - len(row)))
    return q, k, prefix, ids


def _bucket_map(n_bucket, max_dist, two_sided):
    """bucket of every distance key - query in [-max_dist, max_dist]: exact up to a half of a side's buckets, then by the logarithm up to
    max_dist, in whole numbers (log(n / e) / log(m / e) * c >= t  <=>  n^c >= m^t e^(c - t))"""
    side = n_bucket // 2 if two_sided else n_bucket
    e = side // 2
    c = side - e
    out = []
    for d in range(-max_dist, max_dist + 1):
        n = abs(d) if two_sided else max(-d, 0)
        b = n if n < e else min(side - 1, e + max(t for t in range(c + 1) if n ** c >= max_dist ** t * e ** (c - t)))
        out.append(b + (side if two_sided and d > 0 else 0))
    return torch.tensor(out, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)

    h, hk, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["op"] == "norm":
        n = case["rows"]
        qkv = normal(n, (h + 2 * hk) * hd, scale=1.5)            # the in-projection's output: queries, keys and values side by side
        pos = torch.arange(n, device="cuda", dtype=torch.int32)
        if case["far"]:
            pos = torch.randint(0, case["far"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        s = dict(case=case, q=qkv[:, :h * hd].view(n, h, hd), k=qkv[:, h * hd:(h + hk) * hd].view(n, hk, hd), pos=pos,
                 wq=1 + 0.2 * torch.randn(hd, generator=g, device="cuda"), wk=1 + 0.2 * torch.randn(hd, generator=g, device="cuda"),
                 inv_freq=10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"]))
        if case["train"]:
            s.update(gq=normal(n, h, hd), gk=normal(n, hk, hd))
        return s
    ql, kl, prefix, ids = _plan(case)
    nq, nk = sum(ql), sum(kl)

    def whole(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()

    s = dict(case=case, q=normal(nq, h, hd, scale=1.5), k=normal(nk, hk, hd), v=normal(nk, hk, hd), q_off=whole(np.cumsum([0] + ql)),
             k_off=whole(np.cumsum([0] + kl)), max_q=max(ql), max_k=max(kl), slopes=None, table=None, map=None, prefix=None, docs=None)
    if case["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
    if case["buckets"]:
        s["table"] = torch.randn(case["buckets"], h, generator=g, device="cuda")
        s["map"] = _bucket_map(case["buckets"], case["max_dist"], case["two_sided"]).cuda()
    if case["prefix"]:
        s["prefix"] = whole(prefix)
    if case["docs"]:
        s["docs"] = whole(sum(ids, []))
    if case["train"]:
        s["go"] = normal(nq, h, hd)
    return s


def run(state):
    case = state["case"]
    if own:
        return _own_norm(state) if case["op"] == "norm" else _own_attention(state)
    return _plain_norm(state) if case["op"] == "norm" else _plain_attention(state)


# ---- the library's operators -------------------------------------------------------------------------------------------------------------

def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vidsgg-big_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from bigc_hip import sequence
    return sequence


def _own_attention(s):
    lib, c = _library(), s["case"]
    kw = dict(softcap=c["cap"], slopes=s["slopes"], rel_table=s["table"], rel_map=s["map"], causal=c["causal"], window=(c["window"], -1),
              prefix_len=s["prefix"], q_doc=s["docs"], k_doc=s["docs"])
    if not c["train"]:
        return lib.attend(s["q"], s["k"], s["v"], s["q_off"], s["k_off"], s["max_q"], s["max_k"], **kw)
    o, saved = lib.attend(s["q"], s["k"], s["v"], s["q_off"], s["k_off"], s["max_q"], s["max_k"], save=True, **kw)
    dq, dk, dv, dtable = lib.attend_bwd(saved, s["go"])
    return [o, dq, dk, dv] + ([] if dtable is None else [dtable])


def _own_norm(s):
    lib, c = _library(), s["case"]
    args = (s["wq"], s["wk"], s["pos"], s["inv_freq"])
    q, k = lib.head_norm_rope(s["q"], s["k"], *args, interleaved=c["interleaved"])
    if not c["train"]:
        return q, k
    return (q, k) + tuple(lib.head_norm_rope_bwd(s["gq"], s["gk"], s["q"], s["k"], *args, interleaved=c["interleaved"]))


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------

def _rows(off, n, longest):
    """(sequence, longest) row numbers cut to the last row, whether a place holds a row, and (sequence, place) of every row"""
    at = off[:-1, None].long() + torch.arange(longest, device=off.device)
    live = at < off[1:, None]
    row = torch.arange(n, device=off.device)
    seq = torch.bucketize(row, off[1:].long(), right=True)
    return at.clamp(max=n - 1), live, seq, row - off[seq]


def _plain_attention(s):
    c = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    h, hk, hd, S, scale = c["heads"], c["kv_heads"], c["hd"], c["n_seq"], c["hd"] ** -0.5
    Lq, Lk = s["max_q"], s["max_k"]
    qi, qlive, qseq, qrow = _rows(s["q_off"], q.shape[0], Lq)
    ki, klive, kseq, krow = _rows(s["k_off"], k.shape[0], Lk)
    Q = q[qi].float().transpose(1, 2).reshape(S, hk, h // hk * Lq, hd)
    K = k[ki].float().transpose(1, 2)
    V = v[ki].float().transpose(1, 2)
    shift = (s["k_off"][1:] - s["k_off"][:-1]) - (s["q_off"][1:] - s["q_off"][:-1])
    p = torch.arange(Lq, device=q.device) + shift[:, None]
    d = torch.arange(Lk, device=q.device)[None, None] - p[:, :, None]                  # key minus query, (S, Lq, Lk)
    see = torch.ones_like(d, dtype=torch.bool)
    if c["causal"]:
        see &= d <= 0
    if c["window"] >= 0:
        see &= -d <= c["window"]
    if s["prefix"] is not None:
        see |= (torch.arange(Lk, device=q.device) < s["prefix"][:, None])[:, None]
    if s["docs"] is not None:
        dq_, dk_ = s["docs"][qi], s["docs"][ki]
        see &= (dq_[:, :, None] == dk_[:, None, :]) & (dk_ >= 0)[:, None]
    see = (see & qlive[:, :, None] & klive[:, None])[:, None]
    x = (Q @ K.transpose(-1, -2)).view(S, h, Lq, Lk) * scale
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x = t * c["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * d.abs()[:, None]
    if s["table"] is not None:
        R = c["max_dist"]
        x = x + s["table"][s["map"].long()].t()[:, d.clamp(-R, R) + R].transpose(0, 1)
    x = x.masked_fill(~see, float("-inf"))
    m = x.amax(-1, keepdim=True)
    P = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    P = P / P.sum(-1, keepdim=True).clamp(min=1e-30)
    del x, see
    O = (P.view(S, hk, -1, Lk) @ V).view(S, h, Lq, hd)
    o = O[qseq, :, qrow].to(q.dtype)
    if not c["train"]:
        return o
    G = s["go"][qi].float().transpose(1, 2) * qlive[:, None, :, None]
    Gg = G.reshape(S, hk, -1, hd)
    dS = P * ((Gg @ V.transpose(-1, -2)).view(S, h, Lq, Lk) - (G * O).sum(-1, keepdim=True))
    dv = P.view(S, hk, -1, Lk).transpose(-1, -2) @ Gg
    grads = []
    if s["table"] is not None:                                   # sums along the diagonals of equal distance, then by bucket, in 64 bits
        W = Lq + Lk
        skew = torch.nn.functional.pad(dS.flip(2), (0, Lq)).view(S, h, Lq * W)[:, :, :Lq * (W - 1)].view(S, h, Lq, W - 1)
        by_d = skew.sum(2, dtype=torch.float64)                  # column x: place of key - place of query = x - (Lq - 1)
        dist = torch.arange(W - 1, device=q.device) - (Lq - 1) - shift[:, None]
        to = s["map"].long()[dist.clamp(-R, R) + R]
        dt = torch.zeros(c["buckets"], h, dtype=torch.float64, device=q.device)
        grads = [dt.index_add_(0, to.reshape(-1), by_d.transpose(1, 2).reshape(-1, h)).float()]
    if c["cap"]:
        dS = dS * (1 - t * t)
    dS = dS.view(S, hk, -1, Lk) * scale
    dq = (dS @ K).view(S, h, Lq, hd)
    dk = dS.transpose(-1, -2) @ Q
    return [o, dq[qseq, :, qrow].to(q.dtype), dk[kseq, :, krow].to(q.dtype), dv[kseq, :, krow].to(q.dtype)] + grads


def _turn(x, cos, sin, interleaved, back=False):
    """rotates the pairs of the first 2 * cos.shape[-1] columns"""
    r = cos.shape[-1]
    a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if interleaved else (x[..., :r], x[..., r:2 * r])
    sin = -sin if back else sin
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., 2 * r:]], -1)


def _plain_norm(s, eps=1e-6):
    c = s["case"]
    angle = s["pos"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def forward(x, w):
        x = x.float()
        n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
        return _turn(n, cos, sin, c["interleaved"])

    def backward(gy, x, w):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        gn, hat = _turn(gy.float(), cos, sin, c["interleaved"], back=True), x * r
        gw = gn * w
        return (r * (gw - hat * (gw * hat).mean(-1, keepdim=True))), (gn * hat).sum((0, 1), dtype=torch.float64).float()

    t = s["q"].dtype
    out = (forward(s["q"], s["wq"]).to(t), forward(s["k"], s["wk"]).to(t))
    if not c["train"]:
        return out
    dq, dwq = backward(s["gq"], s["q"], s["wq"])
    dk, dwk = backward(s["gk"], s["k"], s["wk"])
    return out + (dq.to(t), dk.to(t), dwq, dwk)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["type"] == "f32" else 2
    h, hk, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["op"] == "norm":
        n = case["rows"] * (h + hk) * hd
        # forward: x in, y out; a training step: x and dy in, y and dx out
        return {"bytes": n * size * (4 if case["train"] else 2) + 4 * case["rows"], "flops": n * (25 if case["train"] else 8)}
    ql, kl, prefix, ids = _plan(case)
    pairs = seen = 0
    for i, n in enumerate(kl):
        p = np.arange(ql[i]) + n - ql[i]
        lo = np.maximum(p - case["window"], 0) if case["window"] >= 0 else np.zeros_like(p)
        hi = p + 1 if case["causal"] else np.full_like(p, n)
        a, b, live = np.zeros_like(p), np.full_like(p, n), np.ones(len(p), bool)
        if case["docs"]:
            d = np.asarray(ids[i])
            a, b, live = np.searchsorted(np.where(d < 0, 1 << 30, d), d, "left"), np.searchsorted(np.where(d < 0, 1 << 30, d), d, "right"), d >= 0
        f = prefix[i] if case["prefix"] else 0
        lo, hi = np.maximum(lo, f), np.maximum(hi, f)            # behind the prefix
        pairs += int(((np.clip(np.minimum(hi, b) - np.maximum(lo, a), 0, None) + np.clip(np.minimum(f, b) - a, 0, None)) * live).sum())
        seen += n - int(lo.min()) + min(f, int(lo.min()))
    rows_q, rows_k = sum(ql) * h * hd * size, seen * hk * hd * size
    if not case["train"]:
        return {"bytes": 2 * rows_q + 2 * rows_k, "flops": 4 * pairs * h * hd}
    return {"bytes": 4 * rows_q + 4 * rows_k, "flops": 14 * pairs * h * hd}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["op"] == "norm" else _exact_attention(s)


def _exact_attention(s):
    c = s["case"]
    qo, ko = s["q_off"].tolist(), s["k_off"].tolist()
    h, group = c["heads"], c["heads"] // c["kv_heads"]
    q, k, v = (s[n].double() for n in "qkv")
    o = torch.zeros_like(q)
    table = s["table"].double() if s["table"] is not None else None
    grads = [torch.zeros_like(x) for x in (q, k, v)] + ([torch.zeros_like(table)] if table is not None else [])
    for i in range(len(qo) - 1):
        (a, b), (e, f) = qo[i:i + 2], ko[i:i + 2]
        dist = torch.arange(f - e, device="cuda").view(1, -1) - torch.arange(b - a, device="cuda").view(-1, 1) - (f - e - b + a)
        near = torch.ones_like(dist, dtype=torch.bool)
        if c["causal"]:
            near = near & (dist <= 0)
        if c["window"] >= 0:
            near = near & (dist >= -c["window"])
        if s["prefix"] is not None:
            near[:, :int(s["prefix"][i])] = True
        if s["docs"] is not None:
            x, y = s["docs"][a:b], s["docs"][e:f]
            near = near & (x.view(-1, 1) == y.view(1, -1)) & (x >= 0).view(-1, 1)
        any_ = near.any(1, keepdim=True)
        for j in range(h):
            leaves = [q[a:b, j], k[e:f, j // group], v[e:f, j // group]] + ([table[:, j]] if table is not None else [])
            leaves = [x.clone().requires_grad_(c["train"]) for x in leaves]
            score = leaves[0] @ leaves[1].t() / c["hd"] ** 0.5
            if c["cap"]:
                score = c["cap"] * torch.tanh(score / c["cap"])
            if s["slopes"] is not None:
                score = score - float(s["slopes"][j]) * dist.abs()
            if table is not None:
                by_distance = leaves[3][s["map"].long()]
                score = score + by_distance[dist.clamp(-c["max_dist"], c["max_dist"]) + c["max_dist"]]
            score = torch.where(near, score, torch.full_like(score, -1e300))
            weight = torch.where(any_, torch.softmax(score, 1), torch.zeros_like(score))
            y = weight @ leaves[2]
            o[a:b, j] = y.detach()
            if c["train"]:
                got = torch.autograd.grad(y, leaves, s["go"][a:b, j].double())
                grads[0][a:b, j] += got[0]
                grads[1][e:f, j // group] += got[1]
                grads[2][e:f, j // group] += got[2]
                if table is not None:
                    grads[3][:, j] += got[3]
    return [o] + grads if c["train"] else o


def _exact_norm(s, eps=1e-6):
    c = s["case"]
    phase = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None, None] * s["inv_freq"])
    r = c["rot"] // 2

    def turned(x, w):
        n = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["hd"] + eps)
        n = n * w
        pair = n[..., :2 * r]
        pair = pair.unflatten(-1, (r, 2)) if c["interleaved"] else pair.unflatten(-1, (2, r)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * phase)
        z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, n[..., 2 * r:]], -1)

    out, grads = [], []
    for name in "qk":
        x, w = s[name].double().requires_grad_(c["train"]), s["w" + name].double().requires_grad_(c["train"])
        y = turned(x, w)
        out.append(y.detach())
        if c["train"]:
            grads += torch.autograd.grad(y, (x, w), s["g" + name].double())
    return tuple(out) if not c["train"] else tuple(out) + (grads[0], grads[2], grads[1], grads[3])
