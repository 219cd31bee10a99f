"""Plain float64 statements of the sequence operators (test infrastructure): one sequence and one head at a time, dense, gradients by autograd.
They have no counterpart in the reference, whose attention knows no order (models/model_0v10.py:109,183)."""
import torch


def seen_matrix(nq, nk, causal=False, window=(-1, -1), prefix=0, q_doc=None, k_doc=None):
    d = torch.arange(nk)[None, :] - (torch.arange(nq)[:, None] + nk - nq)
    near = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        near &= d <= 0
    if window[0] >= 0:
        near &= d >= -window[0]
    if window[1] >= 0:
        near &= d <= window[1]
    near |= (torch.arange(nk) < prefix)[None, :]
    if q_doc is not None:
        near &= (q_doc[:, None] == k_doc[None, :]) & (q_doc >= 0)[:, None]
    return near, d


def attention(q, k, v, q_off, k_off, scale=None, softcap=0.0, slopes=None, rel_table=None, rel_map=None, causal=False, window=(-1, -1),
              prefix_len=None, q_doc=None, k_doc=None, d_o=None, half_eps=0.0):
    """-> dict of float64 results: o, lse and, with d_o, dq, dk, dv, d_rel_table; under "tol_<name>" the bound of every element's error
    for a kernel that takes scores and sums in f32 and rounds P, dS and the results to a type of relative step ``half_eps`` (0: f32).

    The bound: u = 2^-24.  A score is off by at most c = (hd + 16) u (1 + max sum |q_c k_c scale| + max |bias|) (a sum of hd products, the cap and
    the biases added in f32), P by 2 c + (L + 16) u of itself (numerator and denominator), so o by (that + half_eps / 2) sum P |v| and its own
    rounding; dP - delta by (hd + 16) u sum |dO| (|v| + |o|), and by sum |dO| times the error of the o that delta = dO . o is taken from, which for
    half types is one of P in two parts (half_eps^2 instead of half_eps); dS by P times that plus its own relative error; the gradients sum those.

    Below the normal range a rounding step is no longer relative: a P under 2^-126 (f32's and bfloat16's smallest normal number) may be taken as 0,
    which is an absolute error of 2^-126, as large as such a P itself.  f16 reaches down to 2^-14 in steps of 2^-24 below it, so that a kernel that
    rounds to f16 has to scale: with the row's largest P at 2^14 the absolute error is half a step, 2^-25 2^-14 = 2^-39; dS, scaled so that the
    largest lies in [2^13, 2^15), is off by at most 2^-25 2^-13 = 2^-38 of the largest."""
    u = 2.0 ** -24
    n_head, hd, group = q.shape[1], q.shape[2], q.shape[1] // max(1, k.shape[1])
    scale = hd ** -0.5 if scale is None else scale
    qd, kd, vd = q.double(), k.double(), v.double()
    z = torch.zeros_like
    out = dict(o=z(qd), lse=torch.full(q.shape[:2], float("-inf"), dtype=torch.float64), tol_o=z(qd), tol_lse=torch.zeros(q.shape[:2], dtype=torch.float64))
    if d_o is not None:
        out.update(dq=z(qd), dk=z(kd), dv=z(vd), tol_dq=z(qd), tol_dk=z(kd), tol_dv=z(vd))
        if rel_table is not None:
            out.update(d_rel_table=z(rel_table.double()), tol_d_rel_table=z(rel_table.double()))
    r = half_eps / 2
    low = 2.0 ** -39 if half_eps == 2.0 ** -10 else 2.0 ** -126
    low_s = 2.0 ** -38 if half_eps == 2.0 ** -10 else 0.0
    for s in range(len(q_off) - 1):
        a, b, e, f = int(q_off[s]), int(q_off[s + 1]), int(k_off[s]), int(k_off[s + 1])
        if b <= a:
            continue
        near, d = seen_matrix(b - a, f - e, causal, window, 0 if prefix_len is None else int(prefix_len[s]),
                              None if q_doc is None else q_doc[a:b], None if k_doc is None else k_doc[e:f])
        for h in range(n_head):
            hk = h // group
            # a hidden place's value takes no part: rows that nobody sees, and that see nothing, are taken as 0
            sees, seen = near.any(1), near.any(0)
            Q = torch.where(sees[:, None], qd[a:b, h], torch.zeros(())).requires_grad_(d_o is not None)
            K = torch.where(seen[:, None], kd[e:f, hk], torch.zeros(())).requires_grad_(d_o is not None)
            V = torch.where(seen[:, None], vd[e:f, hk], torch.zeros(())).requires_grad_(d_o is not None)
            x = Q @ K.t() * scale
            big = float((Q.detach().abs() @ K.detach().abs().t() * abs(scale)).max()) if f > e else 0.0
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * d.abs()
                big += float((float(slopes[h]) * d.abs() * near).max()) if f > e else 0.0
            T = None
            if rel_table is not None:
                T = rel_table[:, h].double().clone().requires_grad_(d_o is not None)
                R = rel_map.shape[0] // 2
                bias = T[rel_map.long()][d.clamp(-R, R) + R]
                x = x + bias
                fin = bias.detach()[torch.isfinite(bias.detach()) & (bias.detach().abs() < 1e30)]
                big += float(fin.abs().max()) if fin.numel() else 0.0
            x = torch.where(near, x, torch.full_like(x, float("-inf")))
            alive = (x.detach() > float("-inf")).any(1) if f > e else torch.zeros(b - a, dtype=torch.bool)
            safe = torch.where(alive[:, None], x, torch.zeros_like(x))
            P = torch.where(alive[:, None], torch.softmax(safe, 1), torch.zeros_like(x)) if f > e else x
            O = P @ V
            out["o"][a:b, h] = O.detach()
            out["lse"][a:b, h] = torch.where(alive, torch.logsumexp(safe, 1), torch.full((b - a,), float("-inf"), dtype=torch.float64)) .detach() if f > e else float("-inf")
            c = (hd + 16) * u * (1 + big)
            p_err = 2 * c + (f - e + 16) * u
            Pa, Va = P.detach(), V.detach().abs()
            out["tol_o"][a:b, h] = (p_err + r + 2 * u) * (Pa @ Va) + low * Va.sum(0) + (r + u) * O.detach().abs()
            out["tol_lse"][a:b, h] = p_err + 4 * u * torch.nan_to_num(out["lse"][a:b, h], neginf=0.0).abs()
            if d_o is None or f <= e:
                continue
            G = torch.where(sees[:, None], d_o[a:b, h].double(), torch.zeros(()))
            grads = torch.autograd.grad(O, (Q, K, V) + ((T,) if T is not None else ()), G)
            out["dq"][a:b, h] += grads[0]
            out["dk"][e:f, hk] += grads[1]
            out["dv"][e:f, hk] += grads[2]
            Ga = G.abs()
            dP = G @ V.detach().t()
            dS = (Pa * (dP - (G * O.detach()).sum(1, keepdim=True))).abs()
            reach = Ga @ Va.t() + (Ga * (Pa @ Va)).sum(1, keepdim=True)
            o_err = (p_err + r * half_eps + 2 * u) * (Pa @ Va)
            eS = Pa * (Ga * o_err).sum(1, keepdim=True) + Pa * reach * ((hd + 16) * u * 2 + p_err) + dS * 4 * u + near * (low * reach + low_s * dS.max())
            n = (b - a + f - e + 16) * u
            sc = abs(scale) * (1 + 2 * c)
            out["tol_dq"][a:b, h] += sc * ((eS + (r + n) * dS) @ K.detach().abs())
            out["tol_dk"][e:f, hk] += sc * ((eS + (r + n) * dS).t() @ Q.detach().abs())
            out["tol_dv"][e:f, hk] += (p_err + r + n) * (Pa.t() @ Ga) + low * Ga.sum(0)
            if T is not None:
                out["d_rel_table"][:, h] += grads[3]
                m = rel_map.long()[d.clamp(-R, R) + R].reshape(-1)
                total = (n + 64 * u) * dS + eS
                out["tol_d_rel_table"][:, h].index_add_(0, m, torch.where(alive[:, None], total, torch.zeros(())).reshape(-1))
    for name in ("dq", "dk", "dv"):
        if name in out:
            out["tol_" + name] += (r + u) * (out[name].abs() + out["tol_" + name])
    return out


def norm_rope(x, w, pos, inv_freq, eps=1e-6, interleaved=False):
    """x (rows, heads, hd) float64 (may require grad) -> its RMS norm times w, rotated"""
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        n = n * w
    if inv_freq is None:
        return n
    f = inv_freq.shape[0]
    t = pos.double()[:, None, None] * inv_freq.double()
    i = torch.arange(f)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + f)
    a, b = n[..., ia], n[..., ib]
    y = n.clone()
    y[..., ia] = a * torch.cos(t) - b * torch.sin(t)
    y[..., ib] = b * torch.cos(t) + a * torch.sin(t)
    return y
