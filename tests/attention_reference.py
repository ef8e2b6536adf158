"""Attention in 64 bits with its gradients, and how far a kernel may be from them.

With u half a step of the inputs' type (bf16 2^-8... `eps / 2`) and w = 2^-14 for everything that the
kernels do in fp32 (products of up to 128 terms, the exponential, sums: each below 2^-16 relative
to the sums of magnitudes used here, for scores up to ~100):

* a score t itself is an fp32 number, off by 2^-24 |t|, and so is the row's maximum m: where m is
  far from 0 (a bias used as a mask), the row's weights are off by 2^-22 |m| more, relative. (At
  3e38 the scores' differences vanish in 64 bits, too: nothing is added.)
* the weights p are rounded once to the type before P V:  |o' - o| <= u |o| + (u + w) A,
  A = sum_j p_j |v_j|  (the last rounding; the weights' rounding and fp32's).
* the same for dv = sum_i p_ij g_i, with A = sum_i p_ij |g_i|.
* the backward's d = rowsum(g o') takes the rounded o':  |d' - d| <= ed = sum_c |g_c| |o' - o|_c.
  ds = p (dp - d) is off by  E = p ed + w p (|g| |v| + |g| |o|)  and rounded once, u |ds|, before its
  products: |dq' - dq| <= u |dq| + scale sum_j (E + u |ds|)_ij |k_j|, dk alike with |q_i|.
* dbias sums ds in fp32 unrounded: u |dbias| + sum_rows E."""

import torch


class Sums:
    """Results and bounds of one call, gathered per sequence and head."""

    def __init__(self, q, k, bias):
        z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)   # noqa: E731
        self.o, self.dq, self.dk, self.dv = z(q), z(q), z(k), z(k)
        self.eo, self.edq, self.edk, self.edv = z(q), z(q), z(k), z(k)
        if bias is not None:
            self.db, self.edb = z(bias), z(bias)


def head(q, k, v, g, scale, keep, bias, u, w=2.0 ** -14):
    """One head of one sequence in float64: (o, dq, dk, dv, ds) and their bounds before the
    last rounding."""
    k, v = (torch.where(keep.any(0)[:, None], t, torch.zeros_like(t)) for t in (k, v))
    s = q @ k.T * scale
    if bias is not None:
        s = s + bias
    s = torch.where(keep, s, torch.full_like(s, -torch.inf))
    top = s.amax(1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, torch.zeros_like(top), top))
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ v
    w = w + torch.where(top.abs() < 1e30, 2.0 ** -22 * top.abs(), torch.zeros_like(top))
    eo = (u + w) * (p @ v.abs())
    dp = g @ v.T
    d = (g * o).sum(1, keepdim=True)
    ds = p * (dp - d)
    ed = (g.abs() * (u * (o.abs() + eo) + eo)).sum(1, keepdim=True)
    E = p * (ed + w * (g.abs() @ v.abs().T + (g * o).abs().sum(1, keepdim=True)))
    Er = E + u * (ds.abs() + E)
    return ((o, scale * ds @ k, scale * ds.T @ q, p.T @ g, ds),
            (eo, scale * Er @ k.abs(), scale * Er.T @ q.abs(), ((u + w) * p).T @ g.abs(), E))


def close(got, want, off, what):
    """|got - want| <= half a step of got + off, everywhere; NaN nowhere."""
    info = torch.finfo(got.dtype)
    u = info.eps / 2
    bound = u * (want.abs() + off) + off + info.tiny
    err = (got.double() - want).abs()
    assert not got.isnan().any(), what
    over = err - bound
    assert not (over > 0).any(), (what, over.max().item(), err.max().item())


def packed(q, k, v, g, cu_q, cu_k, causal, scale, key_mask=None):
    u = torch.finfo(q.dtype).eps / 2
    r = Sums(q, k, None)
    group = q.shape[1] // k.shape[1]
    q, k, v, g = q.double(), k.double(), v.double(), g.double()
    cu_q, cu_k = cu_q.tolist(), cu_k.tolist()
    for i in range(len(cu_q) - 1):
        a, b, c, d = cu_q[i], cu_q[i + 1], cu_k[i], cu_k[i + 1]
        if a == b or c == d:
            continue
        keep = torch.ones(b - a, d - c, dtype=torch.bool, device=q.device)
        if causal:
            keep = keep.tril((d - c) - (b - a))
        if key_mask is not None:
            keep = keep & key_mask[c:d]
        for h in range(q.shape[1]):
            hk = h // group
            res, off = head(q[a:b, h], k[c:d, hk], v[c:d, hk], g[a:b, h], scale, keep, None, u)
            r.o[a:b, h], r.dq[a:b, h] = res[:2]
            r.eo[a:b, h], r.edq[a:b, h] = off[:2]
            r.dk[c:d, hk] += res[2]
            r.dv[c:d, hk] += res[3]
            r.edk[c:d, hk] += off[2]
            r.edv[c:d, hk] += off[3]
    return r


def pair(q, k, v, g, bias, mask, scale):
    u = torch.finfo(q.dtype).eps / 2
    r = Sums(q, k, bias)
    B, R, N, H, _ = q.shape
    q, k, v, g = q.double(), k.double(), v.double(), g.double()
    for b in range(B):
        bb = min(b, bias.shape[0] - 1) if bias is not None else 0
        for i in range(R):
            keep = torch.ones(N, N, dtype=torch.bool, device=q.device)
            if mask is not None:
                keep = keep & mask[b, i].bool()
            for h in range(H):
                at = (b, i, slice(None), h)
                res, off = head(q[at], k[at], v[at], g[at], scale, keep,
                                None if bias is None else bias[bb, h].double(), u)
                r.o[at], r.dq[at], r.dk[at], r.dv[at] = res[:4]
                r.eo[at], r.edq[at], r.edk[at], r.edv[at] = off[:4]
                if bias is not None:
                    r.db[bb, h] += res[4]
                    r.edb[bb, h] += off[4]
    return r
