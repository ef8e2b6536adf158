"""Timed cases of the layer norm and attention operators.

A case is one call a program makes: a forward, a training step of one operator (forward and
backward, with every gradient returned) or one decoding step. `run` has two forms: the plain
one, elementary torch operations in fp32 rounded once at the end, and the framework's own entry
points in `fast_trimul_b200.functional`. `exact` is the definition in 64 bits.

Operators (`op` of a case):
  layer_norm   y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension
  packed       softmax(q k^T * scale) v of sequences of different lengths stored one behind the
               other, grouped key / value heads, causal (aligned to the last key) or not
  cached       the same for one new token of each sequence over a key / value cache
  pair         attention of every row of a pair representation with an additive pair bias that
               all rows of a batch element share, and a mask of the keys
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # the single representation of the trunk (c_s = 384, N = 384): the smallest call
        {"name": "layer_norm_single", "op": "layer_norm", "rows": 384, "width": 384, "type": "bf16",
         "train": False},
        # the pair representation at N = 1024 in training
        {"name": "layer_norm_pair_train", "op": "layer_norm", "rows": 1024 * 1024, "width": 128,
         "type": "bf16", "train": True},
        # odd width and row count in fp32: a head's norm outside the trunk
        {"name": "layer_norm_odd_train", "op": "layer_norm", "rows": 6151, "width": 1001,
         "type": "fp32", "train": True},
        # ragged prompts, grouped heads, inference
        {"name": "packed_ragged", "op": "packed", "lengths": "4096,1,333,2049,17,1000,640,56",
         "kv_more": 0, "heads": 16, "kv_heads": 4, "dim": 128, "type": "bf16", "causal": True,
         "train": False},
        # a few short sequences over the single representation's heads (16 of 24): latency
        {"name": "packed_short", "op": "packed", "lengths": "129,64,1,200", "kv_more": 0, "heads": 16,
         "kv_heads": 16, "dim": 24, "type": "bf16", "causal": False, "train": False},
        # a ragged training batch in fp16
        {"name": "packed_ragged_train", "op": "packed", "lengths": "1500,2048,7,811,128,1,1777,1920",
         "kv_more": 0, "heads": 12, "kv_heads": 6, "dim": 64, "type": "fp16", "causal": True,
         "train": True},
        # one long sequence in training
        {"name": "packed_long_train", "op": "packed", "lengths": "8192", "kv_more": 0, "heads": 16,
         "kv_heads": 4, "dim": 128, "type": "bf16", "causal": True, "train": True},
        # one new token of one short sequence: latency
        {"name": "cached_short", "op": "cached", "lengths": "501", "capacity": 1024, "heads": 16,
         "kv_heads": 4, "dim": 64, "type": "fp16"},
        # one new token of sixteen long sequences of different lengths: the cache's bandwidth
        {"name": "cached_long", "op": "cached",
         "lengths": "16384,16001,15000,14337,16384,9000,12345,16000,16383,11111,13000,16384,15555,8191,"
                    "16200,14000",
         "capacity": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16"},
        # triangle attention of the trunk (N = 384, 4 heads of 32) in inference, padded crop
        {"name": "pair_trunk", "op": "pair", "batch": 1, "rows": 384, "length": 384, "valid": 371,
         "heads": 4, "dim": 32, "type": "bf16", "train": False},
        # triangle attention in training, a length that is no multiple of a tile
        {"name": "pair_train", "op": "pair", "batch": 1, "rows": 250, "length": 250, "valid": 250,
         "heads": 4, "dim": 32, "type": "bf16", "train": True},
        # attention of the single representation with pair bias (16 heads of 24) in training
        {"name": "pair_single_train", "op": "pair", "batch": 2, "rows": 1, "length": 1001, "valid": 990,
         "heads": 16, "dim": 24, "type": "bf16", "train": True},
    ]


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "packed", "packed", "cached", "pair", "pair"])
    kind = rng.choice(["bf16", "fp16"])
    train = rng.random() < 0.5
    if op == "layer_norm":
        width = _between(rng, 16, 8192)
        rows = _between(rng, 1, max(1, 2 ** 26 // width))
        return {"op": op, "rows": rows, "width": width, "type": rng.choice(["bf16", "fp16", "fp32"]),
                "train": train}
    dim = rng.choice([16, 24, 32, 40, 64, 80, 96, 128])
    if op == "pair":
        length = _between(rng, 8, 448)
        single = rng.random() < 0.3
        if single:
            length = _between(rng, 8, 1200)
        return {"op": op, "batch": rng.choice([1, 1, 2]) if length < 300 or single else 1,
                "rows": 1 if single else length, "length": length,
                "valid": rng.randint(max(1, length // 2), length),
                "heads": rng.choice([4, 8, 16]) if single else 4, "dim": dim if single else rng.choice([16, 32]),
                "type": kind, "train": train}
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    if kv_heads * group > 32:
        group = 4
    if op == "cached":
        batch = _between(rng, 1, 32)
        capacity = _between(rng, 64, 16384)
        lengths = [_between(rng, 1, capacity) for _ in range(batch)]
        return {"op": op, "lengths": ",".join(map(str, lengths)), "capacity": capacity,
                "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "type": kind}
    if kv_heads * group > 16:
        group = 2 if kv_heads == 8 else 4
    count = rng.randint(1, 8)
    longest = _between(rng, 8, 4096)
    lengths = [longest] + [_between(rng, 1, longest) for _ in range(count - 1)]
    rng.shuffle(lengths)
    return {"op": op, "lengths": ",".join(map(str, lengths)),
            "kv_more": rng.choice([0, 0, _between(rng, 1, 512)]),
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "type": kind,
            "causal": rng.random() < 0.7, "train": train}


# ----------------------------------------------------------------------------- inputs
def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case)
    s["leaves"] = []
    if case["op"] == "layer_norm":
        w = case["width"]
        s["x"] = (rand(case["rows"], w) * 1.5 + 0.3).to(t)
        s["weight"] = (1 + 0.1 * rand(w)).to(t)
        s["bias"] = (0.1 * rand(w)).to(t)
        if case["train"]:
            s["grad"] = rand(case["rows"], w).to(t)
            s["leaves"] = [s[k].requires_grad_() for k in ("x", "weight", "bias")]
        return s
    h, d = case["heads"], case["dim"]
    if case["op"] == "pair":
        b, r, n = case["batch"], case["rows"], case["length"]
        # one projection's output, as a trunk's layer splits it
        qkv = rand(b, r, n, 3, h, d).to(t)
        s["q"], s["k"], s["v"] = (x.detach() for x in qkv.unbind(3))
        s["bias"] = rand(b, h, n, n).to(t)
        keep = torch.arange(n, device="cuda") < case["valid"]
        s["mask"] = keep.expand(b, r, n).contiguous()
        if r > 1:   # the padded rows of a crop have no key left at all
            s["mask"] &= keep[:r].view(1, r, 1)
        if case["train"]:
            s["grad"] = rand(b, r, n, h, d).to(t)
            s["leaves"] = [s[k].requires_grad_() for k in ("q", "k", "v", "bias")]
        return s
    hk, lens = case["kv_heads"], _lengths(case)
    if case["op"] == "cached":
        b, cap = len(lens), case["capacity"]
        s["q"] = rand(b, h, d).to(t)
        s["k"] = rand(b, cap, hk, d).to(t)
        s["v"] = rand(b, cap, hk, d).to(t)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return s
    klens = [n + case["kv_more"] for n in lens]

    def ends(ls):
        c = [0]
        for n in ls:
            c.append(c[-1] + n)
        return torch.tensor(c, dtype=torch.int32, device="cuda")

    s["cu_q"], s["cu_k"] = ends(lens), ends(klens)
    s["most_q"], s["most_k"] = max(lens), max(klens)
    s["q"] = rand(sum(lens), h, d).to(t)
    s["k"] = rand(sum(klens), hk, d).to(t)
    s["v"] = rand(sum(klens), hk, d).to(t)
    if case["train"]:
        s["grad"] = rand(sum(lens), h, d).to(t)
        s["leaves"] = [s[k].requires_grad_() for k in ("q", "k", "v")]
    return s


# -------------------------------------------------------------------------- the calls
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


def _run_own(s):
    from fast_trimul_b200 import functional as F
    op = s["op"]
    with torch.set_grad_enabled(bool(s["leaves"])):
        if op == "layer_norm":
            out = F.layer_norm(s["x"], s["weight"], s["bias"])
        elif op == "packed":
            out = F.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"])
        elif op == "cached":
            out = F.cached_attention(s["q"], s["k"], s["v"], s["lengths"])
        else:
            out = F.pair_attention(s["q"], s["k"], s["v"], s["bias"], mask=s["mask"])
    if not s["leaves"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, s["leaves"], s["grad"])]


def _plain_layer_norm(s, eps=1e-5):
    t = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    out = (xh * w + b).to(t)
    if not s["leaves"]:
        return [out]
    g = s["grad"].float()
    gy = g * w
    dx = rstd * (gy - gy.mean(-1, keepdim=True) - xh * (gy * xh).mean(-1, keepdim=True))
    return [out, dx.to(t), (g * xh).sum(0, dtype=torch.float64).to(t), g.sum(0, dtype=torch.float64).to(t)]


def _softmax(scores, keep):
    """Weights of each row over the keys in `keep`; a row without keys has none."""
    scores = scores.masked_fill_(~keep, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, torch.ones_like(total), total))


def _attend(q, k, v, grad, keep, scale, bias=None):
    """out, and (dq, dk, dv, ds) where `grad` is given; q, k, v, grad (..., length, dim) in fp32."""
    s = (q @ k.transpose(-1, -2)).mul_(scale)
    if bias is not None:
        s += bias
    p = _softmax(s, keep)
    out = p @ v
    if grad is None:
        return out, None
    dv = p.transpose(-1, -2) @ grad
    dp = grad @ v.transpose(-1, -2)
    ds = dp.sub_((grad * out).sum(-1, keepdim=True)).mul_(p)
    return out, ((ds @ k) * scale, (ds.transpose(-1, -2) @ q) * scale, dv, ds)


def _plain_pair(s):
    t = s["q"].dtype
    heads_first = lambda x: x.detach().float().transpose(2, 3)   # noqa: E731  (b, r, h, n, d)
    q, k, v = (heads_first(s[x]) for x in ("q", "k", "v"))
    g = heads_first(s["grad"]) if s["leaves"] else None
    out, grads = _attend(q, k, v, g, s["mask"][:, :, None, None, :], s["dim"] ** -0.5,
                         s["bias"].detach().float()[:, None])
    back = lambda x: x.transpose(2, 3).to(t).contiguous()        # noqa: E731
    if grads is None:
        return [back(out)]
    dq, dk, dv, ds = grads
    return [back(out), back(dq), back(dk), back(dv), ds.sum(1).to(t)]


def _padded(x, cu, most):
    """Packed rows (tokens, heads, dim) as (sequences, heads, most, dim) in fp32, with the rows' places."""
    at = torch.arange(most, device=x.device) + cu[:-1, None].long()
    ok = at < cu[1:, None]
    at = at.clamp_(max=x.shape[0] - 1)
    return (x.detach()[at].float() * ok[..., None, None]).transpose(1, 2), at, ok


def _plain_packed(s):
    t, group = s["q"].dtype, s["heads"] // s["kv_heads"]
    q, at_q, ok_q = _padded(s["q"], s["cu_q"], s["most_q"])
    k, at_k, ok_k = _padded(s["k"], s["cu_k"], s["most_k"])
    v = _padded(s["v"], s["cu_k"], s["most_k"])[0]
    split = lambda x: x.unflatten(1, (s["kv_heads"], group))     # noqa: E731
    keep = ok_k[:, None, None, None, :]
    if s["causal"]:
        nq, nk = s["cu_q"].diff(), s["cu_k"].diff()
        last = torch.arange(s["most_q"], device=q.device) + (nk - nq)[:, None]
        keep = keep & (torch.arange(s["most_k"], device=q.device) <= last[:, None, None, :, None])
    g = split(_padded(s["grad"], s["cu_q"], s["most_q"])[0]) if s["leaves"] else None
    out, grads = _attend(split(q), k[:, :, None], v[:, :, None], g, keep, s["dim"] ** -0.5)

    def packed(x, at, ok, tokens):
        y = torch.zeros(tokens, x.shape[1], x.shape[3], dtype=t, device=x.device)
        y[at[ok]] = x.transpose(1, 2)[ok].to(t)
        return y

    out = packed(out.flatten(1, 2), at_q, ok_q, s["q"].shape[0])
    if grads is None:
        return [out]
    dq, dk, dv, _ = grads
    return [out, packed(dq.flatten(1, 2), at_q, ok_q, s["q"].shape[0]),
            packed(dk.sum(2), at_k, ok_k, s["k"].shape[0]), packed(dv.sum(2), at_k, ok_k, s["k"].shape[0])]


def _plain_cached(s):
    b, h, d = s["q"].shape
    hk = s["kv_heads"]
    q = s["q"].float().view(b, hk, h // hk, d)
    k, v = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    keep = (torch.arange(s["capacity"], device=q.device) < s["lengths"][:, None])[:, None, None]
    out, _ = _attend(q, k, v, None, keep, d ** -0.5)
    return [out.reshape(b, h, d).to(s["q"].dtype)]


_PLAIN = {"layer_norm": _plain_layer_norm, "packed": _plain_packed, "cached": _plain_cached, "pair": _plain_pair}


# ---------------------------------------------------------------- the work of a pass
def _pairs_seen(nq, nk, causal):
    """Query / key pairs of one sequence."""
    if not causal:
        return nq * nk
    first = nk - nq + 1          # keys that the first query sees
    if first >= 1:
        return nq * (first + nk) // 2
    return nk * (nk + 1) // 2


def work(case):
    e = 4 if case["type"] == "fp32" else 2
    if case["op"] == "layer_norm":
        n = case["rows"] * case["width"]
        if case["train"]:   # x and the gradient in, y, dx, dw and db out
            return {"bytes": e * (4 * n + 4 * case["width"]), "flops": 19 * n}
        return {"bytes": e * (2 * n + 2 * case["width"]), "flops": 8 * n}
    d, h = case["dim"], case["heads"]
    if case["op"] == "pair":
        b, r, n = case["batch"], case["rows"], case["length"]
        x, bias = b * r * n * h * d, b * h * n * n
        seen = b * (case["valid"] if r > 1 else r) * h * n * case["valid"]
        if case["train"]:
            return {"bytes": e * (8 * x + 2 * bias) + b * r * n, "flops": 14 * d * seen}
        return {"bytes": e * (4 * x + bias) + b * r * n, "flops": 4 * d * seen}
    hk, lens = case["kv_heads"], _lengths(case)
    if case["op"] == "cached":
        n = sum(lens)
        return {"bytes": e * (2 * n * hk * d + 2 * len(lens) * h * d) + 4 * len(lens), "flops": 4 * d * h * n}
    klens = [n + case["kv_more"] for n in lens]
    seen = h * sum(_pairs_seen(a, b, case["causal"]) for a, b in zip(lens, klens))
    q, k = sum(lens) * h * d, sum(klens) * hk * d
    if case["train"]:
        return {"bytes": e * (4 * q + 4 * k) + 8 * (len(lens) + 1), "flops": 14 * d * seen}
    return {"bytes": e * (2 * q + 2 * k) + 8 * (len(lens) + 1), "flops": 4 * d * seen}


# ------------------------------------------------------------------ 64 bits, by itself
def _exact_head(q, k, v, g, scale, allowed, bias):
    """One head of one sequence: out and its gradients (dq, dk, dv, ds), all in 64 bits."""
    z = torch.einsum("id,jd->ij", q, k) * scale
    if bias is not None:
        z = z + bias
    z = torch.where(allowed, z, torch.full_like(z, -math.inf))
    p = torch.nan_to_num(torch.softmax(z, dim=1), nan=0.0)
    out = torch.einsum("ij,jd->id", p, v)
    if g is None:
        return (out,)
    dp = torch.einsum("id,jd->ij", g, v)
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    return (out, scale * torch.einsum("ij,jd->id", ds, k), scale * torch.einsum("ij,id->jd", ds, q),
            torch.einsum("ij,id->jd", p, g), ds)


def exact(case, seed):
    if case["op"] == "layer_norm":
        if case["rows"] * case["width"] > 2 ** 28:
            return None
    else:
        w = work(case)["flops"]
        if w > 4e12:     # the 64-bit products of more than this take too long
            return None
    s = prepare(case, seed)
    big = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    train = bool(s["leaves"])
    if case["op"] == "layer_norm":
        x, wt, bs = big["x"], big["weight"], big["bias"]
        var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        n = (x - mean) / sd
        out = [wt * n + bs]
        if train:
            u = big["grad"] * wt
            out += [(u - u.mean(-1, keepdim=True) - n * (u * n).mean(-1, keepdim=True)) / sd,
                    torch.einsum("rc,rc->c", big["grad"], n), torch.einsum("rc->c", big["grad"])]
        return out
    h, d = case["heads"], case["dim"]
    scale = 1.0 / math.sqrt(d)
    q, k, v, g = big["q"], big["k"], big["v"], big.get("grad")
    if case["op"] == "cached":
        out = torch.zeros_like(q)
        for b, n in enumerate(_lengths(case)):
            for i in range(h):
                j = i // (h // case["kv_heads"])
                ok = torch.ones(1, n, dtype=torch.bool, device=q.device)
                out[b, i] = _exact_head(q[b, i:i + 1], k[b, :n, j], v[b, :n, j], None, scale, ok, None)[0][0]
        return [out]
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    if case["op"] == "pair":
        db = torch.zeros_like(big["bias"])
        if case["batch"] * case["rows"] * h > 6000:
            return None
        for b in range(case["batch"]):
            for r in range(case["rows"]):
                ok = s["mask"][b, r][None, :].expand(case["length"], -1)
                for i in range(h):
                    at = (b, r, slice(None), i)
                    res = _exact_head(q[at], k[at], v[at], g[at] if train else None, scale, ok, big["bias"][b, i])
                    out[at] = res[0]
                    if train:
                        dq[at], dk[at], dv[at] = res[1:4]
                        db[b, i] += res[4]
        return [out, dq, dk, dv, db] if train else [out]
    a = c = 0
    for n in _lengths(case):
        m = n + case["kv_more"]
        ok = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if case["causal"]:
            ok = torch.tril(ok, diagonal=m - n)
        for i in range(h):
            j = i // (h // case["kv_heads"])
            res = _exact_head(q[a:a + n, i], k[c:c + m, j], v[c:c + m, j], g[a:a + n, i] if train else None,
                              scale, ok, None)
            out[a:a + n, i] = res[0]
            if train:
                dq[a:a + n, i] = res[1]
                dk[c:c + m, j] += res[2]
                dv[c:c + m, j] += res[3]
        a, c = a + n, c + m
    return [out, dq, dk, dv] if train else [out]
