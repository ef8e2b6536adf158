"""The attention kernels against 64 bits, with bounds derived in attention_reference.py."""

import math

import pytest
import torch

import attention_reference as ref

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

BF, HF = torch.bfloat16, torch.float16


def gen(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, device="cuda", generator=g)


def ends(lens, first=0):
    c = [first]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device="cuda")


def check_waits():
    from fast_trimul_b200.ops.attention import attention_error_word
    attention_error_word().check()


def train(f, leaves, g, *a, **k):
    ls = [t.detach().requires_grad_() for t in leaves]
    out = f(*ls, *a, **k)
    return [out.detach(), *torch.autograd.grad(out, ls, g)]


def check_packed(q, k, v, cu_q, cu_k, causal=True, key_mask=None, scale=None):
    from fast_trimul_b200.functional import packed_attention
    g = gen(9)(*q.shape).to(q.dtype)
    got = train(packed_attention, (q, k, v), g, cu_q, cu_k, causal=causal, key_mask=key_mask, scale=scale)
    check_waits()
    w = ref.packed(q, k, v, g, cu_q, cu_k, causal, q.shape[2] ** -0.5 if scale is None else scale, key_mask)
    for name, a, want, off in zip(("o", "dq", "dk", "dv"), got, (w.o, w.dq, w.dk, w.dv),
                                  (w.eo, w.edq, w.edk, w.edv)):
        ref.close(a, want, off, name)
    with torch.no_grad():
        assert torch.equal(got[0], packed_attention(q, k, v, cu_q, cu_k, causal=causal, key_mask=key_mask, scale=scale))
    again = train(packed_attention, (q, k, v), g, cu_q, cu_k, causal=causal, key_mask=key_mask, scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


def qkv(rows, krows, h, hk, d, dtype, seed=0):
    r = gen(seed)
    return r(rows, h, d).to(dtype), r(krows, hk, d).to(dtype), r(krows, hk, d).to(dtype)


LENS = [[1], [2, 1, 1], [127], [128], [129], [64, 64, 63], [300, 1, 128, 257], [5, 0, 130, 0]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("h,hk,d,dtype", [(2, 2, 64, BF), (4, 2, 128, HF), (6, 2, 24, BF), (8, 1, 96, BF)])
def test_packed_lengths(lens, causal, h, hk, d, dtype):
    cu = ends(lens)
    check_packed(*qkv(sum(lens), sum(lens), h, hk, d, dtype), cu, cu, causal)


@pytest.mark.parametrize("d", [8, 16, 32, 40, 56, 64, 72, 80, 112, 120, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_packed_head_dimensions(d, dtype):
    cu = ends([150, 33])
    check_packed(*qkv(183, 183, 4, 2, d, dtype, d), cu, cu)


@pytest.mark.parametrize("h,hk", [(1, 1), (3, 1), (5, 1), (7, 1), (12, 4), (16, 1), (33, 1), (64, 1), (128, 1), (65, 1)])
def test_packed_head_groups(h, hk):
    cu = ends([70, 1, 140])
    check_packed(*qkv(211, 211, h, hk, 32, BF, h), cu, cu)


@pytest.mark.parametrize("lens,klens", [([1, 1, 1], [1, 130, 1000]), ([16, 3], [400, 3]), ([40, 200], [7, 130]),
                                        ([9, 0, 5], [0, 20, 300])], ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_packed_other_keys_than_queries(lens, klens, causal):
    got = check_packed(*qkv(sum(lens), sum(klens), 4, 2, 64, BF), ends(lens), ends(klens), causal)
    if lens[0] == 40 and causal:      # 33 queries in front of the first key: no keys, zeros
        assert (got[0][:33] == 0).all() and (got[1][:33] == 0).all()


def test_packed_rows_of_no_sequence_are_zero_and_not_read():
    q, k, v = qkv(300, 280, 4, 2, 64, BF)
    for t, lo, hi in ((q, 7, 250), (k, 20, 260), (v, 20, 260)):
        t[:lo] = float("nan")
        t[hi:] = float("inf")
    cu_q, cu_k = ends([100, 143], 7), ends([140, 100], 20)
    from fast_trimul_b200.functional import packed_attention
    g = gen(4)(*q.shape).to(BF)
    got = train(packed_attention, (q, k, v), g, cu_q, cu_k)
    check_waits()
    clean = [torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (q, k, v)]
    want = train(packed_attention, clean, g, cu_q, cu_k)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, lo, hi in ((got[0], 7, 250), (got[1], 7, 250), (got[2], 20, 260), (got[3], 20, 260)):
        assert (a[:lo] == 0).all() and (a[hi:] == 0).all()


def test_packed_neighbours_do_not_leak():
    """NaN or infinity in one sequence stays in it, also where the tiles overlap it."""
    q, k, v = qkv(90, 90, 2, 2, 32, BF)
    g = gen(5)(*q.shape).to(BF)
    from fast_trimul_b200.functional import packed_attention
    cu = ends([30, 31, 29])
    want = train(packed_attention, (q, k, v), g, cu, causal=False)
    q[40, 1], k[45], v[50], g[44] = float("nan"), float("inf"), float("nan"), float("inf")
    got = train(packed_attention, (q, k, v), g, cu, causal=False)
    for a, b in zip(got, want):
        assert torch.equal(a[:30], b[:30]) and torch.equal(a[61:], b[61:])


@pytest.mark.parametrize("causal", [False, True])
def test_packed_key_mask(causal):
    lens = [200, 50, 1, 131]
    q, k, v = qkv(sum(lens), sum(lens), 4, 2, 64, BF)
    mask = torch.rand(sum(lens), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) > 0.4
    mask[200:250] = False              # a sequence without any key
    mask[:130] = False                 # a whole tile without one
    cu = ends(lens)
    got = check_packed(q, k, v, cu, cu, causal, mask)
    assert (got[0][200:250] == 0).all() and (got[2][200:250] == 0).all()
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("nan"), float("inf")
    again = check_packed(q, k2, v2, cu, cu, causal, mask)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_packed_scales_and_large_scores():
    lens = [130, 70]
    q, k, v = qkv(200, 200, 2, 2, 64, BF)
    cu = ends(lens)
    check_packed(q, k, v, cu, cu, scale=0.0)          # uniform weights
    check_packed(q, k, v, cu, cu, scale=1.0)          # scores of some tens
    # a row whose maximum keeps growing from tile to tile, past the 2^8 of the lazy rescale
    q, k, v = qkv(500, 500, 2, 2, 64, BF, 3)
    q = q.abs() * 0.1
    k = k.abs() * 0.1 * torch.linspace(0.1, 12, 500, device="cuda")[:, None, None].to(BF)
    check_packed(q, k, v, ends([500]), ends([500]), causal=False, scale=1.0)


def test_packed_layouts():
    from fast_trimul_b200.functional import packed_attention
    r = gen()
    cu = ends([100, 60])
    wide = r(160, 3, 4, 64).to(BF)
    q, k, v = wide.unbind(1)                                          # views of one projection
    assert not q.is_contiguous()
    base = packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(base, packed_attention(q, k, v, cu))
    t = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)      # noqa: E731  heads first
    assert torch.equal(base, packed_attention(t(q), t(k), t(v), cu))
    odd = torch.empty(160 * 4 * 64 + 1, dtype=BF, device="cuda")[1:].view(160, 4, 64)
    odd.copy_(q)                                                      # 2-byte aligned
    assert torch.equal(base, packed_attention(odd, k, v, cu))
    gap = torch.empty(160, 4, 68, dtype=BF, device="cuda")[..., :64]  # strides of no whole vectors
    gap.copy_(k)
    assert torch.equal(base, packed_attention(q, gap, v, cu))
    apart = torch.empty(160, 4, 128, dtype=BF, device="cuda")[..., ::2]
    apart.copy_(v)
    assert torch.equal(base, packed_attention(q, k, apart, cu))
    assert torch.equal(packed_attention(q, k[:, :1], v[:, :1], cu),
                       packed_attention(q, k[:, :1].contiguous(), v[:, :1].contiguous(), cu))
    one = k[:, :1].expand(-1, 4, -1)                                  # a broadcast head
    assert torch.equal(packed_attention(q, one, one, cu), packed_attention(q, one.contiguous(), one.contiguous(), cu))
    assert torch.equal(packed_attention(q, k, v, cu.long()), base)
    grads = train(packed_attention, (q, k, v), r(1, 1, 64).to(BF).expand(160, 4, 64), cu)   # broadcast gradient
    assert all(not x.isnan().any() for x in grads)


def test_packed_arrays_that_point_outside_are_clamped():
    """What a caller's mistake leaves in the device arrays must not touch other memory: the
    kernels clamp to the tensors (guarded here by bytes around the outputs' neighbours)."""
    from fast_trimul_b200.functional import packed_attention
    q, k, v = qkv(100, 100, 2, 2, 64, BF)
    for bad in ([0, 50, 1000], [-5, 50, 100], [0, 80, 40], [90, 20, 2 ** 31 - 1], [-(2 ** 31), 0, 100]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out = train(packed_attention, (q, k, v), torch.ones_like(q), cu)
        check_waits()
        assert out[0].shape == q.shape
    good = ends([50, 50])
    check_packed(q, k, v, good, good)


def test_packed_many_short_sequences():
    lens = [(i * 7) % 13 for i in range(700)]
    cu = ends(lens)
    q, k, v = qkv(sum(lens), sum(lens), 2, 1, 32, BF)
    from fast_trimul_b200.functional import packed_attention
    out = packed_attention(q, k, v, cu)
    a, b = cu[401].item(), cu[431].item()
    part = ends(lens[401:431])
    assert torch.equal(out[a:b], packed_attention(q[a:b], k[a:b], v[a:b], part))
    check_packed(q[a:b], k[a:b], v[a:b], part, part)


@pytest.mark.parametrize("h,hk,lens,klens", [(8, 1, [900], [900]), (16, 1, [700, 90], [300, 900]), (8, 2, [640, 1, 513], [640, 1, 513])],
                         ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_packed_few_key_tiles_split_their_queries(h, hk, lens, klens, causal):
    """Shapes whose key tiles are too few for the GPU: parts of the queries are summed, and rows of
    no sequence stay zero."""
    q, k, v = qkv(sum(lens) + 9, sum(klens) + 13, h, hk, 64, BF)
    k[sum(klens) + 5:], v[:5] = float("nan"), float("inf")
    got = check_packed(q, k, v, ends(lens, 4), ends(klens, 5), causal)
    for g in got[2:]:
        assert (g[:5] == 0).all() and (g[sum(klens) + 5:] == 0).all()


def test_gradients_against_differences():
    """The kernels' gradients along a direction against differences of the 64-bit forward."""
    cu = ends([37])
    q, k, v = qkv(37, 37, 2, 1, 16, HF, 5)
    g = gen(6)(*q.shape).to(HF)
    from fast_trimul_b200.functional import packed_attention
    grads = train(packed_attention, (q, k, v), g, cu)[1:]
    dirs = [gen(10 + i)(*t.shape).double() for i, t in enumerate((q, k, v))]
    h = 1e-4
    f = lambda s: (ref.packed(*(t.double() + s * d for t, d in zip((q, k, v), dirs)), g.double(), cu, cu, True,   # noqa: E731
                              0.25).o * g.double()).sum()
    slope = ((f(h) - f(-h)) / (2 * h)).item()
    mine = sum((a.double() * d).sum() for a, d in zip(grads, dirs)).item()
    size = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs)).item()
    assert abs(slope - mine) < 2 * 2 ** -11 * size      # each term is off by a few half steps at most


@pytest.mark.parametrize("n, d, dtype", [(128, 64, torch.float16), (400, 32, BF), (96, 128, BF)])
def test_gradients_lose_no_more_than_two_roundings(n, d, dtype):
    # dS and the result are each rounded once, independently and by the same relative size, so
    # the error's norm is sqrt(2) = 1.41 times the result's rounding alone; 1.5 leaves 6 % for the
    # spread over a few thousand elements. (rowsum(grad * out) of the rounded output gave 1.55.)
    from fast_trimul_b200.functional import packed_attention
    q, k, v = (t.detach().requires_grad_() for t in qkv(n, n, 4, 4, d, dtype))
    g = gen(9)(n, 4, d).to(dtype)
    got = torch.autograd.grad(packed_attention(q, k, v, ends([n])), (q, k), g)
    x = [t.detach().double().transpose(0, 1).requires_grad_() for t in (q, k, v)]
    s = (x[0] @ x[1].transpose(1, 2)) * d ** -0.5
    s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
    want = torch.autograd.grad(s.softmax(-1) @ x[2], x[:2], g.double().transpose(0, 1))
    check_waits()
    for a, b in zip(got, want):
        b = b.transpose(0, 1)
        assert (a.double() - b).norm() <= 1.5 * (b.to(dtype).double() - b).norm()


def test_only_the_gradients_that_are_asked_for():
    from fast_trimul_b200.functional import packed_attention
    q, k, v = qkv(200, 200, 4, 2, 64, BF)
    cu, g = ends([150, 50]), gen(2)(200, 4, 64).to(BF)
    all_ = train(packed_attention, (q, k, v), g, cu)
    for i in range(3):
        ls = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (one,) = torch.autograd.grad(packed_attention(*ls, cu), ls[i], g)
        assert torch.equal(one, all_[1 + i])


# ----------------------------------------------------------------------------- cached
def check_cached(q, kc, vc, lens, scale=None):
    from fast_trimul_b200.functional import cached_attention
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = cached_attention(q, kc, vc, lt, scale=scale)
    check_waits()
    u = torch.finfo(q.dtype).eps / 2
    B, H, D = q.shape
    group = H // kc.shape[2]
    want, off = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = max(0, min(lens[b], kc.shape[1]))
        if n == 0:
            continue
        keep = torch.ones(1, n, dtype=torch.bool, device="cuda")
        for h in range(H):
            kk, vv = kc[b, :n, h // group].double(), vc[b, :n, h // group].double()
            res, o = ref.head(q[b, h:h + 1].double(), kk, vv, torch.zeros(1, D, dtype=torch.float64, device="cuda"),
                              D ** -0.5 if scale is None else scale, keep, None, u)
            want[b, h], off[b, h] = res[0][0], o[0][0]
    ref.close(out, want, off, "cached")
    assert torch.equal(out, cached_attention(q, kc, vc, lt, scale=scale))
    return out


@pytest.mark.parametrize("lens", [[1], [128], [129], [500], [0], [1, 0, 300, 128, 2], [512] * 9, [3] * 70], ids=str)
@pytest.mark.parametrize("h,hk,d,dtype", [(4, 4, 64, BF), (8, 2, 128, HF), (7, 1, 40, BF)])
def test_cached_lengths(lens, h, hk, d, dtype):
    r = gen(len(lens))
    q = r(len(lens), h, d).to(dtype)
    kc, vc = r(len(lens), 512, hk, d).to(dtype), r(len(lens), 512, hk, d).to(dtype)
    for b, n in enumerate(lens):          # behind the length: anything
        kc[b, n:], vc[b, n:] = float("nan"), float("inf")
    check_cached(q, kc, vc, lens)


@pytest.mark.parametrize("batch,length", [(1, 40000), (2, 9001), (3, 20000)])
def test_cached_long(batch, length):
    r = gen(batch)
    q = r(batch, 8, 64).to(BF)
    kc, vc = r(batch, length, 2, 64).to(BF), r(batch, length, 2, 64).to(BF)
    check_cached(q, kc, vc, [length - 37 * b for b in range(batch)])


def test_cached_layouts_and_clamped_lengths():
    from fast_trimul_b200.functional import cached_attention
    r = gen()
    q, kc, vc = r(3, 8, 64).to(BF), r(3, 300, 2, 64).to(BF), r(3, 300, 2, 64).to(BF)
    lens = [300, 17, 130]
    base = check_cached(q, kc, vc, lens)
    heads_first = kc.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack([kc, vc], 2)                       # (B, L, 2, heads, dim)
    lt = torch.tensor(lens, device="cuda")
    assert torch.equal(base, cached_attention(q, heads_first, vc, lt))
    assert torch.equal(base, cached_attention(q, both[:, :, 0], both[:, :, 1], lt))
    assert torch.equal(base, cached_attention(q.transpose(0, 1).contiguous().transpose(0, 1), kc, vc, lt))
    over = torch.tensor([9999, 17, 130], device="cuda")
    assert torch.equal(base, cached_attention(q, kc, vc, over))
    under = cached_attention(q, kc, vc, torch.tensor([-4, 17, -2 ** 31], dtype=torch.int64, device="cuda"))
    check_waits()
    assert (under[[0, 2]] == 0).all() and torch.equal(under[1], base[1])


def test_cached_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the last sequence starts behind 4 GB."""
    cap = 1 << 20
    kc = torch.empty(2, cap, 9, 128, dtype=BF, device="cuda")
    vc = torch.empty(2, cap, 9, 128, dtype=BF, device="cuda")
    r = gen(1)
    q = r(2, 9, 128).to(BF)
    for t in (kc, vc):
        t[0, :200] = r(200, 9, 128).to(BF)
        t[1, :333] = r(333, 9, 128).to(BF)
    check_cached(q, kc, vc, [200, 333])
    kc[1, -128:], vc[1, -128:] = 0, 1
    from fast_trimul_b200.functional import cached_attention
    out = cached_attention(q[1:], kc[1:, -128:], vc[1:, -128:], torch.tensor([128], device="cuda"))
    assert torch.equal(out, torch.ones_like(out))


def test_packed_offsets_past_32_bits():
    from fast_trimul_b200.functional import packed_attention
    rows = (1 << 31) // 1024 + 500
    big = torch.zeros(rows, 8, 128, dtype=BF, device="cuda")
    r = gen(2)
    big[-300:] = r(300, 8, 128).to(BF)
    cu = ends([300], rows - 300)
    out = packed_attention(big, big, big, cu)
    small = big[-300:].clone()
    assert torch.equal(out[-300:], packed_attention(small, small, small, ends([300])))
    assert (out[:1000] == 0).all()


def test_a_prompt_token_by_token():
    """A prompt at once, and the same tokens one by one over a growing cache, in a captured graph
    that replays with new lengths."""
    from fast_trimul_b200.functional import cached_attention, packed_attention
    n, h, hk, d = 200, 8, 2, 64
    q, k, v = qkv(n, n, h, hk, d, HF, 7)
    whole = packed_attention(q, k, v, ends([n]))
    kc, vc = torch.zeros(1, 256, hk, d, dtype=HF, device="cuda"), torch.zeros(1, 256, hk, d, dtype=HF, device="cuda")
    qin, lens = q[:1].clone(), torch.ones(1, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        cached_attention(qin, kc, vc, lens)
        with torch.cuda.graph(graph, stream=s):
            out = cached_attention(qin, kc, vc, lens)
    torch.cuda.current_stream().wait_stream(s)
    for t in range(n):
        kc[0, t], vc[0, t] = k[t], v[t]
        qin.copy_(q[t:t + 1])
        lens.fill_(t + 1)
        graph.replay()
        # each side is off by two half steps at most (its weights' and its last rounding)
        assert (out.float() - whole[t:t + 1].float()).abs().max() < 4 * 2 ** -11 * v[:t + 1].abs().max().float()
    check_waits()


# ------------------------------------------------------------------------------- pair
def check_pair(q, k, v, bias, mask=None, scale=None):
    from fast_trimul_b200.functional import pair_attention
    g = gen(8)(*q.shape).to(q.dtype)
    leaves = (q, k, v) if bias is None else (q, k, v, bias)
    f = (lambda a, b, c, m: pair_attention(a, b, c, None, m, scale=scale)) if bias is None else \
        (lambda a, b, c, d, m: pair_attention(a, b, c, d, m, scale=scale))
    got = train(f, leaves, g, mask)
    check_waits()
    w = ref.pair(q, k, v, g, bias, mask, q.shape[-1] ** -0.5 if scale is None else scale)
    want = [(w.o, w.eo), (w.dq, w.edq), (w.dk, w.edk), (w.dv, w.edv)]
    if bias is not None:
        want.append((w.db, w.edb))
    for name, a, (x, off) in zip(("o", "dq", "dk", "dv", "dbias")[:len(want)], got, want, strict=True):
        ref.close(a, x, off, name)
    again = train(f, leaves, g, mask)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


def pair_inputs(b, r, n, h, d, dtype, seed=0, biases=None):
    x = gen(seed)
    q, k, v = x(b, r, n, 3, h, d).to(dtype).unbind(3)
    return q, k, v, x(biases or b, h, n, n).to(dtype)


@pytest.mark.parametrize("n", [1, 2, 31, 33, 128, 129, 250, 301])
@pytest.mark.parametrize("h,d,dtype", [(4, 24, BF), (2, 64, HF), (2, 96, BF)])
def test_pair_a_bias_of_one_row_alone(n, h, d, dtype):
    # its gradient is dS itself; masked keys, whatever they hold, and a row without any
    q, k, v, bias = pair_inputs(2, 1, n, h, d, dtype, n)
    mask = gen(n)(2, 1, n) > 0
    mask[1] = False
    bad = torch.where(mask[..., None, None], v, torch.full_like(v, float("nan")))
    check_pair(q, k, v, bias)
    got = check_pair(q, k, bad, bias, mask)
    assert torch.equal(got[4][1], torch.zeros_like(got[4][1]))
    # the bias' gradient alone (from another kernel: within a rounding), and all but it
    from fast_trimul_b200.functional import pair_attention
    b = bias.clone().requires_grad_()
    g = gen(8)(*q.shape).to(dtype)
    (alone,) = torch.autograd.grad(pair_attention(q, k, v, b), b, g)
    all_of = train(pair_attention, (q, k, v, bias), g)
    assert (alone.float() - all_of[4].float()).norm() <= 1e-2 * all_of[4].float().norm() + 1e-6
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    for a, c in zip(torch.autograd.grad(pair_attention(*x, bias), x, g), all_of[1:4]):
        assert torch.equal(a, c)


@pytest.mark.parametrize("n", [1, 7, 8, 64, 127, 128, 129, 200])
@pytest.mark.parametrize("h,d,dtype", [(4, 32, BF), (2, 64, HF), (3, 24, BF), (2, 128, BF)])
def test_pair_lengths(n, h, d, dtype):
    check_pair(*pair_inputs(1, 3, n, h, d, dtype, n))


@pytest.mark.parametrize("b,r", [(1, 1), (2, 1), (2, 5), (1, 40)])
@pytest.mark.parametrize("shared", [False, True])
def test_pair_rows_share_the_bias(b, r, shared):
    q, k, v, bias = pair_inputs(b, r, 70, 4, 32, BF, r, biases=1 if shared else None)
    mask = torch.rand(b, r, 70, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) > 0.3
    mask[0, 0] = False
    got = check_pair(q, k, v, bias, mask)
    assert (got[0][0, 0] == 0).all()


def test_pair_without_a_bias():
    q, k, v, _ = pair_inputs(2, 3, 90, 2, 32, BF)
    check_pair(q, k, v, None)
    mask = torch.ones(2, 3, 90, device="cuda")
    mask[:, :, 60:] = 0
    check_pair(q, k, v, None, mask)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_pair_bias_of_the_lowest_value_and_of_infinity(dtype):
    """A bias used as a mask: the type's lowest value everywhere leaves the row's softmax over
    the (equal) lowest scores, -infinity leaves nothing."""
    q, k, v, bias = pair_inputs(1, 2, 150, 2, 32, dtype, 3)
    low = torch.finfo(dtype).min
    bias[:, :, :, 100:] = low
    bias[:, :, 5] = low
    check_pair(q, k, v, bias)
    bias[:, :, 6] = -float("inf")
    bias[:, 1, 7:, :50] = -float("inf")
    got = check_pair(q, k, v, bias)
    assert (got[0][:, :, 6] == 0).all() and (got[4][:, :, 6] == 0).all()
    # (not through check_pair: a key that -infinity hides is still read, so it stays finite)


def test_pair_masked_keys_may_hold_anything():
    q, k, v, bias = pair_inputs(1, 4, 140, 2, 32, BF, 4)
    mask = torch.rand(1, 4, 140, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) > 0.3
    mask[0, 2] = False
    a = check_pair(q, k, v, bias, mask)
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("inf"), float("nan")
    b = check_pair(q, k2, v2, bias, mask)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_pair_bias_layouts():
    from fast_trimul_b200.functional import pair_attention
    q, k, v, bias = pair_inputs(2, 3, 72, 4, 32, BF, 5)
    base = pair_attention(q, k, v, bias)
    last = bias.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)        # heads last, as a linear gives it
    assert torch.equal(base, pair_attention(q, k, v, last))
    assert torch.equal(pair_attention(q, k, v, bias[:1]), pair_attention(q, k, v, bias[:1].expand(2, -1, -1, -1)))
    t = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)            # noqa: E731
    q2, k2, v2, b2 = pair_inputs(1, 72, 72, 4, 32, BF, 6)
    assert torch.equal(pair_attention(q2, k2, v2, b2), pair_attention(t(q2), t(k2), t(v2), b2))
    odd = pair_inputs(1, 2, 75, 2, 16, BF, 7)
    out = train(pair_attention, odd, torch.ones_like(odd[0]))
    assert out[4].shape == (1, 2, 75, 75) and out[4].is_contiguous()


# ------------------------------------------------------- streams, graphs, refusals, failure
def test_two_streams_at_once():
    from fast_trimul_b200.functional import packed_attention
    sets = [(qkv(900, 900, 4, 2, 64, BF, s), ends([500, 400])) for s in range(2)]
    g = gen(1)(900, 4, 64).to(BF)
    want = [train(packed_attention, x, g, cu) for x, cu in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = train(packed_attention, sets[i][0], g, sets[i][1])
    torch.cuda.synchronize()
    check_waits()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", ["packed", "pair"])
def test_training_step_in_a_graph(kind):
    from fast_trimul_b200.functional import packed_attention, pair_attention
    if kind == "packed":
        leaves, rest, f = qkv(300, 300, 4, 2, 64, BF), (ends([200, 100]),), packed_attention
    else:
        leaves, rest, f = pair_inputs(1, 6, 100, 2, 32, BF), (), pair_attention
    g = gen(1)(*leaves[0].shape).to(BF)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    static = [t.detach().clone().contiguous().requires_grad_() for t in leaves]
    with torch.cuda.stream(s):
        torch.autograd.grad(f(*static, *rest), static, g)
        with torch.cuda.graph(graph, stream=s):
            out = f(*static, *rest)
            grads = torch.autograd.grad(out, static, g)
    torch.cuda.current_stream().wait_stream(s)
    for scale in (1.0, 0.5):
        with torch.no_grad():
            for a, b in zip(static, leaves):
                a.copy_(b * scale)
        graph.replay()
        want = train(f, [b * scale for b in leaves], g, *rest)
        assert torch.equal(out.detach(), want[0])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[1:]))
    check_waits()


def test_two_graphs_do_not_share_scratch():
    from fast_trimul_b200.functional import cached_attention
    r = gen(3)
    sets = [(r(2, 8, 64).to(BF), r(2, 4000, 2, 64).to(BF), r(2, 4000, 2, 64).to(BF)) for _ in range(2)]
    lens = torch.tensor([4000, 3500], dtype=torch.int32, device="cuda")
    want = [cached_attention(*x, lens) for x in sets]
    graphs, outs, streams = [], [], []
    for x in sets:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
            outs.append(cached_attention(*x, lens))
        graphs.append(graph)
        streams.append(s)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    check_waits()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refusals():
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import cached_attention, packed_attention, pair_attention
    q, k, v = qkv(40, 40, 4, 2, 64, BF)
    cu = ends([40])
    for bad in (lambda: packed_attention(q.float(), k.float(), v.float(), cu),
                lambda: packed_attention(q[..., :60], k[..., :60], v[..., :60], cu),
                lambda: packed_attention(torch.zeros(4, 2, 136, dtype=BF, device="cuda"), *[torch.zeros(4, 2, 136, dtype=BF, device="cuda")] * 2, ends([4])),
                lambda: packed_attention(torch.zeros(4, 129, 8, dtype=BF, device="cuda"), *[torch.zeros(4, 1, 8, dtype=BF, device="cuda")] * 2, ends([4])),
                lambda: cached_attention(q[:1].float(), k[None].float(), v[None].float(), cu[1:])):
        with pytest.raises(_lib.NativeDeclined):
            bad()
    for bad in (lambda: packed_attention(q, k.half(), v.half(), cu),
                lambda: packed_attention(q, k, v, cu.cpu()),
                lambda: packed_attention(q, k.cpu(), v.cpu(), cu),
                lambda: pair_attention(q[None, None], q[None, None], q[None, None], torch.zeros(1, 4, 40, 40, device="cuda")),
                lambda: cached_attention(q[:1], k[None], v[None], cu[1:].cpu())):
        with pytest.raises(ValueError):
            bad()


def test_nothing_to_attend_to_gives_zeros_whatever_the_inputs_hold():
    from fast_trimul_b200.functional import packed_attention
    bad = torch.full((3, 2, 8), float("nan"), dtype=BF, device="cuda", requires_grad=True)
    for out in (packed_attention(bad, bad, bad, ends([])),
                packed_attention(bad, bad[:0], bad[:0], ends([3]), ends([0]))):
        assert torch.equal(out, torch.zeros_like(bad))
        (grad,) = torch.autograd.grad(out.sum(), bad)
        assert torch.equal(grad, torch.zeros_like(bad))


def test_the_first_call_of_a_gpu_is_not_captured():
    # its error word would be zeroed by the graph's replay alone
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.ops.attention import AttentionErrorWord
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(_lib.NativeDeclined):
            AttentionErrorWord(torch.device("cuda", 0))


@pytest.mark.parametrize("kind", ["packed", "pair", "layer_norm"])
def test_second_derivatives_are_refused(kind):
    # a gradient taken with create_graph is right, and differentiating it raises
    from fast_trimul_b200.functional import layer_norm, packed_attention, pair_attention
    if kind == "packed":
        leaves, f = qkv(40, 40, 4, 2, 64, BF), lambda *x: packed_attention(*x, ends([40]))
    elif kind == "pair":
        leaves, f = pair_inputs(1, 2, 24, 2, 32, BF), pair_attention
    else:
        r = gen(4)
        leaves, f = [r(5, 64).to(BF), r(64), r(64)], layer_norm
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    g = gen(1)(*leaves[0].shape).to(BF)
    want = torch.autograd.grad(f(*leaves), leaves, g)
    got = torch.autograd.grad(f(*leaves), leaves, g, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(sum(x.float().sum() for x in got), leaves)
    got = torch.autograd.grad(f(*leaves), leaves, g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        sum(x.float().sum() for x in got).backward()


@pytest.mark.parametrize("kind", ["packed", "pair", "layer_norm"])
def test_a_captured_backward_of_leaves_that_an_eager_graph_holds_is_refused(kind):
    from fast_trimul_b200.functional import layer_norm, packed_attention, pair_attention
    if kind == "packed":
        leaves, f = qkv(40, 40, 4, 2, 64, BF), lambda *x: packed_attention(*x, cu)
        cu = ends([40])
    elif kind == "pair":
        leaves, f = pair_inputs(1, 2, 24, 2, 32, BF), pair_attention
    else:
        r = gen(4)
        leaves, f = [r(5, 64).to(BF), r(64), r(64)], layer_norm
    leaves = [t.detach().clone().contiguous().requires_grad_() for t in leaves]
    g = gen(1)(*leaves[0].shape).to(BF)
    want = torch.autograd.grad(f(*leaves), leaves, g)
    eager = f(*leaves)                      # lives over the capture
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            out = f(*leaves)                # a forward may be captured
            with pytest.raises(RuntimeError, match="cannot be captured"):
                torch.autograd.grad(out, leaves, g)
    torch.cuda.current_stream().wait_stream(s)
    graph.replay()
    assert torch.equal(out, eager)
    got = torch.autograd.grad(eager, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_waits()


def test_a_withheld_tile_is_reported_and_the_next_call_is_right(monkeypatch):
    """A bounded wait that expires (a test switch withholds one K tile) ends the kernel, and the
    next call raises; nothing faults, and afterwards results are right."""
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import packed_attention
    q, k, v = qkv(64, 64, 2, 2, 64, BF)
    cu = ends([64])
    want = packed_attention(q, k, v, cu)
    monkeypatch.setenv("FTM_TEST_STALL", "attention")
    packed_attention(q, k, v, cu)
    monkeypatch.delenv("FTM_TEST_STALL")
    torch.cuda.synchronize()
    with pytest.raises(_lib.NativeKernelError):
        packed_attention(q, k, v, cu)
    assert torch.equal(packed_attention(q, k, v, cu), want)
    check_waits()


@pytest.mark.parametrize("kernel", ["dq", "dkv"])
@pytest.mark.parametrize("bias", [False, True])
def test_a_withheld_tile_of_a_backward_is_reported(monkeypatch, kernel, bias):
    """One block's first tile is withheld while the others work: its waits expire, its warps leave
    together, and the others see the error at a wait of theirs, whichever that is."""
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import pair_attention
    x = [t.detach().requires_grad_() for t in pair_inputs(1, 60, 200, 4, 32, BF)]
    if not bias:
        x = x[:3] + [None]
    g = gen(2)(1, 60, 200, 4, 32).to(BF)
    grads = lambda: torch.autograd.grad(pair_attention(*x), [t for t in x if t is not None], g)   # noqa: E731
    want = grads()
    monkeypatch.setenv("FTM_TEST_STALL", "attention_" + kernel)
    grads()
    monkeypatch.delenv("FTM_TEST_STALL")
    torch.cuda.synchronize()
    with pytest.raises(_lib.NativeKernelError):
        grads()
    assert all(torch.equal(a, b) for a, b in zip(grads(), want))
    check_waits()


@pytest.mark.parametrize("seqs, nq, nk, h, hk, d, causal, bias", [
    (3, 50, 200, 4, 2, 64, 1, 0), (2, 200, 50, 6, 2, 128, 1, 0), (2, 129, 300, 4, 4, 32, 0, 1),
    (4, 1, 130, 2, 2, 24, 0, 2), (2, 300, 129, 2, 2, 128, 0, 1), (6, 70, 90, 2, 2, 16, 0, 3)])
def test_the_uniform_form_of_the_c_entries(seqs, nq, nk, h, hk, d, causal, bias):
    """Sequences of one length with other numbers of keys than queries; `bias` rows share one."""
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.ops.attention import attention_error_word
    lib, e = _lib.load(), attention_error_word()
    q, k, v = qkv(seqs * nq, seqs * nk, h, hk, d, BF, seqs)
    q, k, v = (t.detach().contiguous() for t in (q, k, v))
    g = gen(3)(seqs * nq, h, d).to(BF)
    wide, n = (nk + 7) // 8 * 8, seqs // bias if bias else 0
    b = gen(4)(n, h, nq, wide).to(BF) if bias else None
    new = lambda *s: torch.full(s, float("nan"), dtype=BF, device="cuda")   # noqa: E731
    out, low, dq, dk, dv = new(*q.shape), new(*q.shape), new(*q.shape), new(*k.shape), new(*k.shape)
    db, st = new(n, h, nq, nk), torch.empty(seqs * nq, h, 2, device="cuda")
    p = _lib.Attention(dtype=_lib.BF16, heads=h, kv_heads=hk, head_dim=d, causal=causal, scale=d ** -0.5,
                       sequences=seqs, q_len=nq, kv_len=nk, q_rows=seqs * nq, kv_rows=seqs * nk, q=q.data_ptr(),
                       q_row_stride=h * d, q_head_stride=d, k=k.data_ptr(), k_row_stride=hk * d, k_head_stride=d,
                       v=v.data_ptr(), v_row_stride=hk * d, v_head_stride=d, out=out.data_ptr(), stats=st.data_ptr(),
                       out_low=low.data_ptr())
    if bias:
        p.bias, p.bias_seqs, p.bias_row_stride = b.data_ptr(), bias, wide
        p.bias_head_stride, p.bias_batch_stride = nq * wide, h * nq * wide
    s = torch.cuda.current_stream().cuda_stream
    assert lib.ftm_attention_workspace_bytes(p, 1) == 0
    size = lib.ftm_attention_bwd_workspace_bytes(p, 1 if bias else 0)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert lib.ftm_attention_fwd(p, 1, None, 0, e.ptr, e.host_ptr, s) == _lib.OK
    assert lib.ftm_attention_bwd(p, g.data_ptr(), h * d, d, None, 0, ws.data_ptr(), size, dq.data_ptr(), dk.data_ptr(),
                                 dv.data_ptr(), db.data_ptr() if bias else None, e.ptr, e.host_ptr, s) == _lib.OK
    check_waits()
    w = ref.Sums(q, k, db if bias else None)
    keep = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
    if causal:
        keep = keep.tril(nk - nq)
    x = [t.double() for t in (q, k, v, g)]
    for i in range(seqs):
        a, c = slice(i * nq, (i + 1) * nq), slice(i * nk, (i + 1) * nk)
        for j in range(h):
            jk = j // (h // hk)
            m = b[i // bias, j, :, :nk].double() if bias else None
            res, off = ref.head(x[0][a, j], x[1][c, jk], x[2][c, jk], x[3][a, j], d ** -0.5, keep, m, 2.0 ** -8)
            w.o[a, j], w.dq[a, j], w.eo[a, j], w.edq[a, j] = res[0], res[1], off[0], off[1]
            w.dk[c, jk] += res[2]
            w.dv[c, jk] += res[3]
            w.edk[c, jk] += off[2]
            w.edv[c, jk] += off[3]
            if bias:
                w.db[i // bias, j] += res[4]
                w.edb[i // bias, j] += off[4]
    for name, got, want, off in (("o", out, w.o, w.eo), ("dq", dq, w.dq, w.edq), ("dk", dk, w.dk, w.edk),
                                 ("dv", dv, w.dv, w.edv), *((("dbias", db, w.db, w.edb),) if bias else ())):
        ref.close(got, want, off, name)


# ----------------------------------------------------------------- the operators together
def test_attention_block_trains_like_the_formula():
    """Norm, projections, packed attention and residual together, as a model uses them, against
    the same block in fp32 on the CPU: outputs, and gradients of every parameter."""
    from fast_trimul_b200 import FastLayerNorm
    from fast_trimul_b200.functional import packed_attention
    torch.manual_seed(0)
    c, h, hk, d = 64, 4, 2, 16
    norm, qkv_, out_ = FastLayerNorm(c), torch.nn.Linear(c, (h + 2 * hk) * d), torch.nn.Linear(h * d, c)
    mods = torch.nn.ModuleList([norm, qkv_, out_]).to(BF)
    x0 = torch.randn(150, c).to(BF)
    lens = [100, 1, 49]

    def run(device, dtype):
        ms = torch.nn.ModuleList([FastLayerNorm(c), torch.nn.Linear(c, (h + 2 * hk) * d), torch.nn.Linear(h * d, c)])
        ms.load_state_dict(mods.state_dict())
        ms.to(device=device, dtype=dtype)
        x = x0.to(device=device, dtype=dtype).requires_grad_()
        y = ms[1](ms[0](x))
        q, k, v = (t.unflatten(-1, (-1, d)) for t in y.split([h * d, hk * d, hk * d], -1))
        o = packed_attention(q, k, v, ends(lens).to(device))
        z = x + ms[2](o.flatten(1))
        z.float().square().mean().backward()
        return [z.detach().float().cpu(), x.grad.float().cpu(), *[p.grad.float().cpu() for p in ms.parameters()]]

    for a, b in zip(run("cuda", BF), run("cpu", torch.float32)):
        # six bf16 roundings in a row at most, each 2^-9 of a root mean square
        assert (a - b).norm() <= 6 * 2 ** -8 * b.norm() + 1e-6


@pytest.mark.parametrize("masked", [False, True])
def test_fused_trunk_equals_the_plain_one(masked):
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.pairformer import PairFormerTrunk
    torch.manual_seed(0)
    n, blocks = 72, 2
    a = PairFormerTrunk(blocks, 384, 128).cuda().to(BF).eval()
    b = PairFormerTrunk(blocks, 384, 128, fused=True).cuda().to(BF).eval()
    b.load_state_dict(a.state_dict())
    r = gen(3)
    s, z = r(1, n, 384).to(BF), r(1, n, n, 128).to(BF)
    mask = torch.ones(1, n, n, device="cuda", dtype=BF)
    m = 60 if masked else n
    mask[:, m:] = 0
    mask[:, :, m:] = 0
    before = _lib.stats["calls"]
    with torch.no_grad():
        s1, z1 = a(s, z, mask)
        s2, z2 = b(s, z, mask)
    check_waits()
    assert _lib.stats["calls"] >= before + blocks * 8
    x, y = z1[:, :m, :m].float(), z2[:, :m, :m].float()
    assert ((x - y).abs().mean() / x.abs().mean()).item() < 2e-2     # both trunks run in bf16
    if not masked:
        assert ((s1.float() - s2.float()).abs().mean() / s1.float().abs().mean()).item() < 2e-2


def test_fused_trunk_trains():
    from fast_trimul_b200.pairformer import PairFormerTrunk
    torch.manual_seed(1)
    ref_trunk = PairFormerTrunk(1, 384, 128)
    s, z = torch.randn(1, 40, 384), torch.randn(1, 40, 40, 128)
    grads = []
    for fused, device, dtype in ((False, "cpu", torch.float32), (True, "cuda", BF)):
        t = PairFormerTrunk(1, 384, 128, fused=fused)
        t.load_state_dict(ref_trunk.state_dict())
        t.to(device=device, dtype=dtype)
        zz = z.clone().to(device=device, dtype=dtype).requires_grad_()
        a, b = t(s.to(device=device, dtype=dtype), zz)
        (a.float().square().mean() + b.float().square().mean()).backward()
        grads.append({"z": zz.grad.float().cpu(), **{k: p.grad.float().cpu() for k, p in t.named_parameters()}})
    for k, want in grads[0].items():
        # a chain of some 30 bf16 roundings of 2^-9 each; small gradients ride on large terms
        assert (grads[1][k] - want).norm() <= 0.1 * want.norm() + 1e-5, k


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 250, 1001])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_pad_rows_copies_every_element(cols, shift):
    """Rows at every alignment, the last one ending with its buffer."""
    from fast_trimul_b200 import _lib
    lib = _lib.load()
    rows, wide = 13, (cols + 7) // 8 * 8
    buf = torch.arange(rows * cols + shift, device="cuda").to(torch.int16)
    src = buf[shift:].view(rows, cols)
    dst = torch.full((rows, wide), -1, dtype=torch.int16, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    assert lib.ftm_pad_rows(src.data_ptr(), cols, dst.data_ptr(), wide, rows, cols, s) == _lib.OK
    assert torch.equal(dst[:, :cols], src)
    assert lib.ftm_pad_rows(src.data_ptr(), cols - 1, dst.data_ptr(), wide, rows, cols, s) == _lib.BAD_SHAPE
    assert lib.ftm_pad_rows(src.data_ptr(), cols, dst.data_ptr(), wide + 1, rows, cols, s) == _lib.BAD_SHAPE
