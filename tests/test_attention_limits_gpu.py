"""Attention on the GPU where numbers get small, large or many: against 64 bits."""

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


def train(f, leaves, g, *a, **k):
    from fast_trimul_b200.ops.attention import attention_error_word
    ls = [t.detach().requires_grad_() for t in leaves]
    out = f(*ls, *a, **k)
    got = [out.detach(), *torch.autograd.grad(out, ls, g)]
    attention_error_word().check()
    return got


# ------------------------------------------------------------------- many keys, many heads
def test_keys_times_the_heads_of_a_group_pass_32_bits():
    """One query of 128 heads on one, 17 000 000 keys in front of it: 128 times the distance of
    the first key is more than 2^31. (Bounds: the weights' sum of 17e6 terms runs over 133 000
    tiles; each addition is off by half a step of a sum of up to 2^25, 1 in 2^24 of it, with either
    sign: 2^-24 sqrt(133 000) < 2^-15, within the 2^-14 of the reference.)"""
    from fast_trimul_b200.functional import packed_attention
    n, h, d = 17_000_000, 128, 8
    r = gen(1)
    q, k, v, g = r(1, h, d).to(BF), r(n, 1, d).to(BF), r(n, 1, d).to(BF), r(1, h, d).to(BF)
    cu_q, cu_k = ends([1]), ends([n])
    got = train(packed_attention, (q, k, v), g, cu_q, cu_k)
    assert (got[2][:1000] != 0).any(1).all() and (got[3][:1000] != 0).any(1).all()
    w = ref.packed(q, k, v, g, cu_q, cu_k, True, d ** -0.5)
    for name, a, want, off in zip(("o", "dq", "dk", "dv"), got, (w.o, w.dq, w.dk, w.dv),
                                  (w.eo, w.edq, w.edk, w.edv)):
        ref.close(a, want, off, name)


# ------------------------------------------------------------------- gradients of any size in fp16
def exact(q, k, v, g, bias=None, keep=None, scale=None):
    """dq, dk, dv (and dbias) in 64 bits; q, k, v, g (..., length, dim), grouped heads repeated."""
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    b = None if bias is None else bias.detach().double().requires_grad_()
    s = x[0] @ x[1].transpose(-1, -2) * (q.shape[-1] ** -0.5 if scale is None else scale)
    if b is not None:
        s = s + b
    if keep is not None:
        s = s.masked_fill(~keep, -torch.inf)
    return torch.autograd.grad(s.softmax(-1) @ x[2], x if b is None else [*x, b], g.double())


def roundings(got, want):
    """The error's norm over that of the result's own rounding (subnormal steps included)."""
    assert not got.isnan().any() and not got.isinf().any()
    return ((got.double() - want).norm() / (want.to(got.dtype).double() - want).norm()).item()


# dS, or the weights, and the result are each rounded once, independently and by the same relative
# size: sqrt(2) = 1.41 times the result's rounding alone, and nearer to 1 where the result itself is
# subnormal. 1.5 leaves 6 % for the spread over the elements.
MOST = 1.5


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e3])
@pytest.mark.parametrize("d", [64, 128])
def test_fp16_gradients_of_any_size(size, d):
    from fast_trimul_b200.functional import packed_attention
    nq, nk, h = 256, 4096, 2
    r = gen(2)
    q, k, v, g = r(nq, h, d).to(HF), r(nk, h, d).to(HF), r(nk, h, d).to(HF), (size * r(nq, h, d)).to(HF)
    got = train(packed_attention, (q, k, v), g, ends([nq]), ends([nk]), causal=False)
    want = exact(*(t.transpose(0, 1) for t in (q, k, v, g)))
    for name, a, b in zip(("dq", "dk", "dv"), got[1:], want):
        assert roundings(a, b.transpose(0, 1)) <= MOST, name


def test_fp16_weights_of_many_keys():
    """Weights below fp16's normal numbers: 2^-15 on average."""
    from fast_trimul_b200.functional import packed_attention
    nq, nk, h, d = 128, 32768, 1, 64
    r = gen(3)
    q, k, v, g = r(nq, h, d).to(HF), r(nk, h, d).to(HF), r(nk, h, d).to(HF), r(nq, h, d).to(HF)
    got = train(packed_attention, (q, k, v), g, ends([nq]), ends([nk]), causal=False)
    want = exact(*(t.transpose(0, 1) for t in (q, k, v, g)))
    for name, a, b in zip(("dq", "dk", "dv"), got[1:], want):
        assert roundings(a, b.transpose(0, 1)) <= MOST, name


def test_fp16_gradients_of_a_scaled_loss_do_not_overflow():
    """dS far above 65504 between operands and results that fp16 holds."""
    from fast_trimul_b200.functional import packed_attention
    nq, nk, h, d = 64, 4, 2, 64
    r = gen(4)
    q, k = (0.01 * r(nq, h, d)).to(HF), (0.01 * r(nk, h, d)).to(HF)
    v, g = (10 * r(nk, h, d)).to(HF), (4000 * r(nq, h, d)).to(HF)
    got = train(packed_attention, (q, k, v), g, ends([nq]), ends([nk]), causal=False)
    want = exact(*(t.transpose(0, 1) for t in (q, k, v, g)))
    for name, a, b in zip(("dq", "dk", "dv"), got[1:], want):
        assert roundings(a, b.transpose(0, 1)) <= MOST, name


def test_fp16_sequences_whose_gradients_differ_in_size():
    from fast_trimul_b200.functional import packed_attention
    n, h, d = 1024, 2, 64
    r = gen(5)
    q, k, v, g = (r(2 * n, h, d).to(HF) for _ in range(4))
    g[n:] *= 1e-3
    got = train(packed_attention, (q, k, v), g, ends([n, n]))
    keep = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    for at in (slice(0, n), slice(n, 2 * n)):
        want = exact(*(t[at].transpose(0, 1) for t in (q, k, v, g)), keep=keep)
        for name, a, b in zip(("dq", "dk", "dv"), got[1:], want):
            assert roundings(a[at], b.transpose(0, 1)) <= MOST, (name, at)


@pytest.mark.parametrize("r, n, d", [(1, 500, 24), (6, 300, 32), (1, 300, 96), (5, 200, 128)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 300.0])
def test_fp16_gradients_of_any_size_with_a_bias(r, n, d, size):
    # the bias' gradient is rounded once more at most (one row alone: dS and its step down)
    from fast_trimul_b200.functional import pair_attention
    x = gen(6)
    q, k, v = x(1, r, n, 3, 2, d).to(HF).unbind(3)
    bias, g = x(1, 2, n, n).to(HF), (size * x(1, r, n, 2, d)).to(HF)
    got = train(pair_attention, (q, k, v, bias), g)
    want = exact(*(t.transpose(2, 3) for t in (q, k, v, g)), bias=bias.unsqueeze(1))
    for name, a, b in zip(("dq", "dk", "dv"), got[1:], want):
        assert roundings(a, b.transpose(2, 3)) <= MOST, name
    assert roundings(got[4], want[3].squeeze(1)) <= MOST, "dbias"


def test_fp16_rows_that_do_not_count_change_nothing():
    """Masked keys, and rows of no sequence, may hold anything: the same bits."""
    from fast_trimul_b200.functional import packed_attention
    lens, h, d = [200, 131], 2, 64
    n = sum(lens)
    r = gen(7)
    q, k, v, g = (r(n + 20, h, d).to(HF) for _ in range(4))
    g *= 1e-3
    mask = torch.rand(n + 20, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) > 0.3
    cu = ends(lens, 10)
    want = train(packed_attention, (q, k, v), g, cu, key_mask=mask)
    for bad in (float("nan"), float("inf"), 65504.0):
        k2, v2, q2, g2 = k.clone(), v.clone(), q.clone(), g.clone()
        for t in (k2, v2, q2, g2):
            t[:10], t[n + 10:] = bad, bad
        k2[~mask], v2[~mask] = bad, bad
        got = train(packed_attention, (q2, k2, v2), g2, cu, key_mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# -------------------------------------------------------------------- derivatives that are not formed
def operators():
    """Each operator with inputs, for the calls below: name, call, tensors."""
    from fast_trimul_b200.functional import cached_attention, layer_norm, packed_attention, pair_attention
    r = gen(8)
    t = lambda *s: r(*s).to(BF)   # noqa: E731
    lens = torch.tensor([5, 3], dtype=torch.int32, device="cuda")
    return [("layer_norm", layer_norm, [t(5, 64), r(64), r(64)]),
            ("layer_norm, copied", lambda x, w, b: layer_norm(x.transpose(0, 1), w, b), [t(64, 5), r(64), r(64)]),
            ("packed", lambda *x: packed_attention(*x, ends([40])), [t(40, 2, 32) for _ in range(3)]),
            ("pair", pair_attention, [t(1, 2, 24, 2, 32) for _ in range(3)] + [t(1, 2, 24, 24)]),
            ("cached", lambda *x: cached_attention(*x, lens), [t(2, 4, 32), t(2, 9, 2, 32), t(2, 9, 2, 32)])]


@pytest.mark.parametrize("op", range(5))
def test_forward_mode_derivatives_are_refused(op):
    # a result without a tangent would be read as a derivative of zero
    import torch.autograd.forward_ad as fwd
    name, f, inputs = operators()[op]
    for i in range(len(inputs)):
        with fwd.dual_level():
            x = list(inputs)
            x[i] = fwd.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*x)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                f(*x)
            if name != "cached":
                y = [t.detach().clone().requires_grad_() for t in inputs]
                y[i] = fwd.make_dual(y[i], torch.ones_like(y[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*y)
        f(*inputs)                   # and without the tangent it runs
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, tuple(inputs), tuple(torch.ones_like(t) for t in inputs))


@pytest.mark.parametrize("op", range(4))
def test_a_gradient_with_a_tangent_is_refused(op):
    import torch.autograd.forward_ad as fwd
    _, f, inputs = operators()[op]
    leaves = [t.detach().clone().requires_grad_() for t in inputs]
    with fwd.dual_level():
        out = f(*leaves)
        g = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, leaves, g)


@pytest.mark.parametrize("n", [24, 25])          # read in place, and padded
@pytest.mark.parametrize("leaf", [True, False])
def test_a_second_derivative_in_the_bias_is_refused(n, leaf):
    from fast_trimul_b200.functional import pair_attention
    r = gen(9)
    q, k, v = (r(1, 2, n, 2, 32).to(BF).requires_grad_() for _ in range(3))
    w = r(1, 2, n, n).to(BF).requires_grad_()
    bias = w if leaf else w * 2
    (dq,) = torch.autograd.grad(pair_attention(q, k, v, bias), q, torch.ones_like(q), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(dq.float().sum(), w, allow_unused=True)


def test_lengths_and_ends_past_32_bits_are_clamped_not_wrapped():
    from fast_trimul_b200.functional import cached_attention, packed_attention
    r = gen(10)
    q, k, v = r(3, 4, 32).to(BF), r(3, 140, 2, 32).to(BF), r(3, 140, 2, 32).to(BF)
    got = cached_attention(q, k, v, torch.tensor([2 ** 32 + 3, 2 ** 31, -2 ** 32 + 4], device="cuda"))
    assert torch.equal(got, cached_attention(q, k, v, torch.tensor([140, 140, 0], device="cuda")))
    q, k, v = r(50, 4, 32).to(BF), r(50, 2, 32).to(BF), r(50, 2, 32).to(BF)
    got = packed_attention(q, k, v, torch.tensor([0, 20, 2 ** 32 + 1], device="cuda"))
    assert torch.equal(got, packed_attention(q, k, v, ends([20, 30])))


# ------------------------------------------------------------------- failures and several threads
def test_a_failure_is_reported_to_every_thread_once(monkeypatch):
    """A withheld tile of one thread's call: its waits expire, kernels of all streams give up, and the
    other thread hears of it at its next call as well; afterwards both get right results."""
    import concurrent.futures
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import packed_attention
    r = gen(11)
    q, k, v = (r(64, 2, 64).to(BF) for _ in range(3))
    cu, side = ends([64]), torch.cuda.Stream()
    want = packed_attention(q, k, v, cu)
    torch.cuda.synchronize()

    def other():
        with torch.cuda.stream(side):
            out = packed_attention(q, k, v, cu)
        side.synchronize()
        return out

    with concurrent.futures.ThreadPoolExecutor(max_workers=1) as pool:
        assert torch.equal(pool.submit(other).result(), want)
        monkeypatch.setenv("FTM_TEST_STALL", "attention")
        packed_attention(q, k, v, cu)
        monkeypatch.delenv("FTM_TEST_STALL")
        torch.cuda.synchronize()
        with pytest.raises(_lib.NativeKernelError):
            packed_attention(q, k, v, cu)
        assert torch.equal(packed_attention(q, k, v, cu), want)
        with pytest.raises(_lib.NativeKernelError):
            pool.submit(other).result()
        assert torch.equal(pool.submit(other).result(), want)


@pytest.mark.parametrize("h, hk, n", [(8, 1, 900), (16, 2, 640), (65, 1, 300), (3, 3, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_fp16_small_gradients_of_grouped_heads(h, hk, n, causal):
    """Query tiles split between blocks, groups that do not divide a tile, and K and V that are views of one
    projection."""
    from fast_trimul_b200.functional import packed_attention
    r, d = gen(12), 64
    q, kv, g = r(n, h, d).to(HF), r(n, 2, hk, d).to(HF), (1e-3 * r(n, h, d)).to(HF)
    k, v = kv.unbind(1)
    got = train(packed_attention, (q, k, v), g, ends([n]), causal=causal)
    keep = torch.ones(n, n, dtype=torch.bool, device="cuda")
    x = [t.transpose(0, 1) for t in (q, k, v, g)]
    x[1], x[2] = (t.repeat_interleave(h // hk, 0) for t in x[1:3])
    want = list(exact(*x, keep=keep.tril() if causal else keep))
    want[1:] = [t.unflatten(0, (hk, h // hk)).sum(1) for t in want[1:]]
    for name, a, b in zip(("dq", "dk", "dv"), got[1:], want):
        b = b.transpose(0, 1)
        if n == 1:         # one key, whose weight is 1 whatever q and k: dv is g, and dS what fp32 leaves of 0
            assert torch.equal(a, g) if name == "dv" else (a.double() - b).abs().max() <= 2 ** -14 * 1e-3 * 64 * 16
            continue
        assert roundings(a, b) <= MOST, name


def test_fp16_gradients_of_zeros():
    from fast_trimul_b200.functional import packed_attention
    q, k, v, g = (gen(13)(70, 2, 32).to(HF) for _ in range(4))
    cu, zero = ends([40, 30]), torch.zeros_like(q)
    assert all((t == 0).all() for t in train(packed_attention, (q, k, v), zero, cu)[1:])
    got = train(packed_attention, (q, k, zero), g, cu)
    assert (got[1] == 0).all() and (got[2] == 0).all() and not got[3].isnan().any() and (got[3] != 0).any()


def test_more_sequences_than_32_bits_count_are_refused():
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import packed_attention
    q = gen(14)(8, 2, 32).to(BF)
    cu = torch.zeros(2 ** 32 + 3, dtype=torch.int32, device="cuda")      # cut to 32 bits: two sequences
    cu[-1] = 8
    with pytest.raises(_lib.NativeDeclined):
        packed_attention(q, q, q, cu)


def test_cached_a_batch_of_many_sequences():
    """Each (sequence, head) is one tile here, so the same bits as in small batches."""
    from fast_trimul_b200.functional import cached_attention
    r, n = gen(15), 16384
    q, k, v = r(n, 16, 8).to(BF), r(n, 40, 8, 8).to(BF), r(n, 40, 8, 8).to(BF)
    lens = torch.arange(n, device="cuda", dtype=torch.int32) % 41
    got = cached_attention(q, k, v, lens)
    for at in (slice(0, 500), slice(8000, 8300), slice(n - 77, n)):
        assert torch.equal(got[at], cached_attention(q[at], k[at], v[at], lens[at]))
