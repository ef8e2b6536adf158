"""The attention operators without a GPU: the torch path against 64 bits, the refusals of the
Python entry points, the C entry points' argument checks, and the fused trunk."""

import ctypes

import pytest
import torch

import attention_reference as ref
from fast_trimul_b200 import _lib
from fast_trimul_b200.functional import cached_attention, packed_attention, pair_attention


def gen(seed=0):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g)


def ends(lens, first=0):
    return torch.tensor([first] + [first + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,klens", [([5, 1, 9], [5, 1, 9]), ([3, 4], [7, 4]), ([6, 2], [2, 5]), ([4, 0, 3], [4, 2, 0])])
def test_packed_matches_64_bits_with_gradients(lens, klens, causal):
    r = gen()
    q, k, v = r(sum(lens) + 2, 4, 8), r(sum(klens) + 1, 2, 8), r(sum(klens) + 1, 2, 8)
    g = r(*q.shape)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, ends(lens, 1), ends(klens), causal=causal)
    grads = torch.autograd.grad(out, leaves, g)
    w = ref.packed(q.detach(), k.detach(), v.detach(), g, ends(lens, 1), ends(klens), causal, 8 ** -0.5)
    assert torch.allclose(out.double(), w.o, atol=1e-5)
    for a, b in zip(grads, (w.dq, w.dk, w.dv)):
        assert torch.allclose(a.double(), b, atol=1e-5)


def test_pair_and_cached_match_64_bits():
    r = gen(1)
    q, k, v, g = (r(2, 3, 6, 2, 4) for _ in range(4))
    bias, mask = r(2, 2, 6, 6), torch.rand(2, 3, 6) > 0.3
    mask[0, 1] = False
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    out = pair_attention(*leaves, mask.float())
    grads = torch.autograd.grad(out, leaves, g)
    w = ref.pair(q.detach(), k.detach(), v.detach(), g, bias.detach(), mask, 0.5)
    assert torch.allclose(out.double(), w.o, atol=1e-5) and (out[0, 1] == 0).all()
    for a, b in zip(grads, (w.dq, w.dk, w.dv, w.db)):
        assert torch.allclose(a.double(), b, atol=1e-5)
    kc, vc, qc = r(3, 9, 2, 4), r(3, 9, 2, 4), r(3, 4, 4)
    lens = torch.tensor([9, 0, 4])
    kc[2, 4:] = float("nan")         # behind the length: never seen
    vc[2, 4:] = float("inf")
    o = cached_attention(qc, kc, vc, lens)
    assert (o[1] == 0).all()
    for b in (0, 2):
        n = int(lens[b])
        one = packed_attention(qc[b:b + 1], kc[b, :n], vc[b, :n], torch.tensor([0, 1]), torch.tensor([0, n]))
        assert torch.allclose(o[b:b + 1], one, atol=1e-6)


def test_masked_keys_count_as_absent_whatever_they_hold():
    r = gen(2)
    q, k, v = r(7, 2, 8), r(7, 2, 8), r(7, 2, 8)
    mask = torch.tensor([1, 0, 1, 1, 0, 1, 1], dtype=torch.bool)
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("nan"), float("inf")
    a = packed_attention(q, k, v, ends([7]), causal=False, key_mask=mask)
    b = packed_attention(q, k2, v2, ends([7]), causal=False, key_mask=mask)
    assert torch.equal(a, b)


def test_refusals():
    r = gen()
    q, k, cu = r(6, 4, 8), r(6, 2, 8), ends([6])
    for bad in (lambda: packed_attention(q[0], k, k, cu),                          # dimensions
                lambda: packed_attention(q, k, k[:, :, :4], cu),                   # k and v differ
                lambda: packed_attention(q[:, :3], k, k, cu),                      # 3 heads on 2
                lambda: packed_attention(q, k.double(), k.double(), cu),           # types differ
                lambda: packed_attention(q, k, k, cu.float()),
                lambda: packed_attention(q, k, k, cu[None]),
                lambda: packed_attention(q, k[:5], k[:5], cu),                     # whose rows?
                lambda: packed_attention(q, k, k, cu, ends([3, 3])),
                lambda: packed_attention(q, k, k, cu, scale=-1.0),
                lambda: packed_attention(q, k, k, cu, scale=float("nan")),
                lambda: packed_attention(q, k, k, cu, key_mask=torch.ones(5)),
                lambda: cached_attention(q, k[None], k[None], cu[:1]),
                lambda: cached_attention(q[:1], k[None], k[None], torch.tensor([1, 2])),
                lambda: cached_attention(q[:1], k[None], k[None], torch.tensor([1.0])),
                lambda: cached_attention(q[:1].requires_grad_(), k[None], k[None], torch.tensor([1])),
                lambda: pair_attention(q, q, q, None),
                lambda: pair_attention(q[None, None], q[None, None], q[None, None], r(1, 4, 5, 6)),
                lambda: pair_attention(q[None, None], q[None, None], q[None, None], r(2, 4, 6, 6)),
                lambda: pair_attention(q[None, None], q[None, None], q[None, None], None, torch.ones(1, 6))):
        with pytest.raises(ValueError):
            bad()


def test_no_sequences_and_no_rows():
    r = gen()
    q, k = r(5, 2, 8), r(5, 2, 8)
    assert torch.equal(packed_attention(q, k, k, torch.tensor([0])), torch.zeros_like(q))
    assert packed_attention(q[:0], k[:0], k[:0], torch.tensor([0, 0])).shape == (0, 2, 8)
    assert torch.equal(packed_attention(q, k[:0], k[:0], ends([5]), torch.tensor([0, 0])), torch.zeros_like(q))
    assert cached_attention(q[:0], r(0, 4, 2, 8), r(0, 4, 2, 8), torch.tensor([], dtype=torch.int32)).shape == (0, 2, 8)
    assert pair_attention(r(1, 0, 4, 2, 8), r(1, 0, 4, 2, 8), r(1, 0, 4, 2, 8), r(1, 2, 4, 4)).shape == (1, 0, 4, 2, 8)


def test_nothing_to_attend_to_gives_zeros_whatever_the_inputs_hold():
    bad = torch.full((3, 2, 8), float("nan"), requires_grad=True)
    for out in (packed_attention(bad, bad, bad, torch.tensor([0])),
                packed_attention(bad, bad[:0], bad[:0], ends([3]), torch.tensor([0, 0])),
                packed_attention(bad, bad, bad, torch.tensor([0, 3]), torch.tensor([1, 1]))):
        assert torch.equal(out, torch.zeros_like(bad))
        (grad,) = torch.autograd.grad(out.sum(), bad)
        assert torch.equal(grad, torch.zeros_like(bad))


def test_c_entry_points_check_their_arguments_before_the_device():
    lib = _lib.load()
    p = 1 << 20     # a 256-byte aligned address, never dereferenced

    def prob(**kw):
        a = dict(dtype=_lib.BF16, heads=4, kv_heads=2, head_dim=64, causal=1, scale=0.125, sequences=3, q_len=0,
                 kv_len=0, q_rows=100, kv_rows=100, cu_q=p, cu_k=p, kv_lengths=None, q=p, q_row_stride=256,
                 q_head_stride=64, k=p, k_row_stride=128, k_head_stride=64, k_batch_stride=0, v=p,
                 v_row_stride=128, v_head_stride=64, v_batch_stride=0, key_mask=None, bias=None, bias_seqs=0,
                 bias_row_stride=0, bias_head_stride=0, bias_batch_stride=0, out=p, stats=p)
        a.update(kw)
        return _lib.Attention(**a)

    def fwd(ws=p, n=1 << 30, err=p, **kw):
        return lib.ftm_attention_fwd(prob(**kw), 1, ws, n, err, None, None)

    assert fwd() == _lib.UNSUPPORTED_ARCH or torch.cuda.is_available()
    uniform = dict(cu_q=None, cu_k=None, q_len=50, kv_len=50, sequences=2)
    pair = dict(uniform, heads=2, causal=0, bias=p, bias_seqs=1, bias_row_stride=56, bias_head_stride=2800,
                bias_batch_stride=5600)
    cache = dict(cu_q=None, cu_k=None, kv_lengths=p, q_len=1, sequences=100, causal=0, stats=None,
                 k_batch_stride=12800, v_batch_stride=12800)
    S, A, D, L, W = _lib.BAD_SHAPE, _lib.BAD_ARGUMENT, _lib.BAD_DTYPE, _lib.BAD_ALIGN, _lib.BAD_WORKSPACE
    for want, kw in (
            (D, dict(dtype=_lib.F32)), (A, dict(scale=-1.0)), (A, dict(scale=float("inf"))), (A, dict(q=None)),
            (S, dict(heads=3)), (S, dict(heads=0)), (S, dict(heads=258, kv_heads=2)), (S, dict(head_dim=60)),
            (S, dict(head_dim=136)), (S, dict(head_dim=0)), (S, dict(sequences=0)), (S, dict(q_rows=0)),
            (S, dict(q_rows=1 << 31)), (A, dict(cu_k=None)), (A, dict(bias=p)), (L, dict(q_row_stride=252)),
            (L, dict(k_head_stride=0)), (L, dict(q=p + 2)), (L, dict(out=p + 8)), (L, dict(stats=p + 4)),
            (S, dict(uniform, q_len=49)), (S, dict(uniform, kv_len=0)), (S, dict(pair, heads=4)),
            (S, dict(pair, bias_seqs=0)), (S, dict(pair, sequences=2, bias_seqs=3)), (L, dict(pair, bias_row_stride=50)),
            (L, dict(pair, bias=p + 2)), (A, dict(cache, stats=p)), (A, dict(cache, causal=1)),
            (A, dict(cache, key_mask=p)), (S, dict(cache, sequences=99)), (L, dict(cache, k_batch_stride=0))):
        assert fwd(**kw) == want, kw
    assert fwd(err=None) == A
    if not torch.cuda.is_available():
        return          # from here on the device is looked at first
    assert fwd(ws=None) == W and fwd(n=8) == W


def test_a_bias_with_a_causal_call_is_refused():
    p = 1 << 20
    prob = _lib.Attention(dtype=_lib.BF16, heads=2, kv_heads=2, head_dim=64, causal=1, scale=0.125, sequences=2,
                          q_len=50, kv_len=50, q_rows=100, kv_rows=100, q=p, q_row_stride=128, q_head_stride=64, k=p,
                          k_row_stride=128, k_head_stride=64, v=p, v_row_stride=128, v_head_stride=64, bias=p,
                          bias_seqs=1, bias_row_stride=56, bias_head_stride=2800, bias_batch_stride=5600, out=p)
    assert _lib.load().ftm_attention_fwd(prob, 0, None, 0, p, None, None) == _lib.BAD_ARGUMENT
    prob.causal = 0
    assert _lib.load().ftm_attention_fwd(prob, 0, None, 0, None, None, None) == _lib.BAD_ARGUMENT   # no error word
    prob.bias_row_stride = 50
    assert _lib.load().ftm_attention_fwd(prob, 0, None, 0, p, None, None) == _lib.BAD_ALIGN


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.ftm_attention_workspace_bytes(None, 0) == 0
    assert lib.ftm_attention_bwd_workspace_bytes(None, 0) == 0


@pytest.mark.parametrize("masked", [False, True])
def test_fused_trunk_equals_the_plain_one(masked):
    from fast_trimul_b200.pairformer import PairFormerTrunk
    torch.manual_seed(0)
    a = PairFormerTrunk(2, 32, 16)
    b = PairFormerTrunk(2, 32, 16, fused=True)
    b.load_state_dict(a.state_dict())
    s, z = torch.randn(2, 9, 32), torch.randn(2, 9, 9, 16)
    mask = None
    if masked:
        mask = torch.ones(2, 9, 9)
        mask[:, 7:] = 0
        mask[:, :, 7:] = 0
    with torch.no_grad():
        s1, z1 = a(s, z, mask)
        s2, z2 = b(s, z, mask)
    n = 7 if masked else 9
    assert torch.allclose(z1[:, :n, :n], z2[:, :n, :n], atol=1e-4)
    if not masked:      # the single attention has no mask: padded rows of z reach it
        assert torch.allclose(s1, s2, atol=1e-4)


def test_torch_extension_loads_and_leaves_cpu_calls_alone():
    ext = _lib.torch_ext()
    x = torch.randn(3, 8)
    assert ext.layer_norm(x, None, None, 1e-5) is None
    q = torch.randn(4, 2, 8)
    cu = ends([4])
    assert ext.packed(q, q, q, cu, cu, True, None, None) is None
    assert ext.cached(q, q[:, None], q[:, None], torch.ones(4, dtype=torch.int32), None) is None
    assert ext.pair(q[None, None], q[None, None], q[None, None], None, None, None) is None
    n = _lib.stats["calls"]
    _lib.stats["calls"] += 2
    assert _lib.stats["calls"] == n + 2
