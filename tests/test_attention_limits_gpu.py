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
