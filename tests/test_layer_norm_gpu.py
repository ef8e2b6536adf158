"""layer_norm on the GPU against the formula in 64 bits.

Tolerances, with u = 2^-24 the unit of fp32, in which the kernel works. Sums of a row run over
at most 16 terms per thread and trees of at most 5 + 4 levels, so a mean of terms t is off by
at most ~30 u max|t|. Per row with r = 1 / sqrt(var + eps):
* x - mu is off by ~32 u max|x|, hence h = (x - mu) r by dh = 100 u (1 + r max|x|) (r itself is
  off by ~40 u relative). y is off by max|w| dh and one rounding to its type, half a step.
* dx = r (v - mean(v) - h mean(v h)), v = g w: each of the three terms is off by at most
  ~40 u max|v| or max|v| dh (mean(v h) and h are both at most ~max|v| and, times h, max|h|
  bounded as |h| <= sqrt(C)): r max|v| (1 + max|h|) 2 dh in all -- a row of nearly equal values
  has a large r, and its dx is large or cancels.
* a column sum of R terms t over rows runs over at most R / 64 + 64 additions: off by
  (R / 64 + 64) u sum|t|, and dw further by sum |g| dh."""

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def formula(x, w, b, eps, g=None):
    """y, or (y, dx, dw, db) and how far each may be off before its rounding."""
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - mu) * r
    w_ = torch.ones_like(x[..., :1]) if w is None else w.double()
    y = h * w_ + (0 if b is None else b.double())
    if g is None:
        return y
    g = g.double()
    v = g * w_
    dx = r * (v - v.mean(-1, keepdim=True) - h * (v * h).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, t.shape[-1])   # noqa: E731
    top = lambda t: t.abs().amax(-1, keepdim=True)   # noqa: E731
    u = 2.0 ** -24
    dh = 100 * u * (1 + r * top(x))
    adds = (flat(x).shape[0] / 64 + 64) * u
    off = (w_.abs().amax() * dh + 2 * u * top(y), r * top(v) * (1 + top(h)) * 2 * dh,
           adds * flat((g * h).abs()).sum(0) + flat(g.abs() * dh).sum(0), adds * flat(g.abs()).sum(0))
    return (y, dx, flat(g * h).sum(0), flat(g).sum(0)), off


def close(got, want, off):
    """|got - want| <= half a step of got's type + off."""
    half = torch.finfo(got.dtype).eps / 2
    least = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps    # a subnormal's step
    over = (got.double() - want).abs() - (half * (want.abs() + off) + off + least)
    assert not (over > 0).any(), over.max().item()


def make(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    c = shape[-1]
    return ((r(*shape) * 1.5 + 0.3).to(dtype), (1 + 0.2 * r(c)).to(dtype), (0.2 * r(c)).to(dtype),
            r(*shape).to(dtype))


def check(x, w, b, g, eps=1e-5):
    from fast_trimul_b200.functional import layer_norm
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    lx = next(it)
    lw = next(it) if w is not None else None
    lb = next(it) if b is not None else None
    y = layer_norm(lx, lw, lb, eps)
    grads = torch.autograd.grad(y, leaves, g)
    wants, offs = formula(x, w, b, eps, g)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    given = (True, True, w is not None, b is not None)
    wanted = [z for z, there in zip(zip(wants, offs), given) if there]
    for got, (want, off) in zip((y.detach(), *grads), wanted, strict=True):
        close(got, want, off)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)
    again = torch.autograd.grad(layer_norm(lx, lw, lb, eps), leaves, g)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))      # the same bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 2, 7, 16, 64, 100, 128, 129, 256, 384, 501, 512, 768, 1000, 1001,
                                   1024, 2047, 2048, 2049, 4096, 5000, 8191, 8192, 8193, 10000])
def test_widths(width, dtype):
    check(*make((37, width), dtype, width))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 33, 1000, 4099])
@pytest.mark.parametrize("width", [24, 128, 384, 700])
def test_row_counts(rows, width, dtype):
    check(*make((rows, width), dtype, rows))


def test_many_rows_sum_accurately():
    check(*make((2, 300, 301, 128), torch.bfloat16))


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_optional_parameters(which):
    x, w, b, g = make((50, 200), torch.float32)
    check(x, w if which == "weight" else None, b if which == "bias" else None, g)


@pytest.mark.parametrize("xd", DTYPES)
@pytest.mark.parametrize("wd", DTYPES)
def test_mixed_types(xd, wd):
    x, _, _, g = make((65, 130), xd)
    _, w, b, _ = make((65, 130), wd)
    check(x, w, b, g)


def test_layouts_and_alignment():
    x, w, b, g = make((40, 3, 256), torch.bfloat16)
    check(x[..., :128], w[:128], b[:128], g[..., :128])               # a slice of wider rows
    check(x[..., 1:130], w[1:130], b[1:130], g[..., 1:130])           # 2-byte aligned pointers
    check(x[..., 2:130], w[2:130], b[2:130], g[..., 2:130])           # 4-byte aligned
    check(x.transpose(0, 1), w, b, g.transpose(0, 1))                 # not one row stride
    check(x[::2], w, b, g[1::2])
    check(x[:, :1].expand(-1, 3, -1), w, b, g)                        # repeated rows
    check(x[:, :, ::2], w[::2], b[::2], g[:, :, ::2])                 # elements apart
    check(x[0, 0], w, b, g[0, 0])                                     # one dimension
    check(x, w, b, g[:1, :1].expand_as(x))                            # a broadcast gradient


def test_empty_and_special_values():
    from fast_trimul_b200.functional import layer_norm
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
    x = torch.randn(6, 130, device="cuda")
    ref = layer_norm(x)
    x[1, 3], x[4, 129] = float("nan"), float("inf")
    y = layer_norm(x)                            # a bad row stays one row
    assert torch.equal(y[[0, 2, 3, 5]], ref[[0, 2, 3, 5]]) and y[[1, 4]].isnan().all()
    c = torch.full((3, 96), 2.5, device="cuda", dtype=torch.float16)
    assert torch.equal(layer_norm(c), torch.zeros_like(c))           # variance 0
    big = torch.full((2, 128), 6e4, device="cuda", dtype=torch.float16)
    big[:, ::2] = -6e4                           # squares past fp16's range
    assert torch.allclose(layer_norm(big).abs(), torch.ones_like(big), atol=1e-3)


def test_only_the_gradients_that_are_asked_for():
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import layer_norm
    x, w, b, g = make((70, 128), torch.float32)
    _, dxr, dwr, dbr = formula(x, w, b, 1e-5, g)[0]
    n = _lib.stats["kernel_launches"]
    lx = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(layer_norm(lx, w, b), lx, g)
    assert _lib.stats["kernel_launches"] == n + 2          # forward, backward; no reduction
    assert torch.allclose(dx.double(), dxr, atol=1e-4)
    lw, lb = w.detach().requires_grad_(), b.detach().requires_grad_()
    dw, db = torch.autograd.grad(layer_norm(x, lw, lb), (lw, lb), g)
    assert torch.allclose(dw.double(), dwr, atol=1e-3) and torch.allclose(db.double(), dbr, atol=1e-3)


def test_gradient_against_differences():
    from fast_trimul_b200.functional import layer_norm
    x, w, b, g = make((5, 33), torch.float32, 3)
    lx = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(layer_norm(lx, w, b), lx, g)
    d = torch.randn_like(x).double()
    h = 1e-5
    f = lambda t: (formula(t, w, b, 1e-5) * g.double()).sum()   # noqa: E731
    slope = (f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
    assert abs(slope - (dx.double() * d).sum()) < 1e-3 * max(1, abs(slope))


def test_graph_capture_streams_and_refusals():
    from fast_trimul_b200 import _lib
    from fast_trimul_b200.functional import layer_norm
    x, w, b, g = make((64, 384), torch.bfloat16)
    want = layer_norm(x, w, b)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    xin = x.clone().requires_grad_()
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(layer_norm(xin, w, b), xin, g)
        with torch.cuda.graph(graph, stream=s):
            y = layer_norm(xin, w, b)
            (dx,) = torch.autograd.grad(y, xin, g)
    torch.cuda.current_stream().wait_stream(s)
    graph.replay()
    first = dx.clone()
    assert torch.equal(y, want)
    with torch.no_grad():
        xin.copy_(x * 2 + 1)
    graph.replay()
    assert torch.equal(y.detach(), layer_norm(x * 2 + 1, w, b)) and not torch.equal(first, dx)
    with torch.cuda.stream(s):
        other = layer_norm(x, w, b)
    s.synchronize()
    assert torch.equal(other, want)
    with pytest.raises(_lib.NativeDeclined):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(x, w.cpu())
    with pytest.raises(ValueError):
        layer_norm(x, w[:-1])
