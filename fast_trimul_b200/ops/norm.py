"""Layer norm over the last dimension, forward and backward on the sm_100a kernels.

`layer_norm(x, weight, bias, eps)` takes any width, any leading dimensions and any mix of
fp32 / fp16 / bf16 between x and its parameters; `FastLayerNorm` is the module form, with
`nn.LayerNorm`'s parameters and state dict. On a CUDA tensor the kernels run (statistics
and sums in fp32, the result rounded once to x's type); elsewhere torch's formula does.
"""

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .. import _lib

_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def device_guard(t):
    """The library launches on the current device: make it `t`'s (nothing to do, and
    nothing paid, when it already is)."""
    return _NO_GUARD if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


class _NoGuard:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def _rows(t, width):
    """`t` as rows of `width` contiguous elements a fixed stride apart, copied only when its
    layout is not that; and the stride."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if width > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    try:
        t = t.view(-1, width)
    except RuntimeError:
        t = t.contiguous().view(-1, width)
    return t, (t.stride(0) if t.shape[0] > 1 else width)


def _checked(x, weight, bias, eps):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm needs a last dimension to normalise, got {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{name} is on {p.device}, x on {x.device}")
    if x.is_cuda:
        for name, p in (("x", x), ("weight", weight), ("bias", bias)):
            if p is not None and p.dtype not in _DT:
                raise _lib.NativeDeclined(f"layer_norm takes fp32, fp16 and bf16, got {p.dtype} for {name}")


def _forward(x, weight, bias, eps, keep_stats):
    lib = _lib.load()
    width = x.shape[-1]
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows = x.numel() // width
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep_stats else None
    if rows:
        x2, stride = _rows(x, width)
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        with device_guard(x):
            _lib.check(lib.ftm_layer_norm_fwd(
                x2.data_ptr(), _DT[x.dtype], stride, None if w is None else w.data_ptr(),
                0 if w is None else _DT[w.dtype], None if b is None else b.data_ptr(),
                0 if b is None else _DT[b.dtype], eps, out.data_ptr(),
                None if stats is None else stats.data_ptr(), rows, width,
                torch.cuda.current_stream().cuda_stream), "ftm_layer_norm_fwd")
        _lib.stats["calls"] += 1
        _lib.stats["kernel_launches"] += 1
    return out, stats


class _LayerNorm(torch.autograd.Function):
    """Forward that keeps (mean, rstd) of each row; backward in one pass over x and the
    gradient plus the reduction of the parameters' gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_like = None if bias is None else bias.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        width = x.shape[-1]
        rows = x.numel() // width
        dev = x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        make = torch.empty if rows else torch.zeros
        dw = make(width, dtype=weight.dtype, device=dev) if need_w else None
        db = make(width, dtype=ctx.bias_like, device=dev) if need_b else None
        if rows and (need_x or need_w or need_b):
            lib = _lib.load()
            x2, xs = _rows(x, width)
            g2, gs = _rows(grad if grad.dtype == x.dtype else grad.to(x.dtype), width)
            w = None if weight is None else weight.contiguous()
            with device_guard(x):
                nbytes = lib.ftm_layer_norm_bwd_workspace_bytes(rows, width) if need_w or need_b else 0
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
                _lib.check(lib.ftm_layer_norm_bwd(
                    x2.data_ptr(), _DT[x.dtype], xs, g2.data_ptr(), gs,
                    None if w is None else w.data_ptr(), 0 if w is None else _DT[w.dtype],
                    stats.data_ptr(), None if dx is None else dx.data_ptr(),
                    None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                    0 if db is None else _DT[db.dtype], None if ws is None else ws.data_ptr(), nbytes,
                    rows, width, torch.cuda.current_stream().cuda_stream), "ftm_layer_norm_bwd")
            _lib.stats["kernel_launches"] += 2 if nbytes else 1
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over x's last dimension.

    x: (..., width) fp32, fp16 or bf16; weight, bias: (width,) of any of these types, or
    None. Returns x's shape and type. Differentiable once in x, weight and bias; the
    gradients have their inputs' types and are the same bits on every call. Rows may be
    strided (a slice of a wider tensor is read in place); other layouts are copied first."""
    _checked(x, weight, bias, eps)
    if not x.is_cuda:
        if all(p is None or p.dtype == x.dtype for p in (weight, bias)):
            return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)
        f = lambda p: None if p is None else p.float()   # noqa: E731
        return F.layer_norm(x.float(), (x.shape[-1],), f(weight), f(bias), eps).to(x.dtype)
    if torch.is_grad_enabled() and any(p is not None and p.requires_grad for p in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


class FastLayerNorm(nn.LayerNorm):
    """`nn.LayerNorm` over one last dimension (same parameters, init and state dict) that
    runs `layer_norm`."""

    def __init__(self, width, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(width, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device,
                         dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("FastLayerNorm normalises one dimension")

    def forward(self, x):
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"expected a last dimension of {self.normalized_shape[0]}, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
