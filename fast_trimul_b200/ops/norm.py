"""Layer norm over the last dimension, forward and backward on the sm_100a kernels.

`layer_norm(x, weight, bias, eps)` takes any width, any leading dimensions and any mix of
fp32 / fp16 / bf16 between x and its parameters; `FastLayerNorm` is the module form, with
`nn.LayerNorm`'s parameters and state dict. On a CUDA tensor the kernels run (statistics
and sums in fp32, the result rounded once to x's type); elsewhere torch's formula does.
"""

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _lib

_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


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


def _formula(x, weight, bias, eps):
    if all(p is None or p.dtype == x.dtype for p in (weight, bias)):
        return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)
    f = lambda p: None if p is None else p.float()   # noqa: E731
    return F.layer_norm(x.float(), (x.shape[-1],), f(weight), f(bias), eps).to(x.dtype)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over x's last dimension.

    x: (..., width) fp32, fp16 or bf16, on a GPU of at most 2^30 - 1024 columns; weight, bias:
    (width,) of any of these types, or None. Returns x's shape and type. Differentiable once in
    x, weight and bias (tangents, of forward mode, are refused on a GPU); the gradients have
    their inputs' types and are the same bits on every call. Rows may be strided (a slice of a
    wider tensor is read in place); other layouts are copied first."""
    if x.is_cuda:
        for name, p in (("x", x), ("weight", weight), ("bias", bias)):
            if p is not None and p.dtype not in _DT:
                raise _lib.NativeDeclined(f"layer_norm takes fp32, fp16 and bf16, got {p.dtype} for {name}")


def _formula(x, weight, bias, eps):
    if all(p is None or p.dtype == x.dtype for p in (weight, bias)):
        return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)
    f = lambda p: None if p is None else p.float()   # noqa: E731
    return F.layer_norm(x.float(), (x.shape[-1],), f(weight), f(bias), eps).to(x.dtype)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over x's last dimension.

    x: (..., width) fp32, fp16 or bf16, on a GPU of at most 2^30 - 1024 columns; weight, bias: (width,) of any of these types, or
    None. Returns x's shape and type. Differentiable once in x, weight and bias (tangents,
    of forward mode, are refused on a GPU); the gradients have their inputs' types and are
    the same bits on every call. Rows may be strided (a slice of a wider tensor is read in
    place); other layouts are copied first."""
    if x.is_cuda:
        try:
            out = _lib.torch_ext().layer_norm(x, weight, bias, eps)
        except RuntimeError as e:
            _lib.check_raised(e)
        if out is not None:
            return out
    _checked(x, weight, bias, eps)
    if not x.is_cuda or x.numel() == 0:
        return _formula(x, weight, bias, eps)
    dense = lambda p: None if p is None else p.contiguous()   # noqa: E731
    try:
        out = _lib.torch_ext().layer_norm(x.contiguous(), dense(weight), dense(bias), eps)
    except RuntimeError as e:
        _lib.check_raised(e)
    if out is None:
        raise _lib.NativeDeclined(f"layer_norm of {tuple(x.shape)}")
    return out


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
