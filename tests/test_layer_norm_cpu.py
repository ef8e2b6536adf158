"""layer_norm without a GPU: the torch path against the formula in 64 bits, the refusals,
the module's state dict, and the C entry points' argument checks."""

import ctypes

import pytest
import torch

import fast_trimul_b200 as ft
from fast_trimul_b200 import _lib
from fast_trimul_b200.functional import layer_norm


def formula(x, w, b, eps):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    h = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    return h * (1 if w is None else w.double()) + (0 if b is None else b.double())


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("affine", [False, True])
def test_cpu_path_matches_the_formula(dtype, tol, affine):
    torch.manual_seed(0)
    x = torch.randn(3, 5, 33).to(dtype)
    w = torch.randn(33) if affine else None       # fp32 parameters of a bf16 input too
    b = torch.randn(33) if affine else None
    y = layer_norm(x, w, b, 1e-5)
    assert y.dtype == dtype and y.shape == x.shape
    assert (y.double() - formula(x, w, b, 1e-5)).abs().max() < tol * 4


def test_module_has_layer_norms_parameters_and_results():
    torch.manual_seed(1)
    ref = torch.nn.LayerNorm(24)
    mod = ft.FastLayerNorm(24)
    torch.nn.init.normal_(ref.weight)
    mod.load_state_dict(ref.state_dict())
    x = torch.randn(7, 24)
    assert torch.equal(mod(x), ref(x))
    assert ft.nn.FastLayerNorm is ft.FastLayerNorm
    with pytest.raises(ValueError):
        mod(torch.randn(7, 25))
    with pytest.raises(ValueError):
        ft.FastLayerNorm((2, 3))


@pytest.mark.parametrize("args", [
    (torch.randn(4, 8), torch.ones(7), None, 1e-5),
    (torch.randn(4, 8), None, torch.ones(8, 1), 1e-5),
    (torch.randn(4, 8), None, None, -1.0),
    (torch.randn(4, 8), None, None, float("nan")),
    (torch.tensor(1.0), None, None, 1e-5),
    (torch.randn(4, 0), None, None, 1e-5),
])
def test_refusals(args):
    with pytest.raises(ValueError):
        layer_norm(*args)


def test_c_entry_points_check_their_arguments_before_the_device():
    lib = _lib.load()
    p = ctypes.c_void_p(1 << 20)       # never dereferenced
    odd = ctypes.c_void_p((1 << 20) + 1)
    fwd, bwd = lib.ftm_layer_norm_fwd, lib.ftm_layer_norm_bwd
    assert fwd(None, 0, 8, None, 0, None, 0, 1e-5, p, None, 4, 8, None) == _lib.BAD_ARGUMENT
    assert fwd(p, 0, 8, None, 0, None, 0, -1.0, p, None, 4, 8, None) == _lib.BAD_ARGUMENT
    assert fwd(p, 0, 8, None, 0, None, 0, 1e-5, p, None, 0, 8, None) == _lib.BAD_SHAPE
    assert fwd(p, 0, 8, None, 0, None, 0, 1e-5, p, None, 4, 0, None) == _lib.BAD_SHAPE
    assert fwd(p, 0, -8, None, 0, None, 0, 1e-5, p, None, 4, 8, None) == _lib.BAD_SHAPE
    assert fwd(p, 3, 8, None, 0, None, 0, 1e-5, p, None, 4, 8, None) == _lib.BAD_DTYPE
    assert fwd(p, 0, 8, p, 7, None, 0, 1e-5, p, None, 4, 8, None) == _lib.BAD_DTYPE
    assert fwd(odd, 1, 8, None, 0, None, 0, 1e-5, p, None, 4, 8, None) == _lib.BAD_ALIGN
    assert lib.ftm_layer_norm_bwd_workspace_bytes(0, 8) == 0
    need = lib.ftm_layer_norm_bwd_workspace_bytes(5, 8)
    assert need == 5 * 2 * 8 * 4       # a partial row per block, never more blocks than rows

    def back(dx=p, dw=p, db=p, ws=p, n=need, rows=5, width=8, dbt=0):
        return bwd(p, 0, 8, p, 8, p, 0, p, dx, dw, db, dbt, ws, n, rows, width, None)
    assert back(dx=None, dw=None, db=None) == _lib.BAD_ARGUMENT
    assert back(ws=None) == _lib.BAD_WORKSPACE
    assert back(n=need - 1) == _lib.BAD_WORKSPACE
    assert back(rows=0) == _lib.BAD_SHAPE
    assert back(dbt=9) == _lib.BAD_DTYPE
