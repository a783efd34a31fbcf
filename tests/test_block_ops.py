"""Layer norm, dropout and GELU operators, what can be checked without a GPU: refusals of the C ABI before any device work,
shapes without data, refusals of the Python functions, and the modules' arguments."""
import ctypes

import pytest
import torch

from mamtorch_b200 import _lib


def test_c_abi_refuses_bad_arguments_before_any_device_work():
    L = _lib.lib()
    one = ctypes.c_void_p(64)   # never dereferenced
    odd = ctypes.c_void_p(65)

    def fwd(x=one, pitch=8, res=None, res_pitch=0, w=None, b=None, pd=0, eps=1e-5, rate=0.0, at=None, y=one, s=None,
            stats=None, rows=4, width=8, dtype=0):
        return L.mam_layer_norm_fwd(x, pitch, res, res_pitch, w, b, pd, eps, rate, 1, at, y, s, stats, rows, width, dtype, None)

    for bad in (dict(x=None), dict(y=None), dict(rows=0), dict(rows=-1), dict(width=0), dict(dtype=3), dict(dtype=-1),
                dict(pd=1), dict(dtype=1, pd=2), dict(eps=-1.0), dict(eps=float("nan")), dict(rate=0.5), dict(res=one),
                dict(s=one), dict(pitch=7), dict(res=one, s=one, res_pitch=7), dict(res=one, s=one, res_pitch=8, rate=1.0),
                dict(res=one, s=one, res_pitch=8, rate=-0.1), dict(x=odd), dict(w=odd), dict(stats=ctypes.c_void_p(68)),
                dict(res=one, s=one, res_pitch=8, rate=0.5, at=ctypes.c_void_p(68))):
        assert fwd(**bad) == 1, bad
    assert fwd(rows=2 ** 31) == 2 and fwd(width=2 ** 30 + 1, pitch=2 ** 30 + 1) == 2

    def bwd(gy=one, gs=None, s=one, pitch=8, stats=one, w=None, pd=0, rate=0.0, ds=one, dx=None, dw=None, db=None, rows=4,
            width=8, dtype=0):
        return L.mam_layer_norm_bwd(gy, gs, s, pitch, stats, w, pd, rate, 1, None, ds, dx, dw, db, rows, width, dtype, None, 0,
                                    None)

    for bad in (dict(s=None), dict(stats=None), dict(ds=None), dict(rows=0), dict(width=-3), dict(dtype=9), dict(pitch=7),
                dict(rate=0.5), dict(dx=one, rate=1.0), dict(pd=2), dict(gs=odd), dict(dw=odd), dict(stats=ctypes.c_void_p(68))):
        assert bwd(**bad) == 1, bad
    for f in (lambda **k: L.mam_dropout_add(k.get("x", one), None, k.get("y", one), k.get("n", 8), k.get("t", 0),
                                            k.get("rate", 0.5), 1, None, None),
              lambda **k: L.mam_gelu_fwd(k.get("x", one), k.get("y", one), k.get("n", 8), k.get("t", 0), k.get("rate", 0.5), 1,
                                         None, None),
              lambda **k: L.mam_gelu_bwd(one, k.get("x", one), k.get("y", one), k.get("n", 8), k.get("t", 0),
                                         k.get("rate", 0.5), 1, None, None)):
        for bad in (dict(x=None), dict(y=None), dict(n=0), dict(n=-1), dict(t=5), dict(rate=1.0), dict(rate=-1.0),
                    dict(rate=float("nan")), dict(x=odd), dict(y=odd)):
            assert f(**bad) == 1, bad
    assert L.mam_gelu_bwd(None, one, one, 8, 0, 0.0, 1, None, None) == 1


def test_workspace_query():
    L = _lib.lib()
    assert L.mam_layer_norm_bwd_workspace_bytes(0, 8) == 0 and L.mam_layer_norm_bwd_workspace_bytes(8, 0) == 0
    assert L.mam_layer_norm_bwd_workspace_bytes(1, 64) == 2 * 64 * 4
    # a row of each sum for each SM at most
    assert L.mam_layer_norm_bwd_workspace_bytes(100000, 768) == 148 * 2 * 768 * 4


def test_shapes_without_data():
    import mamtorch_b200  # noqa: F401

    ops = torch.ops.mamtorch_b200
    x = torch.empty(3, 5, 8, device="meta", dtype=torch.bfloat16)
    w = torch.empty(8, device="meta")
    assert ops.layer_norm(x, w, w, 1e-5).shape == x.shape
    y, s = ops.dropout_add_layer_norm(x, x, w, None, 1e-5, 0.5, 1, None)
    assert y.shape == s.shape == x.shape and y.dtype == s.dtype == x.dtype
    assert ops.dropout(x, None, 0.5, 1, None).shape == x.shape and ops.gelu(x, 0.0, 0, None).dtype == x.dtype
    out = ops.layer_norm_forward(x, None, w, w, 1e-5, 0.0, 0, None, True)
    assert out[1].shape == (15, 2) and out[1].dtype == torch.float32


def test_cpu_tensors_and_bad_rates_fail_loudly():
    from mamtorch_b200.nn import functional as MF

    x = torch.randn(3, 8, requires_grad=True)
    for f in (MF.layer_norm, MF.gelu, lambda v: MF.dropout(v, 0.5, 1), lambda v: MF.dropout_add_layer_norm(v, v)):
        with pytest.raises(NotImplementedError):
            f(x)
        with pytest.raises(NotImplementedError), torch.no_grad():
            f(x)
    for rate in (-0.5, 1.0, float("nan")):
        with pytest.raises(ValueError):
            MF.gelu(x, rate)


def test_block_arguments_and_state():
    from mamtorch_b200.nn.vit import MAMMlpBlock, MAMMlpStack

    keys = ["fc1.bias", "fc1.weight", "fc2.bias", "fc2.weight", "norm.bias", "norm.weight"]
    assert sorted(MAMMlpBlock(8, 16).state_dict()) == keys
    assert sorted(MAMMlpBlock(8, 16, fused=True, drop_rate=0.1).state_dict()) == keys
    for bad in (dict(drop_rate=0.1), dict(fused=True, drop_rate=1.0), dict(fused=True, drop_rate=-0.1)):
        with pytest.raises(ValueError):
            MAMMlpBlock(8, 16, **bad)
    for bad in (dict(depth=0), dict(depth=2, residual=False)):
        with pytest.raises(ValueError):
            MAMMlpStack(hidden=8, intermediate=16, **bad)
    stack = MAMMlpStack(3, 8, 16, drop_rate=0.1, vcon_steps=2)
    assert len(stack.state_dict()) == 3 * 6 + 2
    stack.vcon_step()
    assert all(b.fc1.beta == 0.5 and b.fc2.beta == 0.5 for b in stack.blocks)
    torch.manual_seed(0)
    a = stack.blocks[0].drop_args()
    torch.manual_seed(0)
    assert stack.blocks[0].drop_args() == a and a[0] == 0.1
    assert stack.eval().blocks[0].drop_args() == (0.0, None)
