"""Refusals of the sequence operators and of their entry points, and the layers' host side (no GPU needed)."""
import ctypes
import os

import pytest
import torch

import sinabs_exodus_b200 as ex
from sinabs_exodus_b200 import _lib, _seq


@pytest.fixture(scope="module")
def lib():
    from sinabs_exodus_b200 import build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


def scan_args(nb=2, T=5, M=8, N=4, G=2, kind=torch.float32):
    return dict(x=torch.zeros(nb, T, M, dtype=kind), dt=torch.zeros(nb, T, M, dtype=kind), A=torch.zeros(M, N),
                B=torch.zeros(nb, T, G, N, dtype=kind), C=torch.zeros(nb, T, G, N, dtype=kind))


@pytest.mark.parametrize("change,error,text", [
    (dict(x=torch.zeros(2, 5)), ValueError, "3D"),
    (dict(x=torch.zeros(2, 5, 8, dtype=torch.float64)), ValueError, "float32, bfloat16 or float16"),
    (dict(x=[1.0]), TypeError, "tensor"),
    (dict(dt=torch.zeros(2, 5, 7)), ValueError, "'dt' must have shape"),
    (dict(dt=torch.zeros(2, 5, 8, dtype=torch.bfloat16)), ValueError, "'dt' must be float32"),
    (dict(A=torch.zeros(8, 5)), ValueError, "'A' must have shape"),
    (dict(A=torch.zeros(8, 4, dtype=torch.bfloat16)), ValueError, "'A' must be float32"),
    (dict(B=torch.zeros(2, 5, 3, 4)), ValueError, "groups"),
    (dict(B=torch.zeros(2, 4, 2, 4)), ValueError, "'B' must have shape"),
    (dict(C=torch.zeros(2, 5, 2, 3)), ValueError, "'C' must have shape"),
    (dict(C=torch.zeros(2, 5, 1, 4)), ValueError, "'C' must have shape"),
    (dict(D=torch.zeros(7)), ValueError, "'D' must have shape"),
    (dict(z=torch.zeros(2, 5, 4)), ValueError, "'z' must have shape"),
    (dict(dt_bias=torch.zeros(8, dtype=torch.float16)), ValueError, "'dt_bias' must be float32"),
    (dict(h0=torch.zeros(2, 8, 3)), ValueError, "'h0' must have shape"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError, "'lengths' must have shape"),
    (dict(lengths=torch.zeros(2)), ValueError, "'lengths' must be int32 or int64"),
    (dict(lengths=[1, 2]), TypeError, "'lengths' must be a tensor"),
    ({}, _lib.ExodusLibraryError, "only run on CUDA"),
])
def test_selective_scan_refuses(change, error, text):
    with pytest.raises(error, match=text):
        ex.selective_scan(**{**scan_args(), **change})


def test_selective_scan_refuses_too_many_states():
    with pytest.raises(ValueError, match="1 to 128 states"):
        ex.selective_scan(**scan_args(N=129))
    with pytest.raises(ValueError, match="1 to 128 states"):
        ex.selective_scan(**scan_args(N=0))


@pytest.mark.parametrize("change,error,text", [
    (dict(h=torch.zeros(2, 8, 3)), ValueError, "'h' must have shape"),
    (dict(h=torch.zeros(2, 8, 4, dtype=torch.float16)), ValueError, "'h' must be float32"),
    (dict(h=torch.zeros(2, 4, 8).transpose(1, 2)), ValueError, "contiguous in its channels"),
    (dict(h=torch.zeros(1, 8, 4).expand(2, 8, 4)), ValueError, "overlap"),
    (dict(x=torch.zeros(2, 1, 8)), ValueError, "2D"),
    (dict(B=torch.zeros(2, 8)), ValueError, "shape"),
    ({}, _lib.ExodusLibraryError, "only run on CUDA"),
])
def test_selective_step_refuses(change, error, text):
    a = {k: (v[:, 0] if v.ndim > 2 else v) for k, v in scan_args().items()}
    with pytest.raises(error, match=text):
        ex.selective_step(**{"h": torch.zeros(2, 8, 4), **a, **change})


@pytest.mark.parametrize("change,error,text", [
    (dict(x=torch.zeros(2, 8)), ValueError, "3D"),
    (dict(weight=torch.zeros(7, 4)), ValueError, "'weight' must have shape"),
    (dict(weight=torch.zeros(8, 9)), ValueError, "1 to 8 steps"),
    (dict(weight=torch.zeros(8, 0)), ValueError, "1 to 8 steps"),
    (dict(weight=torch.zeros(8, 4, dtype=torch.float16)), ValueError, "'weight' must be"),
    (dict(bias=torch.zeros(8, dtype=torch.bfloat16)), ValueError, "'bias' must be float32"),
    (dict(bias=torch.zeros(9)), ValueError, "'bias' must have shape"),
    (dict(state=torch.zeros(2, 4, 8)), ValueError, "'state' must have shape"),
    (dict(state=torch.zeros(2, 3, 8, dtype=torch.bfloat16)), ValueError, "'state' must be float32"),
    (dict(lengths=torch.zeros(2)), ValueError, "'lengths'"),
    (dict(activation="relu"), ValueError, "'activation'"),
    ({}, _lib.ExodusLibraryError, "only run on CUDA"),
])
def test_causal_conv_refuses(change, error, text):
    with pytest.raises(error, match=text):
        ex.causal_conv(**{"x": torch.zeros(2, 5, 8), "weight": torch.zeros(8, 4), **change})


@pytest.mark.parametrize("change,error,text", [
    (dict(state=torch.zeros(2, 2, 8)), ValueError, "'state' must have shape"),
    (dict(state=torch.zeros(2, 8, 3).transpose(1, 2)), ValueError, "contiguous in its rows"),
    (dict(state=torch.zeros(1, 3, 8).expand(2, 3, 8)), ValueError, "overlap"),
    (dict(x=torch.zeros(2, 1, 8)), ValueError, "2D"),
    ({}, _lib.ExodusLibraryError, "only run on CUDA"),
])
def test_causal_conv_step_refuses(change, error, text):
    with pytest.raises(error, match=text):
        ex.causal_conv_step(**{"state": torch.zeros(2, 3, 8), "x": torch.zeros(2, 8), "weight": torch.zeros(8, 4), **change})


@pytest.mark.parametrize("change,error,text", [
    (dict(x=torch.zeros(8)), ValueError, "at least 2"),
    (dict(x=torch.zeros(2, 8, dtype=torch.int32)), ValueError, "float32, bfloat16 or float16"),
    (dict(num_groups=3), ValueError, "divide"),
    (dict(num_groups=0), ValueError, "divide"),
    (dict(x=torch.zeros(1, 16385), num_groups=1), ValueError, "at most 16384"),
    (dict(weight=torch.zeros(7)), ValueError, "'weight' must have shape"),
    (dict(weight=torch.zeros(8, dtype=torch.float16)), ValueError, "'weight' must be"),
    (dict(activation="gelu"), ValueError, "'activation'"),
    (dict(eps=-1.0), ValueError, "'eps'"),
    (dict(eps=float("nan")), ValueError, "'eps'"),
    ({}, _lib.ExodusLibraryError, "only run on CUDA"),
])
def test_group_norm_refuses(change, error, text):
    with pytest.raises(error, match=text):
        ex.group_norm(**{"x": torch.zeros(2, 3, 8), "num_groups": 2, **change})


def test_group_norm_refuses_parameters_of_two_types():
    with pytest.raises(ValueError, match="one type"):
        ex.group_norm(torch.zeros(2, 8, dtype=torch.bfloat16), 2, torch.ones(8), torch.zeros(8, dtype=torch.bfloat16))


def test_contiguity_helper_takes_views():
    t = torch.zeros(3, 4, 20)
    assert _seq.channels_contiguous(t[..., 3:9]) .data_ptr() == t[..., 3:9].data_ptr()
    assert _seq.channels_contiguous(t.transpose(1, 2)).is_contiguous()
    g = t[..., 2:14].unflatten(-1, (3, 4))
    assert _seq.channels_contiguous(g, 2).data_ptr() == g.data_ptr()
    assert _seq.channels_contiguous(g[:, :, ::2], 2).is_contiguous()
    assert _seq.channels_contiguous(t[..., :1].expand(3, 4, 6)).is_contiguous()


def rows(p=64, sb=64, st=16):
    return ctypes.byref(_lib.Rows(p, sb, st))


def test_scan_entry_points_validate_before_any_cuda_call(lib):
    p, r, null = ctypes.c_void_p(64), rows(), None

    def forward(y=p, h=p, x=r, A=p, ws=null, ws_bytes=0, dtype=0, B=1, T=8, M=8, N=4, G=1):
        return lib.exb_selective_forward(y, h, null, x, r, A, r, r, null, null, null, null, null, 1, ws, ws_bytes, dtype, B, T, M, N, G, 0, null)

    def refused(st, code, text):
        assert st == code and text in lib.exb_last_error(), (st, lib.exb_last_error())

    refused(forward(y=null), 1, b"y is required")
    refused(forward(A=null), 1, b"A is required")
    refused(forward(x=null), 1, b"x is required")
    refused(forward(x=rows(0)), 1, b"x is required")
    refused(forward(x=rows(66)), 2, b"x is not aligned")
    refused(forward(x=rows(64, -1)), 1, b"negative stride")
    refused(forward(dtype=3), 1, b"element type")
    refused(forward(B=-1), 1, b"negative size")
    refused(forward(N=129), 1, b"states")
    refused(forward(N=0), 1, b"states")
    refused(forward(G=3), 1, b"groups")
    refused(forward(G=0), 1, b"groups")
    need = lib.exb_selective_workspace_bytes(1, 4096, 8, 4, 1, 0)
    assert need > 0
    refused(forward(T=4096), 1, b"bytes of workspace")
    refused(forward(T=4096, ws=p, ws_bytes=need - 1), 1, b"bytes of workspace")
    assert forward(B=0) == 0 and forward(T=0) == 0 and forward(M=0) == 0
    assert lib.exb_selective_workspace_bytes(1, 8, 8, 4, 3, 0) == 0 and lib.exb_selective_workspace_bytes(0, 8, 8, 4, 1, 1) == 0
    assert lib.exb_selective_checkpoint_floats(2, 9, 8, 5) == 2 * 2 * 8 * 8

    def backward(dx=p, dz=null, z=null, ckpt=p, ws=p, ws_bytes=1 << 40):
        return lib.exb_selective_backward(dx, p, p, p, p, null, dz, null, null, r, null, ckpt, r, r, p, r, r, null, z, null, null, 1, ws, ws_bytes,
                                          0, 1, 8, 8, 4, 1, 0, null)

    refused(backward(dx=null), 1, b"dx is required")
    refused(backward(ckpt=null), 1, b"ckpt is required")
    refused(backward(z=r), 1, b"dz is required")
    refused(backward(ws=null), 1, b"bytes of workspace")
    refused(backward(ws_bytes=8), 1, b"bytes of workspace")
    refused(backward(ckpt=ctypes.c_void_p(68)), 2, b"ckpt is not aligned")

    refused(lib.exb_selective_step(p, p, 31, r, r, p, r, r, null, null, null, 1, 0, 2, 8, 4, 1, 0, null), 1, b"overlap")
    refused(lib.exb_selective_step(null, p, 32, r, r, p, r, r, null, null, null, 1, 0, 2, 8, 4, 1, 0, null), 1, b"y is required")
    assert lib.exb_selective_step(p, p, 32, r, r, p, r, r, null, null, null, 1, 0, 0, 8, 4, 1, 0, null) == 0


def test_conv_and_norm_entry_points_validate_before_any_cuda_call(lib):
    p, r, null = ctypes.c_void_p(64), rows(), None

    def refused(st, code, text):
        assert st == code and text in lib.exb_last_error(), (st, lib.exb_last_error())

    def conv(y=p, w=p, act=0, dtype=0, B=1, T=8, M=8, W=4):
        return lib.exb_causal_conv_forward(y, null, r, w, null, null, null, act, 1, dtype, B, T, M, W, 0, null)

    refused(conv(y=null), 1, b"y is required")
    refused(conv(w=null), 1, b"weight is required")
    refused(conv(W=9), 1, b"filters")
    refused(conv(W=0), 1, b"filters")
    refused(conv(act=2), 1, b"activation")
    refused(conv(dtype=7), 1, b"element type")
    refused(conv(T=-1), 1, b"negative size")
    assert conv(T=0) == 0
    refused(lib.exb_causal_conv_backward(p, p, null, null, r, null, r, p, null, null, null, 0, 1, null, 0, 0, 1, 8, 8, 4, 0, null), 1, b"workspace")
    refused(lib.exb_causal_conv_step(p, p, 23, r, p, null, 0, 1, 0, 2, 8, 4, 0, null), 1, b"overlap")
    refused(lib.exb_causal_conv_step(p, null, 24, r, p, null, 0, 1, 0, 2, 8, 4, 0, null), 1, b"state is required")

    def norm(y=p, act=0, eps=1e-5, R=2, S=3, C=8, G=2, ws=null, ws_bytes=0):
        return lib.exb_group_norm_forward(y, p, p, r, null, null, eps, act, 1, ws, ws_bytes, 0, R, S, C, G, 0, null)

    refused(norm(y=null), 1, b"y is required")
    refused(norm(G=3), 1, b"groups")
    refused(norm(C=16385, G=1), 1, b"at most 16384")
    refused(norm(act=3), 1, b"activation")
    refused(norm(eps=-1.0), 1, b"eps")
    refused(norm(R=-1), 1, b"negative size")
    refused(lib.exb_group_norm_backward(p, null, null, r, r, p, p, null, null, 0, 1, null, 0, 0, 2, 3, 8, 2, 0, null), 1, b"workspace")
    assert norm(R=0) == 0 and norm(S=0) == 0


def test_layers_host_side():
    layer = ex.layers.SelectiveLeak(8, num_states=4, groups=2)
    assert layer.h is None and "h" not in layer.state_dict() and layer.inner_channels == 16
    s = torch.nn.functional.softplus(layer.step_bias)
    assert (s >= 0.001 * 0.999).all() and (s <= 0.1 * 1.001).all()
    with pytest.raises(ValueError, match="'groups'"):
        ex.layers.SelectiveLeak(8, groups=3)
    with pytest.raises(ValueError, match="'norm_groups'"):
        ex.layers.SelectiveLeak(8, norm_groups=3)
    with pytest.raises(ValueError, match="step sizes"):
        ex.layers.SelectiveLeak(8, step_min=0.0)
    with pytest.raises(ValueError, match="SelectiveLeak takes"):
        layer(torch.zeros(2, 3, 9))
    with pytest.raises(_lib.ExodusLibraryError, match="only run on CUDA"):
        layer(torch.zeros(2, 3, 8))
    assert "activation='silu'" in repr(ex.layers.GroupNorm(2, 8, activation="silu"))
    with pytest.raises(ValueError, match="'activation'"):
        ex.layers.GroupNorm(2, 8, activation="tanh")
    with pytest.raises(ValueError, match="made for 8 channels"):
        ex.layers.GroupNorm(2, 8)(torch.zeros(2, 9))
    with pytest.raises(ValueError, match="dimensions"):
        ex.layers.GroupNorm(2, 8)(torch.zeros(8))


@pytest.mark.parametrize("name", ["dt", "A", "B", "C"])
def test_what_the_scan_cannot_do_without(name):
    with pytest.raises(TypeError, match=f"'{name}' must be a tensor"):
        ex.selective_scan(**{**scan_args(), name: None})
    a = {k: (v[:, 0] if v.ndim > 2 else v) for k, v in scan_args().items()}
    with pytest.raises(TypeError, match=f"'{name}' must be a tensor"):
        ex.selective_step(**{"h": torch.zeros(2, 8, 4), **a, name: None})


def test_steps_need_their_state():
    a = {k: (v[:, 0] if v.ndim > 2 else v) for k, v in scan_args().items()}
    with pytest.raises(TypeError, match="'h' must be a tensor"):
        ex.selective_step(None, **a)
    with pytest.raises(TypeError, match="'state' must be a tensor"):
        ex.causal_conv_step(None, torch.zeros(2, 8), torch.zeros(8, 4))
    with pytest.raises(TypeError, match="'weight' must be a tensor"):
        ex.causal_conv(torch.zeros(2, 5, 8), None)
    with pytest.raises(TypeError, match="'weight' must be a tensor"):
        ex.group_norm(torch.zeros(2, 8), 2, [1.0] * 8)
