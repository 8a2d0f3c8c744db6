"""residual_norm, norm_gate, gated_linear and rotary without a GPU: registration, Meta inference, refusals of the Python implementations and the C ABI's
status codes (nothing is launched)."""

import ctypes
import math
import os
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import ops_rec
from ops_rec import _layer, _native

OPS = torch.ops.ops_rec


def test_reached_through_the_public_groups():
    a, t = ops_rec.ascendc.activation, ops_rec.ascendc.attention
    assert a.residual_norm is OPS.residual_norm and a.norm_gate is OPS.norm_gate and t.rotary is OPS.rotary
    for name in ("residual_norm", "residual_norm_backward", "norm_gate", "norm_gate_backward", "gated_linear", "gated_linear_backward"):
        assert name in a.__all__
    assert "rotary" in t.__all__ and callable(ops_rec.rotary_frequencies)


def test_the_library_exports_what_the_header_declares():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = open(os.path.join(root, "include", "ops_rec_layer_mi355.h")).read()
    declared = set(re.findall(r"HSTU_API\s+[\w\s\*]+?\b(\w+)\s*\(", header))
    assert declared == set(_native.LAYER_SYMBOLS)
    for name in declared:
        getattr(_native.load(), name)


def test_meta_inference():
    x, r, g = torch.empty(5, 24, device="meta", dtype=torch.bfloat16), torch.empty(5, 24, device="meta"), torch.empty(24, device="meta")
    y, s = OPS.residual_norm(x, r, g)
    assert (y.shape, y.dtype, s.shape, s.dtype) == ((5, 24), torch.bfloat16, (5, 24), torch.float32)
    assert OPS.norm_gate(x, x, g).dtype == torch.bfloat16 and OPS.norm_gate(x, x, g, None, r).dtype == torch.float32
    grads = OPS.residual_norm_backward(y, s, x, None, s, g, g, True, torch.bfloat16, 1e-5, False)
    assert [tuple(t.shape) for t in grads] == [(5, 24), (5, 24), (24,), (24,), (24,)] and grads[0].dtype == torch.bfloat16 and grads[1].dtype == torch.float32
    grads = OPS.residual_norm_backward(y, None, x, x, None, g, None, False, torch.bfloat16, 1e-5, False)
    assert [tuple(t.shape) for t in grads] == [(0,), (5, 24), (24,), (0,), (0,)]
    x, w = torch.empty(5, 24, device="meta", dtype=torch.float16), torch.empty(80, 24, device="meta", dtype=torch.float16)
    assert [tuple(t.shape) for t in OPS.gated_linear(x, w, None, "gelu", True)] == [(5, 40), (0,)]
    wide = torch.empty(5, 200, device="meta", dtype=torch.float16), torch.empty(80, 200, device="meta", dtype=torch.float16)
    assert [tuple(t.shape) for t in OPS.gated_linear(*wide, None, "gelu", True)] == [(5, 40), (5, 120)] and OPS.gated_linear(*wide)[1].shape == (0,)
    grads = OPS.gated_linear_backward(torch.empty(5, 40, device="meta"), x, w, None, x, "silu", [True, False, True])
    assert [tuple(t.shape) for t in grads] == [(5, 24), (0,), (0,)]
    q, k = torch.empty(7, 4, 16, device="meta"), torch.empty(7, 2, 16, device="meta")
    f = torch.empty(8, device="meta", dtype=torch.float64)
    assert [t.shape for t in OPS.rotary(q, k, f, torch.empty(3, device="meta", dtype=torch.int32))] == [q.shape, k.shape]
    for bad in (lambda: OPS.residual_norm(x[0], r, g), lambda: OPS.residual_norm(x, r[:3], g), lambda: OPS.norm_gate(x[0], x, g), lambda: OPS.rotary(q[0], k, f)):
        with pytest.raises(RuntimeError):
            bad()


def test_fake_tensors_that_record_gradients():
    with FakeTensorMode():
        x = torch.empty(5, 24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        g = torch.empty(24, device="cuda", requires_grad=True)
        y, s = OPS.residual_norm(x, x.detach(), g)
        assert y.requires_grad and s.requires_grad
        assert OPS.norm_gate(x, None, g).requires_grad and not OPS.norm_gate(x.detach(), None, g.detach()).requires_grad
        q = torch.empty(5, 2, 8, device="cuda", requires_grad=True)
        f, offs = torch.empty(4, device="cuda", dtype=torch.float64), torch.empty(3, device="cuda", dtype=torch.int32)
        assert OPS.rotary(q, q, f, offs)[0].requires_grad
        with pytest.raises(NotImplementedError, match="frequencies"):
            OPS.rotary(q, q, f.requires_grad_(True), offs)
        with torch.no_grad():
            assert not OPS.rotary(q, q, f, offs)[0].requires_grad
        hidden, mixed = OPS.gated_linear(x, torch.empty(32, 24, device="cuda", dtype=torch.bfloat16), None, "silu", True)
        assert hidden.requires_grad and not mixed.requires_grad


def test_refusals_of_the_norms():
    x, g = torch.zeros(4, 24), torch.ones(24)
    norm, gate = _layer.residual_norm, _layer.norm_gate
    wide = torch.zeros(1, 16385)
    for call, text in [
        (lambda: norm(x[0], x, g), "x should be 2D"),
        (lambda: norm(x.double(), x, g), "unsupported dtype"),
        (lambda: norm(x[:, :0], x[:, :0], g[:0]), "columns"),
        (lambda: norm(x, x[:3], g), "residual must have the shape of x"),
        (lambda: norm(x, x.half(), g), "residual must be float32 or of the dtype of x"),
        (lambda: norm(x.bfloat16(), x.half(), g), "residual must be float32 or of the dtype of x"),
        (lambda: norm(x, x, g[:3]), "gamma must have x.size\\(1\\) elements"),
        (lambda: norm(x, x, g.half()), "gamma must be float32 or of the dtype of x"),
        (lambda: norm(x.half(), x.half(), g, g.half()), "beta must have the dtype of gamma"),
        (lambda: norm(x, x, g, None, g[None]), "scale must have x.size\\(1\\) elements"),
        (lambda: norm(x, x, g, None, None, -1.0), "epsilon must not be negative"),
        (lambda: norm(x, x, g, None, None, math.nan), "epsilon must not be negative"),
        (lambda: norm(wide, wide, wide[0]), "at most 16384 columns share a mean"),
        (lambda: norm(x, x, g), "x must be a GPU tensor"),
        (lambda: gate(x, x[:, :3], g), "gate must have the shape of x"),
        (lambda: gate(x, x.half(), g), "gate must have the dtype of x"),
        (lambda: gate(x, x, g, None, None, 1.0, 5), "multiple of groups"),
        (lambda: gate(x, x, g, None, None, 1.0, 0), "multiple of groups"),
        (lambda: gate(torch.zeros(1, (1 << 20) + 8), None, g, None, None, 1.0, 128), "at most 2\\^20"),
        (lambda: gate(torch.zeros(1, 1).expand(1 << 27, 16), None, g, None, None, 1.0, 16), "rows \\* groups must stay below"),
        (lambda: gate(x.half(), None, g, None, x.bfloat16()), "residual must be float32 or of the dtype of x"),
        (lambda: gate(x, None, g), "x must be a GPU tensor"),
        (lambda: _layer.norm_gate_backward(x, x.half(), None, g, None, False, 1.0, 1, 1e-5, False, False), "grad must have the dtype of x"),
        (lambda: _layer.residual_norm_backward(x, x, x, None, None, g, None, False, torch.float32, 1e-5, False), "needs the sum"),
        (lambda: _layer.residual_norm_backward(x, x, x, x, None, g, None, False, torch.float32, 1e-5, False), "the sum is given where the stream is float32"),
        (lambda: _layer.residual_norm_backward(x, x, None, None, x, g, g, False, torch.float32, 1e-5, False), "x must be given"),
        (lambda: _layer.residual_norm_backward(x[:3], x, x, None, x, g, g, False, torch.float32, 1e-5, False), "y_grad must be"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_refusals_of_rotary():
    q, f, offs = torch.zeros(6, 2, 8), torch.ones(4, dtype=torch.float64), torch.tensor([0, 6])
    for call, text in [
        (lambda: _layer.rotary(q[0], q, f, offs), "3D"),
        (lambda: _layer.rotary(q, q.half(), f, offs), "q and k must both be"),
        (lambda: _layer.rotary(q.double(), q.double(), f, offs), "q and k must both be"),
        (lambda: _layer.rotary(q, q[:5], f, offs), "same rows and head dim"),
        (lambda: _layer.rotary(q, q, f.float(), offs), "float64"),
        (lambda: _layer.rotary(q, q, f[:0], offs), "at least one"),
        (lambda: _layer.rotary(q, q, torch.ones(5, dtype=torch.float64), offs), "at most headDim / 2"),
        (lambda: _layer.rotary(q, q, f), "seq_offset or positions must be given"),
        (lambda: _layer.rotary(q, q, f, offs, None, torch.zeros(6, dtype=torch.int64)), "not both"),
        (lambda: _layer.rotary(q, q, f, None, offs, torch.zeros(6, dtype=torch.int64)), "start goes with seq_offset"),
        (lambda: _layer.rotary(q, q, f, offs.float()), "int32 or int64"),
        (lambda: _layer.rotary(q, q, f, offs[:1]), "at least two element"),
        (lambda: _layer.rotary(q, q, f, offs, offs), "start must have an element per sequence"),
        (lambda: _layer.rotary(q, q, f, None, None, offs), "positions must have an element per row"),
        (lambda: _layer.rotary(q, q, f, offs), "q must be a GPU tensor"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_refusals_of_gated_linear():
    x, w, b = torch.zeros(4, 24).half(), torch.zeros(32, 24).half(), torch.zeros(32).half()
    call, back = _layer.gated_linear, _layer.gated_linear_backward
    odd = torch.zeros(4, 20).half()
    for fn, text in [
        (lambda: call(x[0], w), "x should be 2D"),
        (lambda: call(x, w[0]), "weight should be 2D"),
        (lambda: call(x.float(), w.float()), "x must be float16 or bfloat16"),
        (lambda: call(x, w.bfloat16()), "weight must have the dtype of x"),
        (lambda: call(x, w, b, "relu"), "activation must be one of"),
        (lambda: call(x, w[:31]), "weight must be \\[2 \\* inner, 24\\]"),
        (lambda: call(x, w[:, :16]), "weight must be \\[2 \\* inner, 24\\]"),
        (lambda: call(x, w[:24]), "multiples of 8"),
        (lambda: call(odd, torch.zeros(32, 20).half()), "multiples of 8"),
        (lambda: call(x[:, :0], w[:, :0]), "multiples of 8"),
        (lambda: call(torch.zeros(2, 8).half(), torch.zeros(2 * ((1 << 21) + 8), 8).half()), "at most 2\\^21"),
        (lambda: call(x, w, b[:31]), "bias must have 2 \\* inner elements"),
        (lambda: call(x, w, b.float()), "bias must have the dtype of x"),
        (lambda: call(x, w, b), "x must be a GPU tensor"),
        (lambda: back(torch.zeros(4, 15).half(), x, w, b, b[:0], "silu", [True] * 3), "grad must be"),
        (lambda: back(torch.zeros(4, 16), x, w, b, b[:0], "silu", [True] * 3), "grad must be"),
        (lambda: back(torch.zeros(4, 16).half(), x, w, b, b, "silu", [True] * 3), "mixed must be empty or"),
        (lambda: back(torch.zeros(4, 16).half(), x, w, b, b[:0], "silu", [True]), "wanted must have three"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            fn()


def test_frequencies():
    f, m = ops_rec.rotary_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 100.0**-0.25, 0.1, 100.0**-0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(ops_rec.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0)[0], f / 4)
    b, _ = ops_rec.rotary_frequencies(8, base=100.0, scaling="base", factor=4.0)
    assert b[0] == 1.0 and abs(b[-1] / f[-1] * 4.0 - 1) < 1e-12  # the highest stays, the lowest falls by the factor
    base = ops_rec.rotary_frequencies(64)[0]
    p, m = ops_rec.rotary_frequencies(64, scaling="parts", factor=8.0, original_length=4096)
    turns = base * 4096 / (2 * math.pi)
    assert torch.equal(p[turns > 40], base[turns > 40]) and torch.allclose(p[turns < 0.7], base[turns < 0.7] / 8)
    assert (p <= base).all() and (p >= base / 8 * (1 - 1e-12)).all() and (p[1:] < p[:-1]).all() and abs(m - (1 + 0.1 * math.log(8.0))) < 1e-15
    for kw in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=-1.0), dict(rotary_dim=8, factor=0.0), dict(rotary_dim=8, scaling="no"),
               dict(rotary_dim=2, scaling="base"), dict(rotary_dim=8, scaling="parts"), dict(rotary_dim=8, scaling="parts", original_length=64, fast=1.0)):  # fmt: skip
        with pytest.raises(RuntimeError):
            ops_rec.rotary_frequencies(**kw)


def _norm_params():
    p = _native.ResidualNormParams()
    p.struct_size = ctypes.sizeof(p)
    p.x = p.residual = p.gamma = p.y = p.sum = 0x1000  # never dereferenced
    p.rows, p.cols, p.x_stride, p.residual_stride = 10, 64, 64, 64
    p.dtype, p.stream_dtype, p.affine_dtype, p.epsilon = _native.DT_BF16, _native.DT_FP32, _native.DT_FP32, 1e-5
    return p


def _gate_params():
    p = _native.NormGateParams()
    p.struct_size = ctypes.sizeof(p)
    p.x = p.gamma = p.out = 0x1000
    p.rows, p.cols, p.x_stride, p.groups, p.residual_scale = 10, 64, 64, 4, 1.0
    p.dtype = p.stream_dtype = p.affine_dtype = _native.DT_BF16
    p.epsilon = 1e-5
    return p


def _rotary_params():
    p = _native.RotaryParams()
    p.struct_size = ctypes.sizeof(p)
    p.q = p.k = p.q_out = p.k_out = p.frequencies = p.seq_offset = 0x1000
    p.rows, p.heads_q, p.heads_k, p.dim, p.pairs, p.n_offsets = 10, 2, 2, 64, 32, 3
    return p


def _gated_params():
    p = _native.GatedLinearParams()
    p.struct_size = ctypes.sizeof(p)
    p.x = p.weight = p.hidden = 0x1000
    p.rows, p.cols, p.inner, p.dtype = 10, 64, 128, _native.DT_BF16
    return p


@pytest.mark.parametrize(
    "name,make,changes",
    [
        ("gated_linear_fwd", _gated_params,
         [("struct_size", 4, 161002), ("x", None, 161001), ("weight", None, 161001), ("hidden", None, 161001), ("rows", 0, 161002), ("cols", 60, 161002),
          ("inner", 0, 161002), ("inner", (1 << 21) + 8, 161002), ("cols", (1 << 21) + 8, 161002), ("dtype", _native.DT_FP32, 161002),
          ("activation", 3, 161002), ("activation", -1, 161002), ("x", 0x1008, 161002), ("bias", 0x1002, 161002)]),
        ("residual_norm_fwd", _norm_params,
         [("struct_size", 4, 161002), ("x", None, 161001), ("residual", None, 161001), ("gamma", None, 161001), ("y", None, 161001), ("sum", None, 161001),
          ("rows", 0, 161002), ("cols", 0, 161002), ("cols", 16385, 161002), ("rows", 1 << 31, 161002), ("x_stride", -1, 161002), ("dtype", 3, 161002),
          ("stream_dtype", _native.DT_FP16, 161002), ("affine_dtype", _native.DT_FP16, 161002), ("epsilon", -1.0, 161002), ("epsilon", math.nan, 161002)]),
        ("norm_gate_fwd", _gate_params,
         [("struct_size", 4, 161002), ("x", None, 161001), ("gamma", None, 161001), ("out", None, 161001), ("groups", 0, 161002), ("groups", 5, 161002), ("cols", 1 << 22, 161002),
          ("stream_dtype", _native.DT_FP32, 161002), ("gate_stride", -8, 161002), ("rows", 1 << 30, 161002)]),
        ("rotary_fwd", _rotary_params,
         [("struct_size", 4, 161002), ("q", None, 161001), ("frequencies", None, 161001), ("seq_offset", None, 161002), ("positions", 0x1000, 161002),
          ("dtype", 3, 161002), ("rows", 0, 161002), ("heads_q", 0, 161002), ("heads_k", 65537, 161002), ("dim", 1, 161002), ("pairs", 33, 161002),
          ("pairs", 0, 161002), ("n_offsets", 1, 161002), ("q_stride_row", -1, 161002), ("start_dtype", 2, 161002)]),
    ],
)  # fmt: skip
def test_c_abi_refuses_before_any_device_call(name, make, changes):
    call = getattr(_native.load(), name)
    assert call(None, None) == 161001
    for field, value, code in changes:
        p = make()
        setattr(p, field, value)
        assert call(ctypes.byref(p), None) == code, (field, value, _native.last_error())


def test_c_abi_of_the_backward():
    lib = _native.load()
    p = _native.ResidualNormBwdParams()
    p.struct_size = ctypes.sizeof(p)
    p.fwd = _norm_params()
    p.sum = p.y_grad = p.sum_grad = p.x_grad = p.residual_grad = p.gamma_grad = 0x1000
    size = ctypes.c_uint64(0)
    assert lib.residual_norm_bwd_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0
    one = size.value
    assert one > 0 and one % (64 * 4) == 0
    p.beta_grad, p.fwd.scale, p.scale_grad = 0x1000, 0x1000, 0x1000
    assert lib.residual_norm_bwd_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0 and size.value == 3 * one
    assert lib.residual_norm_bwd(ctypes.byref(p), None, 0, None) == 161004 and "workspace" in _native.last_error()
    p.sum = None
    assert lib.residual_norm_bwd_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 161001
    p.sum, p.fwd.scale = 0x1000, None  # scale_grad without scale
    assert lib.residual_norm_bwd_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 161002
    w = _native.GatedLinearBwdParams()
    w.struct_size = ctypes.sizeof(w)
    w.fwd = _gated_params()
    assert lib.gated_linear_bwd_workspace_size(ctypes.byref(w), ctypes.byref(size)) == 161001  # no mixed, no grad
    w.fwd.mixed = w.grad = w.weight_grad = 0x1000
    assert lib.gated_linear_bwd_workspace_size(ctypes.byref(w), ctypes.byref(size)) == 0 and size.value >= 10 * 256 * 2
    assert lib.gated_linear_bwd(ctypes.byref(w), 0x1000, size.value - 1, None) == 161004
    assert lib.gated_linear_bwd(ctypes.byref(w), 0x1008, size.value, None) == 161004
    kept = size.value
    w.fwd.mixed = w.fwd.hidden = None  # g and u are multiplied again
    assert lib.gated_linear_bwd_workspace_size(ctypes.byref(w), ctypes.byref(size)) == 0 and size.value == kept
    w.bias_grad = 0x1000  # (two rows of column sums of both projections)
    assert lib.gated_linear_bwd_workspace_size(ctypes.byref(w), ctypes.byref(size)) == 0 and size.value >= kept + 2 * 256 * 4
    assert lib.gated_linear_fwd(ctypes.byref(w.fwd), None) == 161001  # (a forward writes one of the two)
    w.x_grad = 0x1004
    assert lib.gated_linear_bwd_workspace_size(ctypes.byref(w), ctypes.byref(size)) == 161002
    g = _native.NormGateBwdParams()
    g.struct_size = ctypes.sizeof(g)
    g.fwd = _gate_params()
    g.out_grad = g.x_grad = g.gamma_grad = 0x1000
    assert lib.norm_gate_bwd_workspace_size(ctypes.byref(g), ctypes.byref(size)) == 0 and size.value > 0
    g.gate_grad = 0x1000  # without a gate
    assert lib.norm_gate_bwd_workspace_size(ctypes.byref(g), ctypes.byref(size)) == 161001
