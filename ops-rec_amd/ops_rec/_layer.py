"""Operators around HSTU attention in a layer, beside those of ``_activation``.  Extensions: the reference has none of the kind.

``residual_norm(x, residual, gamma, beta, scale)``: the residual sum and the norm in front of a block, ``norm_gate(x, gate, gamma, beta, residual)``: the
norm behind it, by parts of a row, with its gate and back onto the stream; ``gated_linear(x, weight, bias)``: both projections of a gated
feed-forward block with activation and product -- all with gradients (``ops_rec.ascendc.activation``);
``rotary(q, k, frequencies, seq_offset)``: rotary positions on jagged queries and keys (``ops_rec.ascendc.attention``), with
``rotary_frequencies`` for the table of frequencies, stretched for contexts longer than those a model was trained on.

Registered as operators of ``torch.ops.ops_rec``; device tensors in canonical form go to the native kernels of
``csrc/torch_binding_layer.cpp``, everything else comes here, where the checks and conversions are.  The autograd formulas are here too; for
device tensors C++ nodes with the same formulas stand in front of them where the binding is built.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad

from . import _native
from ._ops import _DTYPE_CODE, _PYTHON_KERNELS, _check, _lib_def, _lib_meta, _ptr
from ._paged_fp8 import _aligned, _call

NORM_MAX_LEN = 16384  # columns that share a mean, at most
MAX_NORM_COLUMNS = 1 << 20
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)

_lib_def.define("residual_norm(Tensor x, Tensor residual, Tensor gamma, Tensor? beta=None, Tensor? scale=None, float epsilon=1e-5, bool rms=False) -> "
                "(Tensor, Tensor)")  # fmt: skip
_lib_def.define("residual_norm_backward(Tensor? y_grad, Tensor? sum_grad, Tensor? x, Tensor? residual, Tensor? sum, Tensor gamma, Tensor? scale, "
                "bool has_beta, ScalarType x_dtype, float epsilon, bool rms) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")  # fmt: skip
_lib_def.define("norm_gate(Tensor x, Tensor? gate, Tensor gamma, Tensor? beta=None, Tensor? residual=None, float residual_scale=1.0, int groups=1, "
                "float epsilon=1e-5, bool rms=False, bool silu=False) -> Tensor")  # fmt: skip
_lib_def.define("norm_gate_backward(Tensor grad, Tensor x, Tensor? gate, Tensor gamma, Tensor? beta, bool has_residual, float residual_scale, int groups, "
                "float epsilon, bool rms, bool silu) -> (Tensor, Tensor, Tensor, Tensor)")  # fmt: skip
_lib_def.define("rotary(Tensor q, Tensor k, Tensor frequencies, Tensor? seq_offset=None, Tensor? start=None, Tensor? positions=None, "
                "bool interleaved=False, float magnitude=1.0, bool inverse=False) -> (Tensor, Tensor)")  # fmt: skip
_lib_def.define("gated_linear(Tensor x, Tensor weight, Tensor? bias=None, str activation='silu', bool keep=False) -> (Tensor, Tensor)")
_lib_def.define("gated_linear_backward(Tensor grad, Tensor x, Tensor weight, Tensor? bias, Tensor mixed, str activation, bool[3] wanted) -> "
                "(Tensor, Tensor, Tensor)")  # fmt: skip


def _on_device(device, named) -> None:
    _check(device.type == "cuda", f"{named[0][0]} must be a GPU tensor, but it is on {device}")
    for name, t in named:
        _check(t is None or t.device == device, f"{name} must be on the device of {named[0][0]} ({device}), but it is on {getattr(t, 'device', None)}")


def _no_tangents(op, *tensors) -> None:
    """No formulas for forward-mode differentiation: a tangent would be lost."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{op}: forward-mode differentiation is not implemented; do not pass inputs with a tangent")


def _rows(t: Optional[torch.Tensor]):
    """``t`` with the values of a row side by side; rows stay where they are."""
    return t if t is None or t.stride(-1) == 1 or t.size(-1) <= 1 else t.contiguous()


def _dense(t: Optional[torch.Tensor]):
    return None if t is None else t.contiguous()


# ---------------------------------------------------------------------------------------------------- norms ----


def _norm_shapes(x, gamma, beta, epsilon, groups, **planes) -> None:
    _check(x.dim() == 2, "The x should be 2D")
    _check(x.dtype in _FLOATS, f"unsupported dtype {x.dtype}")
    _check(0 < x.size(1) <= MAX_NORM_COLUMNS, f"x must have columns, at most 2^20, but it is {list(x.shape)}")
    for name, t in planes.items():
        _check(t is None or t.shape == x.shape, f"{name} must have the shape of x ({list(x.shape)}), but it is {list(getattr(t, 'shape', ()))}")
    _check(int(groups) >= 1 and x.size(1) % int(groups) == 0, f"the columns ({x.size(1)}) must be a multiple of groups, but groups is {groups}")
    _check(x.size(1) // int(groups) <= NORM_MAX_LEN, f"at most {NORM_MAX_LEN} columns share a mean, but there are {x.size(1) // int(groups)}")
    _check(x.size(0) * int(groups) < 1 << 31, f"rows * groups must stay below 2^31, but there are {x.size(0)} rows and {groups} groups")
    _check(float(epsilon) >= 0.0, f"epsilon must not be negative, but it is {epsilon}")


def _norm_columns(x, **columns) -> None:
    """gamma, beta and scale: a value per column, of one type, fp32 or that of x."""
    gamma = columns["gamma"]
    _check(gamma.dtype in (torch.float32, x.dtype), f"gamma must be float32 or of the dtype of x, but it is {gamma.dtype}")
    for name, t in columns.items():
        if t is not None:
            _check(t.dim() == 1 and t.numel() == x.size(1), f"{name} must have x.size(1) elements ({x.size(1)}), but it is {list(t.shape)}")
            _check(t.dtype == gamma.dtype, f"{name} must have the dtype of gamma ({gamma.dtype}), but it is {t.dtype}")


def _stream_dtype(x, residual) -> None:
    _check(residual is None or residual.dtype in (torch.float32, x.dtype),
           f"residual must be float32 or of the dtype of x, but it is {getattr(residual, 'dtype', None)}")  # fmt: skip


def _residual_norm_checks(x, residual, gamma, beta, scale, epsilon) -> None:
    _norm_shapes(x, gamma, beta, epsilon, 1, residual=residual)
    _norm_columns(x, gamma=gamma, beta=beta, scale=scale)
    _stream_dtype(x, residual)


def _describe_residual_norm(p, x, residual, gamma, beta, scale, epsilon, rms, shape, dtype, stream_dtype):
    p.struct_size, p.rms = ctypes.sizeof(p), int(bool(rms))
    p.x, p.residual, p.gamma, p.beta, p.scale = _ptr(x), _ptr(residual), _ptr(gamma), _ptr(beta), _ptr(scale)
    p.rows, p.cols = shape
    p.x_stride = x.stride(0) if x is not None else 0
    p.residual_stride = residual.stride(0) if residual is not None else 0
    p.dtype, p.stream_dtype, p.affine_dtype, p.epsilon = _DTYPE_CODE[dtype], _DTYPE_CODE[stream_dtype], _DTYPE_CODE[gamma.dtype], float(epsilon)


def residual_norm(x, residual, gamma, beta=None, scale=None, epsilon=1e-5, rms=False):
    """``sum = residual + scale * x`` and ``y = norm(sum) * gamma + beta`` over rows [rows, cols]: what stands in front of a block of a layer,
    ``x`` being the block before's output.  Returns ``(y, sum)``, ``y`` in the type of ``x``, ``sum`` in that of ``residual``.

    ``norm`` takes mean and variance over the columns, or with ``rms`` the root mean square alone.  x is fp32, bf16 or fp16, the residual stream of
    the same type or fp32, gamma, beta and scale (one value per column) all fp32 or all of the type of x.  Rows may be strided; arithmetic is fp32, and
    y is the norm of the sum as it is before it is rounded."""
    _no_tangents("residual_norm", x, residual, gamma, beta, scale)
    _residual_norm_checks(x, residual, gamma, beta, scale, epsilon)
    _on_device(x.device, (("x", x), ("residual", residual), ("gamma", gamma), ("beta", beta), ("scale", scale)))
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    if x.size(0) == 0:
        return y, total
    xc, rc, gc, bc, sc = _rows(x), _rows(residual), _dense(gamma), _dense(beta), _dense(scale)
    p = _native.ResidualNormParams()
    _describe_residual_norm(p, xc, rc, gc, bc, sc, epsilon, rms, x.shape, x.dtype, residual.dtype)
    p.y, p.sum = y.data_ptr(), total.data_ptr()
    _call("residual_norm_fwd", p, x.device, workspace=False)
    return y, total


def residual_norm_meta(x, residual, gamma, beta=None, scale=None, epsilon=1e-5, rms=False):
    _check(x.dim() == 2, "The x should be 2D")
    _check(x.shape == residual.shape, "residual must have the shape of x")
    return x.new_empty(x.shape), x.new_empty(x.shape, dtype=residual.dtype)


def residual_norm_backward(y_grad, sum_grad, x, residual, sum, gamma, scale, has_beta, x_dtype, epsilon, rms):  # noqa: A002
    """Gradients of ``residual_norm``'s x, residual, gamma, beta and scale, those that the call has.  Gradients that are None count as zeros.  The
    norm is taken again of ``sum`` where the stream is fp32 (x is then needed for scale only), of ``residual`` and ``x`` otherwise.
    Where x's gradient is the residual's (no scale, one type), it comes back empty, as does what has no input."""
    given = sum if sum is not None else residual
    _check(given is not None, "residual_norm_backward needs the sum of an fp32 stream, or the residual of another")
    shape, device, stream_dtype = given.shape, given.device, given.dtype
    _check(len(shape) == 2 and shape[1] > 0, "the sum should be 2D")
    _check(x_dtype in _FLOATS and stream_dtype in (torch.float32, x_dtype), f"unsupported dtypes {x_dtype} and {stream_dtype}")
    _check((sum is not None) == (stream_dtype == torch.float32), "the sum is given where the stream is float32, and only there")
    _check(x is not None or (sum is not None and scale is None), "x must be given with a scale, and where the stream is not float32")
    for name, t, dtype in (("y_grad", y_grad, x_dtype), ("sum_grad", sum_grad, stream_dtype), ("x", x, x_dtype)):
        _check(t is None or (t.shape == shape and t.dtype == dtype), f"{name} must be {list(shape)} of {dtype}")
    like = torch.empty(0, dtype=x_dtype, device="meta").new_empty(shape)
    _residual_norm_checks(like, like.new_empty(shape, dtype=stream_dtype), gamma, None, scale, epsilon)
    _on_device(device, (("the sum", given), ("y_grad", y_grad), ("sum_grad", sum_grad), ("x", x), ("gamma", gamma), ("scale", scale)))
    apart = scale is not None or stream_dtype != x_dtype
    x_grad = torch.empty(shape if apart else (0,), dtype=x_dtype, device=device)
    residual_grad = torch.empty(shape, dtype=stream_dtype, device=device)
    make = torch.zeros if shape[0] == 0 else torch.empty
    gamma_grad, beta_grad, scale_grad = (make(shape[1] if there else 0, dtype=gamma.dtype, device=device) for there in (True, has_beta, scale is not None))
    if shape[0] != 0:
        # (tensors live until the call returns: the names hold what _describe took addresses of)
        xc, rc, sc, gc, cc, yg, sg = _rows(x), _rows(residual), _dense(sum), _dense(gamma), _dense(scale), _dense(y_grad), _dense(sum_grad)
        p = _native.ResidualNormBwdParams()
        p.struct_size = ctypes.sizeof(p)
        _describe_residual_norm(p.fwd, xc, None if sum is not None else rc, gc, None, cc, epsilon, rms, shape, x_dtype, stream_dtype)
        p.sum, p.y_grad, p.sum_grad = _ptr(sc), _ptr(yg), _ptr(sg)
        p.x_grad, p.residual_grad = _ptr(x_grad), residual_grad.data_ptr()
        p.gamma_grad, p.beta_grad, p.scale_grad = gamma_grad.data_ptr(), _ptr(beta_grad), _ptr(scale_grad)
        _call("residual_norm_bwd", p, device)
    return x_grad, residual_grad, gamma_grad, beta_grad, scale_grad


def residual_norm_backward_meta(y_grad, sum_grad, x, residual, sum, gamma, scale, has_beta, x_dtype, epsilon, rms):  # noqa: A002
    given = sum if sum is not None else residual
    apart = scale is not None or given.dtype != x_dtype
    columns = (given.size(1) if there else 0 for there in (True, has_beta, scale is not None))
    return (given.new_empty(given.shape if apart else (0,), dtype=x_dtype), given.new_empty(given.shape), *(gamma.new_empty((n,)) for n in columns))


def _residual_norm_setup(ctx, inputs, output):
    x, residual, gamma, beta, scale, epsilon, rms = inputs
    total = output[1]
    wide = total.dtype == torch.float32
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x if scale is not None or not wide else None, None if wide else residual, total if wide else None, gamma, scale)
    ctx.rest = (beta is not None, x.dtype, epsilon, rms)


def _residual_norm_grad(ctx, y_grad, sum_grad):
    x, residual, total, gamma, scale = ctx.saved_tensors
    if y_grad is None and sum_grad is None:
        return (None,) * 7
    dx, dr, dg, db, ds = torch.ops.ops_rec.residual_norm_backward(y_grad, sum_grad, x, residual, total, gamma, scale, *ctx.rest)
    apart = scale is not None or dr.dtype != ctx.rest[1]
    return dx if apart else dr, dr, dg, db if ctx.rest[0] else None, ds if scale is not None else None, None, None


def _norm_gate_checks(x, gate, gamma, beta, residual, groups, epsilon) -> None:
    _norm_shapes(x, gamma, beta, epsilon, groups, gate=gate, residual=residual)
    _norm_columns(x, gamma=gamma, beta=beta)
    _check(gate is None or gate.dtype == x.dtype, f"gate must have the dtype of x, but it is {getattr(gate, 'dtype', None)}")
    _stream_dtype(x, residual)


def _describe_norm_gate(p, x, gate, gamma, beta, residual_scale, groups, epsilon, rms, silu, stream_dtype):
    p.struct_size, p.rms = ctypes.sizeof(p), int(bool(rms))
    p.x, p.gate, p.gamma, p.beta = _ptr(x), _ptr(gate), _ptr(gamma), _ptr(beta)
    p.rows, p.cols = x.shape
    p.x_stride, p.gate_stride = x.stride(0), gate.stride(0) if gate is not None else 0
    p.groups, p.silu, p.dtype, p.stream_dtype, p.affine_dtype = int(groups), int(bool(silu)), _DTYPE_CODE[x.dtype], _DTYPE_CODE[stream_dtype], _DTYPE_CODE[gamma.dtype]
    p.epsilon, p.residual_scale = float(epsilon), float(residual_scale)


def norm_gate(x, gate, gamma, beta=None, residual=None, residual_scale=1.0, groups=1, epsilon=1e-5, rms=False, silu=False):
    """``m * gate`` with ``m = norm(x) * gamma + beta`` over rows [rows, cols]: what stands behind attention in a layer.  The norm (mean and variance,
    or the root mean square with ``rms``) goes over each of ``groups`` equal parts of a row: a head's values, with as many groups as heads.
    ``gate`` None is a gate of 1; with ``silu`` the gate is silu(gate).  With ``residual`` the result goes back onto the stream:
    ``residual + residual_scale * m * gate``, in the residual's type; without, ``residual_scale`` is not used and the result has the type of x.

    x is fp32, bf16 or fp16, the gate the same, the residual the same or fp32, gamma and beta (one value per column) both fp32 or both
    of the type of x.  Rows may be strided; arithmetic is fp32, rounded once."""
    _no_tangents("norm_gate", x, gate, gamma, beta, residual)
    _norm_gate_checks(x, gate, gamma, beta, residual, groups, epsilon)
    _on_device(x.device, (("x", x), ("gate", gate), ("gamma", gamma), ("beta", beta), ("residual", residual)))
    stream_dtype = x.dtype if residual is None else residual.dtype
    out = torch.empty(x.shape, dtype=stream_dtype, device=x.device)
    if x.size(0) == 0:
        return out
    xc, uc, rc, gc, bc = _rows(x), _rows(gate), _rows(residual), _dense(gamma), _dense(beta)
    p = _native.NormGateParams()
    _describe_norm_gate(p, xc, uc, gc, bc, residual_scale, groups, epsilon, rms, silu, stream_dtype)
    p.residual, p.residual_stride = _ptr(rc), rc.stride(0) if rc is not None else 0
    p.out = out.data_ptr()
    _call("norm_gate_fwd", p, x.device, workspace=False)
    return out


def norm_gate_meta(x, gate, gamma, beta=None, residual=None, residual_scale=1.0, groups=1, epsilon=1e-5, rms=False, silu=False):
    _check(x.dim() == 2, "The x should be 2D")
    return x.new_empty(x.shape, dtype=x.dtype if residual is None else residual.dtype)


def norm_gate_backward(grad, x, gate, gamma, beta, has_residual, residual_scale, groups, epsilon, rms, silu):
    """Gradients of ``norm_gate``'s x, gate, gamma and beta (empty where the call has no gate, no beta); the residual's is ``grad`` itself."""
    _norm_gate_checks(x, gate, gamma, beta, grad, groups, epsilon)
    _check(has_residual or grad.dtype == x.dtype, f"without a residual grad must have the dtype of x, but it is {grad.dtype}")
    _on_device(x.device, (("x", x), ("grad", grad), ("gate", gate), ("gamma", gamma), ("beta", beta)))
    x_grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    gate_grad = torch.empty(x.shape if gate is not None else (0,), dtype=x.dtype, device=x.device)
    make = torch.zeros if x.size(0) == 0 else torch.empty
    gamma_grad, beta_grad = (make(x.size(1) if there else 0, dtype=gamma.dtype, device=x.device) for there in (True, beta is not None))
    if x.size(0) != 0:
        xc, uc, dc, gc, bc = _rows(x), _rows(gate), _dense(grad), _dense(gamma), _dense(beta)
        p = _native.NormGateBwdParams()
        p.struct_size = ctypes.sizeof(p)
        _describe_norm_gate(p.fwd, xc, uc, gc, bc, residual_scale, groups, epsilon, rms, silu, grad.dtype)
        p.fwd.residual = dc.data_ptr() if has_residual else None  # (says that there is one)
        p.out_grad, p.x_grad, p.gate_grad = dc.data_ptr(), x_grad.data_ptr(), _ptr(gate_grad)
        p.gamma_grad, p.beta_grad = gamma_grad.data_ptr(), _ptr(beta_grad)
        _call("norm_gate_bwd", p, x.device)
    return x_grad, gate_grad, gamma_grad, beta_grad


def norm_gate_backward_meta(grad, x, gate, gamma, beta, has_residual, residual_scale, groups, epsilon, rms, silu):
    return (x.new_empty(x.shape), x.new_empty(x.shape if gate is not None else (0,)), gamma.new_empty((x.size(1),)),
            gamma.new_empty((x.size(1) if beta is not None else 0,)))  # fmt: skip


def _norm_gate_setup(ctx, inputs, output):
    x, gate, gamma, beta, residual, residual_scale, groups, epsilon, rms, silu = inputs
    ctx.save_for_backward(x, gate, gamma, beta)
    ctx.rest = (residual is not None, residual_scale, groups, epsilon, rms, silu)


def _norm_gate_grad(ctx, grad):
    x, gate, gamma, beta = ctx.saved_tensors
    dx, du, dg, db = torch.ops.ops_rec.norm_gate_backward(grad, x, gate, gamma, beta, *ctx.rest)
    return dx, du if gate is not None else None, dg, db if beta is not None else None, grad if ctx.rest[0] else None, None, None, None, None, None


# --------------------------------------------------------------------------------------------------- rotary ----


def rotary_frequencies(rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=0, fast=32.0, slow=1.0, device=None):
    """``(frequencies, magnitude)`` for ``rotary``: frequency ``j`` of ``rotary_dim / 2`` is ``base ** (-2 j / rotary_dim)`` radians per position, fp64 on
    ``device``.  For contexts ``factor`` times as long as those a model was trained on:

    ``"linear"``  positions are divided by ``factor``;
    ``"base"``    the base grows by ``factor ** (rotary_dim / (rotary_dim - 2))``: the lowest frequency falls by ``factor``, the highest stays;
    ``"parts"``   frequencies of more than ``fast`` turns over ``original_length`` positions stay, those of fewer than ``slow`` are divided by ``factor``,
                  a blend by the index between; the magnitude becomes ``1 + 0.1 ln(factor)``."""
    _check(int(rotary_dim) >= 2 and int(rotary_dim) % 2 == 0, f"rotary_dim must be even and positive, but it is {rotary_dim}")
    _check(float(base) > 0 and float(factor) > 0, f"base and factor must be positive, but they are {base} and {factor}")
    _check(scaling in ("none", "linear", "base", "parts"), f"scaling must be 'none', 'linear', 'base' or 'parts', but it is {scaling!r}")
    dim = int(rotary_dim)
    if scaling == "base":
        _check(dim > 2, "scaling 'base' needs a rotary_dim above 2")
        base = float(base) * float(factor) ** (dim / (dim - 2))
    j = torch.arange(dim // 2, dtype=torch.float64)
    frequencies = float(base) ** (-2.0 * j / dim)
    magnitude = 1.0
    if scaling == "linear":
        frequencies = frequencies / float(factor)
    elif scaling == "parts":
        _check(int(original_length) > 0 and 0 < float(slow) < float(fast), "scaling 'parts' needs original_length > 0 and 0 < slow < fast")
        _check(float(base) > 1.0, f"scaling 'parts' needs a base above 1, but it is {base}")

        def index(turns):  # of the frequency that makes so many turns over the original length
            return dim * math.log(int(original_length) / (2 * math.pi * turns)) / (2 * math.log(float(base)))

        low, high = max(math.floor(index(float(fast))), 0), min(math.ceil(index(float(slow))), dim - 1)
        ramp = ((j - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        frequencies = frequencies * (1 - ramp) + frequencies / float(factor) * ramp
        magnitude = 1.0 + 0.1 * math.log(float(factor)) if float(factor) > 1.0 else 1.0
    return frequencies.to(device) if device is not None else frequencies, magnitude


def _rotary_checks(q, k, frequencies, seq_offset, start, positions) -> None:
    _check(q.dim() == 3 and k.dim() == 3, "The q and k should be 3D in jagged layout")
    _check(q.dtype in _FLOATS and k.dtype == q.dtype, f"q and k must both be float32, bfloat16 or float16, but they are {q.dtype} and {k.dtype}")
    _check(k.size(0) == q.size(0) and k.size(2) == q.size(2), f"q and k must have the same rows and head dim, but they are {list(q.shape)} and {list(k.shape)}")
    _check(1 <= q.size(1) <= 65536 and 1 <= k.size(1) <= 65536 and 2 <= q.size(2) <= 65536, f"heads expect in [1, 65536], headDim in [2, 65536], but q is {list(q.shape)}")
    _check(frequencies.dim() == 1 and frequencies.dtype == torch.float64, f"frequencies must be a vector of float64, but it is {list(frequencies.shape)} of {frequencies.dtype}")
    _check(1 <= frequencies.numel() and 2 * frequencies.numel() <= q.size(2), f"frequencies must have at least one and at most headDim / 2 elements, but there are {frequencies.numel()}")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("rotary: frequencies is a non-differentiable input; do not pass one with requires_grad=True")
    _check((seq_offset is None) != (positions is None), "seq_offset or positions must be given, and not both")
    _check(start is None or seq_offset is not None, "start goes with seq_offset")
    for name, t in (("seq_offset", seq_offset), ("start", start), ("positions", positions)):
        _check(t is None or (t.dim() == 1 and t.dtype in (torch.int32, torch.int64)), f"{name} must be a vector of int32 or int64")
    _check(positions is None or positions.numel() == q.size(0), f"positions must have an element per row ({q.size(0)})")
    _check(seq_offset is None or seq_offset.numel() >= 2, "seq_offset params error should have at least two element.")
    _check(start is None or start.numel() == seq_offset.numel() - 1, "start must have an element per sequence")


def _index_code(t):
    return _native.IDX_I64 if t is not None and t.dtype == torch.int64 else _native.IDX_I32


def rotary(q, k, frequencies, seq_offset=None, start=None, positions=None, interleaved=False, magnitude=1.0, inverse=False):
    """Rotary positions on ``q`` [rows, heads, dim] and ``k`` [rows, heads_k, dim]: each pair ``(a, b)`` of the first ``2 * len(frequencies)`` values of a head becomes
    ``magnitude * (a cos t - b sin t, b cos t + a sin t)``, ``t`` the row's position times the pair's frequency; the other values stay.  Pairs are
    ``(j, j + len(frequencies))``, or with ``interleaved`` ``(2 j, 2 j + 1)``.  ``inverse`` turns the other way (what gradients go through).

    The position of a row is its place in its sequence, ``seq_offset[b] : seq_offset[b + 1]``, plus ``start[b]`` where that is given (the rows a
    cache holds already); or ``positions[row]``, for everything else (targets that stand at one place, gaps).  Rows of no sequence come
    out as zeros.  ``frequencies`` is fp64 (``rotary_frequencies``), and angles are formed in 64 bits.  q and k are fp32, bf16 or fp16, with any strides
    whose last is 1; the results are new and contiguous."""
    _no_tangents("rotary", q, k, frequencies)
    _rotary_checks(q, k, frequencies, seq_offset, start, positions)
    _on_device(q.device, (("q", q), ("k", k), ("frequencies", frequencies), ("seq_offset", seq_offset), ("start", start), ("positions", positions)))
    q_out, k_out = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    if q.size(0) == 0:
        return q_out, k_out
    qc, kc, fc, oc, sc, pc = _rows(q), _rows(k), _dense(frequencies), _dense(seq_offset), _dense(start), _dense(positions)
    p = _native.RotaryParams()
    p.struct_size, p.dtype = ctypes.sizeof(p), _DTYPE_CODE[q.dtype]
    p.q, p.k, p.q_out, p.k_out = qc.data_ptr(), kc.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    p.frequencies, p.positions, p.seq_offset, p.start = fc.data_ptr(), _ptr(pc), _ptr(oc), _ptr(sc)
    p.rows, p.heads_q, p.heads_k, p.dim, p.pairs = q.size(0), q.size(1), k.size(1), q.size(2), frequencies.numel()
    p.n_offsets = seq_offset.numel() if seq_offset is not None else 0
    p.q_stride_row, p.q_stride_head, p.k_stride_row, p.k_stride_head = qc.stride(0), qc.stride(1), kc.stride(0), kc.stride(1)
    p.magnitude, p.interleaved, p.inverse = float(magnitude), int(bool(interleaved)), int(bool(inverse))
    p.positions_dtype, p.seq_offset_dtype, p.start_dtype = _index_code(positions), _index_code(seq_offset), _index_code(start)
    _call("rotary_fwd", p, q.device, workspace=False)
    return q_out, k_out


def rotary_meta(q, k, frequencies, seq_offset=None, start=None, positions=None, interleaved=False, magnitude=1.0, inverse=False):
    _check(q.dim() == 3 and k.dim() == 3, "The q and k should be 3D in jagged layout")
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _rotary_setup(ctx, inputs, output):
    _, _, frequencies, seq_offset, start, positions, interleaved, magnitude, inverse = inputs
    ctx.save_for_backward(frequencies, seq_offset, start, positions)
    ctx.rest = (interleaved, magnitude, not inverse)


def _rotary_grad(ctx, q_grad, k_grad):
    dq, dk = torch.ops.ops_rec.rotary(q_grad, k_grad, *ctx.saved_tensors, *ctx.rest)
    return dq, dk, None, None, None, None, None, None, None


# --------------------------------------------------------------------------------------- gated projections ----

ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}
MAX_GATED_COLUMNS = 1 << 21
# Up to so many columns of x a backward multiplies again and nothing is kept for it: forward and backward of 29028 rows, 96 -> 3352, 983 us with mixed and 611
# without, 44986 rows, 168 -> 456, 226 and 172; 65536 rows, 256 -> 1024, 458 and 481, 20292 rows, 512 -> 2048, 384 and 437.
KEPT_COLUMNS = 192


def _gated_linear_checks(x, weight, bias, activation) -> None:
    _check(x.dim() == 2, "The x should be 2D")
    _check(weight.dim() == 2, "The weight should be 2D")
    _check(x.dtype in (torch.bfloat16, torch.float16), f"x must be float16 or bfloat16, got {x.dtype}")
    _check(weight.dtype == x.dtype, "weight must have the dtype of x")
    _check(activation in ACTIVATIONS, f"activation must be one of {sorted(ACTIVATIONS)}, but it is {activation!r}")
    cols, inner = x.size(1), weight.size(0) // 2
    _check(weight.size(0) % 2 == 0 and weight.size(1) == cols, f"weight must be [2 * inner, {cols}], but it is {list(weight.shape)}")
    _check(8 <= cols <= MAX_GATED_COLUMNS and cols % 8 == 0 and 8 <= inner <= MAX_GATED_COLUMNS and inner % 8 == 0 and inner * cols < 1 << 29,
           f"the columns of x and of hidden must be multiples of 8, at most 2^21, with a product below 2^29, but they are {cols} and {inner}")  # fmt: skip
    _check(x.size(0) < 1 << 31, f"at most 2^31 - 1 rows, but there are {x.size(0)}")
    if bias is not None:
        _check(bias.dim() == 1 and bias.numel() == 2 * inner, f"bias must have 2 * inner elements ({2 * inner}), but it is {list(bias.shape)}")
        _check(bias.dtype == x.dtype, "bias must have the dtype of x")


def _describe_gated_linear(p, x, weight, bias, hidden, mixed, activation):
    p.struct_size, p.activation = ctypes.sizeof(p), ACTIVATIONS[activation]
    p.x, p.weight, p.bias, p.hidden, p.mixed = _ptr(x), _ptr(weight), _ptr(bias), _ptr(hidden), _ptr(mixed)
    p.rows, p.cols, p.inner, p.dtype = x.size(0), x.size(1), weight.size(0) // 2, _DTYPE_CODE[x.dtype]


def gated_linear(x, weight, bias=None, activation="silu", keep=False):
    """``hidden = act(g) * u`` with ``(g, u) = x @ weight^T + bias``: both projections of a gated feed-forward block, its activation and the
    product, for x [rows, cols] and weight [2 * inner, cols], the rows of g first.  Returns ``(hidden, mixed)``, mixed empty unless ``keep``.

    Mixed is for the backward pass alone, which reads g and u out of it: 24 bits of each, as int16 [rows, 3 * inner] in an order of their own.
    No gradient flows through it: it does not require one.  A call in training passes ``keep=True``; without it, as a block that saves memory may
    prefer, the backward multiplies again, which takes 14 % more of a training step at 512 columns of x and 26 % at 2048.  Up to 192 columns that is faster,
    and mixed is empty either way.  ``activation`` is "silu", "gelu" (by its tanh form) or "sigmoid".  x, weight and bias are all bf16 or all fp16; cols
    and inner are multiples of 8.  Sums are fp32, and hidden is taken of them.  The backward's products multiply gradients of g and u that are rounded
    to the type of x, in fp16 scaled by a power of two that keeps the largest in its range."""
    _no_tangents("gated_linear", x, weight, bias)
    _gated_linear_checks(x, weight, bias, activation)
    _on_device(x.device, (("x", x), ("weight", weight), ("bias", bias)))
    inner = weight.size(0) // 2
    hidden = torch.empty((x.size(0), inner), dtype=x.dtype, device=x.device)
    mixed = torch.empty((x.size(0), 3 * inner) if keep and x.size(1) > KEPT_COLUMNS else (0,), dtype=torch.int16, device=x.device)
    if x.size(0) != 0:
        xc, wc, bc = _aligned(x), _aligned(weight), None if bias is None else _aligned(bias)
        p = _native.GatedLinearParams()
        _describe_gated_linear(p, xc, wc, bc, hidden, mixed, activation)
        _call("gated_linear_fwd", p, x.device, workspace=False)
    return hidden, mixed


def gated_linear_meta(x, weight, bias=None, activation="silu", keep=False):
    _check(x.dim() == 2, "The x should be 2D")
    _check(weight.dim() == 2, "The weight should be 2D")
    return x.new_empty((x.size(0), weight.size(0) // 2)), x.new_empty(
        (x.size(0), 3 * (weight.size(0) // 2)) if keep and x.size(1) > KEPT_COLUMNS else (0,), dtype=torch.int16)  # fmt: skip


def gated_linear_backward(grad, x, weight, bias, mixed, activation, wanted):
    """Gradients of ``gated_linear``'s x, weight and bias, those that are ``wanted``, the others empty.  ``mixed`` is what the call returned; if it is
    empty, g and u are multiplied again."""
    _gated_linear_checks(x, weight, bias, activation)
    _check(len(wanted) == 3, "wanted must have three elements")
    rows, inner = x.size(0), weight.size(0) // 2
    _check(tuple(grad.shape) == (rows, inner) and grad.dtype == x.dtype, f"grad must be {[rows, inner]} of the dtype of x")
    _check(mixed.numel() == 0 or (tuple(mixed.shape) == (rows, 3 * inner) and mixed.dtype == torch.int16),
           f"mixed must be empty or {[rows, 3 * inner]} of int16")  # fmt: skip
    _on_device(x.device, (("x", x), ("grad", grad), ("weight", weight), ("bias", bias), ("mixed", mixed)))
    make = torch.zeros if rows == 0 else torch.empty
    shapes = ((rows, x.size(1)), tuple(weight.shape), (2 * inner,))
    there = (wanted[0], wanted[1], wanted[2] and bias is not None)
    grads = tuple(make(shape if want else (0,), dtype=x.dtype, device=x.device) for shape, want in zip(shapes, there))
    if rows != 0 and any(there):
        xc, wc, bc, dc = _aligned(x), _aligned(weight), None if bias is None else _aligned(bias), _aligned(grad)
        p = _native.GatedLinearBwdParams()
        p.struct_size = ctypes.sizeof(p)
        mc = _aligned(mixed) if mixed.numel() != 0 else None
        _describe_gated_linear(p.fwd, xc, wc, bc, None, mc, activation)
        p.grad = dc.data_ptr()
        p.x_grad, p.weight_grad, p.bias_grad = (_ptr(t) for t in grads)
        _call("gated_linear_bwd", p, x.device)
    return grads


def gated_linear_backward_meta(grad, x, weight, bias, mixed, activation, wanted):
    there = (wanted[0], wanted[1], wanted[2] and bias is not None)
    shapes = (x.shape, weight.shape, (weight.size(0),))
    return tuple(x.new_empty(shape if want else (0,)) for shape, want in zip(shapes, there))


def _gated_linear_setup(ctx, inputs, output):
    x, weight, bias, activation, _ = inputs
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.activation = activation


def _gated_linear_grad(ctx, grad, _):
    x, weight, bias, mixed = ctx.saved_tensors
    if grad is None:
        return (None,) * 5
    wanted = [bool(w) for w in ctx.needs_input_grad[:3]]
    got = torch.ops.ops_rec.gated_linear_backward(grad, x, weight, bias, mixed, ctx.activation, wanted)
    there = (wanted[0], wanted[1], wanted[2] and bias is not None)
    return (*(t if want else None for t, want in zip(got, there)), None, None)


for _name, _kernel, _meta in (("residual_norm", residual_norm, residual_norm_meta),
                              ("residual_norm_backward", residual_norm_backward, residual_norm_backward_meta),
                              ("norm_gate", norm_gate, norm_gate_meta),
                              ("norm_gate_backward", norm_gate_backward, norm_gate_backward_meta),
                              ("rotary", rotary, rotary_meta),
                              ("gated_linear", gated_linear, gated_linear_meta),
                              ("gated_linear_backward", gated_linear_backward, gated_linear_backward_meta)):  # fmt: skip
    _PYTHON_KERNELS[_name] = _kernel
    _lib_meta.impl(_name, _meta)
for _name, _setup, _grad in (("residual_norm", _residual_norm_setup, _residual_norm_grad), ("norm_gate", _norm_gate_setup, _norm_gate_grad),
                             ("rotary", _rotary_setup, _rotary_grad), ("gated_linear", _gated_linear_setup, _gated_linear_grad)):  # fmt: skip
    torch.library.register_autograd(f"ops_rec::{_name}", _grad, setup_context=_setup)
