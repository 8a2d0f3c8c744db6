"""gated_linear's backward where tests/test_layer_gated_linear.py does not go: values that are not finite, the ends of fp16, every tile of its products, what is kept above
192 columns of x, and the largest sizes."""

import ctypes
import math

import pytest
import torch

import ops_rec
import layer_reference as R
from ops_rec import _dispatch, _layer, _native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A = ops_rec.ascendc.activation
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _memory_goes_back():
    """Cached blocks go back to the device after each test: tests that count what the allocator takes find it as they expect it."""
    yield
    torch.cuda.empty_cache()


def randn(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def act(name, z):
    if name == "gelu":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    return torch.sigmoid(z) * (z if name == "silu" else 1)


def growth(n):
    """Of a sum of n products in fp32, relative to the sum of their magnitudes: n / 2^24 at most, and in trees and chains whose errors do not all go one way
    2^-18 up to 2^12 products and sqrt(n) / 2^24 beyond."""
    return max(2.0**-18, math.sqrt(n) * 2.0**-24)


def definition(x, w, b, dh, activation):
    """The gradients of x, weight and bias in 64 bits, on the device of the inputs, each with the room of a kernel that multiplies d_mixed in the inputs' type.

    g and u are off by what their sums in fp32 are, and cut to 24 bits; the activations and their slopes have slopes of 1.13 at most, and the hardware's exponential
    and reciprocal are off by 2^-22.  d_mixed is rounded by half a step, in fp16 at a scale at which a step from zero is 2^-22 of its largest value at most."""
    half, inner = R.HALF_STEP[x.dtype], dh.size(1)
    x64, w64, dh64 = x.double(), w.double(), dh.double()
    b64 = torch.zeros(2 * inner, dtype=torch.float64, device=x.device) if b is None else b.double()
    mixed, size = x64 @ w64.t() + b64, x64.abs() @ w64.abs().t() + b64.abs()
    (g, u), (eg, eu) = mixed.chunk(2, dim=1), (growth(x.size(1)) * size).chunk(2, dim=1)
    gl = g.detach().clone().requires_grad_(True)
    a = act(activation, gl)
    (slope,) = torch.autograd.grad(a.sum(), gl)
    a = a.detach()
    d = torch.cat([dh64 * u * slope, dh64 * a], dim=1)
    rg, ru = (2.0**-15 * (t.abs() + e) + e for t, e in ((g, eg), (u, eu)))
    room = torch.cat([dh64.abs() * (slope.abs() * ru + 1.13 * rg * (u.abs() + ru)), dh64.abs() * 1.13 * rg], dim=1) + 2.0**-20 * d.abs()
    rounded = room + half * (d.abs() + room) + (2.0**-22 * d.abs().max() if x.dtype == FP16 else 0.0)
    n = x.size(0)
    return ((d @ w64, rounded @ w64.abs() + growth(2 * inner) * (d.abs() @ w64.abs())),
            (d.t() @ x64, rounded.t() @ x64.abs() + growth(n) * (d.abs().t() @ x64.abs())),
            (d.sum(0), room.sum(0) + growth(n) * d.abs().sum(0)))  # fmt: skip


def compare(got, want, what):
    ref, room = want
    assert got.shape == ref.shape, what
    room = R.HALF_STEP[got.dtype] * ref.abs() * (1 + 2.0**-7) + room + (2.0**-25 if got.dtype == FP16 else 0.0)
    off = (got.detach().double() - ref).abs()
    bad = ~(off <= room)
    assert not bad.any(), (what, int(bad.sum()), off[bad].max().item(), room[bad].min().item())


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("cols", [64, 200])  # g and u multiplied again, and kept
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_gate_that_is_nan_has_gradients_that_are(activation, cols, dtype):
    g = torch.Generator().manual_seed(cols)
    x, w, dh = torch.randn(20, cols, generator=g).to(dtype), (torch.randn(48, cols, generator=g) / cols**0.5).to(dtype), torch.randn(20, 24, generator=g).to(dtype)
    bias = torch.zeros(48, dtype=dtype)
    bias[3] = float("nan")  # one unit's gate
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, bias)]
    hidden, mixed = A.gated_linear(*leaves, activation, True)
    assert (mixed.numel() != 0) == (cols == 200)
    dx, dw, db = torch.autograd.grad(hidden, leaves, dh.to(DEV))
    unit = torch.zeros(48, dtype=torch.bool, device=DEV)
    unit[[3, 27]] = True  # its gate and what the gate multiplies
    assert torch.equal(torch.isnan(hidden), unit[:24].expand(20, 24))
    assert torch.equal(torch.isnan(db), unit) and torch.equal(torch.isnan(dw), unit[:, None].expand(48, cols)) and torch.isnan(dx).all()


def repeated(pattern, rows):
    """The rows of ``pattern`` again and again."""
    period = pattern.size(0)
    out = torch.empty(rows, pattern.size(1), dtype=pattern.dtype, device=DEV)
    whole = rows // period
    out[: whole * period].view(whole, period, -1).copy_(pattern.expand(whole, *pattern.shape))
    out[whole * period :] = pattern[: rows - whole * period]
    return out


def is_repeated(t, pattern):
    step = 512 * pattern.size(0)
    return all(torch.equal(t[at : at + step], repeated(pattern, min(step, t.size(0) - at))) for at in range(0, t.size(0), step))


def test_more_tiles_than_a_launch_has_workgroups():
    """The most rows there may be: 2^24 tiles of 128 rows, of 256 threads each, where a launch has less than 2^32 threads."""
    rows = (1 << 31) - 1
    g = torch.Generator().manual_seed(1)
    x, w, dh = torch.randn(1 << 16, 8, generator=g).to(BF16).to(DEV), torch.randn(16, 8, generator=g).to(BF16).to(DEV), torch.randn(1 << 16, 8, generator=g).to(BF16).to(DEV)
    want = A.gated_linear(x, w)[0]
    dx = A.gated_linear_backward(dh, x, w, None, torch.empty(0, dtype=torch.int16, device=DEV), "silu", [True, False, False])[0]
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 172 GB")
    many = repeated(x, rows)
    hidden = A.gated_linear(many, w)[0]
    assert is_repeated(hidden, want)
    del hidden
    got = A.gated_linear_backward(repeated(dh, rows), many, w, None, torch.empty(0, dtype=torch.int16, device=DEV), "silu", [True, False, False])[0]
    assert is_repeated(got, dx)


def ends_of_fp16(kind, cols, gen):
    """x, weight, bias and the gradient of hidden in fp16, whose d_mixed is past 65504 ("past"), among the subnormals ("small"), or below all of them ("below"), while the
    gradients of x and weight are well inside."""
    rows, inner = 700, 72
    grad, x, w, b = {"past": (2.0**13, 2.0**-11, 2.0**-7, 16.0), "small": (2.0**-12, 2.0**4, 2.0**-4, 2.0**-5), "below": (2.0**-24, 2.0**8, 2.0**-8, 2.0**-10)}[kind]
    bias = randn(gen, 2 * inner, dtype=FP16, std=b)
    weight = randn(gen, 2 * inner, cols, dtype=FP16, std=w)
    if kind != "past":  # (u as small as its bias)
        weight[inner:] = 0
    if kind == "below":  # (and gates of about a half)
        weight[:inner] *= 2.0**-4
    return randn(gen, rows, cols, dtype=FP16, std=x), weight, bias, randn(gen, rows, inner, dtype=FP16, std=grad)


@pytest.mark.parametrize("kind", ["past", "small", "below"])
@pytest.mark.parametrize("cols,keep", [(64, False), (200, True), (200, False)])
def test_the_ends_of_fp16(kind, cols, keep):
    g = torch.Generator().manual_seed(cols)
    x, w, b, dh = (t.to(DEV) for t in ends_of_fp16(kind, cols, g))
    want = definition(x, w, b, dh, "silu")
    assert all(t[0].abs().max() < 60000 for t in want[:2])
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    hidden, mixed = A.gated_linear(*leaves, b, "silu", keep)
    assert (mixed.numel() != 0) == keep
    for got, ref, name in zip(torch.autograd.grad(hidden, leaves, dh), want, ("x", "weight")):
        compare(got, ref, name)


@pytest.mark.parametrize("cols", [64, 200])
def test_a_captured_step_follows_the_size_of_its_gradients(cols):
    gen = torch.Generator().manual_seed(3)
    x, w, b, dh = (t.to(DEV) for t in ends_of_fp16("past", cols, gen))
    dh.mul_(2.0**-10)

    def step():
        mixed = A.gated_linear(x, w, b, "silu", True)[1]
        return A.gated_linear_backward(dh, x, w, b, mixed, "silu", [True, True, False])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for by in (1.0, 2.0**10, 2.0**-25, 2.0**12, 2.0**3):
        dh.mul_(by)
        graph.replay()
        torch.cuda.synchronize()
        want = definition(x, w, b, dh, "silu")
        for got, ref, eager, name in zip(outs[:2], want, step(), ("x", "weight")):
            assert torch.equal(got, eager)
            compare(got, ref, name)


def test_both_implementations_keep_from_the_same_width_on():
    limit = _layer.KEPT_COLUMNS
    assert _dispatch.binding is not None and _dispatch.binding.kept_columns() == limit
    for cols in (limit - 8, limit, limit + 8):
        g = torch.Generator().manual_seed(cols)
        x, w, dh = (randn(g, *shape, dtype=BF16, std=0.3).to(DEV) for shape in ((130, cols), (80, cols), (130, 40)))
        native, python = A.gated_linear(x, w, None, "silu", True), _layer.gated_linear(x, w, None, "silu", True)
        assert all(torch.equal(a, b) for a, b in zip(native, python)) and (native[1].numel() != 0) == (cols > limit)
        meta = torch.ops.ops_rec.gated_linear(x.to("meta"), w.to("meta"), None, "silu", True)
        assert [t.shape for t in meta] == [t.shape for t in native]
        want = definition(x, w, None, dh, "silu")
        got = A.gated_linear_backward(dh, x, w, None, native[1], "silu", [True, True, False])
        for a, b, ref, name in zip(got, _layer.gated_linear_backward(dh, x, w, None, python[1], "silu", [True, True, False]), want, ("x", "weight")):
            assert torch.equal(a, b)
            compare(a, ref, name)


def planned(rows, cols, inner, dtype=BF16, kept=False):
    """(part, kernel, whether its depth is cut) of the three parts of a backward"""
    p = _native.GatedLinearBwdParams()
    p.struct_size = ctypes.sizeof(p)
    none = torch.empty(0)
    _layer._describe_gated_linear(p.fwd, torch.empty(rows, cols, dtype=dtype, device="meta"), torch.empty(2 * inner, cols, dtype=dtype, device="meta"), None, none, none, "silu")
    p.fwd.x = p.fwd.weight = p.grad = p.x_grad = p.weight_grad = 0x1000  # never dereferenced
    p.fwd.mixed = 0x1000 if kept else None
    parts, chunks = [], ctypes.c_int64(0)
    for part in range(3):
        name = _native.load().gated_linear_bwd_kernel_name(ctypes.byref(p), part, ctypes.byref(chunks))
        parts.append((part, name.decode().replace("gated_gemm_", ""), chunks.value > 1))
    return parts


# what is left over differs in every dimension of every tile: rows, columns of x, columns of hidden
TILES = [(16, 8, 8), (16, 8, 416), (669, 8, 8), (4115, 8, 568), (16669, 8, 8), (18694, 8, 72), (17358, 136, 8), (4297, 136, 1568), (22779, 280, 8), (11595, 160, 1728),
         (25679, 272, 8), (17548, 152, 1536), (18, 400, 4120), (5786, 2952, 8), (16, 4232, 1016), (11203, 520, 3744)]  # fmt: skip


def test_every_tile_of_the_backward_is_among_them():
    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("planned for 256 compute units")
    tiles = {0: ["64x128", "128x128", "128x256"], 1: ["64x128", "128x128", "128x256", "192x256", "256x256"], 2: ["128x128", "128x256", "256x256"]}
    expected = {(part, name, cut) for part, names in tiles.items() for name in names for cut in ((False, True) if part != 0 else (False,))}
    assert {entry for size in TILES for entry in planned(*size)} == expected


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,cols,inner", TILES)
def test_every_tile_of_the_backward(rows, cols, inner, dtype):
    g = torch.Generator().manual_seed(rows + cols)
    x, w = randn(g, rows, cols, dtype=dtype).to(DEV), randn(g, 2 * inner, cols, dtype=dtype, std=1.5 / math.sqrt(cols)).to(DEV)
    b, dh = randn(g, 2 * inner, dtype=dtype, std=0.5).to(DEV), randn(g, rows, inner, dtype=dtype).to(DEV)
    mixed = A.gated_linear(x, w, b, "silu", True)[1]
    want = definition(x, w, b, dh, "silu")
    for kept in [torch.empty(0, dtype=torch.int16, device=DEV)] + ([mixed] if mixed.numel() else []):
        for got, ref, name in zip(A.gated_linear_backward(dh, x, w, b, kept, "silu", [True] * 3), want, ("x", "weight", "bias")):
            compare(got, ref, (name, kept.numel() != 0))


@pytest.mark.parametrize("keep", [True, False])
def test_rows_of_d_mixed_that_fill_a_descriptor(keep):
    """256 rows of 2^22 columns are the 2^31 bytes that a tile of the x gradient may ask for; a gradient on a few columns alone, so that these are what the sums are made of."""
    rows, cols, inner = 500, 200, 1 << 21
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert planned(rows, cols, inner)[1:] == [(1, "256x256", True), (2, "256x256", True)]
    g = torch.Generator().manual_seed(3)
    some = torch.tensor([0, 1, 255, 70000, inner // 2 - 1, inner // 2, inner - 256, inner - 1], device=DEV)
    both = torch.cat([some, some + inner])
    x, few, dh = randn(g, rows, cols, dtype=BF16).to(DEV), randn(g, 16, cols, dtype=BF16, std=0.1).to(DEV), randn(g, rows, 8, dtype=BF16).to(DEV)
    weight, grad = torch.zeros(2 * inner, cols, dtype=BF16, device=DEV), torch.zeros(rows, inner, dtype=BF16, device=DEV)
    weight[both], grad[:, some] = few, dh
    hidden, mixed = A.gated_linear(x, weight, None, "silu", keep)
    assert (mixed.numel() != 0) == keep
    dx, dw, _ = A.gated_linear_backward(grad, x, weight, None, mixed, "silu", [True, True, False])
    want = definition(x, few, None, dh, "silu")
    compare(dx, want[0], "x")
    compare(dw[both], want[1], "weight")
    dw[both] = 0
    assert torch.count_nonzero(dw) == 0


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gradients_from_what_was_kept(activation, bias, rows, dtype):
    """All that are wanted, and each choice of them: the same bits, and nothing in the place of the others."""
    g = torch.Generator().manual_seed(rows)
    cols, inner = 200, 264
    x, w = randn(g, rows, cols, dtype=dtype).to(DEV), randn(g, 2 * inner, cols, dtype=dtype, std=1.5 / math.sqrt(cols)).to(DEV)
    b, dh = randn(g, 2 * inner, dtype=dtype, std=0.5).to(DEV) if bias else None, randn(g, rows, inner, dtype=dtype).to(DEV)
    mixed = A.gated_linear(x, w, b, activation, True)[1]
    assert mixed.numel() != 0
    grads = A.gated_linear_backward(dh, x, w, b, mixed, activation, [True, True, True])
    for got, ref, name in list(zip(grads, definition(x, w, b, dh, activation), ("x", "weight", "bias")))[: 3 if bias else 2]:
        compare(got, ref, name)
    assert bias or grads[2].numel() == 0
    for n in range(7):
        wanted = [bool(n & 1), bool(n & 2), bool(n & 4)]
        got = A.gated_linear_backward(dh, x, w, b, mixed, activation, wanted)
        assert all(torch.equal(a, full) if want else a.numel() == 0 for a, full, want in zip(got, grads, wanted))
    # through autograd, with inputs that need no gradient
    leaves = [t if t is None else t.clone() for t in (x, w, b)]
    for frozen in range(3 if bias else 2):
        for i, t in enumerate(leaves):
            if t is not None:
                t.requires_grad_(i != frozen)
        needed = [i for i, t in enumerate(leaves) if t is not None and i != frozen]
        hidden = A.gated_linear(*leaves, activation, True)[0]
        for i, got in zip(needed, torch.autograd.grad(hidden, [leaves[i] for i in needed], dh)):
            assert torch.equal(got, grads[i])


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("cols", [64, 200])
def test_gradients_of_gates_far_out(activation, cols):
    """Gates whose exponentials overflow and underflow: their slopes are 0, 1 or those of the definition, and nothing is NaN."""
    inner = 8
    gates = torch.tensor([0.0, 200.0, -200.0, 1e30, -1e30, 3e38, -3e38, 60.0], dtype=BF16)
    bias = torch.cat([gates, torch.ones(inner, dtype=BF16)]).to(DEV)
    x, w = torch.zeros(6, cols, dtype=BF16, device=DEV), torch.zeros(2 * inner, cols, dtype=BF16, device=DEV)
    x[:, 0] = 1.0
    mixed = A.gated_linear(x, w, bias, activation, True)[1]
    assert (mixed.numel() != 0) == (cols == 200)
    dx, dw, db = A.gated_linear_backward(torch.ones(6, inner, dtype=BF16, device=DEV), x, w, bias, mixed, activation, [True, True, True])
    z = torch.where(gates.double().abs() > 1000, 1000.0 * gates.double().sign(), gates.double()).requires_grad_(True)
    (slope,) = torch.autograd.grad(act(activation, z).sum(), z)
    value = torch.where(gates > 1000, gates.double() if activation != "sigmoid" else torch.ones(()).double(), act(activation, z.detach()))
    want = 6 * torch.cat([slope, value])  # six rows, each with u = 1 and a gradient of 1
    fits = want.abs() < 3.3e38
    for got in (db.double().cpu(), dw[:, 0].double().cpu()):
        assert torch.allclose(got[fits], want[fits], rtol=2.0**-7, atol=2.0**-126) and not torch.isnan(got).any()
    assert torch.count_nonzero(dw[:, 1:]) == 0 and torch.count_nonzero(dx) == 0


@pytest.mark.parametrize("filled", [0x7E, 0xFF])  # 8.5e37, NaN
@pytest.mark.parametrize("rows,cols,inner", [(5, 200, 40), (300, 200, 264), (1000, 64, 1000), (2500, 72, 520)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_workspaces_that_hold_something(rows, cols, inner, dtype, filled):
    """What a workspace held before reaches nothing: neither the gradients nor the power of two that fp16 is scaled by."""
    g = torch.Generator().manual_seed(rows)
    x, w = randn(g, rows, cols, dtype=dtype).to(DEV), randn(g, 2 * inner, cols, dtype=dtype, std=1.5 / math.sqrt(cols)).to(DEV)
    b, dh = randn(g, 2 * inner, dtype=dtype, std=0.5).to(DEV), randn(g, rows, inner, dtype=dtype).to(DEV)
    mixed = A.gated_linear(x, w, b, "silu", True)[1]
    want = A.gated_linear_backward(dh, x, w, b, mixed, "silu", [True] * 3)
    got = [torch.empty_like(t).fill_(-1.0) for t in want]
    p = _native.GatedLinearBwdParams()
    p.struct_size = ctypes.sizeof(p)
    _layer._describe_gated_linear(p.fwd, x, w, b, None, mixed if mixed.numel() else None, "silu")
    p.grad, p.x_grad, p.weight_grad, p.bias_grad = (t.data_ptr() for t in (dh, *got))
    lib, size = _native.load(), ctypes.c_uint64(0)
    assert lib.gated_linear_bwd_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0
    space = torch.full((size.value + 512,), filled, dtype=torch.uint8, device=DEV)
    assert lib.gated_linear_bwd(ctypes.byref(p), space.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream) == 0, _native.last_error()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(bool(torch.isfinite(t).all()) for t in got)
    assert bool((space[size.value :] == filled).all())
