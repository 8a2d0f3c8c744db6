"""gated_linear, forward and backward, against its definition in 64 bits.

Room, beside half a step of the output: sums of n products in fp32 are off by at most n * 2^-24 of the sum of their magnitudes, and the matrix units add
in trees and chains whose errors do not all go one way: 2^-18 of it is allowed up to 2^12 products, and sqrt(n) / 2^24 beyond.  The hardware's
exponential and reciprocal are off by 2^-22 at most.  The backward reads g and u cut to 24 bits, 2^-15 of them at most, and multiplies gradients rounded
to the type: their errors are bounded term by term (in ``check``)."""

import math

import pytest
import torch

import ops_rec
from ops_rec import _native
import layer_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A = ops_rec.ascendc.activation
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _memory_goes_back():
    """Cached blocks go back to the device after each test: tests that count what the allocator takes find it as they expect it."""
    yield
    torch.cuda.empty_cache()


def act(name, z):
    if name == "gelu":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    return torch.sigmoid(z) * (z if name == "silu" else 1)


def inputs(rows, cols, inner, dtype, bias, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g).to(dtype)
    w = (torch.randn(2 * inner, cols, generator=g) * 1.5 / math.sqrt(cols)).to(dtype)
    b = (torch.randn(2 * inner, generator=g) * 0.5).to(dtype) if bias else None
    return x, w, b, torch.randn(rows, inner, generator=g).to(dtype)


def growth(n):
    return max(2.0**-18, math.sqrt(n) * 2.0**-24)


def compare(got, ref, room, what):
    assert got.shape == ref.shape, what
    step = R.HALF_STEP[got.dtype]
    room = step * ref.abs() * (1 + 2.0**-7) + room + (2.0**-25 if got.dtype == FP16 else 0.0)
    bad = ~((got.detach().double().cpu() - ref).abs() <= room)
    assert not bad.any(), (what, int(bad.sum()), (got.detach().double().cpu() - ref).abs()[bad].max().item(), room[bad].min().item())


def read(kept):
    """g and u out of mixed: their upper 16 bits, then for every 8 columns the third bytes of g and of u."""
    kept = kept.detach().cpu()
    rows, inner = kept.size(0), kept.size(1) // 3
    high = kept[:, : 2 * inner].int() << 16
    low = kept.view(torch.uint8)[:, 4 * inner :].reshape(rows, inner // 8, 2, 8).transpose(1, 2).reshape(rows, 2 * inner).int() << 8
    return (high | low).view(torch.float32)


def check(rows, cols, inner, dtype, activation="silu", bias=True, keep=True, backward=True, seed=0):
    x, w, b, dh = inputs(rows, cols, inner, dtype, bias, seed)
    x64, w64, b64, dh64 = (None if t is None else t.double() for t in (x, w, b, dh))
    mixed = x64 @ w64.t() + (0 if b is None else b64)
    size = x64.abs() @ w64.abs().t() + (0 if b is None else b64.abs())
    g, u = mixed.chunk(2, dim=1)
    err = growth(cols) * size  # of g and u before rounding
    eg, eu = err.chunk(2, dim=1)
    a = act(activation, g)
    dev = [None if t is None else t.to(DEV).requires_grad_(backward) for t in (x, w, b)]
    hidden, kept = A.gated_linear(*dev, activation, keep)
    keep = keep and cols > 192  # (else a backward multiplies again)
    assert hidden.dtype == dtype and hidden.is_contiguous() and tuple(kept.shape) == ((rows, 3 * inner) if keep else (0,)) and kept.dtype == torch.int16
    # (slopes of the activations are at most 1.13)
    compare(hidden, a * u, 1.13 * eg * u.abs() + a.abs() * eu + 2.0**-20 * (a * u).abs(), "hidden")
    if keep:
        compare(read(kept), mixed, err + 2.0**-15 * (mixed.abs() + err), "mixed")
    if not backward:
        return
    gl = g.clone().requires_grad_(True)
    (slope,) = torch.autograd.grad(act(activation, gl).sum(), gl)
    d_mixed = torch.cat([dh64 * u * slope, dh64 * a], dim=1)
    # what cutting g and u to 24 bits (and their sums' errors) does to the gradients: the second derivatives of the activations are at most 1.13
    half = R.HALF_STEP[dtype]
    rg, ru = (2.0**-15 * (t.abs() + e) + e for t, e in ((g, eg), (u, eu)))
    room_d = torch.cat([dh64.abs() * (slope.abs() * ru + 1.13 * rg * (u.abs() + ru)), dh64.abs() * 1.13 * rg], dim=1) + 2.0**-20 * d_mixed.abs()
    rounded = room_d + half * (d_mixed.abs() + room_d) + (2.0**-25 if dtype == FP16 else 0.0)
    grads = torch.autograd.grad(hidden, [t for t in dev if t is not None], dh.to(DEV))
    compare(grads[0], d_mixed @ w64, rounded @ w64.abs() + growth(2 * inner) * (d_mixed.abs() @ w64.abs()), "x")
    compare(grads[1], d_mixed.t() @ x64, rounded.t() @ x64.abs() + growth(rows) * (d_mixed.abs().t() @ x64.abs()), "weight")
    if bias:
        compare(grads[2], d_mixed.sum(0), room_d.sum(0) + growth(rows) * d_mixed.abs().sum(0), "bias")


SIZES = [(1, 8, 8), (1, 512, 256), (2, 72, 40), (16, 64, 136), (17, 520, 24), (33, 128, 320), (64, 1000, 16), (65, 8, 8), (70, 200, 72), (128, 256, 264),
         (129, 40, 1000), (300, 264, 136), (1000, 72, 520), (513, 1032, 8), (257, 520, 2056)]  # fmt: skip


@pytest.mark.parametrize("rows,cols,inner", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sizes(rows, cols, inner, dtype):
    check(rows, cols, inner, dtype, seed=rows + cols)
    check(rows, cols, inner, dtype, "gelu", bias=False, keep=False, seed=rows + inner)


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("rows", [5, 40, 200])
def test_activations(activation, rows):
    for dtype in (BF16, FP16):
        check(rows, 64, 72, dtype, activation, seed=rows)


@pytest.mark.parametrize("rows,cols,inner", [(4096, 256, 512), (20000, 64, 128), (2000, 1024, 1408)])
def test_larger(rows, cols, inner):
    check(rows, cols, inner, BF16, seed=1)


def name(rows, cols, inner):
    p = _native.GatedLinearParams()
    x = torch.empty(0)
    ops_rec._layer._describe_gated_linear(p, torch.empty(rows, cols, dtype=BF16, device="meta"), torch.empty(2 * inner, cols, dtype=BF16, device="meta"), None, x, x, "silu")
    p.x = p.weight = p.hidden = 0x1000
    return _native.load().gated_linear_fwd_kernel_name(p).decode()


def test_every_tile_of_the_forward():
    seen = set()
    for rows, cols, inner in ((64, 64, 64), (200, 64, 256), (700, 64, 2048), (8300, 72, 2056), (4096, 2056, 2048)):
        seen.add(name(rows, cols, inner))
        check(rows, cols, inner, BF16, backward=False, seed=3)
        check(rows, cols, inner, FP16, "gelu", backward=False, bias=False, seed=4)
    assert len(seen) == 5, seen


def test_the_widest():
    """2^21 columns, where a tile's rows of d_mixed fill a descriptor; a gradient on a few columns alone, so that these are what the sums are made of."""
    rows, inner = 260, 1 << 21
    g = torch.Generator().manual_seed(3)
    x, weight = torch.randn(rows, 8, generator=g).to(BF16), torch.zeros(2 * inner, 8, dtype=BF16)
    some = torch.tensor([0, 1, 255, 70000, inner // 2 - 1, inner // 2, inner - 256, inner - 1])
    both = torch.cat([some, some + inner])
    weight[both] = torch.randn(16, 8, generator=g).to(BF16)
    dh = torch.randn(rows, 8, generator=g).to(BF16)
    wide = torch.zeros(rows, inner, dtype=BF16, device=DEV)
    wide[:, some.to(DEV)] = dh.to(DEV)
    leaves = [x.to(DEV).requires_grad_(True), weight.to(DEV).requires_grad_(True)]
    hidden = A.gated_linear(*leaves, None, "silu", True)[0]
    dx, dw = torch.autograd.grad(hidden, leaves, wide)
    x64, w64, dh64 = x.double(), weight[both].double(), dh.double()
    gate, up = (x64 @ w64.t()).chunk(2, dim=1)
    s = torch.sigmoid(gate)
    compare(hidden.detach()[:, some.to(DEV)], gate * s * up, 2.0**-17 * (x64.abs() @ w64.abs().t()).max() * (gate.abs() + up.abs()), "hidden")
    d = torch.cat([dh64 * up * s * (1 + gate * (1 - s)), dh64 * gate * s], dim=1)
    room = 2.0**-8 * d.abs() + 2.0**-13 * d.abs().max()  # (its rounding; g and u are cut by 2^-15 of them at most, and off by their sums)
    compare(dx, d @ w64, room @ w64.abs() + 2.0**-18 * (d.abs() @ w64.abs()), "x")
    compare(dw[both.to(DEV)], d.t() @ x64, room.t() @ x64.abs() + 2.0**-18 * (d.t().abs() @ x64.abs()), "weight")
    dw[both.to(DEV)] = 0
    assert torch.count_nonzero(dw) == 0


@pytest.mark.parametrize("inner", [1000, 4000, 6000, 8000])
@pytest.mark.parametrize("rows", [16, 31, 33, 64, 80, 96])
def test_few_rows(rows, inner):
    """Every number of blocks of rows with 8, 16, 24 and 32 columns of hidden a workgroup, over depths that end inside a run and inside an operand."""
    for cols in (72, 200):
        assert name(rows, cols, inner) == "gated_few_rows"
        check(rows, cols, inner, BF16 if inner % 3 else FP16, "silu", backward=False, seed=rows)


def test_values_far_out():
    # gates whose exponentials overflow and underflow, and that are not finite
    x = torch.eye(8, dtype=BF16, device=DEV)
    w = torch.zeros(16, 8, dtype=BF16, device=DEV)
    gates = torch.tensor([0.0, 200.0, -200.0, 1e30, -1e30, float("inf"), float("nan"), 60.0], dtype=BF16, device=DEV)
    w[0], w[8:] = gates, 1.0
    for activation in ("silu", "gelu", "sigmoid"):
        got = A.gated_linear(x, w, None, activation)[0][:, 0].double().cpu()
        g = gates.double().cpu()
        # x holds zeros beside the one: a row meets its own gate, and 0 * (infinity, NaN) from the others
        assert torch.isnan(got).all()
        w[0] = torch.where(torch.isfinite(gates), gates, torch.zeros_like(gates))
        got = A.gated_linear(x, w, None, activation)[0][:, 0].double().cpu()
        want = act(activation, torch.where(torch.isfinite(g), g, torch.zeros_like(g)))
        want = torch.where(g.abs() > 100, torch.where(g > 0, torch.ones_like(g) if activation == "sigmoid" else g, torch.zeros_like(g)), want)
        want = torch.where(torch.isfinite(g), want, act(activation, torch.zeros_like(g)))
        assert torch.allclose(got, want, rtol=2.0**-8, atol=1e-30), (activation, got, want)
        dx, dw, _ = A.gated_linear_backward(torch.ones(8, 8, dtype=BF16, device=DEV), x, w, None, A.gated_linear(x, w, None, activation, True)[1], activation, [True, True, False])
        assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
        w[0] = gates


def test_rows_stay_alone():
    x, w, b, _ = (None if t is None else t.to(DEV) for t in inputs(300, 64, 72, BF16, True, 7))
    clean = A.gated_linear(x, w, b)[0]
    for rows in (300, 40):
        bad = x[:rows].clone()
        bad[17, 5] = float("nan")
        got, want = A.gated_linear(bad, w, b)[0], A.gated_linear(x[:rows], w, b)[0]
        rest = [i for i in range(rows) if i != 17]
        assert torch.equal(got[rest], want[rest]) and torch.isnan(got[17]).all()
    assert torch.equal(A.gated_linear(x, w, b)[0], clean)


def test_views_and_no_rows():
    x, w, b, dh = (t.to(DEV) for t in inputs(90, 72, 40, FP16, True, 9))
    wide = torch.zeros(90, 80, dtype=FP16, device=DEV)
    wide[:, 3:75] = x
    odd = torch.zeros(80 * 72 + 1, dtype=FP16, device=DEV)
    odd[1:] = w.flatten()
    assert torch.equal(A.gated_linear(wide[:, 3:75], odd[1:].view(80, 72), b)[0], A.gated_linear(x, w, b)[0])
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    hidden, mixed = A.gated_linear(*leaves, "silu", True)
    hidden.sum().backward()  # (a gradient that comes as an expanded view)
    want = A.gated_linear_backward(torch.ones_like(hidden), x, w, b, mixed.detach(), "silu", [True, True, True])
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))
    for wanted in ([True, False, False], [False, True, False], [False, False, True], [False, False, False]):
        got = A.gated_linear_backward(torch.ones_like(hidden), x, w, b, mixed.detach(), "silu", wanted)
        assert all(torch.equal(a, g) if want_it else a.numel() == 0 for a, g, want_it in zip(got, want, wanted))
    check(90, 72, 40, FP16, keep=False, seed=9)  # (g and u multiplied again)
    frozen = A.gated_linear(leaves[0], w, b, "silu", True)[0]
    (dx,) = torch.autograd.grad(frozen, leaves[0], dh)
    assert torch.equal(dx, A.gated_linear_backward(dh, x, w, b, mixed.detach(), "silu", [True, False, False])[0])
    assert frozen.requires_grad and not A.gated_linear(*leaves, "silu", True)[1].requires_grad  # (no gradient flows through mixed)
    none = torch.empty(0, 72, dtype=FP16, device=DEV, requires_grad=True)
    hidden, mixed = A.gated_linear(none, leaves[1], leaves[2], "silu", True)
    assert hidden.shape == (0, 40) and mixed.shape == (0,)
    dx, dw = torch.autograd.grad(hidden, [none, leaves[1]], hidden.detach())
    assert dx.shape == (0, 72) and torch.count_nonzero(dw) == 0 and dw.shape == w.shape


def test_the_same_bits_every_time_and_across_batches():
    x, w, b, dh = (t.to(DEV) for t in inputs(1500, 256, 264, BF16, True, 5))
    hidden, mixed = A.gated_linear(x, w, b, "silu", True)
    grads = A.gated_linear_backward(dh, x, w, b, mixed, "silu", [True, True, True])
    for _ in range(3):
        h, m = A.gated_linear(x, w, b, "silu", True)
        assert torch.equal(h, hidden) and torch.equal(m, mixed)
        assert all(torch.equal(a, c) for a, c in zip(A.gated_linear_backward(dh, x, w, b, mixed, "silu", [True, True, True]), grads))
    assert torch.equal(A.gated_linear(x, w, b)[0], hidden)
