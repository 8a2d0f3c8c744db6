"""residual_norm and norm_gate, forward and backward, against their definitions in 64 bits."""

import pytest
import torch

import ops_rec
import layer_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A = ops_rec.ascendc.activation
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def randn(gen, *shape, dtype=FP32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype)


def leaves(*tensors):
    return [None if t is None else t.to(DEV).requires_grad_(True) for t in tensors]


def columns_magnitude(terms):
    return terms.detach().abs().sum(0)


def check_residual_norm(rows, cols, dtype, stream, affine, rms=False, with_beta=True, with_scale=True, seed=0, offset=0.0, grads=(True, True)):
    g = torch.Generator().manual_seed(seed)
    x, residual = randn(g, rows, cols, dtype=dtype), randn(g, rows, cols, dtype=stream, std=1.5, mean=offset)
    gamma = randn(g, cols, dtype=affine, std=0.2, mean=1.0)
    beta = randn(g, cols, dtype=affine, std=0.2) if with_beta else None
    scale = randn(g, cols, dtype=affine, std=0.2, mean=0.7) if with_scale else None
    dy, dr = randn(g, rows, cols, dtype=dtype), randn(g, rows, cols, dtype=stream)
    ref_in = R.wide(x, residual, gamma, beta, scale)
    ref_y, ref_s = R.residual_norm(*ref_in, rms=rms)
    dev = leaves(x, residual, gamma, beta, scale)
    y, s = A.residual_norm(*dev, 1e-5, rms)
    assert y.dtype == dtype and s.dtype == stream and y.is_contiguous() and s.is_contiguous()
    n = R.norm(ref_s, rms, 1e-5)
    rstd = float(1 / ref_s.detach().var(1, unbiased=False).add(1e-5).sqrt().min()) if not rms else 1.0
    m = ref_y.abs().max().item() + ref_s.abs().max().item() * rstd
    R.check(s, ref_s, ref_s.abs().max().item(), "sum")
    R.check(y, ref_y, m, "y")
    outs = [(o, r, d) for o, r, d, want in ((y, ref_y, dy, grads[0]), (s, ref_s, dr, grads[1])) if want]
    got = torch.autograd.grad([o for o, _, _ in outs], [t for t in dev if t is not None], [d.to(DEV) for _, _, d in outs], allow_unused=True)
    want = torch.autograd.grad([r for _, r, _ in outs], [t for t in ref_in if t is not None], [d.double() for _, _, d in outs], allow_unused=True)
    ds = want[1].detach()
    m = ds.abs().max().item() * (1 + ref_s.abs().max().item() * rstd) + dy.abs().max().item() * gamma.abs().max().item() * rstd
    dy64, n = dy.double(), n.detach()
    terms = {"gamma": dy64 * n, "beta": dy64, "scale": ds * x.double()}
    for name, a, b in zip([k for k, t in zip(("x", "residual", "gamma", "beta", "scale"), dev) if t is not None], got, want):
        b = torch.zeros(a.shape, dtype=torch.float64) if b is None else b
        R.check(a, b, m if name in ("x", "residual") else columns_magnitude(terms[name]) + m, name)


SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (33, 64), (2, 65), (70, 100), (9, 128), (3, 250), (129, 512), (7, 513), (65, 1002), (5, 1024), (3, 2047),
         (4, 3000), (2, 4097), (3, 8192), (2, 8200), (2, 16384)]  # fmt: skip


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,stream,affine", [(BF16, BF16, FP32), (BF16, FP32, FP32), (FP16, FP16, FP16), (FP16, FP32, FP32), (FP32, FP32, FP32)])
def test_residual_norm(rows, cols, dtype, stream, affine):
    check_residual_norm(rows, cols, dtype, stream, affine, seed=rows + cols)
    check_residual_norm(rows, cols, dtype, stream, affine, rms=True, with_beta=False, with_scale=False, seed=rows * cols)


@pytest.mark.parametrize("grads", [(True, False), (False, True)])
@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (FP16, FP32)])
def test_residual_norm_with_one_of_its_gradients(dtype, stream, grads):
    check_residual_norm(37, 200, dtype, stream, FP32, grads=grads)
    check_residual_norm(37, 200, dtype, stream, FP32, with_scale=False, grads=grads)


def test_a_stream_far_from_zero():
    check_residual_norm(40, 512, FP32, FP32, FP32, offset=4096.0)
    check_residual_norm(40, 512, BF16, FP32, FP32, offset=-300.0, with_scale=False)


def test_many_rows():
    check_residual_norm(40000, 40, BF16, BF16, FP32)
    check_norm_gate(30011, 96, BF16, BF16, FP32, groups=4, silu=True)


def check_norm_gate(rows, cols, dtype, stream, affine, groups=1, rms=False, silu=False, with_gate=True, with_beta=True, with_residual=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, gate = randn(g, rows, cols, dtype=dtype, std=0.3), randn(g, rows, cols, dtype=dtype, std=2.0) if with_gate else None
    gamma = randn(g, cols, dtype=affine, std=0.2, mean=1.0)
    beta = randn(g, cols, dtype=affine, std=0.2) if with_beta else None
    residual = randn(g, rows, cols, dtype=stream, std=2.0) if with_residual else None
    d = randn(g, rows, cols, dtype=stream if with_residual else dtype)
    ref_in = R.wide(x, gate, gamma, beta, residual)
    ref = R.norm_gate(*ref_in, 0.25, groups, rms=rms, silu=silu)
    dev = leaves(x, gate, gamma, beta, residual)
    out = A.norm_gate(*dev, 0.25, groups, 1e-5, rms, silu)
    assert out.dtype == d.dtype and out.is_contiguous()
    parts = x.double().view(rows, groups, -1)
    size = (parts * parts).mean(-1) if rms else parts.var(-1, unbiased=False)
    rstd = float(1 / (size + 1e-5).sqrt().min())
    top = (gate.abs().max().item() if with_gate else 1.0) * (1.0 + parts.abs().max().item() * rstd) * (gamma.abs().max().item() + 1.0)
    R.check(out, ref, ref.abs().max().item() + top, "out")
    names = [k for k, t in zip(("x", "gate", "gamma", "beta", "residual"), dev) if t is not None]
    got = torch.autograd.grad([out], [t for t in dev if t is not None], [d.to(DEV)])
    want = torch.autograd.grad([ref], [t for t in ref_in if t is not None], [d.double()])
    act = 1.0 if gate is None else (gate.double() * torch.sigmoid(gate.double()) if silu else gate.double())
    dm = d.double() * act * (0.25 if with_residual else 1.0)
    n = R.norm(parts, rms, 1e-5).reshape(rows, cols)
    terms = {"gamma": dm * n, "beta": dm}
    m = float(d.abs().max()) * top * (1 + rstd)
    for name, a, b in zip(names, got, want):
        R.check(a, b, m if name in ("x", "gate", "residual") else columns_magnitude(terms[name]) + float(dm.abs().max()), name)


@pytest.mark.parametrize("rows,cols,groups", [(1, 1, 1), (3, 6, 3), (5, 56, 7), (33, 64, 1), (70, 512, 4), (9, 1000, 5), (64, 2048, 16), (3, 2050, 2),
                                              (2, 8192, 1), (4, 4096, 1), (5, 20480, 2), (130, 48, 16), (2, 40000, 8)])  # fmt: skip
@pytest.mark.parametrize("dtype,stream,affine", [(BF16, BF16, FP32), (BF16, FP32, BF16), (FP16, FP32, FP32), (FP32, FP32, FP32)])
def test_norm_gate(rows, cols, groups, dtype, stream, affine):
    check_norm_gate(rows, cols, dtype, stream, affine, groups, silu=True, seed=rows + cols)
    check_norm_gate(rows, cols, dtype, stream, affine, groups, rms=True, with_beta=False, with_residual=True, seed=rows)
    check_norm_gate(rows, cols, dtype, stream, affine, groups, with_gate=False, with_residual=rows % 2 == 0, seed=cols)


def test_strided_rows():
    g = torch.Generator().manual_seed(5)
    wide = randn(g, 50, 700, dtype=BF16).to(DEV)
    x, gate, residual = wide[:, 3:203], wide[:, 250:450], wide[::1, 499:699]
    gamma = randn(g, 200).to(DEV)
    for out, same in zip(A.residual_norm(x, residual, gamma), A.residual_norm(x.contiguous(), residual.contiguous(), gamma)):
        assert torch.equal(out, same)
    assert torch.equal(A.norm_gate(x, gate, gamma, None, residual, 0.5, 4), A.norm_gate(x.contiguous(), gate.contiguous(), gamma, None, residual.contiguous(), 0.5, 4))
    across = randn(g, 200, 50, dtype=BF16).to(DEV).t()  # (columns side by side: copied)
    assert torch.equal(A.norm_gate(across, gate, gamma), A.norm_gate(across.contiguous(), gate, gamma))
    one = x[:1].expand(50, 200)  # a row for all
    assert torch.equal(A.residual_norm(one, residual, gamma)[0], A.residual_norm(one.contiguous(), residual, gamma)[0])
    # gradients that come as expanded views, and through strided inputs
    leaf = wide.clone().requires_grad_(True)
    A.norm_gate(leaf[:, 3:203], leaf[:, 250:450], gamma, None, None, 1.0, 4).sum().backward()
    dx, du, _, _ = A.norm_gate_backward(torch.ones(50, 200, dtype=BF16, device=DEV), x, gate, gamma, None, False, 1.0, 4, 1e-5, False, False)
    assert torch.equal(leaf.grad[:, 3:203], dx) and torch.equal(leaf.grad[:, 250:450], du) and torch.count_nonzero(leaf.grad[:, :3]) == 0


def test_no_rows():
    x, gamma = torch.empty(0, 24, device=DEV, requires_grad=True), torch.ones(24, device=DEV, requires_grad=True)
    y, s = A.residual_norm(x, x, gamma)
    assert y.shape == s.shape == (0, 24)
    dx, dg = torch.autograd.grad([y, s], [x, gamma], [y.detach(), s.detach()])
    assert dx.shape == (0, 24) and torch.equal(dg, torch.zeros(24, device=DEV))
    out = A.norm_gate(x, x, gamma, gamma, None, 1.0, 3)
    dx, dg = torch.autograd.grad([out], [x, gamma], [out.detach()])
    assert dx.shape == (0, 24) and torch.equal(dg, torch.zeros(24, device=DEV))


@pytest.mark.parametrize("cols", [40, 100, 512, 1002, 4097])
def test_a_row_that_is_not_finite_stays_alone(cols):
    g = torch.Generator().manual_seed(cols)
    x, residual, gamma = randn(g, 9, cols, dtype=BF16).to(DEV), randn(g, 9, cols, dtype=BF16).to(DEV), randn(g, cols).to(DEV)
    clean = A.residual_norm(x, residual, gamma)[0]
    back = A.residual_norm_backward(x, x, x, residual, None, gamma, None, False, BF16, 1e-5, False)
    for bad in (float("nan"), float("inf")):
        xx = x.clone()
        xx[4, cols - 1] = bad
        y = A.residual_norm(xx, residual, gamma)[0]
        rest = [i for i in range(9) if i != 4]
        assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[4]).any()
        db = A.residual_norm_backward(x, x, xx, residual, None, gamma, None, False, BF16, 1e-5, False)
        assert torch.equal(db[1][rest], back[1][rest]) and torch.isnan(db[1][4]).all()


@pytest.mark.parametrize("cols", [7, 64, 1002, 8200])
def test_a_row_with_nan_has_no_root_mean_square(cols):
    g = torch.Generator().manual_seed(cols)
    x, gamma = randn(g, 5, cols, dtype=BF16).to(DEV), randn(g, cols).to(DEV)
    x[2, cols // 2] = float("nan")
    y, total = A.residual_norm(x, x, gamma, rms=True)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all() and int(torch.isnan(total).sum()) == 1
    assert torch.isnan(A.norm_gate(x, None, gamma, rms=True)[2]).all()
    x[2, cols // 2] = float("inf")
    y = A.norm_gate(x, None, gamma, rms=True)
    assert int(torch.isnan(y[2]).sum()) == 1 and torch.count_nonzero(y[2]) == 1  # inf / inf there, the others' share is 0


def test_rows_of_equal_values():
    gamma, beta = torch.full((64,), 2.0, device=DEV), torch.full((64,), 0.5, device=DEV)
    x = torch.tensor([0.0, 1.0, -3.5, 1000.0], device=DEV)[:, None].repeat(1, 64)
    y, _ = A.residual_norm(x, torch.zeros_like(x), gamma, beta)
    assert torch.equal(y, torch.full_like(y, 0.5))
    assert torch.equal(A.norm_gate(torch.zeros_like(x), None, gamma, None, None, 1.0, 8, 1e-5, True), torch.zeros_like(x))


def test_the_same_bits_every_time_and_in_any_batch():
    g = torch.Generator().manual_seed(3)
    x, residual, gamma = randn(g, 3001, 512, dtype=BF16).to(DEV), randn(g, 3001, 512).to(DEV), randn(g, 512).to(DEV)
    first = A.residual_norm(x, residual, gamma)
    sums = A.residual_norm_backward(x, residual, None, None, first[1], gamma, None, True, BF16, 1e-5, False)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(A.residual_norm(x, residual, gamma), first))
        assert all(torch.equal(a, b) for a, b in zip(A.residual_norm_backward(x, residual, None, None, first[1], gamma, None, True, BF16, 1e-5, False), sums))
    part = A.residual_norm(x[1000:1007], residual[1000:1007], gamma)
    assert torch.equal(part[0], first[0][1000:1007]) and torch.equal(part[1], first[1][1000:1007])


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(11)
    x, residual, gamma, beta, scale = (randn(g, *s).to(DEV) for s in ((3, 24), (3, 24), (24,), (24,), (24,)))
    w, v = randn(g, 3, 24).to(DEV).double(), randn(g, 3, 24).to(DEV).double()

    def loss(*t):
        y, s = A.residual_norm(*t[:2], *t[2:])
        z = A.norm_gate(y, s, t[2], t[3], t[1], 0.5, 3, 1e-5, False, True)
        return (z.double() * w).sum() + (y.double() * v).sum()

    tensors = [t.requires_grad_(True) for t in (x, residual, gamma, beta, scale)]
    grads = torch.autograd.grad(loss(*tensors), tensors)
    step = 2.0**-6
    for i, t in enumerate(tensors):
        direction = randn(g, *t.shape).to(DEV)
        with torch.no_grad():
            ends = [loss(*(u + s * step * direction if j == i else u for j, u in enumerate(tensors))) for s in (1, -1, 2, -2)]
        slope = (8 * (ends[0] - ends[1]) - (ends[2] - ends[3])) / (12 * step)  # (off by step^4)
        exact = (grads[i].double() * direction.double()).sum()
        assert abs(slope - exact) <= 2e-3 * (1 + abs(exact)), (i, slope.item(), exact.item())
