"""residual_norm, norm_gate, rotary and gated_linear in every way in which a program calls them: natively and through the Python
implementations, traced and compiled, captured into graphs, on streams of their own, two at once, into memory that holds NaN, over rows
that overlap, past 2^31 elements."""

import pytest
import torch

import ops_rec
import helpers
from ops_rec import _ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACT, ROTARY = ops_rec.ascendc.activation, ops_rec.ascendc.attention.rotary
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
CHECKS = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
GRAPH = CHECKS + ("test_autograd_registration",)
BACKENDS = ["aot_eager", "inductor"]


@pytest.fixture(autouse=True)
def _memory_goes_back():
    """Cached blocks go back to the device after each test: tests that count what the allocator takes find it as they expect it."""
    yield
    torch.cuda.empty_cache()


def randn(seed, *shape, dtype=FP32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype).to(DEV)


def residual_norm_call(rows=70, cols=200, dtype=BF16, stream=FP32, seed=0):
    tensors = (randn(seed, rows, cols, dtype=dtype), randn(seed + 1, rows, cols, dtype=stream, std=2.0), randn(seed + 2, cols, std=0.1, mean=1.0),
               randn(seed + 3, cols), randn(seed + 4, cols))  # fmt: skip
    return ACT.residual_norm, tensors, (1e-5, False)


def norm_gate_call(rows=70, cols=200, dtype=BF16, stream=FP32, seed=0):
    tensors = (randn(seed, rows, cols, dtype=dtype), randn(seed + 1, rows, cols, dtype=dtype), randn(seed + 2, cols, std=0.1, mean=1.0), randn(seed + 3, cols),
               randn(seed + 4, rows, cols, dtype=stream))  # fmt: skip
    return ACT.norm_gate, tensors, (0.5, 4, 1e-5, False, True)


def rotary_call(rows=70, heads=4, heads_k=2, dim=64, dtype=BF16, seed=0):
    tensors = (randn(seed, rows, heads, dim, dtype=dtype), randn(seed + 1, rows, heads_k, dim, dtype=dtype))
    offsets = torch.tensor([0, rows // 3, rows // 3, rows - 2], device=DEV)
    return ROTARY, tensors, (ops_rec.rotary_frequencies(48, device=DEV)[0], offsets, torch.tensor([7, 0, 100003], device=DEV), None, False, 1.1)


def gated_linear_call(rows=70, cols=256, inner=264, dtype=BF16, seed=0):
    tensors = (randn(seed, rows, cols, dtype=dtype), randn(seed + 1, 2 * inner, cols, dtype=dtype, std=cols**-0.5), randn(seed + 2, 2 * inner, dtype=dtype))
    return lambda *a: ACT.gated_linear(*a)[0], tensors, ("silu", True)


CALLS = {"residual_norm": residual_norm_call, "norm_gate": norm_gate_call, "rotary": rotary_call, "gated_linear": gated_linear_call}
calls = pytest.mark.parametrize("name", list(CALLS))


def listed(outs):
    return [outs] if torch.is_tensor(outs) else list(outs)


def grads_for(outs, seed=50):
    return [randn(seed + i, *o.shape).to(o.dtype) for i, o in enumerate(outs)]


def forward_and_gradients(fn, tensors, rest):
    """Outputs and the gradients of every tensor, for gradients of the outputs that the seed alone makes; leaves of its own every time."""
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    outs = listed(fn(*leaves, *rest))
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, grads_for(outs)))


def same(got, want):
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------- two implementations ----


def operator_calls():
    """(operator, arguments) of every operator, the backward ones among them."""
    _, (x, residual, gamma, beta, scale), _ = residual_norm_call()
    y, total = ACT.residual_norm(x, residual, gamma, beta, scale)
    narrow = residual.to(BF16)
    yield "residual_norm", (x, residual, gamma, beta, scale, 1e-5, False)
    yield "residual_norm", (x, narrow, gamma, None, None, 1e-3, True)
    yield "residual_norm_backward", (randn(9, *x.shape, dtype=BF16), randn(8, *x.shape), x, None, total, gamma, scale, True, BF16, 1e-5, False)
    yield "residual_norm_backward", (randn(9, *x.shape, dtype=BF16), None, None, None, total, gamma, None, False, BF16, 1e-5, True)
    yield "residual_norm_backward", (None, randn(9, *x.shape, dtype=BF16), x, narrow, None, gamma, None, True, BF16, 1e-5, False)
    _, (x, gate, gamma, beta, residual), rest = norm_gate_call()
    yield "norm_gate", (x, gate, gamma, beta, residual, *rest)
    yield "norm_gate", (x, None, gamma, None, None, 1.0, 1, 1e-5, True, False)
    yield "norm_gate_backward", (randn(9, *x.shape), x, gate, gamma, beta, True, *rest)
    yield "norm_gate_backward", (randn(9, *x.shape, dtype=BF16), x, None, gamma, None, False, 1.0, 2, 1e-5, True, False)
    _, (q, k), rest = rotary_call()
    yield "rotary", (q, k, *rest)
    yield "rotary", (q, k, rest[0], None, None, torch.arange(70, dtype=torch.int32, device=DEV), True, 1.0, True)
    _, (x, weight, bias), _ = gated_linear_call()
    hidden, mixed = ACT.gated_linear(x, weight, bias, "gelu", True)
    yield "gated_linear", (x, weight, bias, "gelu", True)
    yield "gated_linear", (x, weight, None, "sigmoid", False)
    yield "gated_linear_backward", (randn(9, *hidden.shape, dtype=BF16), x, weight, bias, mixed, "gelu", [True, True, True])
    yield "gated_linear_backward", (randn(9, *hidden.shape, dtype=BF16), x, weight, None, torch.empty(0, dtype=torch.int16, device=DEV), "silu", [False, True, False])


def test_native_kernels_and_python_implementations_give_the_same_bits():
    for name, args in operator_calls():
        native, python = listed(getattr(torch.ops.ops_rec, name)(*args)), listed(_ops._PYTHON_KERNELS[name](*args))
        assert same(native, python), name
        assert all(a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride() for a, b in zip(native, python)), name


def test_opcheck_of_every_operator():
    for name, args in operator_calls():
        op = getattr(torch.ops.ops_rec, name).default
        if name.endswith("_backward"):
            torch.library.opcheck(op, args, test_utils=CHECKS)
        else:
            leaves = tuple(a.clone().requires_grad_(True) if torch.is_tensor(a) and a.dtype in (BF16, FP32) else a for a in args)
            torch.library.opcheck(op, leaves, test_utils=GRAPH)


@calls
@pytest.mark.parametrize("backend", BACKENDS)
def test_compiled(name, backend):
    fn = None
    torch._dynamo.reset()
    for rows in (70, 33):
        op, tensors, rest = CALLS[name](rows=rows)
        fn = fn or torch.compile(op, backend=backend, fullgraph=True, dynamic=True)
        try:
            got = listed(fn(*tensors, *rest))
            gradients = forward_and_gradients(fn, tensors, rest)
        except torch._dynamo.exc.BackendCompilerFailed as err:
            pytest.skip(f"inductor could not generate code here: {str(err)[:200]}")
        assert same(got, listed(op(*tensors, *rest)))
        assert same(gradients, forward_and_gradients(op, tensors, rest))  # (the operators' own gradients, nothing generated between)


# ------------------------------------------------------------------------------------------------ graphs, streams ----


@calls
@pytest.mark.parametrize("rows", [5, 700])
def test_replays_of_a_captured_step(name, rows):
    """Forward and backward captured together, replayed on other values with eager calls of the same between; leaves of the capture's
    own."""
    make = CALLS[name]
    op, static, rest = make(rows=rows)
    static = [t.clone() for t in static]
    d = grads_for(listed(op(*static, *rest)))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in static]
        outs = listed(op(*leaves, *rest))
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, d))

    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (100, 200, 0, 300):
        values = make(rows=rows, seed=seed)[1]
        for a, b in zip(static, values):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = forward_and_gradients(op, values, rest)
        assert same(got, want), seed


def test_two_graphs_replayed_side_by_side():
    """Each capture has workspaces of its own: replays of both at once on two streams leave each other's results alone."""
    kept = []
    for seed in (0, 40):
        steps = [CALLS[name](rows=900, seed=seed) for name in CALLS]
        want = [forward_and_gradients(*s) for s in steps]
        d = [grads_for(w[: len(w) - len(s[1])]) for w, s in zip(want, steps)]

        def step(steps=steps, d=d):
            got = []
            for (fn, tensors, rest), g in zip(steps, d):
                leaves = [t.detach().requires_grad_(True) for t in tensors]
                outs = listed(fn(*leaves, *rest))
                got.append([o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, g)))
            return got

        side = torch.cuda.Stream(device=DEV)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        kept.append((graph, captured, want, step))  # (step holds what the graph reads)
    streams = [torch.cuda.Stream(device=DEV) for _ in kept]
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, *_), s in zip(kept, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, captured, want, _ in kept:
            assert all(same(a, b) for a, b in zip(captured, want))


@calls
def test_on_streams_of_their_own(name):
    """Two calls at once on two streams, inputs made there too: a launch on another stream would read them too early."""
    streams, got = [torch.cuda.Stream(device=DEV) for _ in range(2)], []
    want = [forward_and_gradients(*CALLS[name](rows=3000, seed=s)) for s in (0, 60)]
    sources = [CALLS[name](rows=3000, seed=s) for s in (0, 60)]
    torch.cuda.synchronize()
    for (op, tensors, rest), s in zip(sources, streams):
        with torch.cuda.stream(s):
            busy = torch.zeros(1 << 26, device=DEV)
            for _ in range(4):
                busy += 1.0  # (some milliseconds before the inputs are there)
            got.append(forward_and_gradients(op, [t.clone() + busy[0].to(t.dtype) * 0 for t in tensors], rest))
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, want))


@calls
@pytest.mark.parametrize("rows", [1, 70, 2500])
def test_memory_that_holds_nan(name, rows, monkeypatch):
    op, tensors, rest = CALLS[name](rows=rows) if name != "rotary" or rows > 6 else CALLS[name](rows=7)
    want = forward_and_gradients(op, tensors, rest)
    helpers.poison_workspace(monkeypatch)
    got = forward_and_gradients(op, tensors, rest)
    assert same(got, want) and all(bool(torch.isfinite(t).all()) for t in got)


# --------------------------------------------------------------------------------------------------- odd layouts ----


def test_rows_that_overlap_and_the_same_tensor_twice():
    """Inputs may be one tensor, one row for all rows, or windows of one row: they are only read."""
    gamma = randn(1, 64, mean=1.0)
    x = randn(2, 40, 64, dtype=BF16)
    assert same(listed(ACT.residual_norm(x, x, gamma)), listed(ACT.residual_norm(x.clone(), x.clone(), gamma)))
    wide = x[:1].expand(40, 64)
    assert same(listed(ACT.residual_norm(wide, x, gamma)), listed(ACT.residual_norm(wide.contiguous(), x, gamma)))
    window = randn(3, 200, dtype=BF16).as_strided((40, 64), (3, 1))
    assert torch.equal(ACT.norm_gate(window, window, gamma), ACT.norm_gate(window.contiguous(), window.contiguous(), gamma))
    q = randn(4, 40, 2, 64, dtype=BF16)
    f, at = ops_rec.rotary_frequencies(64, device=DEV)[0], torch.full((40,), 77, dtype=torch.int32, device=DEV)
    got = ROTARY(q, q, f, positions=at)
    assert torch.equal(got[0], got[1])
    shared = q[:, :1].expand(40, 5, 64)
    assert torch.equal(ROTARY(shared, q, f, positions=at)[0], got[0][:, :1].expand(40, 5, 64))
    # a broadcast input's gradient is the sum of its rows', added by the framework in its own order
    one = x[:1].float().requires_grad_(True)
    many = one.detach().expand(40, 64).contiguous().requires_grad_(True)
    d = randn(5, 40, 64)
    (a,) = torch.autograd.grad(ACT.residual_norm(one.expand(40, 64), x.float(), gamma)[0], one, d)
    (b,) = torch.autograd.grad(ACT.residual_norm(many, x.float(), gamma)[0], many, d)
    assert torch.allclose(a, b.sum(0, keepdim=True), rtol=0, atol=40 * 2.0**-23 * float(b.abs().max()))


def test_gradients_that_are_expanded():
    for name in CALLS:
        op, tensors, rest = CALLS[name]()
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        got = torch.autograd.grad(sum(o.sum() for o in listed(op(*leaves, *rest))), leaves)
        outs = listed(op(*leaves, *rest))
        want = torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
        assert same(got, want), name


def test_past_31_bits_of_elements():
    """Rows far behind the start of a large buffer come out as they do by themselves: strided rows, and outputs of more than 2^31 elements."""
    rows, cols = 2_100_000, 1024  # 2.15e9 elements of 2 bytes
    x = torch.empty(rows, cols, dtype=BF16, device=DEV)
    x.zero_()
    picked = torch.tensor([0, 1, 2_097_150, 2_097_151, 2_097_152, 2_097_153, rows - 2, rows - 1], device=DEV)
    values = randn(1, len(picked), cols, dtype=BF16)
    x[picked] = values
    gamma, beta = randn(2, cols, mean=1.0), randn(3, cols)
    got = ACT.norm_gate(x, x, gamma, beta)
    assert torch.equal(got[picked], ACT.norm_gate(values, values, gamma, beta))
    del got
    y, total = ACT.residual_norm(x, x, gamma, beta)
    want = ACT.residual_norm(values, values, gamma, beta)
    assert torch.equal(y[picked], want[0]) and torch.equal(total[picked], want[1])
    del y, total
    heads = x.view(rows, 8, 128)
    f, at = ops_rec.rotary_frequencies(128, device=DEV)[0], torch.arange(rows, device=DEV)
    got = ROTARY(heads, heads[:, :1], f, positions=at)[0]
    assert torch.equal(got[picked], ROTARY(values.view(-1, 8, 128), values.view(-1, 8, 128)[:, :1], f, positions=at[picked])[0])
    del got
    weight = randn(4, 16, cols, dtype=BF16, std=0.03)
    got = ACT.gated_linear(x, weight)[0]  # (x past 31 bits)
    assert torch.equal(got[picked][:, :], ACT.gated_linear(x[picked.repeat(300)], weight)[0][: len(picked)])
    del x, got
    x = torch.zeros(rows, 8, dtype=BF16, device=DEV)
    x[picked] = values[:, :8]
    weight = randn(5, 2048, 8, dtype=BF16, std=0.3)
    got = ACT.gated_linear(x, weight)[0]  # (hidden past 31 bits)
    assert torch.equal(got[picked], ACT.gated_linear(x[picked.repeat(300)], weight)[0][: len(picked)])


def test_gradients_past_31_bits_of_elements():
    """Gradients on a few rows of a large batch, zeros on the others: their rows come out as in a batch of their own, and columns as the sums over them."""
    rows, cols = 2_100_000, 1024
    picked = torch.tensor([0, 1, 2_097_150, 2_097_151, 2_097_152, 2_097_153, rows - 2, rows - 1], device=DEV)
    few = [randn(i, len(picked), cols, dtype=BF16) for i in range(3)]
    x, gate, grad = (torch.zeros(rows, cols, dtype=BF16, device=DEV) for _ in range(3))
    for t, v in zip((x, gate, grad), few):
        t[picked] = v
    gamma, beta = randn(4, cols, mean=1.0), randn(5, cols)
    rest = (False, 1.0, 1, 1e-5, False, True)
    got, want = ACT.norm_gate_backward(grad, x, gate, gamma, beta, *rest), ACT.norm_gate_backward(few[2], few[0], few[1], gamma, beta, *rest)
    assert all(torch.equal(a[picked], b) for a, b in zip(got[:2], want[:2]))
    assert all(torch.allclose(a, b, rtol=0, atol=2.0**-18 * float(b.abs().max())) for a, b in zip(got[2:], want[2:]))
    got = ACT.residual_norm_backward(grad, gate, x, x, None, gamma, None, True, BF16, 1e-5, False)
    want = ACT.residual_norm_backward(few[2], few[1], few[0], few[0], None, gamma, None, True, BF16, 1e-5, False)
    assert torch.equal(got[1][picked], want[1])
    del x, gate, grad, got
    # d_mixed of 8.6e9 elements
    inner = 2048
    x, grad = torch.zeros(rows, 8, dtype=BF16, device=DEV), torch.zeros(rows, inner, dtype=BF16, device=DEV)
    xs, ds = randn(6, len(picked), 8, dtype=BF16), randn(7, len(picked), inner, dtype=BF16)
    x[picked], grad[picked] = xs, ds
    weight = randn(8, 2 * inner, 8, dtype=BF16, std=0.3)
    dx, dw, _ = ACT.gated_linear_backward(grad, x, weight, None, torch.empty(0, dtype=torch.int16, device=DEV), "sigmoid", [True, True, False])
    x64, w64, d64 = (t.double().cpu() for t in (xs, weight, ds))
    g, u = (x64 @ w64.t()).chunk(2, dim=1)
    a = torch.sigmoid(g)
    d_mixed = torch.cat([d64 * u * a * (1 - a), d64 * a], dim=1)
    # d_mixed is rounded by half a step of its values, 2^-8 of them, and the results by as much again
    for got, want, room in ((dx[picked], d_mixed @ w64, d_mixed.abs() @ w64.abs()), (dw, d_mixed.t() @ x64, d_mixed.abs().t() @ x64.abs())):
        assert bool(((got.double().cpu() - want).abs() <= 2.0**-8 * want.abs() * (1 + 2.0**-7) + (2.0**-8 + 2.0**-17) * room).all())
    dx[picked] = 0
    assert torch.count_nonzero(dx) == 0


def test_second_derivatives_of_a_rotation():
    """A rotation is linear: the gradient of its gradient is a rotation again."""
    _, (q, k), rest = rotary_call(dtype=FP32)
    q, d = q.requires_grad_(True), randn(77, *q.shape).requires_grad_(True)
    (dq,) = torch.autograd.grad(ROTARY(q, k, *rest)[0], q, d, create_graph=True)
    e = randn(78, *q.shape)
    (back,) = torch.autograd.grad(dq, d, e)
    assert torch.equal(back, ROTARY(e, k, *rest)[0])
