"""A layer of the operators around attention, as a model chains them, forward and backward: residual_norm -> in_linear_silu -> rotary ->
hstu_jagged -> norm_gate -> output projection -> residual_norm -> gated_linear -> projection, against the same chain in 64 bits."""

import pytest
import torch

import ops_rec
import layer_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACT, ATT = ops_rec.ascendc.activation, ops_rec.ascendc.attention


@pytest.fixture(autouse=True)
def _memory_goes_back():
    """Cached blocks go back to the device after each test: tests that count what the allocator takes find it as they expect it."""
    yield
    torch.cuda.empty_cache()


def weights(cols, heads, dim, inner, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    hd = heads * dim

    def matrix(n, k):
        return (torch.randn(n, k, generator=g) / k**0.5).to(dtype)

    return dict(gamma1=1.0 + 0.1 * torch.randn(cols, generator=g), beta1=0.1 * torch.randn(cols, generator=g), w_in=matrix(4 * hd, cols),
                b_in=0.1 * torch.randn(4 * hd, generator=g), gamma2=1.0 + 0.1 * torch.randn(hd, generator=g), beta2=0.1 * torch.randn(hd, generator=g),
                w_out=matrix(cols, hd), scale=0.5 + 0.1 * torch.randn(cols, generator=g), gamma3=1.0 + 0.1 * torch.randn(cols, generator=g),
                w_gated=matrix(2 * inner, cols), b_gated=(0.1 * torch.randn(2 * inner, generator=g)).to(dtype), w_down=matrix(cols, inner))  # fmt: skip


def layer(x, stream, w, offsets, heads, dim, longest, frequencies):
    """The layer's output, which the next layer's residual_norm adds to the stream, and the stream."""
    rows, hd = x.size(0), heads * dim
    a, stream = ACT.residual_norm(x, stream, w["gamma1"], w["beta1"])
    u, v, q, k, _ = ACT.distance_in_linear_silu(a, w["w_in"], w["b_in"], [hd] * 4)
    q, k = ATT.rotary(q.view(rows, heads, dim), k.view(rows, heads, dim), frequencies, offsets)
    o = ATT.hstu_jagged(q, k, v.view(rows, heads, dim), None, None, 0, longest, 1.0 / 16, offsets, None, None, 0, dim**-0.5)
    o = ACT.norm_gate(o.view(rows, hd), u, w["gamma2"], w["beta2"], groups=heads)
    b, stream = ACT.residual_norm(o @ w["w_out"].t(), stream, w["gamma3"], scale=w["scale"], rms=True)
    return ACT.gated_linear(b, w["w_gated"], w["b_gated"], "silu", True)[0] @ w["w_down"].t(), stream


def layer_wide(x, stream, w, offsets, heads, dim, frequencies):
    rows, hd = x.size(0), heads * dim
    a, stream = R.residual_norm(x, stream, w["gamma1"], w["beta1"])
    u, v, q, k = torch.nn.functional.silu(a @ w["w_in"].t() + w["b_in"]).split([hd] * 4, dim=1)
    place = R.positions(offsets, None, rows)
    q, k, v = R.rotary(q.reshape(rows, heads, dim), place, frequencies), R.rotary(k.reshape(rows, heads, dim), place, frequencies), v.reshape(rows, heads, dim)
    parts = []
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        s = torch.nn.functional.silu(q[lo:hi].transpose(0, 1) @ k[lo:hi].permute(1, 2, 0) * dim**-0.5) / 16
        parts.append((torch.tril(s) @ v[lo:hi].transpose(0, 1)).transpose(0, 1))
    o = R.norm_gate(torch.cat(parts).reshape(rows, hd), u, w["gamma2"], w["beta2"], groups=heads)
    b, stream = R.residual_norm(o @ w["w_out"].t(), stream, w["gamma3"], None, w["scale"], rms=True)
    g, up = (b @ w["w_gated"].t() + w["b_gated"]).chunk(2, dim=1)
    return (torch.nn.functional.silu(g) * up) @ w["w_down"].t(), stream


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim,cols,inner,lengths", [(2, 64, 64, 96, [5, 130, 1, 77]), (4, 128, 256, 512, [300, 1, 258, 64]), (1, 32, 32, 136, [1])])
def test_a_layer_and_its_gradients(heads, dim, cols, inner, lengths, dtype):
    g = torch.Generator().manual_seed(len(lengths))
    offsets = [0] + torch.tensor(lengths).cumsum(0).tolist()
    rows = offsets[-1]
    w = weights(cols, heads, dim, inner, dtype, heads)
    x, stream = torch.randn(rows, cols, generator=g).to(dtype), torch.randn(rows, cols, generator=g)
    dy, ds = torch.randn(rows, cols, generator=g).to(dtype), torch.randn(rows, cols, generator=g)
    frequencies, _ = ops_rec.rotary_frequencies(dim)
    leaves = {"x": x, "stream": stream, **w}
    on = {n: t.to(DEV).requires_grad_(True) for n, t in leaves.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in leaves.items()}
    outs = layer(on["x"], on["stream"], on, torch.tensor(offsets, dtype=torch.int32, device=DEV), heads, dim, max(lengths), frequencies.to(DEV))
    refs = layer_wide(wide["x"], wide["stream"], wide, offsets, heads, dim, frequencies)
    assert outs[0].dtype == dtype and outs[1].dtype == torch.float32
    got = dict(zip(on, torch.autograd.grad(outs, list(on.values()), [dy.to(DEV), ds.to(DEV)])))
    want = dict(zip(wide, torch.autograd.grad(refs, list(wide.values()), [dy.double(), ds.double()])))
    # What a value has been rounded by, over the whole tensor: half a step of it at most, each time.  The output lies behind nine roundings (a, the
    # projection and its silu, q or k, o, the gated o, its projection, b, hidden, the output) and each of them is carried on with a gain of at
    # most 2 of the relative size over the tensor (the gated norm of a head, whose spread is about its size, the products of two rounded values);
    # a gradient comes back through as many again, with the same gains.
    for name, a, b, roundings in [("out", outs[0], refs[0], 9), ("sum", outs[1], refs[1], 9)] + [(n, got[n], want[n], 18) for n in on]:
        a, b = a.detach().double().cpu(), b.detach()
        assert a.shape == b.shape
        assert float((a - b).norm()) <= 2 * roundings * R.HALF_STEP[dtype] * float(b.norm()), name
