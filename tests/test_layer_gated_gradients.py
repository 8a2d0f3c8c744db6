"""gated_linear's backward where tests/test_layer_gated_linear.py does not go: values that are not finite, the ends of fp16, every tile of its products, what is kept above
192 columns of x, and the largest sizes."""

import pytest
import torch

import ops_rec

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A = ops_rec.ascendc.activation
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _memory_goes_back():
    """Cached blocks go back to the device after each test: tests that count what the allocator takes find it as they expect it."""
    yield
    torch.cuda.empty_cache()


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
