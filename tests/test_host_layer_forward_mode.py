"""Forward-mode differentiation through the operators of a layer: they have no formulas for it, and say so instead of losing the tangent (no GPU needed)."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

import ops_rec  # noqa: F401  (defines the operators)
from ops_rec import _layer

OPS = torch.ops.ops_rec


def calls(device):
    """name -> (call, its differentiable inputs)"""
    half = dict(dtype=torch.bfloat16, device=device)
    x, r, g = torch.zeros(5, 24, **half), torch.zeros(5, 24, device=device), torch.ones(24, device=device)
    q, f, offs = torch.zeros(5, 2, 8, device=device), torch.ones(4, dtype=torch.float64, device=device), torch.zeros(3, dtype=torch.int32, device=device)
    w, b = torch.zeros(32, 24, **half), torch.zeros(32, **half)
    return {
        "residual_norm": (lambda fn, t: fn(*t), [x, r, g, g + 1, g + 2]),
        "norm_gate": (lambda fn, t: fn(*t), [x, x + 1, g, g + 1, r]),
        "rotary": (lambda fn, t: fn(*t, f, offs), [q, q + 1]),
        "gated_linear": (lambda fn, t: fn(*t, "silu", True), [x, w, b]),
    }


@pytest.mark.parametrize("name,count", [("residual_norm", 5), ("norm_gate", 5), ("rotary", 2), ("gated_linear", 3)])
@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("through_the_dispatcher", [True, False])
def test_a_tangent_is_refused(name, count, recorded, through_the_dispatcher):
    def every(call, inputs, fn):
        assert len(inputs) == count
        with forward_ad.dual_level():
            for i, t in enumerate(inputs):
                for grad_mode in (True, False):
                    dual = forward_ad.make_dual(t, torch.ones_like(t))
                    rest = [u.detach().requires_grad_(recorded) if j != i else dual for j, u in enumerate(inputs)]
                    with torch.set_grad_enabled(grad_mode), pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
                        call(fn, rest)

    if through_the_dispatcher:
        with FakeTensorMode():
            call, inputs = calls("cuda")[name]
            every(call, inputs, getattr(OPS, name))
            call(getattr(OPS, name), inputs)  # (without a tangent, inside a level or not, nothing changes)
            with forward_ad.dual_level():
                call(getattr(OPS, name), inputs)
    else:
        call, inputs = calls("cpu")[name]
        every(call, inputs, getattr(_layer, name))
