"""The layer operators in 64 bits, by their definitions, for the tests: forward with torch.float64, gradients by autograd."""

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def wide(*tensors):
    return [None if t is None else t.detach().double().cpu().requires_grad_(True) for t in tensors]


def norm(s, rms, eps):
    if rms:
        return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    c = s - s.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)


def residual_norm(x, residual, gamma, beta=None, scale=None, eps=1e-5, rms=False):
    s = residual + (x if scale is None else scale * x)
    y = norm(s, rms, eps) * gamma
    return (y if beta is None else y + beta), s


def norm_gate(x, gate, gamma, beta=None, residual=None, residual_scale=1.0, groups=1, eps=1e-5, rms=False, silu=False):
    m = norm(x.view(x.size(0), groups, -1), rms, eps).reshape(x.shape) * gamma
    if beta is not None:
        m = m + beta
    if gate is not None:
        m = m * (gate * torch.sigmoid(gate) if silu else gate)
    return m if residual is None else residual + residual_scale * m


def rotary(t, position, frequencies, interleaved=False, magnitude=1.0):
    """``position`` [rows] in 64 bits, NaN where a row has none (its result is 0)."""
    n = frequencies.numel()
    angle = torch.nan_to_num(position)[:, None, None] * frequencies
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    a, b = (t[..., 0 : 2 * n : 2], t[..., 1 : 2 * n : 2]) if interleaved else (t[..., :n], t[..., n : 2 * n])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)
    out = torch.cat([turned, t[..., 2 * n :]], dim=-1)
    return torch.where(torch.isnan(position)[:, None, None], torch.zeros_like(out), out)


def positions(offsets, start, rows):
    place = torch.full((rows,), float("nan"), dtype=torch.float64)
    for b, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        place[lo:hi] = torch.arange(hi - lo, dtype=torch.float64) + (start[b] if start is not None else 0)
    return place


def check(got, ref, magnitude, what=""):
    """Half a step of the type, and 2^-18 of ``magnitude`` for what fp32 arithmetic leaves: sums of up to 64 terms per lane and tree, each
    rounding at most 2^-24 of the sum of magnitudes."""
    assert got.shape == ref.shape, what
    got64, ref = got.detach().double().cpu(), ref.detach()
    room = HALF_STEP[got.dtype] * ref.abs() * (1 + 2.0**-7) + 2.0**-18 * magnitude
    if got.dtype == torch.float16:
        room = room + 2.0**-25  # half a step among the subnormals
    bad = ~((got64 - ref).abs() <= room)
    assert not bad.any(), (what, int(bad.sum()), (got64 - ref).abs()[bad].max().item(), float(torch.as_tensor(room).expand_as(bad)[bad].min()))
