"""The cosines and sines that rotary multiplies fp32 values by, read out of it, against those of the angles in 64 bits."""

import pytest
import torch

import ops_rec

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("far", [1, 1000, 1 << 20])
@pytest.mark.parametrize("interleaved", [False, True])
def test_cosines_and_sines_are_off_by_their_rounding(far, interleaved):
    """Pairs (1, 0) come out as (cosine, sine).  The library's are within a unit in the last place, 2^-24 of values up to 1, and what is added for the rest of the
    angle is rounded once more: 1.5 of it.  Over all angles roundings to nearest have a root mean square of 0.25 of it; the library's own error may be as much."""
    rows, pairs = 20000, 32
    g = torch.Generator().manual_seed(far)
    places = torch.randint(0, 4096 * far, (rows,), generator=g)
    frequencies, _ = ops_rec.rotary_frequencies(2 * pairs, base=50.0)
    q = torch.zeros(rows, 1, 2 * pairs, device=DEV)
    (q[..., 0::2] if interleaved else q[..., :pairs]).fill_(1.0)
    out = ops_rec.ascendc.attention.rotary(q, q, frequencies.to(DEV), positions=places.to(DEV), interleaved=interleaved)[0][:, 0].double().cpu()
    c, s = (out[:, 0::2], out[:, 1::2]) if interleaved else (out[:, :pairs], out[:, pairs:])
    angle = places.double()[:, None] * frequencies
    # (the angle itself is off by 2^-53 of it in 64 bits on either side, and so is its fraction of a turn)
    room = 4 * angle.max().item() * 2.0**-53
    off = torch.stack([c - torch.cos(angle), s - torch.sin(angle)]).abs()
    assert off.max() <= 1.5 * 2.0**-24 + room, off.max().item() * 2**24
    assert (off**2).mean().sqrt() <= 0.36 * 2.0**-24 + room, (off**2).mean().sqrt().item() * 2**24
