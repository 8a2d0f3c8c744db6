"""rotary against its definition in 64 bits."""

import pytest
import torch

import ops_rec
import layer_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
rotary = ops_rec.ascendc.attention.rotary
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def check(got, t, place, frequencies, interleaved, magnitude):
    ref = R.rotary(t.double(), place, frequencies, interleaved, magnitude)
    # cosine and sine to 2^-18 at most, and their products to half a step
    R.check(got, ref, t.double().abs().max().item() * magnitude)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(2, 1), (16, 8), (64, 32), (96, 32), (128, 64), (50, 25), (50, 11), (72, 20), (256, 128), (130, 3), (40, 16)])
def test_layouts(dtype, interleaved, dim, pairs):
    g = torch.Generator().manual_seed(dim + pairs)
    lengths = [5, 0, 1, 33, 2, 0]
    offs = [0]
    for n in lengths:
        offs.append(offs[-1] + n)
    rows = offs[-1] + 3  # the last three rows are in no sequence
    q, k = torch.randn(rows, 4, dim, generator=g).to(dtype), torch.randn(rows, 2, dim, generator=g).to(dtype)
    frequencies, _ = ops_rec.rotary_frequencies(2 * pairs)
    start = [0, 9, 100003, 7, 1 << 20, 0]
    for index in (torch.int32, torch.int64):
        qo, ko = rotary(q.to(DEV), k.to(DEV), frequencies.to(DEV), torch.tensor(offs, dtype=index, device=DEV), torch.tensor(start, dtype=torch.int64, device=DEV),
                        None, interleaved, 1.25)  # fmt: skip
        place = R.positions(offs, start, rows)
        for got, t in ((qo, q), (ko, k)):
            check(got, t, place, frequencies, interleaved, 1.25)
            assert torch.count_nonzero(got[-3:]) == 0
            assert torch.equal(got[: offs[-1], :, 2 * pairs :].cpu(), t[: offs[-1], :, 2 * pairs :])


@pytest.mark.parametrize("heads,heads_k", [(1, 1), (3, 1), (7, 5), (16, 16), (9, 2)])
@pytest.mark.parametrize("rows", [1, 2, 63, 4097])
def test_heads_and_rows(rows, heads, heads_k):
    g = torch.Generator().manual_seed(rows + heads)
    q, k = torch.randn(rows, heads, 64, generator=g).to(BF16), torch.randn(rows, heads_k, 64, generator=g).to(BF16)
    frequencies, _ = ops_rec.rotary_frequencies(64, base=500.0)
    place = torch.randint(0, 1 << 24, (rows,), generator=g)
    for index in (torch.int32, torch.int64):
        qo, ko = rotary(q.to(DEV), k.to(DEV), frequencies.to(DEV), positions=place.to(index).to(DEV))
        check(qo, q, place.double(), frequencies, False, 1.0)
        check(ko, k, place.double(), frequencies, False, 1.0)


def test_positions_far_out():
    # 2^40 positions: in 32 bits the angle itself would be off by thousands of turns
    place = torch.tensor([0, 1, (1 << 24) + 1, (1 << 31) + 7, (1 << 40) + 3, -5])
    q = torch.randn(6, 2, 32, generator=torch.Generator().manual_seed(0))
    frequencies, _ = ops_rec.rotary_frequencies(32)
    out, _ = rotary(q.to(DEV), q.to(DEV), frequencies.to(DEV), positions=place.to(DEV))
    # angles of 2^40 radians are off by 2^-13 in 64 bits already: each side its own rounding of the product
    room = 2.0 * place.abs().max().double() * 2.0**-52
    ref = R.rotary(q.double(), place.double(), frequencies)
    assert (out.double().cpu() - ref).abs().max() <= room * q.abs().max() + 2.0**-18
    R.check(out[:4], ref[:4], 4.0)
    assert torch.equal(out[0].cpu(), q[0])  # (position 0 turns nothing)


@pytest.mark.parametrize("batch", [1, 2, 7, 8, 9, 63, 64, 65, 511, 2048])
def test_sequences_are_found(batch):
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 4, (batch,), generator=g).tolist()
    lengths[-1] += 1
    offs = [2]  # (two rows ahead of the first sequence)
    for n in lengths:
        offs.append(offs[-1] + n)
    rows = offs[-1] + 2
    q = torch.ones(rows, 1, 2)
    start = torch.randint(0, 1000, (batch,), generator=g)
    out, _ = rotary(q.to(DEV), q.to(DEV), torch.ones(1, dtype=torch.float64, device=DEV), torch.tensor(offs, dtype=torch.int32, device=DEV),
                    start.to(torch.int32).to(DEV))  # fmt: skip
    check(out, q, R.positions(offs, start.tolist(), rows), torch.ones(1, dtype=torch.float64), False, 1.0)
    assert torch.count_nonzero(out[:2]) == 0 and torch.count_nonzero(out[-2:]) == 0


def test_strides_and_rows_that_are_not_finite():
    g = torch.Generator().manual_seed(2)
    mixed = torch.randn(40, 1000, generator=g).to(BF16).to(DEV)  # queries and keys as parts of a projection's row
    q, k = mixed[:, 5:517].view(40, 4, 128), mixed[:, 600:856].view(40, 2, 128)
    frequencies = ops_rec.rotary_frequencies(96, device=DEV)[0]
    offs = torch.tensor([0, 11, 40], dtype=torch.int32, device=DEV)
    for interleaved in (False, True):
        for got, same in zip(rotary(q, k, frequencies, offs, interleaved=interleaved), rotary(q.contiguous(), k.contiguous(), frequencies, offs, interleaved=interleaved)):
            assert torch.equal(got, same)
    by_heads = q.contiguous().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rotary(by_heads, k, frequencies, offs)[0], rotary(q, k, frequencies, offs)[0])
    across = q.contiguous().transpose(1, 2).contiguous().transpose(1, 2)  # (values of a head apart: copied)
    assert torch.equal(rotary(across, k, frequencies, offs)[0], rotary(q, k, frequencies, offs)[0])
    clean = rotary(q, k, frequencies, offs)[0]
    bad = q.contiguous().clone()
    bad[7, 1, 3] = float("nan")
    bad[39, 0, 100] = float("inf")
    out = rotary(bad, k, frequencies, offs)[0]
    changed = torch.zeros(40, 4, 128, dtype=torch.bool, device=DEV)
    changed[7, 1, [3, 51]] = True
    changed[39, 0, 100] = True
    assert torch.equal(torch.where(changed, torch.zeros_like(out), out), torch.where(changed, torch.zeros_like(clean), clean))
    # rows of no sequence are zeros, whatever they hold
    short = torch.tensor([0, 7], dtype=torch.int32, device=DEV)
    assert torch.count_nonzero(rotary(bad, k, frequencies, short)[0][7:]) == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(dtype, interleaved):
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(30, 4, 40, generator=g).to(dtype), torch.randn(30, 1, 40, generator=g).to(dtype)
    dq, dk = torch.randn(30, 4, 40, generator=g).to(dtype), torch.randn(30, 1, 40, generator=g).to(dtype)
    frequencies, offs, start = ops_rec.rotary_frequencies(24)[0], [0, 12, 12, 28], [5, 0, 1000]
    place = R.positions(offs, start, 30)
    dev = [t.to(DEV).requires_grad_(True) for t in (q, k)]
    args = (frequencies.to(DEV), torch.tensor(offs, device=DEV), torch.tensor(start, device=DEV), None, interleaved, 1.5)
    outs = rotary(*dev, *args)
    got = torch.autograd.grad(outs, dev, [dq.to(DEV), dk.to(DEV)], retain_graph=True)
    for t, d, a in ((q, dq, got[0]), (k, dk, got[1])):
        leaf = t.double().requires_grad_(True)
        ref = torch.autograd.grad(R.rotary(leaf, place, frequencies, interleaved, 1.5), leaf, d.double())[0]
        R.check(a, ref, 1.5 * d.double().abs().max().item())
    # a gradient of one output alone
    only = torch.autograd.grad(outs[0], dev, dq.to(DEV), retain_graph=True)
    assert torch.equal(only[0], got[0]) and torch.count_nonzero(only[1]) == 0
    # turned there and back: the transpose is the inverse at magnitude 1
    there = rotary(*dev, *args[:5], 1.0)
    back = rotary(*there, *args[:5], 1.0, True)
    assert (back[0][:28].double() - dev[0][:28].double()).abs().max() <= 4 * R.HALF_STEP[dtype] * q.abs().max().double() * 2


def test_no_rows():
    q = torch.empty(0, 2, 8, device=DEV)
    out = rotary(q, q, torch.ones(4, dtype=torch.float64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV))
    assert out[0].shape == out[1].shape == (0, 2, 8)
