"""The 8-bit paged cache away from magnitudes of one: what a cache holds has no type, so a call must do with it what the definition says
whatever the type of q holds.  Against the definition in 64 bits (paged_fp8_reference), or bit for bit where powers of two move from one factor to
another."""

import numpy as np
import pytest
import torch

import ops_rec
import paged_fp8_reference as R
from test_gpu_paged_fp8 import DEV, TYPES, call, check, compare, queries
from test_gpu_paged_fp8_tiles import MOST

pytestmark = pytest.mark.gpu
OPS = ops_rec.ascendc.attention
# the kernel that shares keys, the same in parts and with weights, the one of half the wavefronts, the one of tiles of 128 rows (lens, counts, dim, more)
KERNELS = pytest.mark.parametrize("lens,counts,dim,kw", [
    ([300, 140], [40, 7], 64, {}), ([9000, 40], [1, 3], 64, {}), ([300, 140], [70, 7], 128, dict(weights=True)), ([300, 140], [70, 7], 64, dict(max_q=MOST)),
    ([300, 140, 77, 40], [70, 7, 77, 1], 128, dict(max_q=MOST)), ([300, 140], [5, 7], 256, {})], ids=["keys", "parts", "weights", "half", "tile", "d256"])  # fmt: skip


def cache(lens, dim, seed=1, **kw):
    return R.make(lens, dim=dim, heads_k=2, page=64, seed=seed, device=DEV, **kw)


@TYPES
@KERNELS
@pytest.mark.parametrize("shift", [-40, -9, 17, 60])
def test_a_power_of_two_in_the_scales_is_one_in_the_result(lens, counts, dim, kw, dtype, shift):
    """V 2^shift as large and silu_scale as much smaller, K and alpha likewise: no product changes but by that power, so no bit of the result does."""
    kw, scale, alpha = dict(kw), 1 / 64, 1 / 16
    weights = kw.pop("weights", False)
    q, offs = queries(counts, 2, dim, dtype), R.offsets(counts, device=DEV)

    def run(k_shift, v_shift):
        c = cache(lens, dim)
        c["k_scale"] *= 2.0**k_shift
        c["v_scale"] *= 2.0**v_shift
        w = torch.zeros_like(c["weights"]) if weights else None
        return call(c, q, offs, counts, alpha=alpha * 2.0**-k_shift, silu_scale=scale * 2.0**-v_shift, weights=w, **kw), w

    want, want_w = run(0, 0)
    assert want.isfinite().all() and want.any()
    for k_shift, v_shift in ((shift, 0), (0, shift), (shift, -shift)):
        got, w = run(k_shift, v_shift)
        assert torch.equal(got, want)
        assert not weights or torch.equal(w * 2.0**v_shift, want_w)


@KERNELS
@pytest.mark.parametrize("targets", [False, True], ids=["causal", "targets"])
def test_values_past_the_type_of_q(lens, counts, dim, kw, targets):
    """Values of up to some 1e6 read by fp16 rows, half the blocks of them so: finite outputs are finite, and no row has anything of what it does not see."""
    c = cache(lens, dim)
    c["v_scale"].view(-1)[::2] *= 2.0**14
    kw = dict(kw, targets=[min(n, 30) for n in counts], group=1) if targets else kw
    check(lens, counts, dim=dim, dtype=torch.float16, cache=c, seed=1, silu_scale=1e-7, **kw)


@KERNELS
def test_keys_and_scores_past_the_type_of_q(lens, counts, dim, kw):
    """Keys of up to some 1e6, and scores of a few 1e6, whose weights are scaled down to a type that ends at 65504."""
    c = cache(lens, dim)
    c["k_scale"] *= 2.0**16
    check(lens, counts, dim=dim, dtype=torch.float16, cache=c, seed=1, alpha=1.0, silu_scale=1e-10, **kw)


@KERNELS
def test_rows_of_very_different_weights(lens, counts, dim, kw):
    """Rows of q from 2^-16 to 2^-1 beside each other, blocks of V over 2^16: a row's error is in proportion to its own weights."""
    kw = dict(kw)
    weights = kw.pop("weights", False)
    c = cache(lens, dim)
    n = c["v_scale"].view(-1)
    n *= torch.exp2(torch.arange(n.numel(), device=DEV) * 5 % 17 - 8)
    q, offs = queries(counts, 2, dim, torch.float16), R.offsets(counts, device=DEV)
    q *= torch.exp2(torch.arange(len(q), device=DEV) * 7 % 16 - 16.0).view(-1, 1, 1).half()
    want, off, *_ = R.book(c).attend(q, offs, c["cache_len"], kw.get("max_q", max(counts)), alpha=1.0, silu_scale=2.0**-4)
    # A weight times its block's scales goes into the product as a multiple of 2^-24 of a unit, which rounds by half of that.  The unit puts a bound of
    # the row's scores, 448 dim times its largest value, with the scales of the block at 2^0.8 or above (2^11 / 2^8, and powers of two that
    # may be almost twice what they bound); codes of V are at most 448.
    book, o = R.book(c), offs.tolist()
    for b, s_k in enumerate(lens):
        for h in range(2):
            products = np.concatenate([(book.scales[0] * book.scales[1])[pid, h] for pid in book._pages(b)])[: -(-s_k // 32)]
            bound = 448 * dim * abs(q[o[b] : o[b + 1], h].cpu().double().numpy()).max(1, keepdims=True) * products.sum() * 32
            off[o[b] : o[b + 1], h] += 2.0**-4 * bound * 2.0 ** (-25 - 0.8) * 448
    w = torch.zeros_like(c["weights"]) if weights else None
    compare(call(c, q, offs, counts, alpha=1.0, silu_scale=2.0**-4, weights=w, **kw), want, off)


@pytest.mark.parametrize("dtype,top", [(torch.float16, 65504.0), (torch.bfloat16, 3e5), (torch.bfloat16, 1e30)], ids=["fp16", "bf16-in-the-cache", "1e30"])
@pytest.mark.parametrize("dim,max_q", [(64, None), (128, MOST)], ids=["keys", "tile"])
def test_candidates_past_fp16(dim, max_q, dtype, top):
    """Rows of +-65504, whose codes stand for 65536, and what a cache written in bf16 holds beyond, in one candidate: the others do not see it."""
    lens, counts, targets = [200, 200, 200, 200], [40] * 4, [30] * 4
    c = R.make([n - m for n, m in zip(lens, counts)], room=lens, dim=dim, heads_k=2, page=64, seed=2, device=DEV)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(160, 2, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    v[20, :, ::3], v[20, :, 1::3], v[60, :, 5], k[100, 0, 7] = top, -top, 63488.0, top
    offs = R.offsets(counts, device=DEV)
    OPS.hstu_paged_fp8_append(k, v, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], offs, c["cache_len"], c["page_offsets"], c["page_ids"], 40)
    c["cache_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q, tgt = queries(counts, 2, dim, torch.float16, 4), torch.tensor(targets, dtype=torch.int32, device=DEV)
    kw = dict(group=1, alpha=2.0**-20, silu_scale=2.0**2)
    want, off, *_ = R.book(c).attend(q, offs, c["cache_len"], 40, num_target=tgt, **kw)
    got = call(c, q, offs, counts, num_target=tgt, max_q=max_q, **kw)
    small = torch.from_numpy(abs(want) < 60000)
    assert small[19].all() and small[21].all() and (top > 1e9 or small.all())
    compare(got.cpu()[small], want[small], off[small])
    assert (got.cpu()[torch.from_numpy(abs(want) > 66000)].isinf()).all()


@TYPES
@KERNELS
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 2.0**100], ids=str)
def test_pages_that_are_none_whatever_page_0_holds(lens, counts, dim, kw, dtype, scale):
    """Page 0 is nobody's and holds anything; rows of pages that are not there count as zeros, their keys' weights as nothing."""
    seed = next(i for i in range(1000) if 0 in R.make(lens, dim=32, heads_k=1, page=64, seed=i, spare=2)["free"])
    c = cache(lens, dim, seed=seed)
    c["k_scale"][0], c["v_scale"][0] = scale, scale
    c["page_ids"][1], c["page_ids"][-1] = -1, 1 << 30
    got = check(lens, counts, dim=dim, dtype=dtype, cache=c, seed=1, **kw)
    assert got.isfinite().all()


@pytest.mark.parametrize("old", [0, 3], ids=["new-block", "older-rows"])
def test_rows_at_the_top_of_bf16(old):
    """The largest values of bf16 lie nearer to 256 * 2^120, which no float holds, than to 240 * 2^120, which they become: finite in the cache, after another
    append and after an eviction, and no row has anything of what it does not see."""
    top, n, dim = 3.3895313892515355e38, 40, 64
    c = R.make([old], room=[100], page=64, heads_k=2, dim=dim, seed=2, spare=3, device=DEV, poison=False)
    tensors = c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"]
    k, v = (torch.zeros(n, 2, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k[1, 0, :6] = v[1, 0, :6] = torch.tensor([top, -top, 248 * 2.0**120, 247 * 2.0**120, -232 * 2.0**120, float("inf")], device=DEV)
    v[35, 1, 7] = top
    want = torch.tensor([240.0, -240.0, 240.0, 240.0, -224.0, float("nan")], device=DEV)  # (232 is a tie)

    def row(t, i, head):
        block = t[int(c["page_ids"][i // 64]), head, i % 64 // 32].float()
        return block[i % 32] if block.shape[0] == 32 else block[:, i % 32]

    def check_rows():
        for t, s in ((tensors[0], tensors[2]), (tensors[1].transpose(3, 4).contiguous(), tensors[3])):
            torch.testing.assert_close(row(t, old + 1, 0)[:6], want, rtol=0, atol=0, equal_nan=True)
            assert s[int(c["page_ids"][0]), 0, 0] == 2.0**120
        assert row(tensors[1].transpose(3, 4).contiguous(), old + 35, 1)[7] == 240

    def add(rows, at):
        OPS.hstu_paged_fp8_append(rows[0], rows[1], *tensors, R.offsets([len(rows[0])], device=DEV), torch.tensor([at], dtype=torch.int32, device=DEV),
                                  c["page_offsets"], c["page_ids"], n, c["weights"])  # fmt: skip

    add((k, v), old)
    check_rows()
    add((k[:1], v[:1]), old + 2)  # (into the same block, which is put together again)
    check_rows()
    add((k[2:], v[2:]), old + 2)
    check_rows()
    c["cache_len"] = torch.tensor([old + n], dtype=torch.int32, device=DEV)
    tensors[1].view(torch.uint8)[int(c["page_ids"][0]), 0, 0, 5, old + 1] = 0  # (the value that was infinite)
    tensors[0].view(torch.uint8)[int(c["page_ids"][0]), 0, 0, old + 1, 5] = 0
    q, offs = queries([n], 2, dim, torch.bfloat16), R.offsets([n], device=DEV)
    tgt = torch.tensor([n], dtype=torch.int32, device=DEV)
    got = call(c, q, offs, [n], num_target=tgt, group=1, alpha=2.0**-126, silu_scale=1.0)
    others = [i for i in range(n) if i != 1]  # (scores of the row 1, sums of five products of some 3e38, are past fp32)
    assert got[others].isfinite().all()
    new = torch.tensor(c["free"][:2], dtype=torch.int32, device=DEV)
    before = [tensors[2][int(c["page_ids"][0]), 0, 0].clone(), row(tensors[0], old + 1, 0).clone()]
    OPS.hstu_paged_fp8_evict(*tensors, c["weights"], c["cache_len"], c["page_offsets"], c["page_ids"], torch.tensor([0, 2], dtype=torch.int32, device=DEV), new, 100, 100)
    c["page_ids"] = new
    assert torch.equal(before[1], row(tensors[0], old + 1, 0)) and tensors[2][int(new[0]), 0, 0] == before[0]


def test_every_block_appended_past_32_bits():
    """Blocks, scales and weights of pages beyond 4 GiB of the cache, the last block, which is written in part, among them; and nothing beside them."""
    page, heads, dim = 256, 8, 128
    n = (1 << 32) // (page * heads * dim) + 40
    c = R.make([600], page=page, heads_k=heads, dim=dim, seed=1, device=DEV)
    names, where = ("k_cache", "v_cache", "k_scale", "v_scale", "weights"), torch.tensor([n - 1, 3, n - 5], device=DEV)
    raw = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
    big = dict(c, page_ids=where.to(torch.int32))
    for name in names:
        small = raw(c[name])
        big[name] = torch.full((n, *small.shape[1:]), 7, dtype=small.dtype, device=DEV)
        big[name][where] = small[c["page_ids"].long()]
        big[name] = big[name].view(c[name].dtype)
    k, v = (torch.randn(50, heads, dim, device=DEV).to(torch.bfloat16) for _ in range(2))
    for t in (c, big):
        OPS.hstu_paged_fp8_append(k, v, *(t[name] for name in names[:4]), R.offsets([50], device=DEV), t["cache_len"], t["page_offsets"], t["page_ids"], 50, t["weights"])
    for name in names:
        a, b = raw(c[name])[c["page_ids"].long()], raw(big[name])[where]
        assert torch.equal(a.nan_to_num(-1.0) if a.is_floating_point() else a, b.nan_to_num(-1.0) if b.is_floating_point() else b)
        for beside in (0, 2, 4, n - 6, n - 4, n - 2):
            assert (raw(big[name])[beside] == 7).all()
    book = R.book(dict(c, cache_len=torch.tensor([650])))
    assert all(torch.from_numpy(book.rows(w, 0, h, 650)).isfinite().all() for w in (0, 1) for h in range(heads))


@TYPES
@KERNELS
@pytest.mark.parametrize("k_shift,v_shift", [(-66, -66), (-100, -100), (0, -110), (20, 60)], ids=str)
def test_blocks_of_very_different_scales(lens, counts, dim, kw, dtype, k_shift, v_shift):
    """Every third block nearly nothing (a cache written in bf16 holds it), or so large that an output is it: what the other blocks add stays."""
    c = cache(lens, dim)
    for name, shift in (("k_scale", k_shift), ("v_scale", v_shift)):
        c[name].view(-1)[1::3] *= 2.0**shift
    kw = dict(kw, silu_scale=2.0**-80) if v_shift > 0 and dtype == torch.float16 else kw
    got = check(lens, counts, dim=dim, dtype=dtype, cache=c, seed=1, **kw)
    assert got.isfinite().all() and (dtype == torch.bfloat16 or v_shift > 0 or got[1:].any())


@TYPES
@pytest.mark.parametrize("dim,max_q", [(64, None), (128, MOST), (256, None)], ids=["keys", "tile", "d256"])
def test_rows_that_are_not_finite_leave_the_others_alone(dim, max_q, dtype):
    lens, counts = [200, 140, 77, 40], [40, 7, 77, 1]
    c = cache(lens, dim)
    q, offs = queries(counts, 2, dim, dtype), R.offsets(counts, device=DEV)
    want = call(c, q, offs, counts, max_q=max_q)
    q[7, 1, 3], q[9, 0], q[60, 0, dim - 1] = float("inf"), float("nan"), -float("inf")
    got = call(c, q, offs, counts, max_q=max_q)
    for at in ((7, 1), (9, 0), (60, 0)):
        assert not got[at].isfinite().any()
        got[at] = want[at]
    assert torch.equal(got, want)
