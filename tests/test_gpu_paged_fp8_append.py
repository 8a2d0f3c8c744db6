"""Rows written into the 8-bit paged cache, bit for bit against the definition in 64 bits."""

import pytest
import torch

import ops_rec
import paged_fp8_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
append = lambda *a, **kw: ops_rec.ascendc.attention.hstu_paged_fp8_append(*a, **kw)  # noqa: E731


def rows_of(n, heads, dim, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    # magnitudes over many binades, so that codes reach the subnormals of their block
    k, v = (std * torch.randn(n, heads, dim, generator=g) * torch.exp2(torch.randint(-12, 4, (n, heads, dim), generator=g)) for _ in range(2))
    return k.to(dtype).to(DEV), v.to(dtype).to(DEV)


def tensors(c):
    return c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"]


def check(c, k, v, counts, max_seq_len=None, weights=True):
    b = R.book(c)
    offs = R.offsets(counts, c["cache_len"].dtype, DEV)
    b.append(k, v, offs, c["cache_len"])
    w = c["weights"] if weights else None
    append(k, v, *tensors(c), offs, c["cache_len"], c["page_offsets"], c["page_ids"], max_seq_len or max(max(counts), 1), w)
    b.same(*tensors(c), w)
    return b, offs


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 96, 128, 176, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_head_dims_and_types(dim, dtype):
    old, new = [0, 5, 31, 32, 70], [40, 1, 1, 33, 100]
    c = R.make(old, room=[a + b for a, b in zip(old, new)], page=64, dim=dim, heads_k=2, seed=dim, device=DEV)
    check(c, *rows_of(sum(new), 2, dim, dtype, dim), new)


@pytest.mark.parametrize("page", [32, 96, 256])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("new", [1, 31, 33, 200], ids=str)
def test_pages_index_types_and_counts(page, index, new):
    old = [0, 1, 30, 31, 32, 33, 63, 95, 96, 255, 256]
    counts = [new, 0, 1, new, new, 2, 3, new, 0, 1, new]
    c = R.make(old, room=[a + b for a, b in zip(old, counts)], page=page, heads_k=3, dim=32, seed=page + new, index=index, device=DEV)
    check(c, *rows_of(sum(counts), 3, 32, torch.bfloat16, new), counts, max_seq_len=new + 7)


def test_the_same_rows_again_change_nothing():
    old, new = [20, 61], [9, 70]
    c = R.make(old, room=[29, 131], page=32, seed=4, device=DEV)
    k, v = rows_of(79, 2, 64, torch.bfloat16, 5)
    _, offs = check(c, k, v, new)
    before = [t.clone().view(torch.uint8) for t in tensors(c)]
    append(k, v, *tensors(c), offs, c["cache_len"], c["page_offsets"], c["page_ids"], 70, c["weights"])
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, tensors(c)))


def test_many_single_rows_are_one_call_of_them_all_while_the_scale_stands():
    """One row at a time: live rows go through every change of scale, which rounds only what falls below the block's smallest
    normal code; with rows of one size and the largest first nothing does."""
    n, dim = 40, 64
    k, v = (torch.rand(n, 1, dim, device=DEV).add(1).to(torch.bfloat16) for _ in range(2))
    k[0, 0, 0] = v[0, 0, 0] = 3.0
    k[32, 0, 0] = v[32, 0, 0] = 3.0
    one, all_ = (R.make([0], room=[n], page=64, heads_k=1, dim=dim, device=DEV, seed=1) for _ in range(2))
    length = torch.zeros(1, dtype=torch.int32, device=DEV)
    for i in range(n):
        append(k[i : i + 1], v[i : i + 1], *tensors(one), R.offsets([1], device=DEV), length + i, one["page_offsets"], one["page_ids"], 1)
    append(k, v, *tensors(all_), R.offsets([n], device=DEV), length, all_["page_offsets"], all_["page_ids"], n)
    assert all(torch.equal(a.view(torch.uint8)[one["page_ids"].long()], b.view(torch.uint8)[one["page_ids"].long()]) for a, b in zip(tensors(one), tensors(all_)))


@pytest.mark.parametrize("top", [448.0, 449.0, 1.0, 0.0, 2.0**-120, 2.0**-130, 3e38, 2.0**-133], ids=str)
def test_scales_at_the_borders(top):
    c = R.make([3], room=[40], page=64, heads_k=1, dim=16, seed=2, device=DEV, poison=False)
    c["k_cache"].view(torch.uint8)[:] = 0
    c["v_cache"].view(torch.uint8)[:] = 0x80  # minus zero
    k = torch.zeros(37, 1, 16, dtype=torch.bfloat16, device=DEV)
    k[5, 0, 3], k[6, 0, 4] = -top, top / 3
    check(c, k, k.neg(), [37])


def test_values_that_are_not_finite_become_nan_and_leave_the_others_alone():
    c = R.make([7], room=[60], page=64, heads_k=2, dim=32, seed=3, device=DEV)
    k, v = rows_of(50, 2, 32, torch.float16, 6, std=0.1)
    k[3, 0, 1], k[4, 0, 2], k[30, 1, 7] = float("inf"), float("-inf"), float("nan")
    v[3, 1, 1], v[40, 0, 2] = float("nan"), float("inf")
    check(c, k, v, [50])
    # a live NaN stays one
    c["cache_len"] = torch.tensor([20], dtype=torch.int32, device=DEV)
    check(c, k[:8], v[:8], [8])


def test_strided_rows():
    """Heads out of one wide projection, heads first, and rows that start off a 16-byte border (which are copied)."""
    n, heads, dim = 45, 2, 64
    wide = torch.randn(n, 4 * heads * dim + 4, device=DEV).to(torch.bfloat16)
    k = wide[:, : heads * dim].unflatten(1, (heads, dim))
    v = torch.randn(heads, n, dim, device=DEV).to(torch.bfloat16).transpose(0, 1)
    check(R.make([9], room=[60], heads_k=heads, dim=dim, seed=1, device=DEV), k, v, [n])
    k8 = torch.randn(n, heads * dim * 2, device=DEV).to(torch.bfloat16)[:, 8 : 8 + heads * dim].unflatten(1, (heads, dim))
    check(R.make([9], room=[60], heads_k=heads, dim=dim, seed=1, device=DEV), k8, v, [n])
    odd = wide[:, 4 : 4 + heads * dim].unflatten(1, (heads, dim))
    check(R.make([9], room=[60], heads_k=heads, dim=dim, seed=1, device=DEV), odd, v, [n])
    flat = torch.randn(n * heads * dim + 1, device=DEV).to(torch.bfloat16)[1:].view(n, heads, dim)
    check(R.make([9], room=[60], heads_k=heads, dim=dim, seed=1, device=DEV), flat, k, [n])
    expanded = torch.randn(n, 1, dim, device=DEV).to(torch.bfloat16).expand(n, heads, dim)  # one head for all
    check(R.make([9], room=[60], heads_k=heads, dim=dim, seed=1, device=DEV), expanded, expanded, [n])


def test_rows_without_a_place_are_dropped():
    # the pages hold 64 and 96 rows; page ids that are none; rows past max_seq_len
    c = R.make([60, 10, 5], room=[64, 96, 64], page=32, seed=8, device=DEV)
    k, v = rows_of(120, 2, 64, torch.bfloat16, 9)
    c["page_ids"][1] = 10_000  # the page that row 60 of the first sequence lies in
    c["page_ids"][3] = -1
    check(c, k, v, [30, 80, 10])
    c = R.make([0, 0], room=[64, 64], page=32, seed=8, device=DEV)
    b, offs = R.book(c), R.offsets([40, 50], device=DEV)
    b.append(torch.cat([k[:16], k[40:56]]), torch.cat([v[:16], v[40:56]]), R.offsets([16, 16]), c["cache_len"])
    append(k[:90], v[:90], *tensors(c), offs, c["cache_len"], c["page_offsets"], c["page_ids"], 16, c["weights"])
    b.same(*tensors(c), c["weights"])


def test_nothing_to_write():
    c = R.make([5, 0], room=[64, 32], page=32, seed=8, device=DEV)
    k, v = rows_of(4, 2, 64, torch.bfloat16, 9)
    check(c, k[:0], v[:0], [0, 0])
    check(c, k, v, [0, 0])  # rows that belong to no sequence
    none = R.make([0], room=[0], spare=1, seed=1, device=DEV)  # a sequence without pages
    check(none, k, v, [4])


def test_without_weights():
    c = R.make([5], room=[64], seed=8, device=DEV, weights=False)
    check(c, *rows_of(40, 2, 64, torch.bfloat16, 9), [40], weights=False)


def test_another_stream():
    c = R.make([5], room=[200], seed=8, device=DEV)
    k, v = rows_of(150, 2, 64, torch.bfloat16, 9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        check(c, k, v, [150])
    torch.cuda.current_stream().wait_stream(stream)
