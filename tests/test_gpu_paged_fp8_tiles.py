"""Attention over the 8-bit paged cache where rows are many: workgroups of half the wavefronts and the kernel for tiles of 128 rows, which
a call reaches that allows for enough rows, and keys dealt to several workgroups, by the lengths of up to 64 sequences and alike for more."""

import pytest
import torch

import paged_fp8_reference as R
from test_gpu_paged_fp8 import DEV, TYPES, call, check, queries

pytestmark = pytest.mark.gpu
MOST = 20480  # rows that a call may allow for: 160 tiles of 128, and 4 sequences of 2 key heads then fill the machine with them
WEIGHTS = pytest.mark.parametrize("weights", [False, True], ids=["plain", "weights"])


def kernels_of(run):
    from torch.profiler import ProfilerActivity, profile

    run()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        run()
        torch.cuda.synchronize()
    return " ".join(e.name for e in prof.events())


@pytest.mark.parametrize("dim,max_q,kernel", [(64, 300, "attend_kernel<hstu::bf16_tag, 2, 8,"), (64, MOST, "attend_kernel<hstu::bf16_tag, 2, 4,"),
                                              (128, MOST, "tile_kernel<hstu::bf16_tag, 4>"), (128, 300, "attend_kernel<hstu::bf16_tag, 4, 8,"),
                                              (160, MOST, "attend_kernel<hstu::bf16_tag, 6, 2,"), (256, 300, "attend_kernel<hstu::bf16_tag, 8, 4,")], ids=str)  # fmt: skip
def test_the_kernel_that_these_tests_are_for_is_the_one_that_runs(dim, max_q, kernel):
    c = R.make([700] * 4, dim=dim, seed=1, device=DEV)
    q, offs = queries([300] * 4, 2, dim, torch.bfloat16), R.offsets([300] * 4, device=DEV)
    assert kernel in kernels_of(lambda: call(c, q, offs, [300], max_q=max_q))


@TYPES
@WEIGHTS
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 256])
def test_head_dims(dim, dtype, weights):
    check([1000, 517, 133, 20], [300, 129, 1, 20], dim=dim, dtype=dtype, seed=dim, page=96, max_q=MOST, weights=weights)


@pytest.mark.parametrize("heads,heads_k", [(8, 2), (6, 2), (16, 16), (3, 3)], ids=str)
def test_grouped_heads(heads, heads_k):
    check([200, 70, 331, 40], [200, 3, 90, 33], heads=heads, heads_k=heads_k, dim=112, seed=heads, max_q=MOST)


@pytest.mark.parametrize("rows", [33, 130, 300], ids=lambda n: f"rows{n}")
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (32, 32), (33, 31), (64, 0), (100, 4), (500, 100), (2000, 10), (64, 1000)], ids=str)
def test_windows(rows, window, sinks):
    check([rows + 600, rows, rows + 31, rows + 97], [rows] * 4, window=window, sinks=sinks, dim=128, page=32, seed=window + rows, max_q=MOST)


@WEIGHTS
@pytest.mark.parametrize("group", [1, 3, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)], ids=["all", "window"])
def test_targets(group, window, sinks, weights):
    counts = [140, 100, 43, 600]
    check([540, 164, 133, 700], counts, targets=[100, 100, 3, 500], group=group, window=window, sinks=sinks, heads=4, heads_k=2, dim=128, seed=group,
          max_q=MOST, weights=weights)  # fmt: skip


@WEIGHTS
def test_sequences_without_rows_or_keys(weights):
    check([5, 0, 0, 40, 0, 200], [20, 3, 0, 0, 1, 200], dim=128, seed=1, weights=weights, max_q=MOST)
    c = R.make([0, 10, 300, 31], room=[0, 10, 300, 31], dim=128, seed=2, device=DEV)
    check([0, 10, 300, 31], [2, 4, 400, 31], dim=128, cache=c, weights=weights, max_q=MOST)


@pytest.mark.parametrize("window,targets", [(0, 0), (70, 0), (0, 12)], ids=["causal", "window", "targets"])
def test_what_a_row_does_not_see_reaches_nothing(window, targets):
    """NaN in a key and in a value, one of them among codes behind the last row: only the rows that see it, in the value's dims."""
    lens, counts = [350, 155, 60, 40], [150, 150, 60, 1]
    for which, at in (("k_cache", 200), ("v_cache", 200), ("v_cache", 349), ("v_cache", 351), ("v_cache", 120)):
        c = R.make(lens, dim=128, page=64, seed=9, device=DEV)
        cell = c[which].view(torch.uint8)[int(c["page_ids"][at // 64]), :, at % 64 // 32]
        if which == "k_cache":
            cell[:, at % 32, 3] = 0x7F
        else:
            cell[:, 5, at % 32] = 0xFF
            cell[:, 77, at % 32] = 0x7F
        kw = dict(targets=[targets] * 3 + [0], group=1) if targets else {}
        got = check(lens, counts, dim=128, cache=c, window=window, sinks=2 if window else 0, max_q=MOST, **kw)
        assert which == "k_cache" or not got[..., [0, 16, 31, 127]].isnan().any()
        assert not got[150:].isnan().any()  # the other sequences


def test_keys_past_64_and_past_128_steps():
    check([32 * 150 + 9, 32 * 64, 32 * 65, 32 * 63 + 1], [130, 1, 33, 2], dim=128, page=256, seed=1, max_q=MOST)
    check([32 * 4 * 130 + 9, 32 * 64 * 4, 32], [40, 1, 32], dim=16, page=256, seed=1, max_q=MOST)


def test_pages_that_are_none_and_pages_of_two_sequences():
    c = R.make([200, 290, 300, 290], dim=128, page=32, seed=1, device=DEV)
    ids = c["page_ids"]
    ids[2], ids[9] = -1, 1 << 30
    ids[7], ids[8] = ids[0], ids[1]  # the second sequence begins as the first
    check([200, 290, 300, 290], [150, 200, 1, 290], dim=128, cache=c, max_q=MOST)
    check([200, 290, 300, 290], [150, 200, 1, 290], dim=128, cache=c, weights=True, max_q=MOST)


@TYPES
@WEIGHTS
def test_tiles_of_128_rows_in_parts(dtype, weights):
    """4 x 2 key heads and 85 tiles each: six parts for the four sequences, and the long one's keys are two of them."""
    check([6000, 100, 1030, 40], [300, 100, 130, 1], dim=128, dtype=dtype, page=128, seed=4, max_q=10880, weights=weights)


@WEIGHTS
def test_tiles_of_128_rows_in_parts_of_more_sequences(weights):
    lens = [2500 - 37 * i for i in range(65)]
    check(lens, [140 if i % 9 == 0 else 1 + i % 3 for i in range(65)], heads=1, heads_k=1, dim=128, page=128, seed=5, max_q=1024, weights=weights)


@WEIGHTS
@pytest.mark.parametrize("rows,dim", [(1, 64), (3, 256), (40, 128), (100, 32)], ids=str)
def test_parts_alike_for_more_than_64_sequences(rows, dim, weights):
    lens = [0, 1, 3000, 2999] + [rows + 41 * i for i in range(66)]
    check(lens, [min(rows, n) if i % 5 else 0 for i, n in enumerate(lens)], heads=1, heads_k=1, dim=dim, page=128, seed=6, weights=weights)


@WEIGHTS
@pytest.mark.parametrize("rows,dim", [(100, 128), (70, 64), (257, 256)], ids=str)
def test_several_tiles_of_rows_in_parts(rows, dim, weights):
    check([9000 + rows, 4100], [rows, rows // 2], heads=2, heads_k=1, dim=dim, page=256, seed=7, weights=weights)


@pytest.mark.parametrize("lens", [[5000] * 5, [0, 5000, 0, 5000, 2500], [64] * 6 + [9000], [2049] * 64, [9000]], ids=["equal", "zeros", "one-long", "64", "alone"])
def test_how_keys_are_dealt(lens):
    check(lens, [1] * len(lens), heads=2, heads_k=1, dim=64, page=128, seed=8)


@WEIGHTS
def test_a_window_with_targets_past_the_blocks_it_allows_for(weights):
    """A target sees itself, far behind the window's keys: the last part of a tile takes what the parts before leave."""
    check([9000, 9000], [800, 30], targets=[790, 20], group=2000, window=2100, sinks=40, heads=1, heads_k=1, dim=64, page=128, seed=9, weights=weights)


@pytest.mark.parametrize("dim", [32, 256])
def test_sums_of_weights_that_the_workspace_does_not_hold_at_once(dim):
    """A call that allows for 2^24 keys: 128 MiB for the sums of a tile of 32 rows, of which the launch takes four; ten in three launches."""
    check([700], [300], dim=dim, weights=True, seed=1, max_k=1 << 24)
    check([700, 300], [300, 300], dim=dim, weights=True, seed=1, max_k=1 << 24)
    check([700] + [40] * 4, [300] + [1] * 4, dim=dim, weights=True, seed=1, max_k=1 << 24)  # a tile in a launch


def test_more_tiles_than_a_grid_holds():
    """2048 sequences of 16 heads that may have 20480 rows each: 21 million tiles of 32."""
    lens = [1 + i % 50 for i in range(2048)]
    check(lens, [1 if i % 7 else min(40, n) for i, n in enumerate(lens)], heads=16, heads_k=16, dim=16, page=64, seed=3, max_q=MOST, silu_scale=0.1)


@pytest.mark.parametrize("dim,max_q", [(128, MOST), (128, 10880), (64, 200)], ids=["tiles", "tiles-in-parts", "parts"])
def test_the_same_bits_every_time(dim, max_q):
    lens = [6000, 300, 300, 200]
    c = R.make(lens, dim=dim, page=128, seed=2, device=DEV)
    q, offs = queries([200] * 4, 2, dim, torch.bfloat16), R.offsets([200] * 4, device=DEV)
    first = None
    for _ in range(4):
        w = torch.zeros_like(c["weights"])
        got = (call(c, q, offs, [200], weights=w, max_q=max_q), w)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@TYPES
def test_weights_past_the_type_of_q_are_infinite(dtype):
    """P rounds to infinity there: an output is infinite with the sign of the value, and a row that sees no such key is what it was."""
    c = R.make([1, 40], heads_k=1, dim=32, page=32, seed=1, device=DEV)
    where, offs = [int(c["page_ids"][i]) for i in (0, 1)], R.offsets([1, 1], device=DEV)
    q = queries([1, 1], 1, 32, dtype)
    want = call(c, q, offs, [1], silu_scale=1.0)
    k = c["k_cache"][where[0], 0, 0, 0].float() * c["k_scale"][where[0], 0, 0]
    v = c["v_cache"][where[0], 0, 0, :, 0].float() * c["v_scale"][where[0], 0, 0]
    q[0, 0] = torch.sign(k) * (60000.0 if dtype == torch.float16 else 3e38)
    got = call(c, q, offs, [1], silu_scale=1.0)
    assert torch.equal(got[1], want[1])
    assert (got[0, 0][v > 0] == float("inf")).all() and (got[0, 0][v < 0] == -float("inf")).all()
