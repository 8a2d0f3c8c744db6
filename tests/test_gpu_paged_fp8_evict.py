"""Eviction from the 8-bit paged cache, bit for bit against the definition, and the operators of the cache one after the other."""

import pytest
import torch

import ops_rec
import paged_fp8_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OPS = ops_rec.ascendc.attention


def new_pages(c, lens, keep, page, room=None):
    counts = [-(-min(n, keep, 10**9 if room is None else room) // page) for n in lens]
    assert sum(counts) <= len(c["free"])
    index = c["cache_len"].dtype
    return R.offsets(counts, index, DEV), torch.tensor(c["free"][: sum(counts)], dtype=index, device=DEV)


def check(lens, keep, *, sinks=0, recent=0, page=64, heads_k=2, dim=32, seed=0, index=torch.int32, room=None, change=None, max_k=None):
    spare = sum(-(-min(n, keep) // page) for n in lens) + 1
    c = R.make(lens, page=page, heads_k=heads_k, dim=dim, seed=seed, index=index, spare=spare, device=DEV)
    offs, ids = new_pages(c, lens, keep, page, room)
    if change is not None:
        change(c, ids)
    b = R.book(c)
    want_len, want = b.evict(c["cache_len"], offs, ids, keep, sinks, recent)
    got_len, kept = OPS.hstu_paged_fp8_evict(c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["weights"], c["cache_len"], c["page_offsets"],
                                             c["page_ids"], offs, ids, max_k or max(max(lens), 1), keep, sinks, recent)  # fmt: skip
    assert got_len.dtype == index and kept.dtype == index and kept.shape == (len(lens), keep)
    assert got_len.tolist() == want_len
    assert kept.tolist() == want
    b.same(c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["weights"])
    return c, got_len, kept, offs, ids


@pytest.mark.parametrize("dim", [16, 48, 64, 128, 176, 256])
@pytest.mark.parametrize("page", [32, 96, 256])
def test_head_dims_and_pages(dim, page):
    check([300, 77, 200, 31, 0], 70, sinks=3, recent=20, dim=dim, page=page, seed=dim)


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (32, 0, 0), (33, 10, 10), (40, 40, 0), (40, 0, 40), (40, 100, 100),
                                               (40, 30, 100), (299, 0, 0), (300, 4, 4), (1000, 4, 4)], ids=str)  # fmt: skip
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
def test_budgets(keep, sinks, recent, index):
    check([300, 1, 40, 41, 0, 250], keep, sinks=sinks, recent=recent, seed=keep, index=index, heads_k=1)


@pytest.mark.parametrize("heads_k", [1, 3, 16])
def test_scores_are_sums_over_the_heads_in_their_order(heads_k):
    check([700, 1100], 300, sinks=4, recent=30, heads_k=heads_k, dim=16, seed=heads_k)


@pytest.mark.parametrize("n", [2047, 4100, 9000, 32761, 40001])
def test_long_sequences(n):
    """(more scores than LDS holds among them)"""
    check([n, n // 3], n // 4, sinks=5, recent=n // 20, heads_k=2 if n < 10000 else 1, dim=16, page=256, seed=n)


def test_ties_go_to_the_lower_index():
    def few(c, _):
        c["weights"].copy_((c["weights"].nan_to_num(0) * 3).floor())  # 0, 1 or 2 (0 .. 4 over two heads)

    for keep in (10, 100, 333, 900, 1500):
        check([2000, 1100], keep, recent=5, dim=16, change=few, seed=keep)
    check([2000, 500], 77, dim=16, change=lambda c, _: c["weights"].zero_())
    check([2000, 500], 77, dim=16, change=lambda c, _: c["weights"].copy_(torch.where(c["weights"] > 0.5, -0.0, 0.0)), heads_k=1)


def test_weights_of_any_kind():
    """Negative, infinite, subnormal; NaN counts as less than any."""

    def odd(c, _):
        w = c["weights"]
        pages = c["page_ids"].long()
        w[pages[0], :, ::3] = -1.0
        w[pages[1], :, ::5] = float("inf")
        w[pages[2], :, ::2] = float("nan")
        w[pages[3], 0, 1::7] = float("-inf")
        w[pages[4]] *= 1e-42

    for keep in (20, 150, 280, 400):
        check([500], keep, page=64, dim=16, change=odd, seed=1)


def test_values_that_are_nan_move_as_nan():
    def nan(c, _):
        c["k_cache"].view(torch.uint8)[c["page_ids"][0].item(), 0, 0, 5, 3] = 0x7F
        c["v_cache"].view(torch.uint8)[c["page_ids"][1].item(), 1, 1, 4, 9] = 0xFF

    check([200], 190, change=nan, seed=3)


def test_room_and_page_ids_that_are_none():
    """New pages that hold less than the budget; ids out of range among the old pages (rows of zeros) and the new (nothing written)."""
    check([300, 200], 150, sinks=4, recent=10, room=70, page=32)

    def wild(c, ids):
        c["page_ids"][1], c["page_ids"][4] = -1, 1 << 29
        ids[1] = 1 << 29

    check([300, 200], 150, sinks=4, recent=10, page=32, change=wild)


def test_no_new_pages_at_all():
    c = R.make([100], seed=1, device=DEV)
    none, offs = torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    n, kept = OPS.hstu_paged_fp8_evict(c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["weights"], c["cache_len"], c["page_offsets"],
                                       c["page_ids"], offs, none, 100, 10)  # fmt: skip
    assert n.tolist() == [0] and kept.tolist() == [[-1] * 10]


def test_index_tensors_of_two_types():
    a = R.make([300], page=64, spare=4, seed=5, device=DEV)
    b = R.make([300], page=64, spare=4, seed=5, device=DEV)
    offs, ids = new_pages(a, [300], 100, 64)
    out = []
    for c, convert in ((a, lambda t: t), (b, lambda t: t.long())):
        out.append(OPS.hstu_paged_fp8_evict(c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["weights"], c["cache_len"], c["page_offsets"],
                                            convert(c["page_ids"]), offs, convert(ids), 300, 100, 2, 3))  # fmt: skip
    assert all(x.dtype == torch.int32 and torch.equal(x, y) for x, y in zip(*out))
    assert torch.equal(a["k_cache"].view(torch.uint8), b["k_cache"].view(torch.uint8))


def serve(c, steps, keep, max_k, log=None):
    """A history that grows by steps of new events with candidates behind them, and is cut when it passes its budget."""
    length, offsets, ids = c["cache_len"], c["page_offsets"], c["page_ids"]
    outs = []
    for q, k, v, offs, new, tgt, most, to in steps:
        cache = (c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"])
        OPS.hstu_paged_fp8_append(k, v, *cache, offs, length, offsets, ids, most, c["weights"])
        outs.append(OPS.hstu_paged_fp8(q, *cache, offs, length + new + tgt, offsets, ids, most, max_k, 0.0, tgt, 1, 0.125, 256, 4, c["weights"]))
        length = length + new
        if to is not None:
            length, kept = OPS.hstu_paged_fp8_evict(*cache, c["weights"], length, offsets, ids, *to, max_k, keep, 4, 32)
            offsets, ids = to
            outs += [length, kept]
    return outs


def steps_for(c, lens, heads, heads_k, dim, n_steps, keep, page, seed):
    g = torch.Generator().manual_seed(seed)
    steps, free = [], list(c["free"])
    for i in range(n_steps):
        new, tgt = torch.randint(0, 40, (len(lens),), generator=g), torch.randint(1, 9, (len(lens),), generator=g)
        counts = (new + tgt).tolist()
        q, k, v = (torch.randn(sum(counts), h, dim, generator=g).to(torch.bfloat16).to(DEV) for h in (heads, heads_k, heads_k))
        to = None
        if i % 2 == 1:  # room for the rows kept and for those of the next steps
            counts_to = [-(-(keep + 120) // page)] * len(lens)
            to = (R.offsets(counts_to, device=DEV), torch.tensor(free[: sum(counts_to)], dtype=torch.int32, device=DEV))
            free = free[sum(counts_to) :]
        steps.append((q, k, v, R.offsets(counts, device=DEV), new.int().to(DEV), tgt.int().to(DEV), max(counts), to))
    return steps


def session(seed=0):
    lens, heads, heads_k, dim, page, keep = [150, 3, 290], 4, 2, 64, 32, 128
    c = R.make(lens, room=[n + 160 for n in lens], page=page, heads_k=heads_k, dim=dim, seed=seed, spare=80, device=DEV, poison=False)
    return c, steps_for(c, lens, heads, heads_k, dim, 6, keep, page, seed), keep


def test_the_operators_one_after_the_other():
    """Appending, attending and evicting over several steps, each against the definition on the state that the operators left.
    (The weights of the book follow the operators', within the tolerance of a step, so that the choice is the same.)"""
    c, steps, keep = session()
    length, offsets, ids = c["cache_len"], c["page_offsets"], c["page_ids"]
    for q, k, v, offs, new, tgt, most, to in steps:
        cache = (c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"])
        now = dict(c, page_offsets=offsets, page_ids=ids)
        b = R.book(now)
        b.append(k, v, offs, length)
        OPS.hstu_paged_fp8_append(k, v, *cache, offs, length, offsets, ids, most, c["weights"])
        b.same(*cache, c["weights"])
        want, off, inc, inc_off = b.attend(q, offs, length + new + tgt, most, 0.0, tgt, 1, 0.125, 256, 4)
        before = c["weights"].cpu().double()
        got = OPS.hstu_paged_fp8(q, *cache, offs, length + new + tgt, offsets, ids, most, 600, 0.0, tgt, 1, 0.125, 256, 4, c["weights"])
        assert (torch.from_numpy(want) - got.cpu().double()).abs().le(torch.from_numpy(off)).all()
        total = before + torch.from_numpy(inc)
        assert (total - c["weights"].cpu().double()).abs().le(torch.from_numpy(inc_off) + total * 2.0**-24).all()
        length = length + new
        if to is not None:
            b = R.book(now)
            want_len, want_kept = b.evict(length, *to, keep, 4, 32)
            length, kept = OPS.hstu_paged_fp8_evict(*cache, c["weights"], length, offsets, ids, *to, 600, keep, 4, 32)
            assert length.tolist() == want_len and kept.tolist() == want_kept
            b.same(*cache, c["weights"])
            offsets, ids = to


def test_a_session_captured_and_replayed():
    """Every replay, from the state that the session began with, gives what the eager calls gave; the program works between."""
    c, steps, keep = session(1)
    state = ("k_cache", "v_cache", "k_scale", "v_scale", "weights")
    start = {n: c[n].clone() for n in state}

    def back():
        for n in state:
            c[n].view(torch.uint8).copy_(start[n].view(torch.uint8))

    want = [t.clone() for t in serve(c, steps, keep, 600)]
    end = {n: c[n].clone() for n in state}
    back()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve(c, steps, keep, 600)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serve(c, steps, keep, 600)
    for _ in range(4):
        back()
        torch.randn(1000, 1000, device=DEV).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(c[n].view(torch.uint8), end[n].view(torch.uint8)) for n in state)


def test_sessions_on_two_streams():
    sessions = [session(2), session(3)]
    want = []
    for c, steps, keep in sessions:
        before = {n: c[n].clone() for n in ("k_cache", "v_cache", "k_scale", "v_scale", "weights")}
        want.append([t.clone() for t in serve(c, steps, keep, 600)])
        for n, t in before.items():
            c[n].view(torch.uint8).copy_(t.view(torch.uint8))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sessions], []
    for (c, steps, keep), s in zip(sessions, streams):
        with torch.cuda.stream(s):
            got.append(serve(c, steps, keep, 600))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


@pytest.mark.parametrize("keep", [60, 100, 140, 180, 230])
def test_scores_of_nan_rank_as_minus_infinity(keep):
    """200 of 250 rows score NaN or -infinity, in turn: of those the first stay, whichever they are."""

    def lowest(c, _):
        pages = c["page_ids"].long()
        for i in range(250):
            if i % 5:
                c["weights"][pages[i // 64], :, i % 64] = float("nan") if i % 2 else float("-inf")

    _, _, kept, _, _ = check([250], keep, dim=16, change=lowest, seed=2)
    lowest_kept = [i for i in kept[0].tolist() if i % 5]
    assert lowest_kept == [i for i in range(250) if i % 5][: keep - 50]


@pytest.mark.parametrize("keep", [70, 100_000])
def test_a_longest_length_without_a_limit(keep):
    """(launches and workspace go by what the pages hold)"""
    check([300, 77, 1100], keep, sinks=3, recent=20, seed=keep, max_k=1 << 24)
    check([40001, 33], 10_000, sinks=3, recent=20, heads_k=1, dim=16, page=256, seed=keep, max_k=1 << 24)
