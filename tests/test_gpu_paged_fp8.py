"""Attention over the 8-bit paged cache against the definition in 64 bits, within what its roundings allow
(paged_fp8_reference.Book.attend)."""

import numpy as np
import pytest
import torch

import ops_rec
import helpers
import paged_fp8_reference as R
from ops_rec import _native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


def queries(counts, heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 77)
    return torch.randn(sum(counts), heads, dim, generator=g).to(dtype).to(DEV)


def call(c, q, offs, counts, *, max_q=None, max_k=None, silu_scale=0.0, num_target=None, group=0, alpha=1.0, window=0, sinks=0, weights=None):
    max_q = max_q or max(max(counts), 1)
    max_k = max_k or max(int(c["cache_len"].max()), 1)
    return ops_rec.ascendc.attention.hstu_paged_fp8(
        q, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], offs, c["cache_len"], c["page_offsets"], c["page_ids"], max_q, max_k,
        silu_scale, num_target, group, alpha, window, sinks, weights)  # fmt: skip


def compare(got, want, off):
    got = got.detach().cpu().double().numpy()
    assert got.shape == want.shape
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    bad = np.abs(got - want) > off + 1e-30
    if bad.any():
        worst = np.nanargmax(np.abs(got - want) / (off + 1e-30))
        pytest.fail(f"{bad.sum()} of {bad.size} off, the worst {got.flat[worst]} for {want.flat[worst]}, {off.flat[worst]} allowed; first at {np.argwhere(bad)[0]}")


def check(lens, counts, *, heads=2, heads_k=2, dim=64, page=64, dtype=torch.bfloat16, seed=0, index=torch.int32, weights=False, targets=None, **kw):
    """lens: rows in the cache, the call's own among them."""
    c = kw.pop("cache", None) or R.make(lens, page=page, heads_k=heads_k, dim=dim, seed=seed, index=index, device=DEV)
    q, offs = queries(counts, heads, dim, dtype, seed), R.offsets(counts, index, DEV)
    tgt = torch.tensor(targets, dtype=index, device=DEV) if targets is not None else None
    kw.setdefault("alpha", dim**-0.5)
    ref_kw = {n: v for n, v in kw.items() if n in ("silu_scale", "group", "alpha", "window", "sinks")}
    max_q = kw.get("max_q") or max(max(counts), 1)
    want, off, inc, inc_off = R.book(c).attend(q, offs, c["cache_len"], max_q, num_target=tgt, **ref_kw)
    w = torch.zeros_like(c["weights"]) if weights else None
    if weights:  # the increments are added to what is there; what is not live is left alone
        g = torch.Generator().manual_seed(seed)
        w += torch.rand(w.shape, generator=g).to(DEV)
        before = w.clone()
    with helpers_poison():
        got = call(c, q, offs, counts, num_target=tgt, weights=w, **kw)
    compare(got, want, off)
    if weights:
        live = torch.from_numpy(inc > 0)
        total = before.cpu().double().numpy() + inc
        compare(w, total, inc_off + total * 2.0**-24)
        assert torch.equal(w.cpu()[~live], before.cpu()[~live])
    return got


class helpers_poison:
    """Outputs and workspaces handed out full of NaN."""

    def __enter__(self):
        self.patch = pytest.MonkeyPatch()
        helpers.poison_workspace(self.patch)

    def __exit__(self, *_):
        self.patch.undo()
        torch.use_deterministic_algorithms(False)


@TYPES
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 96, 112, 128, 160, 192, 256])
@pytest.mark.parametrize("rows", [1, 20, 60, 150], ids=lambda n: f"rows{n}")
def test_head_dims_and_rows(dim, dtype, rows):
    """Every head-dim group with every way of dealing rows and keys to wavefronts."""
    check([rows, rows + 33, 1000, 517], [rows, rows, rows, 1], dim=dim, dtype=dtype, heads=2, heads_k=2, seed=dim, page=96)


@TYPES
@pytest.mark.parametrize("heads,heads_k", [(1, 1), (4, 1), (6, 2), (16, 16), (16, 4), (3, 3)], ids=str)
@pytest.mark.parametrize("rows", [1, 9, 70], ids=lambda n: f"rows{n}")
def test_grouped_heads(heads, heads_k, dtype, rows):
    check([200, 70, 131], [rows, 3, rows], heads=heads, heads_k=heads_k, dim=32, dtype=dtype, seed=heads)


@pytest.mark.parametrize("page", [32, 64, 160, 256])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
def test_pages_and_index_types(page, index):
    lens = [1, 31, 32, 33, page - 1, page, page + 1, 2 * page, 700]
    check(lens, [1] * len(lens), page=page, index=index, dim=32, seed=page)
    check(lens, [min(n, 40) for n in lens], page=page, index=index, dim=32, seed=page)


@TYPES
@pytest.mark.parametrize("group", [1, 3, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)], ids=["all", "window"])
@pytest.mark.parametrize("n", [(7, 20), (0, 33), (40, 100)], ids=str)
def test_targets(dtype, group, window, sinks, n):
    new, targets = n
    counts = [new + targets, targets, new + 3]
    check([400 + counts[0], targets + 64, 90 + counts[2]], counts, targets=[targets, targets, 3], group=group, window=window, sinks=sinks,
          dtype=dtype, heads=4, heads_k=2, dim=32, seed=group + new)  # fmt: skip


@pytest.mark.parametrize("rows", [1, 33, 130, 300], ids=lambda n: f"rows{n}")
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (32, 32), (33, 31), (64, 0), (100, 4), (500, 100), (2000, 10), (64, 1000)], ids=str)
def test_windows(rows, window, sinks):
    check([rows + 600, rows, rows + 31, rows + 97], [rows] * 4, window=window, sinks=sinks, dim=32, page=32, seed=window + rows)


@pytest.mark.parametrize("kw", [dict(targets=[5, 900], counts=[10, 1000], group=1), dict(targets=[300, 300], counts=[300, 350], group=7, window=40, sinks=3),
                                dict(targets=[700, 0], counts=[5, 600], group=2)], ids=["many", "groups", "more-targets-than-rows"])  # fmt: skip
def test_long_slates_of_targets(kw):
    """Blocks of targets that a tile's rows do not see at all are skipped."""
    counts = kw.pop("counts")
    check([max(n, 800) + 123 for n in counts], counts, dim=32, heads=1, heads_k=1, seed=3, **kw)


@pytest.mark.parametrize("weights", [False, True], ids=["plain", "weights"])
def test_more_rows_than_keys_and_empty_sequences(weights):
    """Rows before the first key see nothing: zeros.  Sequences without rows, without keys, without pages."""
    check([5, 0, 0, 40, 0], [20, 3, 0, 0, 1], dim=32, seed=1, weights=weights)
    check([100, 0], [300, 70], dim=32, seed=1, weights=weights)
    c = R.make([0, 10], room=[0, 10], dim=32, seed=2, device=DEV)
    check([0, 10], [2, 4], dim=32, cache=c, weights=weights)


@TYPES
@pytest.mark.parametrize("rows", [1, 40, 100, 400], ids=lambda n: f"rows{n}")
@pytest.mark.parametrize("heads,heads_k,dim", [(2, 2, 64), (4, 2, 128), (2, 1, 256)], ids=str)
def test_weights(dtype, rows, heads, heads_k, dim):
    check([rows + 300, rows + 11, rows], [rows, rows, min(rows, 7)], heads=heads, heads_k=heads_k, dim=dim, dtype=dtype, weights=True, seed=rows)


@pytest.mark.parametrize("kw", [dict(window=40, sinks=9), dict(targets=[30, 10], group=4), dict(targets=[60, 10], group=1, window=64, sinks=33), dict(alpha=-0.3)],
                         ids=["window", "targets", "both", "negative-alpha"])  # fmt: skip
@pytest.mark.parametrize("rows", [70, 200], ids=lambda n: f"rows{n}")
def test_weights_under_masks(kw, rows):
    check([rows + 500, rows + 40], [rows, rows - 50], dim=32, weights=True, seed=rows, **kw)


@pytest.mark.parametrize("weights", [False, True], ids=["plain", "weights"])
@pytest.mark.parametrize("rows,dim,dtype", [(1, 128, torch.bfloat16), (40, 64, torch.float16), (3, 256, torch.bfloat16)], ids=["one", "wide", "d256"])
def test_long_keys_dealt_to_several_workgroups(rows, dim, dtype, weights):
    """Few tiles on long keys: parts, added by a second kernel; short sequences in the same call have one part."""
    lens = [9000 + rows, 40 + rows, 1025, 5000]
    check(lens, [rows, rows, 1, rows], heads=1, heads_k=1, dim=dim, dtype=dtype, page=256, weights=weights, seed=rows)


def test_keys_past_64_steps_of_a_wavefront():
    """The places of 64 steps are looked up at a time; here a wavefront has more."""
    check([64 * 32 * 4 + 700], [130], heads=1, heads_k=1, dim=32, page=256, seed=1)
    # many pairs, so that each has its keys to itself
    check([64 * 32 * 8 + 700] + [33] * 15, [1] * 16, heads=16, heads_k=16, dim=16, page=256, seed=1)


@pytest.mark.parametrize("silu_scale,alpha", [(0.0, 1.0), (0.25, 0.5), (1.0, -1.0), (-0.5, 2.0)], ids=str)
def test_scale_and_alpha(silu_scale, alpha):
    check([100, 65], [4, 65], dim=32, silu_scale=silu_scale, alpha=alpha, max_q=80)


@pytest.mark.parametrize("rows", [1, 20, 60, 150], ids=lambda n: f"rows{n}")
@pytest.mark.parametrize("window,targets", [(0, 0), (70, 0), (0, 12)], ids=["causal", "window", "targets"])
def test_what_a_row_does_not_see_reaches_nothing(rows, window, targets):
    """NaN in a key and in a value: the rows that see it are NaN (in the value's dims only), the others are what they were."""
    lens, counts = [rows + 200, rows + 5], [rows, rows]
    targets = min(targets, rows)
    for which, at in (("k_cache", 200), ("v_cache", 200), ("v_cache", 200 + rows - 1), ("v_cache", 120)):
        c = R.make(lens, dim=32, page=64, seed=rows, device=DEV)
        pid = int(c["page_ids"][at // 64])
        cell = c[which].view(torch.uint8)[pid, :, at % 64 // 32]
        if which == "k_cache":
            cell[:, at % 32, 3] = 0x7F
        else:
            cell[:, 5, at % 32] = 0xFF
            cell[:, 17, at % 32] = 0x7F
        kw = dict(targets=[targets, targets], group=1) if targets else {}
        got = check(lens, counts, dim=32, cache=c, window=window, sinks=2 if window else 0, seed=rows, **kw)
        assert which == "k_cache" or not got[..., [0, 16, 31]].isnan().any()
        assert not got[rows:].isnan().any()  # the other sequence


def test_a_page_in_two_sequences():
    """A prefix that sequences share: read by all of them, and weights of all of them added to it."""
    c = R.make([130, 130, 100], dim=32, page=64, seed=1, device=DEV)
    ids = c["page_ids"]
    ids[3], ids[4], ids[6] = ids[0], ids[1], ids[0]  # the second sequence begins as the first, the third with its first page
    check([130, 130, 100], [2, 5, 40], dim=32, cache=c, weights=True, seed=1)


def test_page_ids_that_are_none_read_as_zeros():
    c = R.make([200, 90, 300], dim=32, page=32, seed=1, device=DEV)
    c["page_ids"][2] = -1
    c["page_ids"][9] = 1 << 30
    check([200, 90, 300], [50, 2, 1], dim=32, cache=c, weights=True)


def test_lengths_and_offsets_that_do_not_fit_are_cut():
    """cache_len beyond the pages or negative, page offsets out of range, row offsets past the rows: nothing outside is read or written."""
    c = R.make([64, 64, 64], dim=32, page=64, seed=1, device=DEV)
    q, offs = queries([4, 4, 4], 2, 32, torch.bfloat16), R.offsets([4, 4, 4], device=DEV)
    good = call(c, q, offs, [4])
    long = dict(c, cache_len=torch.tensor([64, 1 << 30, -5], dtype=torch.int32, device=DEV))
    got = call(long, q, offs, [4], max_k=1000)
    assert torch.equal(got[:8], good[:8]) and not got[8:].any()
    wild = dict(c, page_offsets=torch.tensor([0, 1, -3, 1 << 30], dtype=torch.int32, device=DEV))
    got = call(wild, q, offs, [4], max_k=1000)
    assert torch.equal(got[:4], good[:4]) and not got[4:8].any() and not got.isnan().any()
    rows = torch.tensor([0, 4, 100, 8], dtype=torch.int32, device=DEV)
    got = call(c, q, rows, [4], max_k=1000)
    assert torch.equal(got[:4], good[:4]) and not got.isnan().any()


def test_rows_of_no_sequence_are_zeros():
    c = R.make([50, 60], dim=32, seed=1, device=DEV)
    q = queries([20], 2, 32, torch.bfloat16)
    offs = torch.tensor([3, 9, 16], dtype=torch.int32, device=DEV)
    with helpers_poison():
        got = call(c, q, offs, [7])
    assert not got[:3].any() and not got[16:].any() and not got.isnan().any() and got[3:16].any(dim=2).all()
    short = call(c, q, offs, [4], max_q=4, silu_scale=1 / 7)  # rows past the longest length allowed
    assert not short[7:9].any() and not short[13:16].any() and not short.isnan().any()


def test_infinities_stay_where_they_are():
    c = R.make([70, 70], dim=32, seed=1, device=DEV)
    q, offs = queries([40, 1], 2, 32, torch.bfloat16), R.offsets([40, 1], device=DEV)
    want = call(c, q, offs, [40])
    q[7, 1, 3], q[9, 0] = float("inf"), float("nan")
    got = call(c, q, offs, [40])
    assert got[7, 1].isnan().any() and got[9, 0].isnan().all()
    got[7, 1], got[9, 0] = want[7, 1], want[9, 0]
    assert torch.equal(got, want)


def test_large_scores_saturate():
    """silu of large magnitudes: x above, 0 below, no NaN from exp2 past its range."""
    c = R.make([64], dim=32, heads_k=1, seed=1, device=DEV)
    q = 1000 * queries([3], 1, 32, torch.bfloat16)
    got = call(c, q, R.offsets([3], device=DEV), [3], alpha=1.0, silu_scale=1e-3)
    want, off, *_ = R.book(c).attend(q, R.offsets([3]), c["cache_len"], 3, silu_scale=1e-3)
    compare(got, want, off)


def test_a_cache_past_32_bits():
    """A block far beyond 4 GiB of the cache."""
    page, heads, dim = 256, 8, 128
    n = (1 << 32) // (page * heads * dim) + 40
    c = R.make([600], page=page, heads_k=heads, dim=dim, seed=1, device=DEV)
    big = dict(c)
    shape = lambda t: (n, *t.shape[1:])  # noqa: E731
    for name in ("k_cache", "v_cache"):
        big[name] = torch.zeros(shape(c[name]), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    for name in ("k_scale", "v_scale", "weights"):
        big[name] = torch.ones(shape(c[name]), device=DEV)
    where = torch.tensor([n - 1, 3, n - 5], device=DEV)
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        raw = (lambda t: t.view(torch.uint8)) if "cache" in name else (lambda t: t)
        raw(big[name])[where] = raw(c[name])[c["page_ids"].long()]
    big["page_ids"] = where.to(torch.int32)
    q, offs = queries([3], heads, dim, torch.bfloat16), R.offsets([3], device=DEV)
    weights = [torch.zeros_like(c["weights"]), torch.zeros_like(big["weights"])]
    assert torch.equal(call(c, q, offs, [3], weights=weights[0]), call(big, q, offs, [3], weights=weights[1]))
    assert torch.equal(weights[0][c["page_ids"].long()], weights[1][where])
    k, v = (torch.randn(50, heads, dim, device=DEV).to(torch.bfloat16) for _ in range(2))
    for t in (c, big):
        ops_rec.ascendc.attention.hstu_paged_fp8_append(k, v, t["k_cache"], t["v_cache"], t["k_scale"], t["v_scale"], R.offsets([50], device=DEV),
                                                        t["cache_len"], t["page_offsets"], t["page_ids"], 50)  # fmt: skip
    for name in ("k_cache", "v_cache"):
        a, b = c[name].view(torch.uint8)[c["page_ids"].long()], big[name].view(torch.uint8)[where]
        assert torch.equal(a[:, :, :4][:2], b[:, :, :4][:2]) and torch.equal(a[2, :, :4], b[2, :, :4])


@pytest.mark.parametrize("rows,keys", [(1, 9000), (64, 300), (200, 2000)], ids=["parts", "tile", "rows"])
def test_the_same_bits_every_time(rows, keys):
    c = R.make([keys, keys // 2], dim=64, page=128, seed=2, device=DEV)
    q, offs = queries([rows, rows], 2, 64, torch.bfloat16), R.offsets([rows, rows], device=DEV)
    first = None
    for _ in range(4):
        w = torch.zeros_like(c["weights"])
        got = (call(c, q, offs, [rows], weights=w), w)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_strided_and_unaligned_queries_are_copied():
    c = R.make([70, 33], dim=32, seed=1, device=DEV)
    offs = R.offsets([6, 3], device=DEV)
    wide = torch.randn(9, 2, 64, device=DEV).to(torch.bfloat16)
    q = wide[..., 7:39]
    assert torch.equal(call(c, q, offs, [6]), call(c, q.contiguous(), offs, [6]))
    flat = torch.empty(9 * 2 * 32 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(9, 2, 32)
    flat.copy_(q)
    assert torch.equal(call(c, flat, offs, [6]), call(c, q.contiguous(), offs, [6]))
    # index tensors of two types, one of them a slice with a stride
    mixed = dict(c, cache_len=c["cache_len"].long(), page_ids=torch.stack([c["page_ids"]] * 2, 1)[:, 0])
    assert torch.equal(call(mixed, q, offs, [6]), call(c, q, offs, [6]))


def test_the_native_kernel_and_the_python_implementation_agree():
    from ops_rec import _paged_fp8

    c = R.make([400, 33], dim=64, seed=1, device=DEV)
    q, offs = queries([6, 3], 2, 64, torch.bfloat16), R.offsets([6, 3], device=DEV)
    args = (q, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], offs, c["cache_len"], c["page_offsets"], c["page_ids"], 6, 400, 0.0, None, 0,
            0.125, 100, 4)  # fmt: skip
    weights = [torch.zeros_like(c["weights"]) for _ in range(2)]
    assert torch.equal(ops_rec.ascendc.attention.hstu_paged_fp8(*args, weights[0]), _paged_fp8.hstu_paged_fp8(*args, weights[1]))
    assert torch.equal(*weights)


def test_the_workspace_is_asked_for_and_refused_when_short():
    import ctypes

    p = _native.PagedFp8FwdParams()
    c = R.make([9000], dim=64, page=128, seed=1, device=DEV)
    from ops_rec import _paged_fp8

    q, offs = queries([1], 2, 64, torch.bfloat16), R.offsets([1], device=DEV)
    out = torch.full_like(q, 7.0)
    p.struct_size, p.dtype = ctypes.sizeof(p), _native.DT_BF16
    _paged_fp8._describe(p.cache, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], None, c)
    p.q, p.out, p.seq_offset, p.total_q, p.num_heads_q = q.data_ptr(), out.data_ptr(), offs.data_ptr(), 1, 2
    p.max_seq_len_q, p.max_seq_len_k, p.silu_scale, p.alpha = 1, 9000, 1.0, 1.0
    lib, size = _native.load(), ctypes.c_uint64(0)
    assert lib.hstu_paged_fp8_fwd_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0 and size.value > 0
    ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
    assert lib.hstu_paged_fp8_fwd(ctypes.byref(p), ws.data_ptr(), size.value - 1, None) != 0 and b"workspace" in lib.hstu_last_error()
    assert lib.hstu_paged_fp8_fwd(ctypes.byref(p), None, size.value, None) != 0
    torch.cuda.synchronize()
    assert (out == 7.0).all()
