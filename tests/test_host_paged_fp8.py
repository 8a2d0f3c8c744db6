"""The operators of the 8-bit paged cache on the host: schemas, refusals and their words, shapes, and the reference that the GPU tests use."""

import ctypes
import re
import subprocess

import numpy as np
import pytest
import torch

import ops_rec
import paged_fp8_reference as R
from ops_rec import _build, _native, _paged_fp8

OPS = ("hstu_paged_fp8", "hstu_paged_fp8_append", "hstu_paged_fp8_evict")


def cache(pages=3, heads=2, blocks=2, dim=32):
    return dict(k_cache=torch.zeros(pages, heads, blocks, 32, dim).to(torch.float8_e4m3fn), v_cache=torch.zeros(pages, heads, blocks, dim, 32).to(torch.float8_e4m3fn),
                k_scale=torch.ones(pages, heads, blocks), v_scale=torch.ones(pages, heads, blocks))  # fmt: skip


def index(*values):
    return torch.tensor(values, dtype=torch.int32)


def attend_args(**kw):
    return dict(q=torch.zeros(4, 4, 32, dtype=torch.bfloat16), **cache(), seq_offset=index(0, 1, 4), cache_len=index(5, 9), page_offsets=index(0, 1, 2),
                page_ids=index(0, 1), max_seq_len=3, max_seq_len_k=9) | kw  # fmt: skip


def append_args(**kw):
    rows = torch.zeros(4, 2, 32, dtype=torch.float16)
    return dict(k=rows, v=rows, **cache(), seq_offset=index(0, 1, 4), cache_len=index(5, 9), page_offsets=index(0, 1, 2), page_ids=index(0, 1), max_seq_len=3) | kw


def evict_args(**kw):
    return dict(**cache(), weights=torch.zeros(3, 2, 64), cache_len=index(5, 9), page_offsets=index(0, 1, 2), page_ids=index(0, 1),
                new_page_offsets=index(0, 0, 1), new_page_ids=index(2), max_seq_len_k=9, keep=4) | kw  # fmt: skip


ARGS = dict(zip(OPS, (attend_args, append_args, evict_args)))


def test_they_are_reached_through_the_package():
    for name in OPS:
        assert name in ops_rec.ascendc.attention.__all__ and getattr(ops_rec.ascendc.attention, name) is getattr(torch.ops.ops_rec, name)


@pytest.mark.parametrize("name", OPS)
def test_tensors_of_the_host_are_refused(name):
    with pytest.raises((NotImplementedError, RuntimeError)):
        getattr(torch.ops.ops_rec, name)(**ARGS[name]())
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):
        getattr(_paged_fp8, name)(**ARGS[name]())


COMMON = [
    (dict(k_cache=torch.zeros(3, 2, 64, 32).to(torch.float8_e4m3fn)), r"k_cache must be \[num_pages"),
    (dict(k_cache=torch.zeros(3, 2, 2, 16, 32).to(torch.float8_e4m3fn)), "has 32 rows"),
    (dict(v_cache=torch.zeros(3, 2, 2, 64, 32).to(torch.float8_e4m3fn)), "v_cache must be"),
    (dict(k_cache=torch.zeros(3, 2, 2, 32, 32, dtype=torch.uint8)), "k_cache must be torch.float8_e4m3fn"),
    (dict(v_cache=torch.zeros(3, 2, 2, 32, 32).to(torch.float8_e5m2)), "v_cache must be torch.float8_e4m3fn"),
    (dict(k_cache=torch.zeros(2, 3, 2, 32, 32).to(torch.float8_e4m3fn).transpose(0, 1)), "k_cache must be contiguous"),
    (dict(k_scale=torch.ones(3, 2, 2, dtype=torch.float64)), "k_scale must be torch.float32"),
    (dict(v_scale=torch.ones(3, 2, 1)), "v_scale must be"),
    (dict(k_scale=torch.ones(3, 2, 4)[..., ::2]), "k_scale must be contiguous"),
    (dict(weights=torch.zeros(3, 2, 32)), "weights must be"),
    (cache(dim=24), "multiple of 16"),
    (cache(dim=272), "multiple of 16"),
    (cache(heads=17), "headNum"),
    (cache(pages=0), "must not be empty"),
]


@pytest.mark.parametrize("change,words", COMMON, ids=[w for _, w in COMMON])
@pytest.mark.parametrize("name", OPS)
def test_caches_that_are_refused(name, change, words):
    with pytest.raises(RuntimeError, match=words):
        getattr(_paged_fp8, name)(**ARGS[name](**change))


OWN = [
    ("hstu_paged_fp8", dict(q=torch.zeros(4, 4, 32)), "bfloat16 or float16"),
    ("hstu_paged_fp8", dict(q=torch.zeros(4, 128, dtype=torch.bfloat16)), "3D"),
    ("hstu_paged_fp8", dict(q=torch.zeros(4, 4, 64, dtype=torch.bfloat16)), "head dim of the cache"),
    ("hstu_paged_fp8", dict(q=torch.zeros(4, 3, 32, dtype=torch.bfloat16)), "multiple of the cache's"),
    ("hstu_paged_fp8", dict(q=torch.zeros(4, 18, 32, dtype=torch.bfloat16)), "at most 16"),
    ("hstu_paged_fp8", dict(max_seq_len=0), "maxSeqLen"),
    ("hstu_paged_fp8", dict(max_seq_len=20481), "maxSeqLen"),
    ("hstu_paged_fp8", dict(max_seq_len_k=0), "maxSeqLenK"),
    ("hstu_paged_fp8", dict(max_seq_len_k=(1 << 24) + 1), "maxSeqLenK"),
    ("hstu_paged_fp8", dict(num_target=index(1, 1)), "targetGroupSize"),
    ("hstu_paged_fp8", dict(window=-1), "window and sinks"),
    ("hstu_paged_fp8", dict(sinks=-1), "window and sinks"),
    ("hstu_paged_fp8_append", dict(k=torch.zeros(4, 2, 32)), "bfloat16 or float16"),
    ("hstu_paged_fp8_append", dict(v=torch.zeros(4, 2, 32, dtype=torch.bfloat16)), "bfloat16 or float16"),
    ("hstu_paged_fp8_append", dict(v=torch.zeros(3, 2, 32, dtype=torch.float16)), "heads and head dim"),
    ("hstu_paged_fp8_append", dict(max_seq_len=0), "maxSeqLen"),
    ("hstu_paged_fp8_evict", dict(weights=None), "goes by weights"),
    ("hstu_paged_fp8_evict", dict(keep=0), "keep"),
    ("hstu_paged_fp8_evict", dict(sinks=-1), "sinks and recent"),
    ("hstu_paged_fp8_evict", dict(recent=-1), "sinks and recent"),
    ("hstu_paged_fp8_evict", dict(max_seq_len_k=0), "maxSeqLenK"),
]


@pytest.mark.parametrize("name,change,words", OWN, ids=[f"{n}-{w}-{i}" for i, (n, _, w) in enumerate(OWN)])
def test_arguments_that_are_refused(name, change, words):
    with pytest.raises(RuntimeError, match=words):
        getattr(_paged_fp8, name)(**ARGS[name](**change))


@pytest.mark.parametrize("change,words", [
    (dict(cache_len=index(1)), "length per sequence"), (dict(seq_offset=index(0, 4)), "length of page_offsets"), (dict(page_offsets=index(0)), "at least two"),
    (dict(page_offsets=torch.zeros(2050, dtype=torch.int32)), "batchSize"), (dict(page_ids=torch.zeros(2)), "int32 or int64"),
    (dict(cache_len=index(1, 2).view(2, 1)), "one dimension"), (dict(new_page_offsets=index(0, 1)), "length of page_offsets")])  # fmt: skip
def test_index_tensors_that_are_refused(change, words):
    """(what the operators check once the tensors are known to be on a GPU)"""
    with pytest.raises(RuntimeError, match=words):
        _paged_fp8._check_batch(_paged_fp8._index_tensors(dict(cache_len=index(5, 9), page_offsets=index(0, 1, 2), page_ids=index(0, 1)) | change))


def test_index_tensors_of_two_types_become_the_wider():
    got = _paged_fp8._index_tensors(dict(cache_len=index(5, 9), page_ids=torch.tensor([1 << 33])))
    assert all(t.dtype == torch.int64 for t in got.values()) and got["page_ids"].item() == 1 << 33


def test_meta():
    meta = lambda kw: {n: t.to("meta") if torch.is_tensor(t) else t for n, t in kw.items()}  # noqa: E731
    out = torch.ops.ops_rec.hstu_paged_fp8(**meta(attend_args()))
    assert out.shape == (4, 4, 32) and out.dtype == torch.bfloat16
    assert torch.ops.ops_rec.hstu_paged_fp8_append(**meta(append_args())) is None
    n, kept = torch.ops.ops_rec.hstu_paged_fp8_evict(**meta(evict_args()))
    assert n.shape == (2,) and kept.shape == (2, 4) and n.dtype == kept.dtype == torch.int32


# ---- the C ABI: every refusal comes before a launch, so that it needs no GPU ----


def block(params, **kw):
    p = params()
    p.struct_size = ctypes.sizeof(p)
    c = p.cache
    c.k_cache = c.v_cache = 1 << 20
    c.k_scale = c.v_scale = c.cache_len = c.page_offsets = c.page_ids = 1 << 16
    c.num_pages, c.page_size, c.n_page_ids, c.num_heads_k, c.head_dim, c.n_offsets = 4, 64, 4, 2, 32, 3
    if params is _native.PagedFp8FwdParams:
        p.q = p.out = p.seq_offset = 1 << 16
        p.total_q, p.num_heads_q, p.max_seq_len_q, p.max_seq_len_k, p.silu_scale, p.alpha = 8, 2, 4, 100, 1.0, 1.0
    elif params is _native.PagedFp8AppendParams:
        p.k = p.v = p.seq_offset = 1 << 16
        p.total, p.max_seq_len, p.k_stride_row, p.k_stride_head, p.v_stride_row, p.v_stride_head = 8, 4, 64, 32, 64, 32
    else:
        c.weights = p.new_page_offsets = p.new_page_ids = p.new_cache_len = p.kept = 1 << 16
        p.n_new_page_ids, p.max_seq_len_k, p.keep = 2, 100, 50
    for name, value in kw.items():
        setattr(c if name in dict(_native.PagedFp8Cache._fields_) else p, name, value)
    return p


def refused(p):
    lib, size = _native.load(), ctypes.c_uint64(0)
    if isinstance(p, _native.PagedFp8AppendParams):
        rc = lib.hstu_paged_fp8_append(ctypes.byref(p), None)
    else:
        name = "hstu_paged_fp8_fwd" if isinstance(p, _native.PagedFp8FwdParams) else "hstu_paged_fp8_evict"
        rc = getattr(lib, name)(ctypes.byref(p), None, 0, None)
        assert getattr(lib, name + "_workspace_size")(ctypes.byref(p), ctypes.byref(size)) == rc
    assert rc != 0
    return _native.last_error()


ALL = (_native.PagedFp8FwdParams, _native.PagedFp8AppendParams, _native.PagedFp8EvictParams)


@pytest.mark.parametrize("params", ALL, ids=lambda p: p.__name__)
@pytest.mark.parametrize("kw,words", [
    (dict(struct_size=8), "struct_size"), (dict(k_cache=None), "must all be given"), (dict(cache_len=None), "must all be given"), (dict(page_ids=None), "must all be given"),
    (dict(n_offsets=1), "batchSize"), (dict(n_offsets=2050), "batchSize"), (dict(index_dtype=7), "index dtype"), (dict(num_heads_k=17), "head num"),
    (dict(head_dim=24), "multiple of 16"), (dict(head_dim=272), "multiple of 16"), (dict(page_size=48), "page_size"), (dict(page_size=0), "page_size"),
    (dict(num_pages=0), "num_pages"), (dict(num_pages=1 << 30), "blocks"), (dict(k_cache=(1 << 20) + 8), "aligned")], ids=lambda x: str(x)[:40])  # fmt: skip
def test_the_library_refuses_caches(params, kw, words):
    assert words in refused(block(params, **kw))


@pytest.mark.parametrize("params,kw,words", [
    (ALL[0], dict(dtype=2), "bf16 or fp16"), (ALL[0], dict(q=None), "must all be given"), (ALL[0], dict(out=(1 << 16) + 2), "aligned"),
    (ALL[0], dict(num_heads_q=3), "multiple of the cache's"), (ALL[0], dict(max_seq_len_q=0), "maxSeqLen"), (ALL[0], dict(max_seq_len_k=1 << 25), "maxSeqLenK"),
    (ALL[0], dict(num_target=1 << 16), "targetGroupSize"), (ALL[0], dict(window=-1), "window"),
    (ALL[1], dict(dtype=3), "bf16 or fp16"), (ALL[1], dict(v=None), "must all be given"), (ALL[1], dict(k=(1 << 16) + 8), "aligned"),
    (ALL[1], dict(v_stride_row=60), "strides"), (ALL[1], dict(k_stride_head=-32), "strides"), (ALL[1], dict(max_seq_len=0), "maxSeqLen"),
    (ALL[2], dict(weights=None), "weights"), (ALL[2], dict(kept=None), "must all be given"), (ALL[2], dict(keep=0), "keep"), (ALL[2], dict(recent=-1), "recent"),
    (ALL[2], dict(max_seq_len_k=0), "maxSeqLenK"), (ALL[2], dict(n_new_page_ids=-1), "n_new_page_ids")], ids=lambda x: str(x)[:40])  # fmt: skip
def test_the_library_refuses_arguments(params, kw, words):
    assert words in refused(block(params, **kw))


def test_the_library_refuses_null():
    lib = _native.load()
    assert lib.hstu_paged_fp8_append(None, None) != 0 and lib.hstu_paged_fp8_fwd(None, None, 0, None) != 0 and lib.hstu_paged_fp8_evict(None, None, 0, None) != 0
    assert lib.hstu_paged_fp8_fwd_kernel_name(None) is None


# ---- what the compiler has to keep for the attention kernels ----


@pytest.mark.parametrize("source", list(_build.SCORE_SOURCE_FLAGS))
def test_nothing_in_scratch(source, tmp_path):
    try:
        hipcc = _build.hipcc_path()
    except RuntimeError:
        pytest.skip("no hipcc on this host")
    out = tmp_path / "kernels.s"
    subprocess.run([hipcc, *_build.flags_of(source), "--cuda-device-only", "-S", f"{_build.CSRC}/{source}", "-o", str(out)], check=True, capture_output=True,
                   timeout=300)  # fmt: skip
    sizes = re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", out.read_text())
    assert len(sizes) >= 12 and set(sizes) == {"0"}


# ---- the reference itself ----


def test_codes_of_known_values():
    value, scale = R.quantise(np.array([[448.0, -1.0, 0.0, 17.0, 2.0**-9, 2.0**-10, 3 * 2.0**-11, np.inf]]))
    assert scale == 1.0 and np.isnan(value[0, -1])
    assert value[0, :-1].tolist() == [448.0, -1.0, 0.0, 16.0, 2.0**-9, 0.0, 2.0**-9]  # 17 is a tie to the even 16, 2^-10 one to 0
    assert R.quantise(np.array([449.0]))[1] == 2.0 and R.quantise(np.array([0.0]))[1] == 1.0 and R.quantise(np.array([224.0]))[1] == 0.5
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    np.testing.assert_array_equal(R.decode(codes), codes.double().numpy())
    np.testing.assert_array_equal(R.decode(R.encode(R.decode(codes))), R.decode(codes))


@pytest.mark.parametrize("targets,group", [(0, 0), (5, 1), (5, 2), (9, 3), (20, 4)])
def test_the_mask_is_the_built_in_one(targets, group):
    from oracle import hstu_oracle

    book = R.book(R.make([10]))
    for s_q, s_k in ((12, 30), (12, 12), (20, 5)):
        want = hstu_oracle.builtin_mask_pointwise(s_q, s_k, 0, targets, group).astype(bool)
        assert (book.mask(s_q, s_k, targets, group, 0, 0) == want).all()


def test_the_attention_is_the_paged_oracle_s_on_the_same_values():
    """Codes times scales as a cache in fp32, through the oracle of the 16-bit operator."""
    from oracle import hstu_oracle

    c = R.make([70, 33], page=64, heads_k=2, dim=32, seed=3, poison=False)
    b = R.book(c)
    q = torch.randn(20, 4, 32, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    counts, targets = [12, 8], torch.tensor([5, 3], dtype=torch.int32)
    k, v = (torch.from_numpy(np.concatenate([np.stack([b.rows(w, s, h, n) for h in range(2)], 1) for s, n in enumerate([70, 33])])).float() for w in (0, 1))
    want = hstu_oracle.hstu_jagged_forward(q.float(), k, v, mask_type=0, max_seq_len=12, max_seq_len_k=70, seq_offset=R.offsets(counts),
                                           seq_offset_k=R.offsets([70, 33]), num_target=targets, target_group_size=2, alpha=0.2, out_dtype=torch.float32)  # fmt: skip
    got, *_ = b.attend(q, R.offsets(counts), c["cache_len"], 12, 0.0, targets, 2, 0.2)
    np.testing.assert_allclose(got, want.double().numpy(), rtol=1e-4, atol=1e-4 * np.abs(got).max())


def test_an_eviction_s_workspace_goes_by_what_the_pages_hold():
    """A longest length without a limit asks for nothing that four pages of 64 rows cannot fill: scores that LDS holds need no workspace."""
    lib, size = _native.load(), ctypes.c_uint64(1)
    p = block(_native.PagedFp8EvictParams, max_seq_len_k=1 << 24, keep=1 << 24, n_offsets=2049)
    assert lib.hstu_paged_fp8_evict_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0 and size.value == 0
    p = block(_native.PagedFp8EvictParams, max_seq_len_k=1 << 24, n_page_ids=1000)
    assert lib.hstu_paged_fp8_evict_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0 and 2 * 64000 * 4 <= size.value <= 2 * 64100 * 4
    p = block(_native.PagedFp8EvictParams, max_seq_len_k=50000, n_page_ids=1000)
    assert lib.hstu_paged_fp8_evict_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0 and 2 * 50000 * 4 <= size.value <= 2 * 50100 * 4
