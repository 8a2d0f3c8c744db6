"""The 8-bit paged key / value cache: ``hstu_paged_fp8_append`` writes rows into it, ``hstu_paged_fp8`` attends to it,
``hstu_paged_fp8_evict`` keeps what the attention weights say is worth keeping.  An extension: the reference's paged cache
(``hstu_paged``) holds the type of q, twice the bytes.

The cache of one layer, tensors that the program allocates and keeps::

    k_cache          e4m3 [num_pages, heads_k, page_size / 32, 32, dim]    the rows of a block of 32 tokens
    v_cache          e4m3 [num_pages, heads_k, page_size / 32, dim, 32]    the same, tokens innermost
    k_scale, v_scale fp32 [num_pages, heads_k, page_size / 32]             what the codes of a block are multiplied by: powers of two
    weights          fp32 [num_pages, heads_k, page_size]                  accumulated attention weights (optional)

Sequence ``b`` has the pages ``page_ids[page_offsets[b] : page_offsets[b + 1]]``, and its first ``cache_len[b]`` rows in them are
live; what lies behind them may hold anything.  A cache has no type: rows of bf16 and of fp16 write it and read it.

A serving step appends the new rows (and the candidates to be ranked) behind
``cache_len``, attends with the lengths that include them, and goes on from the length that it wants to keep: the next append
overwrites the rest.

Registered as operators of ``torch.ops.ops_rec``; device tensors in canonical form go to the native kernels of
``csrc/torch_binding.cpp``, everything else comes here, where the checks and conversions are.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native
from ._ops import _DTYPE_CODE, _PYTHON_KERNELS, _check, _check_devices, _lib_def, _lib_meta, _max_seq_len_check, _ptr

BLOCK = 32  # tokens that share a scale
MAX_SEQ_LEN_K = 1 << 24
MAX_HEAD_DIM = 256

_CACHE = "Tensor{0} k_cache, Tensor{1} v_cache, Tensor{2} k_scale, Tensor{3} v_scale"
_READ, _WRITTEN = _CACHE.format("", "", "", ""), _CACHE.format("(a!)", "(b!)", "(c!)", "(d!)")
_lib_def.define(
    f"hstu_paged_fp8(Tensor q, {_READ}, Tensor seq_offset, Tensor cache_len, Tensor page_offsets, Tensor page_ids, int max_seq_len, "
    "int max_seq_len_k, float silu_scale=0.0, Tensor? num_target=None, int target_group_size=0, float alpha=1.0, int window=0, "
    "int sinks=0, Tensor(a!)? weights=None) -> Tensor"
)
_lib_def.define(
    f"hstu_paged_fp8_append(Tensor k, Tensor v, {_WRITTEN}, Tensor seq_offset, Tensor cache_len, Tensor page_offsets, Tensor page_ids, "
    "int max_seq_len, Tensor(e!)? weights=None) -> ()"
)
_lib_def.define(
    f"hstu_paged_fp8_evict({_WRITTEN}, Tensor(e!) weights, Tensor cache_len, Tensor page_offsets, Tensor page_ids, "
    "Tensor new_page_offsets, Tensor new_page_ids, int max_seq_len_k, int keep, int sinks=0, int recent=0) -> (Tensor, Tensor)"
)


def _check_cache(k_cache, v_cache, k_scale, v_scale, weights):
    _check(k_cache.dim() == 5 and v_cache.dim() == 5, "k_cache must be [num_pages, heads, page_size / 32, 32, dim], v_cache [num_pages, heads, page_size / 32, dim, 32]")
    pages, heads, blocks, rows, dim = k_cache.shape
    _check(rows == BLOCK, f"a block of k_cache has {BLOCK} rows, but got {rows}")
    _check(tuple(v_cache.shape) == (pages, heads, blocks, dim, BLOCK), f"v_cache must be {[pages, heads, blocks, dim, BLOCK]}, but it is {list(v_cache.shape)}")
    _check(k_cache.numel() > 0, "k_cache must not be empty")
    _check(1 <= heads <= 16, f"headNum expect in [1, 16], but value is {heads}")
    _check(16 <= dim <= MAX_HEAD_DIM and dim % 16 == 0, f"headDim of the 8-bit cache expect a multiple of 16 in [16, {MAX_HEAD_DIM}], but value is {dim}")
    for name, t, dtype, shape in (("k_cache", k_cache, torch.float8_e4m3fn, None), ("v_cache", v_cache, torch.float8_e4m3fn, None),
                                  ("k_scale", k_scale, torch.float32, (pages, heads, blocks)), ("v_scale", v_scale, torch.float32, (pages, heads, blocks)),
                                  ("weights", weights, torch.float32, (pages, heads, blocks * BLOCK))):  # fmt: skip
        if t is None:
            continue
        _check(t.dtype == dtype, f"{name} must be {dtype}, but it is {t.dtype}")
        _check(shape is None or tuple(t.shape) == shape, f"{name} must be {list(shape or ())}, but it is {list(t.shape)}")
        _check(t.is_contiguous(), f"{name} must be contiguous")  # (the cache is never copied)


def _index_tensors(named):
    """Index tensors contiguous and of one type: int32 where they all are, int64 otherwise (a page id is never cut)."""
    for name, t in named.items():
        _check(t.dim() == 1, f"{name} must have one dimension")
        _check(t.dtype in (torch.int32, torch.int64), f"{name} must be int32 or int64, but it is {t.dtype}")
    dtype = torch.int32 if all(t.dtype == torch.int32 for t in named.values()) else torch.int64
    return {name: t.to(dtype).contiguous() for name, t in named.items()}


def _describe(c, k_cache, v_cache, k_scale, v_scale, weights, index):
    pages, heads, blocks, _, dim = k_cache.shape
    c.k_cache, c.v_cache, c.k_scale, c.v_scale = k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
    c.weights = None if weights is None else weights.data_ptr()
    c.cache_len, c.page_offsets = index["cache_len"].data_ptr(), index["page_offsets"].data_ptr()
    c.page_ids = _ptr(index["page_ids"])
    c.num_pages, c.page_size, c.n_page_ids = pages, blocks * BLOCK, index["page_ids"].numel()
    c.num_heads_k, c.head_dim, c.n_offsets = heads, dim, index["page_offsets"].numel()
    c.index_dtype = _native.IDX_I64 if index["cache_len"].dtype == torch.int64 else _native.IDX_I32


def _check_batch(index):
    n = index["page_offsets"].numel()
    _check(n >= 2, "page_offsets params error should have at least two element.")
    _check(n - 1 <= 2048, f"batchSize expect in [1, 2048], but value is {n - 1}")
    _check(index["cache_len"].numel() == n - 1, f"cache_len must have a length per sequence ({n - 1}), but it has {index['cache_len'].numel()}")
    for name in ("seq_offset", "new_page_offsets"):
        if name in index:
            _check(index[name].numel() == n, f"{name} must have the length of page_offsets ({n}), but it has {index[name].numel()}")


def _call(name, params, device, workspace=True):
    """Sizes and allocates the workspace where there is one, and launches."""
    lib = _native.load()
    with torch.cuda.device(device):
        stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
        args = (ctypes.byref(params),)
        if workspace:
            size = ctypes.c_uint64(0)
            rc = getattr(lib, name + "_workspace_size")(ctypes.byref(params), ctypes.byref(size))
            if rc != _native.HSTU_OK:
                raise RuntimeError(f"{name}_workspace_size failed ({rc}): {_native.last_error()}")
            ws = torch.empty(max(size.value, 1), dtype=torch.uint8, device=device)
            args += (ws.data_ptr(), size.value)
        rc = getattr(lib, name)(*args, stream)
    if rc != _native.HSTU_OK:
        raise RuntimeError(f"{name} failed ({rc}): {_native.last_error()}")


def _aligned(t):
    """``t`` contiguous and where the kernels' 16-byte accesses may read it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def hstu_paged_fp8(q, k_cache, v_cache, k_scale, v_scale, seq_offset, cache_len, page_offsets, page_ids, max_seq_len, max_seq_len_k,
                   silu_scale=0.0, num_target=None, target_group_size=0, alpha=1.0, window=0, sinks=0, weights=None):  # fmt: skip
    """HSTU attention of the rows ``q`` [total, heads, dim] (bf16 or fp16) to an 8-bit paged cache in which their own keys and values
    are already: row ``i`` of a sequence's ``s_q`` has the position ``i + cache_len - s_q``.

    The built-in mask of ``hstu_jagged`` without context rows: keys up to the row's position; of the last ``num_target`` rows each
    sees the history and its own group of ``target_group_size``.  With ``window`` > 0 a row sees, of the keys it would see, the last
    ``window`` up to its position (a target row, standing where the first target stands: ``window - 1`` of the history and its
    group) and the first ``sinks``.  ``silu_scale`` 0 means ``1 / max_seq_len``.

    ``weights``, where given, gets for every live key and key head the sum over rows and query heads of the magnitudes of the
    attention weights added to it.  Returns the type and shape of ``q``; rows of no sequence come out as zeros.  There is no backward."""
    _check(q.dim() == 3, "The q should be 3D in jagged layout")
    _check(q.dtype in (torch.bfloat16, torch.float16), f"q must be bfloat16 or float16, but it is {q.dtype}")
    _check_cache(k_cache, v_cache, k_scale, v_scale, weights)
    heads_k, dim = k_cache.size(1), k_cache.size(4)
    _check(q.size(2) == dim, f"q must have the head dim of the cache ({dim}), but it has {q.size(2)}")
    _check(1 <= q.size(1) <= 16 and q.size(1) % heads_k == 0, f"the heads of q must be a multiple of the cache's ({heads_k}), at most 16, but there are {q.size(1)}")
    _max_seq_len_check(int(max_seq_len), "maxSeqLen")
    _check(1 <= int(max_seq_len_k) <= MAX_SEQ_LEN_K, f"maxSeqLenK expect in [1, {MAX_SEQ_LEN_K}], but value is {max_seq_len_k}")
    _check(num_target is None or int(target_group_size) > 0, "targetGroupSize must be greater than 0 when numTarget is defined")
    _check(int(target_group_size) < 1 << 30, f"targetGroupSize expect below 2^30, but value is {target_group_size}")
    _check(int(window) >= 0 and int(sinks) >= 0, f"window and sinks must not be negative, but they are {window} and {sinks}")
    named = {"seq_offset": seq_offset, "cache_len": cache_len, "page_offsets": page_offsets, "page_ids": page_ids}
    if num_target is not None:
        named["num_target"] = num_target
    _check(q.device.type == "cuda", f"q must be a GPU tensor, but it is on {q.device}")
    _check_devices(q.device, (("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale), ("weights", weights),
                              *named.items()))  # fmt: skip
    index = _index_tensors(named)
    _check_batch(index)
    if num_target is not None:
        _check(num_target.numel() == seq_offset.numel() - 1, f"num_target must have a count per sequence ({seq_offset.numel() - 1}), but it has {num_target.numel()}")
    qc = _aligned(q)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if q.numel() == 0:
        return out
    p = _native.PagedFp8FwdParams()
    p.struct_size, p.dtype = ctypes.sizeof(p), _DTYPE_CODE[q.dtype]
    _describe(p.cache, k_cache, v_cache, k_scale, v_scale, weights, index)
    p.q, p.out, p.seq_offset = qc.data_ptr(), out.data_ptr(), index["seq_offset"].data_ptr()
    p.num_target = index["num_target"].data_ptr() if num_target is not None else None
    p.total_q, p.num_heads_q = q.size(0), q.size(1)
    p.max_seq_len_q, p.max_seq_len_k, p.target_group_size = int(max_seq_len), int(max_seq_len_k), int(target_group_size)
    p.window, p.sinks = int(window), int(sinks)
    p.silu_scale = 1.0 / int(max_seq_len) if float(silu_scale) == 0.0 else float(silu_scale)
    p.alpha = float(alpha)
    _call("hstu_paged_fp8_fwd", p, q.device)
    return out


def hstu_paged_fp8_meta(q, k_cache, v_cache, k_scale, v_scale, seq_offset, cache_len, page_offsets, page_ids, max_seq_len, max_seq_len_k,
                        silu_scale=0.0, num_target=None, target_group_size=0, alpha=1.0, window=0, sinks=0, weights=None):  # fmt: skip
    _check(q.dim() == 3, "The q should be 3D in jagged layout")
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _rows(t):
    """``t`` with strides the append kernel reads: whole heads in 16-byte steps."""
    ok = t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0
    return t if ok else _aligned(t)


def hstu_paged_fp8_append(k, v, k_cache, v_cache, k_scale, v_scale, seq_offset, cache_len, page_offsets, page_ids, max_seq_len, weights=None):
    """Writes the rows ``k``, ``v`` [total, heads_k, dim] (bf16 or fp16; head dim contiguous, other strides as they come) into the
    cache: those of sequence ``b``, ``seq_offset[b] : seq_offset[b + 1]``, at the positions from ``cache_len[b]`` on.  ``cache_len`` stays as
    it is.  Rows that the sequence's pages have no room for, and rows past ``max_seq_len``, are dropped.

    Each block of 32 tokens that is written to gets a new scale: the smallest power of two that brings its largest finite
    magnitude, old rows included, to at most 448.  Codes round to nearest even, but never to what no float holds (256 times the largest scale,
    2^120); values that are not finite become NaN.  The rows of a
    written block behind the new end are cleared, and the ``weights`` of new rows and of those, where given, become 0."""
    _check(k.dim() == 3 and v.dim() == 3, "The k and v should be 3D in jagged layout")
    _check(k.dtype in (torch.bfloat16, torch.float16) and v.dtype == k.dtype, f"k and v must both be bfloat16 or float16, but they are {k.dtype} and {v.dtype}")
    _check_cache(k_cache, v_cache, k_scale, v_scale, weights)
    rows = (k.size(0), k_cache.size(1), k_cache.size(4))
    _check(tuple(k.shape) == rows and tuple(v.shape) == rows, f"k and v must have the cache's heads and head dim ({list(rows)}), but they are {list(k.shape)} and {list(v.shape)}")
    _check(1 <= int(max_seq_len) <= MAX_SEQ_LEN_K, f"maxSeqLen expect in [1, {MAX_SEQ_LEN_K}], but value is {max_seq_len}")
    named = {"seq_offset": seq_offset, "cache_len": cache_len, "page_offsets": page_offsets, "page_ids": page_ids}
    _check(k.device.type == "cuda", f"k must be a GPU tensor, but it is on {k.device}")
    for name, t in (("v", v), ("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale), ("weights", weights), *named.items()):
        _check(t is None or t.device == k.device, f"{name} must be on the device of k ({k.device}), but it is on {getattr(t, 'device', None)}")
    index = _index_tensors(named)
    _check_batch(index)
    if k.numel() == 0:
        return
    kc, vc = _rows(k), _rows(v)
    p = _native.PagedFp8AppendParams()
    p.struct_size, p.dtype = ctypes.sizeof(p), _DTYPE_CODE[k.dtype]
    _describe(p.cache, k_cache, v_cache, k_scale, v_scale, weights, index)
    p.k, p.v, p.seq_offset, p.total = kc.data_ptr(), vc.data_ptr(), index["seq_offset"].data_ptr(), k.size(0)
    p.k_stride_row, p.k_stride_head, p.v_stride_row, p.v_stride_head = kc.stride(0), kc.stride(1), vc.stride(0), vc.stride(1)
    p.max_seq_len = int(max_seq_len)
    _call("hstu_paged_fp8_append", p, k.device, workspace=False)


def hstu_paged_fp8_append_meta(k, v, k_cache, v_cache, k_scale, v_scale, seq_offset, cache_len, page_offsets, page_ids, max_seq_len, weights=None):
    _check(k.dim() == 3 and v.dim() == 3, "The k and v should be 3D in jagged layout")


def hstu_paged_fp8_evict(k_cache, v_cache, k_scale, v_scale, weights, cache_len, page_offsets, page_ids, new_page_offsets, new_page_ids,
                         max_seq_len_k, keep, sinks=0, recent=0):  # fmt: skip
    """Moves the rows worth keeping to other pages, ``new_page_ids[new_page_offsets[b] : new_page_offsets[b + 1]]`` of sequence ``b``: at
    most ``keep`` rows each (and no more than those pages hold) -- the first ``sinks``, the last ``recent``, and of the others those
    with the largest sums of ``weights`` over the key heads, NaN counting as minus infinity, ties to the lower index -- in the order they
    were in, with scales of their new blocks and with their weights.  A sequence of no more than ``keep`` rows moves whole.  The old pages are only read: once
    the call is done (in the stream's order) they are the program's to hand out again.  New pages must be no pages that the call reads.

    Returns ``new_cache_len`` [batch] and ``kept`` [batch, keep]: the old indices of the rows that stay, -1 behind them (for what a
    program keeps beside the cache, time stamps say), both of the type of ``cache_len``."""
    _check(weights is not None, "eviction goes by weights, which must be given")
    _check_cache(k_cache, v_cache, k_scale, v_scale, weights)
    _check(1 <= int(max_seq_len_k) <= MAX_SEQ_LEN_K, f"maxSeqLenK expect in [1, {MAX_SEQ_LEN_K}], but value is {max_seq_len_k}")
    _check(1 <= int(keep) <= MAX_SEQ_LEN_K, f"keep expect in [1, {MAX_SEQ_LEN_K}], but value is {keep}")
    _check(int(sinks) >= 0 and int(recent) >= 0, f"sinks and recent must not be negative, but they are {sinks} and {recent}")
    named = {"cache_len": cache_len, "page_offsets": page_offsets, "page_ids": page_ids, "new_page_offsets": new_page_offsets,
             "new_page_ids": new_page_ids}  # fmt: skip
    device = k_cache.device
    _check(device.type == "cuda", f"k_cache must be a GPU tensor, but it is on {device}")
    for name, t in (("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale), ("weights", weights), *named.items()):
        _check(t.device == device, f"{name} must be on the device of k_cache ({device}), but it is on {t.device}")
    index = _index_tensors(named)
    _check_batch(index)
    batch = cache_len.numel()
    new_len = torch.empty(batch, dtype=index["cache_len"].dtype, device=device)
    kept = torch.empty((batch, int(keep)), dtype=index["cache_len"].dtype, device=device)
    p = _native.PagedFp8EvictParams()
    p.struct_size = ctypes.sizeof(p)
    _describe(p.cache, k_cache, v_cache, k_scale, v_scale, weights, index)
    p.new_page_offsets, p.new_page_ids = index["new_page_offsets"].data_ptr(), _ptr(index["new_page_ids"])
    p.new_cache_len, p.kept, p.n_new_page_ids = new_len.data_ptr(), kept.data_ptr(), new_page_ids.numel()
    p.max_seq_len_k, p.keep, p.sinks, p.recent = int(max_seq_len_k), int(keep), int(sinks), int(recent)
    _call("hstu_paged_fp8_evict", p, device)
    return new_len.to(cache_len.dtype), kept.to(cache_len.dtype)


def hstu_paged_fp8_evict_meta(k_cache, v_cache, k_scale, v_scale, weights, cache_len, page_offsets, page_ids, new_page_offsets, new_page_ids,
                              max_seq_len_k, keep, sinks=0, recent=0):  # fmt: skip
    _check(int(keep) >= 1, f"keep expect in [1, {MAX_SEQ_LEN_K}], but value is {keep}")
    return cache_len.new_empty(cache_len.shape), cache_len.new_empty((cache_len.size(0), keep))


for _name, _kernel, _meta in (("hstu_paged_fp8", hstu_paged_fp8, hstu_paged_fp8_meta),
                              ("hstu_paged_fp8_append", hstu_paged_fp8_append, hstu_paged_fp8_append_meta),
                              ("hstu_paged_fp8_evict", hstu_paged_fp8_evict, hstu_paged_fp8_evict_meta)):  # fmt: skip
    _PYTHON_KERNELS[_name] = _kernel
    _lib_meta.impl(_name, _meta)
