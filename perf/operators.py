"""The operators of the 8-bit paged key / value cache, as cases to time: writing new rows into the cache
(``hstu_paged_fp8_append``), attention that reads it (``hstu_paged_fp8``: single rows, candidates, chunks, with a sliding
window, with the attention weights added up per key) and moving the rows that are kept to other pages
(``hstu_paged_fp8_evict``).

The cache of one layer: pages of ``page`` tokens in blocks of 32; ``k_cache`` e4m3 [pages, heads_k, page / 32, 32, dim],
``v_cache`` e4m3 [pages, heads_k, page / 32, dim, 32], a scale per block and head for each, and fp32 ``weights``
[pages, heads_k, page].  The plain forms compute the same from elementary torch operations on padded tensors; ``exact`` goes
sequence by sequence in 64 bits.

A case is a dict of plain values.  ``batch`` sequences have ``lo .. hi`` rows in the cache before the call, spread evenly,
and ``new_lo .. new_hi`` new rows plus ``targets`` candidates in it; the order of the lengths, and every value, comes from
the seed given to ``prepare``.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEVICE = "cuda:0"
_BLOCK = 32  # tokens that share a scale
_TOP = 448.0  # the largest e4m3 value
_FP8 = torch.float8_e4m3fn

_DEFAULTS = dict(kind="attend", dtype="bf16", batch=32, heads=4, heads_k=4, dim=128, page=128, lo=1024, hi=4096, new_lo=1, new_hi=1,
                 targets=0, group=1, window=0, sinks=0, weights=False, keep=0, recent=0)  # fmt: skip


def _case(**values):
    return dict(_DEFAULTS, **values)


def listed():
    return [
        # ---- attention over the cache ----
        # the smallest call in use: the next event of a few users with short histories, where latency counts
        _case(name="attend-one-small", batch=4, dim=64, heads=2, heads_k=2, page=64, lo=100, hi=500),
        # a batch of single new events on ragged histories: bound by the cache's bytes
        _case(name="attend-one", batch=64, page=128, lo=2048, hi=8192),
        # single events of a few users with very long histories and wide heads: few rows, a long axis
        _case(name="attend-one-long", dtype="fp16", batch=3, heads=4, heads_k=2, dim=256, page=256, lo=30011, hi=120011),
        # ranking: some new events and a slate of candidates per request, odd lengths
        _case(name="attend-candidates", dtype="fp16", batch=32, dim=64, page=64, lo=501, hi=4001, new_lo=1, new_hi=16, targets=48),
        # a chunk of new events on a longer history, shared key heads: bound by the matrix and vector units
        _case(name="attend-chunk", batch=16, heads=8, heads_k=4, page=128, lo=2048, hi=8192, new_lo=512, new_hi=512),
        # the same with a sliding window behind a few first tokens, longer histories
        _case(name="attend-window", batch=24, page=128, lo=8192, hi=16384, new_lo=100, new_hi=260, window=1024, sinks=64),
        # candidates whose attention weights are added up per key, for the eviction to go by
        _case(name="attend-weights", batch=32, page=128, lo=2048, hi=4096, new_lo=8, new_hi=32, targets=32, weights=True),
        # ---- writing ----
        # the next event of every user of a batch
        _case(name="append-one", kind="append", batch=64, page=128, lo=100, hi=4096, weights=True),
        # chunks of new events, ragged and not at block borders
        _case(name="append-chunk", kind="append", dtype="fp16", batch=32, heads_k=8, page=256, lo=0, hi=2000, new_lo=500, new_hi=4001),
        # ---- eviction ----
        # a few short histories cut in half
        _case(name="evict-small", kind="evict", batch=4, heads_k=2, dim=64, page=64, lo=300, hi=500, keep=256, sinks=4, recent=64),
        # a batch of long histories cut to a budget, in one call
        _case(name="evict-long", kind="evict", batch=32, heads_k=4, page=128, lo=4096, hi=16384, keep=2048, sinks=16, recent=512),
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "evict"])
    heads_k = rng.choice([1, 2, 4, 4, 8])
    case = _case(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16"]), heads_k=heads_k, heads=heads_k * rng.choice([1, 1, 2, 4]),
                 dim=rng.choice([32, 48, 64, 64, 96, 128, 128, 128, 192, 256]), page=rng.choice([32, 64, 96, 128, 128, 256]))  # fmt: skip
    case["heads"] = min(case["heads"], 16)
    batch, hi = _log_int(rng, 1, 128), _log_int(rng, 40, 16384)
    lo = max(1, int(hi * rng.choice([1.0, rng.uniform(0.1, 0.9)])))
    if kind == "attend":
        shape = rng.choice(["one", "one", "candidates", "chunk"])
        if shape == "candidates":
            case.update(new_lo=0, new_hi=rng.randint(0, 32), targets=rng.randint(1, 64), group=rng.choice([1, 1, 3, 64]))
        elif shape == "chunk":
            case["new_hi"] = _log_int(rng, 64, 600)
            case["new_lo"] = rng.randint(1, case["new_hi"])
        if rng.random() < 0.3:
            case.update(window=_log_int(rng, 16, 2048), sinks=rng.choice([0, 4, rng.randint(1, 100)]))
        case["weights"] = rng.random() < 0.25
    elif kind == "append":
        case.update(lo=0, weights=rng.random() < 0.5)
        case["new_hi"] = rng.choice([1, _log_int(rng, 2, 4096)])
        case["new_lo"] = rng.randint(min(1, case["new_hi"]), case["new_hi"])
        lo = rng.randint(0, hi)
    else:
        case["keep"] = max(1, int(hi * rng.uniform(0.1, 0.9)))
        case["sinks"] = rng.randint(0, min(64, case["keep"] - 1))
        case["recent"] = rng.randint(0, (case["keep"] - case["sinks"]) // 2)
        case["weights"] = True
    while True:
        case.update(batch=batch, lo=min(lo, hi), hi=hi)
        w, longest = work(case), hi + case["new_hi"] + case["targets"]
        pairs = batch * case["heads"] * (case["new_hi"] + case["targets"]) * longest
        held = 2 * batch * longest * heads_k * case["dim"]
        if w["bytes"] <= 4e8 and w["flops"] <= 1e11 and (kind != "attend" or pairs <= 6e8) and held <= 1e9:
            return case
        if batch > 1:
            batch = max(1, int(batch / 1.5))
        else:
            hi = max(64, int(hi / 1.3))


# ------------------------------------------------------------------------------------------------------- inputs ----


def _spread(lo, hi, n):
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    """(rows cached before the call, new rows) of each sequence, candidates among the new ones: the same for every seed."""
    n = case["batch"]
    new = _spread(case["new_lo"], case["new_hi"], n)
    new = new[::2] + new[1::2][::-1]
    return list(zip(_spread(case["lo"], case["hi"], n), [x + case["targets"] for x in new]))


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def _encode(values):
    """Block values [..., 32, dim] (any order of the last two) as e4m3 codes and the blocks' scales: the smallest power of two
    that brings the largest finite magnitude to at most 448; what is not finite becomes NaN."""
    finite = torch.isfinite(values)
    top = torch.where(finite, values, torch.zeros_like(values)).abs().amax(dim=(-1, -2))
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    exponent = (exponent - 9 + (mantissa > 0.875).to(exponent.dtype)).clamp(min=-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), exponent), torch.ones_like(top))
    scaled = torch.where(finite, values / scale[..., None, None], torch.full_like(values, math.nan))
    return scaled.to(_FP8), scale


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(_DEVICE).manual_seed(seed)
    lengths = _lengths(case)
    rng.shuffle(lengths)
    page, dim, heads_k, heads = case["page"], case["dim"], case["heads_k"], case["heads"]
    evict = case["kind"] == "evict"
    old = [a for a, _ in lengths]
    new = [0 if evict else b for _, b in lengths]
    total = [a + b for a, b in zip(old, new)]
    pages = [-(-t // page) for t in total]
    new_pages = [-(-min(t, case["keep"]) // page) for t in total] if evict else []
    n_pages = sum(pages) + sum(new_pages) + 3
    order = list(range(n_pages))
    rng.shuffle(order)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=_DEVICE, dtype=dtype)

    def index(values):
        return torch.tensor(np.asarray(values), dtype=torch.int32, device=_DEVICE)

    blocks = page // _BLOCK
    # rows differ in size as a model's do, and heads from each other
    head_size = 0.25 * torch.arange(1, heads_k + 1, device=_DEVICE).view(-1, 1, 1, 1)
    k_codes, k_scale = _encode(randn(n_pages, heads_k, blocks, _BLOCK, dim) * head_size)
    v_codes, v_scale = _encode(randn(n_pages, heads_k, blocks, dim, _BLOCK) * head_size)
    state = dict(case=case, k_cache=k_codes, v_cache=v_codes, k_scale=k_scale, v_scale=v_scale, page_offsets=index(_offsets(pages)),
                 page_ids=index(order[: sum(pages)]), longest=max(total))  # fmt: skip
    if evict or case["weights"]:
        # accumulated weights fall off steeply: most tokens have little, a few have a lot
        state["weights"] = (randn(n_pages, heads_k, page) * 1.5).exp() * 1e-2
    if evict:
        state.update(cache_len=index(total), new_page_offsets=index(_offsets(new_pages)),
                     new_page_ids=index(order[sum(pages) : sum(pages) + sum(new_pages)]))  # fmt: skip
        return state
    rows, dtype = sum(new), _DTYPES[case["dtype"]]
    state.update(seq_offset=index(_offsets(new)), rows=rows, most=max(max(new), 1))
    if case["kind"] == "append":
        # the projection's outputs: [rows, heads * dim], seen as heads
        state.update(k=(randn(rows, heads_k * dim) * 0.5).to(dtype).view(rows, heads_k, dim),
                     v=(randn(rows, heads_k * dim) * 0.5).to(dtype).view(rows, heads_k, dim), cache_len=index(old))  # fmt: skip
    else:
        state.update(q=randn(rows, heads, dim).to(dtype), cache_len=index(total),
                     num_target=index([case["targets"]] * case["batch"]) if case["targets"] else None)  # fmt: skip
    return state


# -------------------------------------------------------------------------------------------------- plain forms ----


def _index(tensor, at):
    """``tensor[at]`` for e4m3 tensors too."""
    return tensor.view(torch.uint8)[at].view(_FP8) if tensor.dtype == _FP8 else tensor[at]


def _table(offsets, ids, most):
    """Page ids as [batch, most], 0 where a sequence has no such page."""
    at = offsets[:-1, None].long() + torch.arange(most, device=ids.device)
    return torch.where(at < offsets[1:, None], ids[at.clamp(max=ids.numel() - 1)].long(), torch.zeros_like(at))


def _rows_of(s, table, live):
    """K and V of the pages in ``table`` as fp32 [batch, heads_k, tokens, dim], 0 where ``live`` [batch, tokens] is not."""
    live = live[:, None, :, None]
    k = _index(s["k_cache"], table).float() * s["k_scale"][table][..., None, None]
    v = _index(s["v_cache"], table).float() * s["v_scale"][table][..., None, None]
    batch, pages, heads, blocks, _, dim = k.shape
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(batch, heads, -1, dim)
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(batch, heads, -1, dim)
    return torch.where(live, k, torch.zeros_like(k)), torch.where(live, v, torch.zeros_like(v))


def _mask(case, rows, keys, s_q, s_k):
    """Which keys a row sees, [batch, rows, keys]."""
    i, j = torch.arange(rows, device=_DEVICE)[None, :, None], torch.arange(keys, device=_DEVICE)[None, None, :]
    s_q, s_k = s_q.long()[:, None, None], s_k.long()[:, None, None]
    position = i + s_k - s_q
    centre = position
    seen = (j <= position) & (i < s_q) & (j < s_k)
    if case["targets"]:
        first_row, first_key = s_q - case["targets"], s_k - case["targets"]
        target = i >= first_row
        above = torch.div(i - first_row, case["group"], rounding_mode="floor") * case["group"]
        seen = seen & ~(target & (j >= first_key) & (j < first_key + above))
        centre = torch.where(target, first_key, position)
    if case["window"]:
        seen = seen & ((j > centre - case["window"]) | (j < case["sinks"]))
    return seen


def _plain_attend(s):
    case, page = s["case"], s["case"]["page"]
    pages, rows = -(-s["longest"] // page), s["most"]
    keys, offsets = pages * page, s["seq_offset"].long()
    s_q, s_k = offsets[1:] - offsets[:-1], s["cache_len"].long()
    table = _table(s["page_offsets"], s["page_ids"], pages)
    k, v = _rows_of(s, table, torch.arange(keys, device=_DEVICE) < s_k[:, None])
    at = offsets[:-1, None] + torch.arange(rows, device=_DEVICE)
    inside = at < offsets[1:, None]
    batch, heads_k, shared = case["batch"], case["heads_k"], case["heads"] // case["heads_k"]
    q = s["q"].float()[at.clamp(max=s["rows"] - 1)].view(batch, rows, heads_k, shared, -1).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(batch, heads_k, shared * rows, -1), k.transpose(2, 3)) * (case["dim"] ** -0.5)
    p = x / (1 + torch.exp(-x)) * (1.0 / s["most"])
    seen = _mask(case, rows, keys, s_q, s_k)[:, None, None]
    p = torch.where(seen, p.view(batch, heads_k, shared, rows, keys), torch.zeros((), device=_DEVICE))
    out = torch.matmul(p.view(batch, heads_k, shared * rows, keys), v).view(batch, heads_k, shared, rows, -1)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, rows, case["heads"], -1)
    # back to packed rows: a sequence's last row has the largest index that is inside
    flat = torch.zeros((s["rows"] + 1,) + tuple(out.shape[2:]), device=_DEVICE)
    flat[torch.where(inside, at, torch.full_like(at, s["rows"]))] = out
    out = flat[: s["rows"]].to(s["q"].dtype)
    if not case["weights"]:
        return out
    sums = p.abs().sum(dim=(2, 3)).view(batch, heads_k, pages, page).permute(0, 2, 1, 3)
    weights = torch.zeros_like(s["weights"])
    real = torch.arange(pages, device=_DEVICE) < (s["page_offsets"][1:] - s["page_offsets"][:-1])[:, None]
    weights.index_put_((table,), torch.where(real[..., None, None], sums, torch.zeros_like(sums)), accumulate=True)
    return out, weights


def _store(s, table, first, count, values_k, values_v):
    """Blocks ``first`` .. of each sequence from values [batch, heads_k, blocks, 32, dim] (``count`` of them): codes and scales."""
    per_page = s["case"]["page"] // _BLOCK
    n = values_k.shape[2]
    block = first[:, None] + torch.arange(n, device=_DEVICE)
    there = torch.arange(n, device=_DEVICE) < count[:, None]
    at = torch.nonzero(there, as_tuple=True)
    page, sub = table[at[0], (block // per_page)[at]], (block % per_page)[at]
    for cache, scales, values in ((s["k_cache"], s["k_scale"], values_k), (s["v_cache"], s["v_scale"], values_v.transpose(3, 4))):
        codes, scale = _encode(values.transpose(1, 2)[at])
        cache.view(torch.uint8).index_put_((page[:, None], torch.arange(scale.shape[1], device=_DEVICE), sub[:, None]), codes.view(torch.uint8))
        scales.index_put_((page[:, None], torch.arange(scale.shape[1], device=_DEVICE), sub[:, None]), scale)
    return page, sub, at


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    offsets, old = s["seq_offset"].long(), s["cache_len"].long()
    new = offsets[1:] - offsets[:-1]
    first = old // _BLOCK
    count = torch.where(new > 0, (old + new + _BLOCK - 1) // _BLOCK - first, torch.zeros_like(new))
    n = s["most"] // _BLOCK + 2
    table = _table(s["page_offsets"], s["page_ids"], -(-s["longest"] // page) + 1)
    # the blocks touched, their live rows decoded and the new rows put behind them
    per_page = page // _BLOCK
    block = first[:, None] + torch.arange(n, device=_DEVICE)
    pid = torch.gather(table, 1, (block // per_page).clamp(max=table.shape[1] - 1))
    sub = block % per_page
    position = (block[:, :, None] * _BLOCK + torch.arange(_BLOCK, device=_DEVICE)).view(case["batch"], -1)
    fresh = (position >= old[:, None]) & (position < (old + new)[:, None])
    at = (offsets[:-1, None] + position - old[:, None]).clamp(min=0, max=s["rows"] - 1)
    values = []
    for cache, scales, rows, swap in ((s["k_cache"], s["k_scale"], s["k"], False), (s["v_cache"], s["v_scale"], s["v"], True)):
        # [batch, n, heads, 32, dim] -> [batch, heads, n * 32, dim]
        held = _index(cache, (pid[:, :, None], torch.arange(case["heads_k"], device=_DEVICE), sub[:, :, None])).float()
        held = held * scales[pid[:, :, None], torch.arange(case["heads_k"], device=_DEVICE), sub[:, :, None]][..., None, None]
        held = (held.transpose(3, 4) if swap else held).permute(0, 2, 1, 3, 4).reshape(case["batch"], case["heads_k"], n * _BLOCK, -1)
        held = torch.where((position < old[:, None])[:, None, :, None], held, torch.zeros_like(held))
        held = torch.where(fresh[:, None, :, None], rows.float()[at].transpose(1, 2), held)
        values.append(held.view(case["batch"], case["heads_k"], n, _BLOCK, -1))
    page_at, sub_at, where = _store(s, table, first, count, *values)
    out = [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    if case["weights"]:
        w = s["weights"].view(-1, case["heads_k"], per_page, _BLOCK)
        live = (position < old[:, None]).view(case["batch"], n, _BLOCK)[where][:, None]
        heads = torch.arange(case["heads_k"], device=_DEVICE)
        held = w[page_at[:, None], heads, sub_at[:, None]]
        w.index_put_((page_at[:, None], heads, sub_at[:, None]), torch.where(live, held, torch.zeros_like(held)))
        out.append(s["weights"])
    return out


def _plain_evict(s):
    case, page = s["case"], s["case"]["page"]
    pages = -(-s["longest"] // page)
    keys, length = pages * page, s["cache_len"].long()
    table = _table(s["page_offsets"], s["page_ids"], pages)
    held = s["weights"][table].permute(0, 2, 1, 3).reshape(case["batch"], case["heads_k"], keys)
    score = held[:, 0]
    for h in range(1, case["heads_k"]):  # the sum is taken in the order of the heads
        score = score + held[:, h]
    j = torch.arange(keys, device=_DEVICE)
    room = (s["new_page_offsets"][1:] - s["new_page_offsets"][:-1]).long() * page
    budget = torch.minimum(length.clamp(max=case["keep"]), room)
    sinks = budget.clamp(max=case["sinks"])
    recent = (budget - sinks).clamp(max=case["recent"])
    forced = (j < sinks[:, None]) | (j >= (length - recent)[:, None])
    score = torch.where(torch.isnan(score), torch.full_like(score, -math.inf), score)
    score = torch.where(forced, torch.full_like(score, math.inf), score)
    score = torch.where(j < length[:, None], score, torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    chosen = torch.where(j < budget[:, None], order, torch.full_like(order, keys))
    chosen = torch.sort(chosen, dim=1).values[:, : case["keep"]]
    if chosen.shape[1] < case["keep"]:
        chosen = torch.nn.functional.pad(chosen, (0, case["keep"] - chosen.shape[1]), value=keys)
    kept = torch.where(chosen < keys, chosen, torch.full_like(chosen, -1)).to(s["cache_len"].dtype)
    # the rows kept, in whole blocks
    n = -(-case["keep"] // _BLOCK)
    chosen = torch.nn.functional.pad(chosen, (0, n * _BLOCK - case["keep"]), value=keys)
    there, at = chosen < keys, chosen.clamp(max=keys - 1)
    per_page = page // _BLOCK
    pid, sub, slot = torch.gather(table, 1, at // page)[:, None], (at % page // _BLOCK)[:, None], (at % _BLOCK)[:, None]
    head = torch.arange(case["heads_k"], device=_DEVICE)[None, :, None]
    values = []
    for cache, scales, swap in ((s["k_cache"], s["k_scale"], False), (s["v_cache"], s["v_scale"], True)):
        rows = cache.view(torch.uint8)
        rows = (rows.transpose(3, 4) if swap else rows)[pid, head, sub, slot].view(_FP8).float() * scales[pid, head, sub][..., None]
        rows = torch.where(there[:, None, :, None], rows, torch.zeros_like(rows))
        values.append(rows.view(case["batch"], case["heads_k"], n, _BLOCK, -1))
    weights = torch.where(there[:, None], torch.gather(held, 2, at[:, None].expand(-1, case["heads_k"], -1)), torch.zeros((), device=_DEVICE))
    new_table = _table(s["new_page_offsets"], s["new_page_ids"], -(-case["keep"] // page))
    zero = torch.zeros_like(budget)
    page_at, sub_at, where = _store(s, new_table, zero, (budget + _BLOCK - 1) // _BLOCK, *values)
    w = s["weights"].view(-1, case["heads_k"], per_page, _BLOCK)
    w.index_put_((page_at[:, None], head[0, :, 0], sub_at[:, None]), weights.view(case["batch"], case["heads_k"], n, _BLOCK).transpose(1, 2)[where])
    return budget.to(s["cache_len"].dtype), kept, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["weights"]


# -------------------------------------------------------------------------------------------------------- calls ----


def _own_attend(s):
    case = s["case"]
    # a program that adds weights up over several calls begins with a cleared plane
    weights = torch.zeros_like(s["weights"]) if case["weights"] else None
    out = _attention().hstu_paged_fp8(
        s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["seq_offset"], s["cache_len"], s["page_offsets"], s["page_ids"],
        s["most"], s["longest"], 0.0, s["num_target"], case["group"] if case["targets"] else 0, case["dim"] ** -0.5, case["window"],
        case["sinks"], weights)  # fmt: skip
    return (out, weights) if case["weights"] else out


def _own_append(s):
    weights = s["weights"] if s["case"]["weights"] else None
    _attention().hstu_paged_fp8_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["seq_offset"], s["cache_len"],
                                       s["page_offsets"], s["page_ids"], s["most"], weights)  # fmt: skip
    out = [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    return out + [weights] if weights is not None else out


def _own_evict(s):
    case = s["case"]
    length, kept = _attention().hstu_paged_fp8_evict(
        s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["weights"], s["cache_len"], s["page_offsets"], s["page_ids"],
        s["new_page_offsets"], s["new_page_ids"], s["longest"], case["keep"], case["sinks"], case["recent"])  # fmt: skip
    return length, kept, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["weights"]


def _attention():
    if "ops_rec" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "ops-rec_amd"))
        import ops_rec  # noqa: F401
    return sys.modules["ops_rec"].ascendc.attention


def run(state):
    kind = state["case"]["kind"]
    if own:
        return (_own_attend if kind == "attend" else _own_append if kind == "append" else _own_evict)(state)
    return (_plain_attend if kind == "attend" else _plain_append if kind == "append" else _plain_evict)(state)


# --------------------------------------------------------------------------------------------------------- work ----


def work(case):
    dim, heads, heads_k = case["dim"], case["heads"], case["heads_k"]
    moved = flops = 0
    for old, new in _lengths(case):
        if case["kind"] == "evict":
            kept = min(old, case["keep"])
            # the weights of every row, and each row that is kept: read, and written to its new place
            moved += old * heads_k * 4 + 2 * kept * heads_k * (2 * dim + 4)
            continue
        if case["kind"] == "append":
            moved += new * heads_k * dim * 2 * (2 + 1) + -(-new // _BLOCK) * heads_k * 8 + (new * heads_k * 4 if case["weights"] else 0)
            flops += 4 * new * heads_k * dim
            continue
        s_q, s_k, t, g = new, old + new, case["targets"], case["group"]
        i = np.arange(s_q)
        position = i + s_k - s_q
        seen, centre = position + 1, position.copy()
        if t:
            target = i >= s_q - t
            seen = np.where(target, seen - (i - (s_q - t)) // g * g, seen)
            centre = np.where(target, s_k - t, position)
        keys = s_k
        if case["window"] and s_q:
            seen = seen - np.maximum(centre - case["window"] - case["sinks"] + 1, 0)
            keys = s_k - max(int(centre.min()) - case["window"] - case["sinks"] + 1, 0)
        flops += int(seen.sum()) * heads * 4 * dim
        moved += keys * heads_k * 2 * dim + -(-keys // _BLOCK) * heads_k * 8 + 4 * s_q * heads * dim + (keys * heads_k * 8 if case["weights"] else 0)
    return {"bytes": float(moved), "flops": float(flops)}


# -------------------------------------------------------------------------------------------------------- exact ----


def _decoded(codes):
    """e4m3 codes as their values, from the format: sign, four bits of exponent (bias 7), three of fraction; 0x7f is NaN."""
    code = np.arange(256)
    e, m = code >> 3 & 15, code & 7
    value = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0 ** (e - 10.0))
    value = np.where(code & 127 == 127, np.nan, np.where(code & 128, -value, value))
    return torch.from_numpy(value).to(codes.device)[codes.view(torch.uint8).long()]


def _rounded(values, scale):
    """Values over a scale, as the nearest e4m3 value, ties to even."""
    x = values / scale
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0**-6)))
    step = 2.0 ** (e - 3)
    return np.where(np.isfinite(values), np.rint(x / step) * step, np.nan)


def _scale(values):
    top = np.max(np.abs(np.where(np.isfinite(values), values, 0.0)))
    return 2.0 ** max(math.ceil(math.log2(top / _TOP)), -126) if top > 0 else 1.0


class _Books:
    """The cache in 64 bits, row by row."""

    def __init__(self, s):
        self.s, self.page = s, s["case"]["page"]
        self.values = [_decoded(s["k_cache"]).cpu().numpy(), _decoded(s["v_cache"]).cpu().numpy()]
        self.scales = [s["k_scale"].double().cpu().numpy(), s["v_scale"].double().cpu().numpy()]
        self.weights = s["weights"].double().cpu().numpy() if "weights" in s else None

    def block(self, which, pid, h, sub):
        x = self.values[which][pid, h, sub] * self.scales[which][pid, h, sub]
        return x if which == 0 else x.T

    def put(self, which, pid, h, sub, values):
        scale = _scale(values)
        x = _rounded(values, scale)
        self.values[which][pid, h, sub] = x if which == 0 else x.T
        self.scales[which][pid, h, sub] = scale

    def answer(self):
        return [torch.from_numpy(x) for x in self.values + self.scales]


def _exact_attend(s):
    case, page, dim = s["case"], s["case"]["page"], s["case"]["dim"]
    offsets, lens = s["seq_offset"].tolist(), s["cache_len"].tolist()
    firsts, ids = s["page_offsets"].tolist(), s["page_ids"].tolist()
    out = torch.zeros(tuple(s["q"].shape), dtype=torch.float64, device=_DEVICE)
    weights = torch.zeros(tuple(s["weights"].shape), dtype=torch.float64, device=_DEVICE) if case["weights"] else None
    shared = case["heads"] // case["heads_k"]
    for b, s_k in enumerate(lens):
        s_q, mine = offsets[b + 1] - offsets[b], ids[firsts[b] : firsts[b + 1]]
        if not s_q:
            continue
        i, j = torch.arange(s_q, device=_DEVICE)[:, None], torch.arange(s_k, device=_DEVICE)[None]
        place = i + (s_k - s_q)
        sees = j <= place
        around = place
        if case["targets"]:
            t, g = case["targets"], case["group"]
            candidate, other = i >= s_q - t, j >= s_k - t
            same = torch.div(i - (s_q - t), g, rounding_mode="floor") == torch.div(j - (s_k - t), g, rounding_mode="floor")
            sees = torch.where(candidate & other, (j <= place) & same, sees)
            around = torch.where(candidate, torch.full_like(place, s_k - t), place)
        if case["window"]:
            sees = sees & ((around - j < case["window"]) | (j < case["sinks"]))
        for h in range(case["heads_k"]):
            k = (_decoded(s["k_cache"][mine, h]) * s["k_scale"][mine, h].double()[..., None, None]).reshape(-1, dim)[:s_k]
            v = (_decoded(s["v_cache"][mine, h]) * s["v_scale"][mine, h].double()[..., None, None]).transpose(2, 3).reshape(-1, dim)[:s_k]
            for n in range(h * shared, (h + 1) * shared):
                x = s["q"][offsets[b] : offsets[b + 1], n].double() @ k.t() / math.sqrt(dim)
                p = torch.where(sees, x * torch.sigmoid(x) / s["most"], 0.0)
                out[offsets[b] : offsets[b + 1], n] = p @ v
                if weights is not None:
                    sums = torch.zeros(len(mine) * page, dtype=torch.float64, device=_DEVICE)
                    sums[:s_k] = p.abs().sum(0)
                    weights[mine, h] += sums.view(-1, page)
    return out if weights is None else (out, weights)


def _exact_append(s):
    case, page = s["case"], s["case"]["page"]
    books, per_page = _Books(s), page // _BLOCK
    rows = [s["k"].double().cpu().numpy(), s["v"].double().cpu().numpy()]
    offsets, firsts, ids = s["seq_offset"].tolist(), s["page_offsets"].tolist(), s["page_ids"].tolist()
    for b, old in enumerate(s["cache_len"].tolist()):
        end = old + offsets[b + 1] - offsets[b]
        for block in range(old // _BLOCK, -(-end // _BLOCK) if end > old else 0):
            pid, sub, start = ids[firsts[b] + block // per_page], block % per_page, block * _BLOCK
            a, z = max(old, start), min(end, start + _BLOCK)
            for h in range(case["heads_k"]):
                for which in (0, 1):
                    values = np.zeros((_BLOCK, case["dim"]))
                    if a > start:
                        values[: a - start] = books.block(which, pid, h, sub)[: a - start]
                    values[a - start : z - start] = rows[which][offsets[b] + a - old : offsets[b] + z - old, h]
                    books.put(which, pid, h, sub, values)
            if case["weights"]:
                books.weights[pid, :, a - start + sub * _BLOCK : (sub + 1) * _BLOCK] = 0
    return books.answer() + ([torch.from_numpy(books.weights)] if case["weights"] else [])


def _exact_evict(s):
    case, page = s["case"], s["case"]["page"]
    books, per_page = _Books(s), page // _BLOCK
    firsts, ids = s["page_offsets"].tolist(), s["page_ids"].tolist()
    new_firsts, new_ids = s["new_page_offsets"].tolist(), s["new_page_ids"].tolist()
    lens, kept = [], []
    for b, length in enumerate(s["cache_len"].tolist()):
        mine, to = ids[firsts[b] : firsts[b + 1]], new_ids[new_firsts[b] : new_firsts[b + 1]]
        # scores are sums in 32 bits by definition: which rows stay is a matter of their order
        each = s["weights"][mine].cpu().numpy()
        score = each[:, 0].copy()
        for h in range(1, case["heads_k"]):
            score += each[:, h]
        score = score.reshape(-1)[:length]
        budget = min(length, case["keep"], len(to) * page)
        sinks = min(budget, case["sinks"])
        recent = min(budget - sinks, case["recent"])
        stay = set(range(sinks)) | set(range(length - recent, length))
        for j in sorted(range(length), key=lambda j: (-score[j], j)):
            if len(stay) >= budget:
                break
            stay.add(j)
        stay = sorted(stay)
        lens.append(len(stay))
        kept.append(stay + [-1] * (case["keep"] - len(stay)))
        for start in range(0, len(stay), _BLOCK):
            some = stay[start : start + _BLOCK]
            pid, sub = to[start // page], start % page // _BLOCK
            at = [(mine[j // page], j % page // _BLOCK, j % _BLOCK) for j in some]
            pids, subs, slots = (np.array(x) for x in zip(*at))
            for h in range(case["heads_k"]):
                for which in (0, 1):
                    values = np.zeros((_BLOCK, case["dim"]))
                    x = books.values[which]
                    x = x[pids, h, subs, slots] if which == 0 else x[pids, h, subs, :, slots]
                    values[: len(some)] = x * books.scales[which][pids, h, subs][:, None]
                    books.put(which, pid, h, sub, values)
                books.weights[pid, h, sub * _BLOCK : (sub + 1) * _BLOCK] = 0
                books.weights[pid, h, sub * _BLOCK : sub * _BLOCK + len(some)] = books.weights[pids, h, subs * _BLOCK + slots]
    dtype = s["cache_len"].dtype
    return [torch.tensor(lens, dtype=dtype), torch.tensor(kept, dtype=dtype)] + books.answer() + [torch.from_numpy(books.weights)]


def exact(case, seed):
    blocks = sum(-(-(min(a, case["keep"]) if case["kind"] == "evict" else b) // _BLOCK) for a, b in _lengths(case))
    if case["kind"] != "attend" and (blocks * case["heads_k"] > 60_000 or sum(a + b for a, b in _lengths(case)) * case["heads_k"] * case["dim"] > 2e8):
        return None  # block by block on the host: too many of them
    state = prepare(case, seed)
    return (_exact_attend if case["kind"] == "attend" else _exact_append if case["kind"] == "append" else _exact_evict)(state)
