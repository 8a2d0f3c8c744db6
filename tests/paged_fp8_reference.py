"""The 8-bit paged cache in 64 bits on the CPU, written from the operators' definitions: what the tests compare with.

A ``Book`` holds copies of a cache's tensors; ``append``, ``attend`` and ``evict`` do what the operators do, row by row.  ``attend`` also
says how far a correct kernel may be off."""

from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = 32
_CODE = np.arange(256)
_E, _M = _CODE >> 3 & 15, _CODE & 7
# e4m3: sign, 4 bits of exponent with bias 7, 3 of fraction, subnormals; no infinities, 0x7f and 0xff are NaN
_VALUES = np.where(_E == 0, _M * 2.0**-9, (8 + _M) * 2.0 ** (_E - 10.0))
_VALUES = np.where((_CODE & 127) == 127, np.nan, np.where(_CODE & 128, -_VALUES, _VALUES))


def decode(codes):
    return _VALUES[codes.cpu().contiguous().view(torch.uint8).numpy()]


def quantise(values):
    """(code values, scale) of a block."""
    finite = np.where(np.isfinite(values), values, 0.0)
    top = np.abs(finite).max() if finite.size else 0.0
    scale = 2.0 ** max(math.ceil(math.log2(top / 448.0)), -126) if top > 0 else 1.0
    x = finite / scale
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0**-6))) - 3)
    return np.where(np.isfinite(values), np.rint(x / step) * step, np.nan), scale


def encode(values):
    """Code values as codes (NaN: 0x7f)."""
    flat = np.abs(np.nan_to_num(values, nan=0.0)).ravel()
    code = np.searchsorted(_VALUES[:127], flat)
    assert (_VALUES[code] == flat).all()
    code = np.where(np.signbit(values).ravel(), code | 128, code)
    code = np.where(np.isnan(values).ravel(), 127, code)
    return torch.from_numpy(code.reshape(values.shape).astype(np.uint8)).view(torch.float8_e4m3fn)


class Book:
    def __init__(self, k_cache, v_cache, k_scale, v_scale, weights, page_offsets, page_ids):
        self.codes = [decode(k_cache), np.swapaxes(decode(v_cache), 3, 4)]  # both [pages, heads, blocks, 32, dim]
        self.scales = [k_scale.cpu().double().numpy().copy(), v_scale.cpu().double().numpy().copy()]
        self.weights = None if weights is None else weights.cpu().double().numpy().copy()
        self.offsets, self.ids = page_offsets.tolist(), page_ids.tolist()
        self.pages, self.heads, self.blocks, _, self.dim = k_cache.shape
        self.page = self.blocks * BLOCK

    def _pages(self, b, offsets=None, ids=None):
        offsets, ids = offsets or self.offsets, self.ids if ids is None else ids
        return ids[offsets[b] : offsets[b + 1]]

    def rows(self, which, b, h, n):
        """The first n rows of a sequence, [n, dim]; rows of a page that is not there are zeros."""
        out = np.zeros((n, self.dim))
        for i, pid in enumerate(self._pages(b)):
            a, z = i * self.page, min(n, (i + 1) * self.page)
            if a < z and 0 <= pid < self.pages:
                x = self.codes[which][pid, h] * self.scales[which][pid, h][:, None, None]
                out[a:z] = x.reshape(self.page, self.dim)[: z - a]
        return out

    def append(self, k, v, seq_offset, cache_len):
        rows, offsets = (k.cpu().double().numpy(), v.cpu().double().numpy()), seq_offset.tolist()
        for b, old in enumerate(cache_len.tolist()):
            pages = self._pages(b)
            end = min(old + offsets[b + 1] - offsets[b], len(pages) * self.page)
            for blk in range(old // BLOCK, -(-end // BLOCK) if end > old else 0):
                pid, sub, start = pages[blk // self.blocks], blk % self.blocks, blk * BLOCK
                if not 0 <= pid < self.pages:
                    continue
                a, z = max(old, start), min(end, start + BLOCK)
                for h in range(self.heads):
                    for which in (0, 1):
                        x = np.zeros((BLOCK, self.dim))
                        x[: a - start] = (self.codes[which][pid, h, sub] * self.scales[which][pid, h, sub])[: a - start]
                        x[a - start : z - start] = rows[which][offsets[b] + a - old : offsets[b] + z - old, h]
                        self.codes[which][pid, h, sub], self.scales[which][pid, h, sub] = quantise(x)
                if self.weights is not None:
                    self.weights[pid, :, sub * BLOCK + a - start : (sub + 1) * BLOCK] = 0

    def mask(self, s_q, s_k, targets, group, window, sinks):
        i, j = np.arange(s_q)[:, None], np.arange(s_k)[None]
        position = i + s_k - s_q
        seen, centre = j <= position, np.broadcast_to(position, (s_q, 1))
        if targets and group:
            row, key = i - (s_q - targets), j - (s_k - targets)
            seen = seen & ~((row >= 0) & (key >= 0) & (key // group < row // group))
            centre = np.where(row >= 0, s_k - targets, position)
        if window:
            seen = seen & ((j > centre - window) | (j < sinks))
        return seen

    def attend(self, q, seq_offset, cache_len, max_seq_len, silu_scale=0.0, num_target=None, group=0, alpha=1.0, window=0, sinks=0):
        """(out, how far it may be off, weights' increments, how far they may be off), in 64 bits.

        With u the unit roundoff of q's type: P is rounded to it (u |P| each, and at most 2^-25 below the normal fp16 range, in units
        of the weight before its factor alpha * silu_scale), and so is the output (u |O|).  Scores are sums of dim products in
        fp32: off by at most dim 2^-23 sum |q k|, and by 2^-21 of the weight for exp2 (its argument's rounding is of the score's
        kind, 4 units of it counted), reciprocal and products, silu' being at most 1.1; the sums over n keys add n 2^-24 of their
        magnitudes.  fp16 numbers below 2^-14 are multiples of 2^-24, so there a rounding is off by up to 2^-25 whatever the value: of the
        output, and of a code times its scale (K and V as the products take them).  Weights are sums of |P| in fp32 before it is
        rounded."""
        scale = silu_scale or 1.0 / max_seq_len
        u = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[q.dtype]
        under = 2.0**-25 if q.dtype == torch.float16 else 0.0
        x_q, offsets = q.cpu().double().numpy(), seq_offset.tolist()
        out, off = np.zeros(x_q.shape), np.zeros(x_q.shape)
        plane = (self.pages, self.heads, self.page)
        inc, inc_off = np.zeros(plane), np.zeros(plane)
        ratio = x_q.shape[1] // self.heads
        for b, s_k in enumerate(cache_len.tolist()):
            s_q, pages = offsets[b + 1] - offsets[b], self._pages(b)
            s_k = min(s_k, len(pages) * self.page)
            t = num_target.tolist()[b] if num_target is not None else 0
            seen = self.mask(s_q, s_k, t, group, window, sinks)
            for n in range(x_q.shape[1]):
                k, v = self.rows(0, b, n // ratio, s_k), self.rows(1, b, n // ratio, s_k)
                rows = x_q[offsets[b] : offsets[b + 1], n]
                with np.errstate(all="ignore"):
                    s = alpha * np.where(seen, rows @ k.T, 0.0)
                    p = np.where(seen, s / (1 + np.exp(-s)) * scale, 0.0)
                    size = abs(alpha) * np.where(seen, np.abs(rows) @ np.abs(k).T, 0.0)
                    size_k = abs(alpha) * under * np.abs(rows).sum(1, keepdims=True)  # (K's own rounding)
                d_p = np.where(seen, 1.1 * abs(scale) * size_k, 0.0) + np.where(seen, 1.1 * abs(scale) * size * (self.dim + 4) * 2.0**-23 + np.abs(p) * 2.0**-21, 0.0)
                # a key that a row does not see adds nothing to it, whatever the key's row holds
                for r in range(s_q):
                    at = seen[r]
                    out[offsets[b] + r, n] = p[r, at] @ v[at]
                    one = (np.abs(p[r, at]) * (u + s_k * 2.0**-24) + d_p[r, at] + under * abs(alpha * scale)) @ np.abs(v[at])
                    one = one + under * np.abs(p[r, at]).sum()  # (V's)
                    off[offsets[b] + r, n] = one + u * (np.abs(out[offsets[b] + r, n]) + one) + under
                total, slack = np.abs(p).sum(0), d_p.sum(0)
                for i, pid in enumerate(pages):
                    a, z = i * self.page, min(s_k, (i + 1) * self.page)
                    if a < z and 0 <= pid < self.pages:
                        inc[pid, n // ratio, : z - a] += total[a:z]
                        inc_off[pid, n // ratio, : z - a] += slack[a:z] + (s_q * ratio + 2) * 2.0**-24 * total[a:z]
        return out, off, inc, inc_off

    def evict(self, cache_len, new_offsets, new_ids, keep, sinks, recent):
        new_offsets, new_ids = new_offsets.tolist(), new_ids.tolist()
        lens, kept = [], []
        before = [x.copy() for x in self.codes], [x.copy() for x in self.scales], self.weights.copy()
        for b, length in enumerate(cache_len.tolist()):
            pages, to = self._pages(b), self._pages(b, new_offsets, new_ids)
            length = min(length, len(pages) * self.page)
            score = np.zeros(length, dtype=np.float32)
            for j in range(length):
                pid = pages[j // self.page]
                for h in range(self.heads if 0 <= pid < self.pages else 0):
                    w = np.float32(before[2][pid, h, j % self.page])
                    score[j] = w if h == 0 else score[j] + w
            budget = min(length, keep, len(to) * self.page)
            first = min(budget, sinks)
            last = min(budget - first, recent)
            stay = set(range(first)) | set(range(length - last, length))
            for j in sorted(range(length), key=lambda j: (np.inf if np.isnan(score[j]) else -score[j], j)):
                if len(stay) >= budget:
                    break
                stay.add(j)
            stay = sorted(stay)
            lens.append(len(stay))
            kept.append(stay + [-1] * (keep - len(stay)))
            for start in range(0, len(stay), BLOCK):
                pid, sub = to[start // self.page], start % self.page // BLOCK
                if not 0 <= pid < self.pages:
                    continue
                some = stay[start : start + BLOCK]
                for h in range(self.heads):
                    x, w = np.zeros((2, BLOCK, self.dim)), np.zeros(BLOCK)
                    for n, j in enumerate(some):
                        src, at = pages[j // self.page], j % self.page
                        if 0 <= src < self.pages:
                            for which in (0, 1):
                                x[which, n] = before[0][which][src, h, at // BLOCK, at % BLOCK] * before[1][which][src, h, at // BLOCK]
                            w[n] = before[2][src, h, at]
                    for which in (0, 1):
                        self.codes[which][pid, h, sub], self.scales[which][pid, h, sub] = quantise(x[which])
                    self.weights[pid, h, sub * BLOCK : (sub + 1) * BLOCK] = w
        return lens, kept

    def same(self, k_cache, v_cache, k_scale, v_scale, weights=None):
        """Whether the tensors hold exactly what the book does."""
        for which, codes in ((0, decode(k_cache)), (1, np.swapaxes(decode(v_cache), 3, 4))):
            np.testing.assert_array_equal(codes, self.codes[which])
        np.testing.assert_array_equal(k_scale.cpu().double().numpy(), self.scales[0])
        np.testing.assert_array_equal(v_scale.cpu().double().numpy(), self.scales[1])
        if weights is not None:
            np.testing.assert_array_equal(weights.cpu().double().numpy(), self.weights)


def make(lens, *, page=64, heads_k=2, dim=64, room=None, spare=2, seed=0, index=torch.int32, device="cpu", weights=True, poison=True):
    """A cache that holds random rows for sequences of these lengths; pages for ``room`` rows each (default: the lengths).  What is not
    live is NaN, codes, scales and weights alike, in the pages of the sequences too."""
    g = torch.Generator().manual_seed(seed)
    room = room or lens
    counts = [-(-max(r, n) // page) for r, n in zip(room, lens)]
    total, blocks = sum(counts) + spare, page // BLOCK
    order = torch.randperm(total, generator=g).tolist()
    k = torch.full((total, heads_k, blocks, BLOCK, dim), 0x7F, dtype=torch.uint8)
    v = torch.full((total, heads_k, blocks, dim, BLOCK), 0xFF, dtype=torch.uint8)
    scales = [torch.full((total, heads_k, blocks), math.nan), torch.full((total, heads_k, blocks), math.nan)]
    w = torch.full((total, heads_k, page), math.nan)
    at = 0
    for n, count in zip(lens, counts):
        for blk in range(-(-n // BLOCK)):
            pid, sub, live = order[at + blk // blocks], blk % blocks, min(BLOCK, n - blk * BLOCK)
            for h in range(heads_k):
                for which, cache in ((0, k), (1, v)):
                    size = 10 ** (0.5 * torch.randn(1, generator=g).item())
                    codes, scale = quantise((size * torch.randn(BLOCK, dim, generator=g)).double().numpy())
                    codes = encode(codes).view(torch.uint8)
                    if which == 0:
                        cache[pid, h, sub, :live] = codes[:live]
                    else:
                        cache[pid, h, sub, :, :live] = codes[:live].T
                    scales[which][pid, h, sub] = scale
            w[pid, :, sub * BLOCK : sub * BLOCK + live] = torch.rand(heads_k, live, generator=g)
        at += count
    if not poison:
        k, v = torch.where((k & 127) == 127, 0, k), torch.where((v & 127) == 127, 0, v)
        scales, w = [torch.nan_to_num(s, nan=1.0) for s in scales], torch.nan_to_num(w)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=index)
    out = dict(k_cache=k.view(torch.float8_e4m3fn), v_cache=v.view(torch.float8_e4m3fn), k_scale=scales[0], v_scale=scales[1],
               weights=w if weights else None, page_offsets=offsets, page_ids=torch.tensor(order[:at], dtype=index),
               cache_len=torch.tensor(lens, dtype=index))  # fmt: skip
    out["free"] = order[at:]
    return {n: t.to(device) if torch.is_tensor(t) else t for n, t in out.items()}


def book(c):
    return Book(c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["weights"], c["page_offsets"], c["page_ids"])


def offsets(counts, index=torch.int32, device="cpu"):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=index, device=device)
