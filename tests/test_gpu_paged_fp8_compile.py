"""The operators of the 8-bit paged cache under torch.compile and torch.library.opcheck: their schemas say what they write."""

import pytest
import torch

import ops_rec
import paged_fp8_reference as R
from test_gpu_compile import BACKENDS, compiled

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CACHE = ("k_cache", "v_cache", "k_scale", "v_scale")
PAGES = ("cache_len", "page_offsets", "page_ids")


def rows(counts, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(sum(counts), heads, dim, generator=g).to(torch.bfloat16).to(DEV)


def copy(c):
    return {n: c[n].clone() for n in (*CACHE, *PAGES, "weights")}


def test_opcheck():
    c, offs = R.make([70, 33], heads_k=2, dim=32, page=64, seed=1, device=DEV), R.offsets([6, 3], device=DEV)
    cache, pages = tuple(c[n] for n in CACHE), tuple(c[n] for n in PAGES)
    checks = ("test_faketensor", "test_autograd_registration")  # (test_schema multiplies its inputs, which torch does not do for e4m3: the test below)
    ops, q = torch.ops.ops_rec, rows([6, 3], 4, 32, 1)
    for weights in (None, c["weights"]):
        torch.library.opcheck(ops.hstu_paged_fp8.default, (q, *cache, offs, *pages, 6, 70, 0.0, None, 0, 0.2, 20, 2, weights), test_utils=checks)
    k = rows([6, 3], 2, 32, 2)
    room = R.make([70, 33], room=[128, 64], heads_k=2, dim=32, page=64, seed=1, device=DEV)
    torch.library.opcheck(ops.hstu_paged_fp8_append.default, (k, k, *(room[n] for n in CACHE), offs, *(room[n] for n in PAGES), 6, room["weights"]), test_utils=checks)
    spare = R.make([70, 33, 64, 64], heads_k=2, dim=32, page=64, seed=1, device=DEV)
    old = (spare["cache_len"][:2].contiguous(), spare["page_offsets"][:3].contiguous(), spare["page_ids"])
    new = (torch.tensor([3, 4, 5], dtype=torch.int32, device=DEV), spare["page_ids"])
    torch.library.opcheck(ops.hstu_paged_fp8_evict.default, (*(spare[n] for n in CACHE), spare["weights"], *old, *new, 70, 40, 2, 8), test_utils=checks)


def test_each_operator_writes_no_more_than_its_schema_says():
    k, q = rows([6, 3], 2, 32, 2), rows([6, 3], 4, 32, 1)
    offs = R.offsets([6, 3], device=DEV)
    c = R.make([70, 33, 64, 64], room=[128, 64, 64, 64], heads_k=2, dim=32, page=64, seed=1, device=DEV)
    old = (c["cache_len"][:2].contiguous(), c["page_offsets"][:3].contiguous(), c["page_ids"])
    new = (torch.tensor([3, 4, 5], dtype=torch.int32, device=DEV), c["page_ids"].clone())
    cache, ops = tuple(c[n] for n in CACHE), torch.ops.ops_rec
    for op, args in ((ops.hstu_paged_fp8.default, (q, *cache, offs, *old, 6, 70, 0.0, None, 0, 0.2, 20, 2, c["weights"])),
                     (ops.hstu_paged_fp8_append.default, (k, k.clone(), *cache, offs, *old, 6, c["weights"])),
                     (ops.hstu_paged_fp8_evict.default, (*cache, c["weights"], *old, *new, 70, 40, 2, 8))):  # fmt: skip
        before = [t.clone() if isinstance(t, torch.Tensor) else t for t in args]
        out = op(*args)
        outs = [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
        for arg, t, b in zip(op._schema.arguments, args, before):
            if not isinstance(t, torch.Tensor):
                continue
            same = torch.equal(t.view(torch.uint8), b.view(torch.uint8))
            assert same or (arg.alias_info is not None and arg.alias_info.is_write), (op, arg.name)
            assert all(o.untyped_storage().data_ptr() != t.untyped_storage().data_ptr() for o in outs)


@pytest.mark.parametrize("backend", BACKENDS)
def test_a_compiled_step_is_an_eager_one(backend):
    """Append, then attend with weights, in one graph: the attention reads what the append wrote, and the program's tensors change."""
    att = ops_rec.ascendc.attention

    def step(q, k, v, k_cache, v_cache, k_scale, v_scale, weights, offs, cache_len, page_offsets, page_ids, most, longest):
        att.hstu_paged_fp8_append(k, v, k_cache, v_cache, k_scale, v_scale, offs, cache_len, page_offsets, page_ids, most, weights)
        lens = cache_len + (offs[1:] - offs[:-1])
        return att.hstu_paged_fp8(q, k_cache, v_cache, k_scale, v_scale, offs, lens, page_offsets, page_ids, most, longest, 0.1, None, 0, 0.2, 0, 0, weights), lens

    fn = compiled(step, backend)
    start = R.make([70, 33], room=[256, 256], heads_k=2, dim=32, page=64, seed=1, device=DEV)
    eager, graph = copy(start), copy(start)
    for counts in ([6, 3], [1, 1], [9, 40]):
        offs = R.offsets(counts, device=DEV)
        q, k, v = rows(counts, 4, 32, 1), rows(counts, 2, 32, 2), rows(counts, 2, 32, 3)
        got = []
        for f, c in ((step, eager), (fn, graph)):
            y, lens = f(q, k, v, *(c[n] for n in CACHE), c["weights"], offs, *(c[n] for n in PAGES), max(counts), 256)
            c["cache_len"] = lens
            got.append(y)
        assert torch.equal(*got)
    for n in (*CACHE, "weights", "cache_len"):
        assert torch.equal(*(c[n].view(torch.uint8) for c in (eager, graph))), n  # (what is not live may be NaN)


def test_nothing_of_a_graph_stays_in_the_cache():
    """Rows and queries that ask for gradients, which these operators do not give: the program's tensors hold no graph afterwards."""
    c = R.make([70], room=[128], heads_k=2, dim=32, page=64, seed=1, device=DEV)
    offs, att = R.offsets([6], device=DEV), ops_rec.ascendc.attention
    q, k = (rows([6], 2, 32, seed).requires_grad_() for seed in (1, 2))
    att.hstu_paged_fp8_append(k, k, *(c[n] for n in CACHE), offs, *(c[n] for n in PAGES), 6, c["weights"])
    att.hstu_paged_fp8(q, *(c[n] for n in CACHE), offs, *(c[n] for n in PAGES), 6, 70, weights=c["weights"])
    assert not any(c[n].requires_grad or c[n].grad_fn for n in (*CACHE, "weights"))
    with torch.no_grad():
        assert not att.hstu_paged_fp8(q, *(c[n] for n in CACHE), offs, *(c[n] for n in PAGES), 6, 70).requires_grad
