"""GPU: packed rows that belong to no sequence (a step of fixed size that is not full) come out as zeros, lse as -inf."""
import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}

CASES = [  # new, cached, rows before the first sequence, rows after the last, hints
    ([1], [0], 0, 1, dict(max_q=1)),
    ([1, 1, 1], [700, 30, 4], 0, 5, dict(max_q=1)),
    ([1], [1500], 2, 1000, dict(max_q=1)),
    ([1, 0, 2, 0], [40, 9, 300, 5], 0, 17, dict(max_q=2)),
    ([1] * 40, [11 * i for i in range(40)], 0, 300, dict(max_q=1)),
    ([90, 130], [5, 0], 0, 3, dict(max_q=130)),
    ([300], [0], 7, 700, dict(max_q=300)),
    ([150, 1, 1], [60, 333, 2], 0, 40, {}),
    ([0, 0], [50, 0], 0, 33, {}),
]


def _padded(new, ctx, before, after, page=32):
    bt = ref.Batch(new, ctx, page, seed=len(new))
    bt.q_start += before
    return bt, before + bt.n + after


@pytest.mark.parametrize("new,ctx,before,after,hints", CASES)
@pytest.mark.parametrize("dtype,d", [(torch.float16, 128), (torch.bfloat16, 64)])
def test_attention(new, ctx, before, after, hints, dtype, d):
    from vault_b200 import PagedKVCache
    bt, n = _padded(new, ctx, before, after)
    parts = ref.random_cache(1, bt.n_pages, 2, 32, d, seed=3)
    cache = PagedKVCache.wrap(*(t.cuda() for t in parts))
    q = torch.randn(n, 6, d, generator=torch.Generator().manual_seed(4)).to(dtype)
    out = torch.full((n, 6, d), math.nan, dtype=dtype, device="cuda")
    torch.full((n, 6), 7.0, device="cuda")                       # what an allocation of lse's size finds
    got, lse = cache.attention(0, q.cuda(), *bt.cuda(), out=out, return_lse=True, **hints)
    want, want_lse, tol, tol_lse = ref.attention(q, parts, 0, bt, 0, 0, d ** -0.5)
    assert got is out
    assert bool(((out.cpu().double() - want).abs() <= tol + HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]).all())
    lse, seen = lse.cpu().double(), ~torch.isinf(want_lse)
    assert torch.equal(lse[~seen], want_lse[~seen]) and bool(((lse - want_lse).abs()[seen] <= tol_lse[seen]).all())
    cache.check()


@pytest.mark.parametrize("new,ctx,before,after", [c[:4] for c in CASES])
@pytest.mark.parametrize("dtype,d", [(torch.float32, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("turned", [True, False])
def test_append(new, ctx, before, after, dtype, d, turned):
    """The queries of the sequences are what they are without padding, the cache too."""
    from vault_b200 import PagedKVCache, rope_table
    bt, n = _padded(new, ctx, before, after)
    start = ref.random_cache(1, bt.n_pages, 2, 32, d, seed=3)
    x = torch.randn(n, 9, d, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    rope = rope_table(2048, d) if turned else None
    table, kv_len, q_start = bt.cuda()
    both = []
    for lo, hi, starts in ((0, n, q_start), (before, before + bt.n, q_start - before)):
        cache = PagedKVCache.wrap(*(t.cuda() for t in start))
        q_out = torch.full((hi - lo, 5, d), math.nan, dtype=dtype, device="cuda")
        cache.append(0, x[lo:hi, 5:7], x[lo:hi, 7:], table, kv_len, starts, rope=rope, q=x[lo:hi, :5], q_out=q_out)
        cache.check()
        both.append((q_out, cache))
    padded, plain = both
    assert torch.equal(padded[0][before:before + bt.n], plain[0])
    assert bool((padded[0][:before] == 0).all()) and bool((padded[0][before + bt.n:] == 0).all())
    for a, b in ((padded[1].k, plain[1].k), (padded[1].v, plain[1].v), (padded[1].k_scale, plain[1].k_scale),
                 (padded[1].v_scale, plain[1].v_scale)):
        assert torch.equal(a, b)


def test_a_graph_of_fixed_size_follows_its_index_arrays():
    """One captured step of 8 rows, replayed with 5, 0 and 8 of them in use."""
    from vault_b200 import PagedKVCache
    d = 128
    bt = ref.Batch([1] * 8, [40, 3, 100, 7, 64, 15, 16, 0], 16, seed=1)
    parts = ref.random_cache(1, bt.n_pages, 2, 16, d, seed=3)
    cache = PagedKVCache.wrap(*(t.cuda() for t in parts))
    table, kv_len, q_start = bt.cuda()
    q = torch.randn(8, 4, d, generator=torch.Generator().manual_seed(4)).half().cuda()
    whole = cache.attention(0, q, table, kv_len, q_start, max_q=1).clone()
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(0, q, table, kv_len, q_start, max_q=1, out=out)
    for used in (5, 0, 8):
        q_start.copy_(torch.arange(9, dtype=torch.int32).clamp(max=used))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert bool((out[used:] == 0).all()) and torch.equal(out[:used], whole[:used])
