"""GPU: the operators of a decode step captured into one graph, and short chunks of wide groups under a window."""
import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _step(cache, x, hq, hkv, head, table, kv_len, one_each, rope, scores, finished, out_table):
    """One beam-search step: append, attention of every layer, logits, selection, reorder.  The table is updated in place."""
    from vault_b200 import beam_select
    for layer in range(cache.n_layers):
        q = cache.append(layer, x[:, hq:hq + hkv], x[:, hq + hkv:], table, kv_len, one_each, rope=rope, q=x[:, :hq])
        o = cache.attention(layer, q, table, kv_len, one_each, max_q=1, max_kv=4000)
    logits = (o.float().flatten(1) @ head).view(*scores.shape, -1)
    tokens, parents, best, done = beam_select(logits, scores, finished, 3)
    out_table.copy_(cache.reorder(table, kv_len, parents))
    return tokens, parents, best, done


def test_a_captured_step_replays_as_it_runs():
    """Three steps of 2 groups of 4 beams over 3,000 cached tokens, by calls and by replays of one graph: the same bits."""
    from vault_b200 import PagedKVCache, rope_table
    d, hq, hkv, page, rows = 128, 12, 2, 64, 8
    bt = ref.Batch([1] * rows, [3000 + 40 * (r // 4) for r in range(rows)], page, seed=1, extra_cols=2)
    parts = ref.random_cache(2, bt.n_pages, hkv, page, d, seed=2)
    g = torch.Generator().manual_seed(3)
    xs = [torch.randn(rows, hq + 2 * hkv, d, generator=g).half().cuda() for _ in range(3)]
    head = torch.randn(hq * d, 5000, generator=g).cuda()
    rope = rope_table(4096, d)
    one_each = bt.q_start.cuda()

    def start():
        scores = torch.zeros(2, 4, device="cuda")
        scores[:, 1:] = -3.0
        return (PagedKVCache.wrap(*(t.cuda() for t in parts)), torch.empty_like(xs[0]), bt.table.cuda(), bt.kv_len.cuda(), scores,
                torch.zeros(2, 4, dtype=torch.uint8, device="cuda"))

    def drive(run, x, table, kv_len, scores, finished, out_table):
        seen = []
        for step in range(3):
            x.copy_(xs[step])
            tokens, parents, best, done = run()
            seen += [tokens.clone(), parents.clone(), best.clone(), done.clone()]
            scores.copy_(best), finished.copy_(done), table.copy_(out_table), kv_len.add_(1)
        return seen

    cache, x, table, kv_len, scores, finished = start()
    out_table = torch.empty_like(table)
    args = (hq, hkv, head, table, kv_len, one_each, rope, scores, finished, out_table)
    want = drive(lambda: _step(cache, x, *args), x, table, kv_len, scores, finished, out_table)
    want += [table.clone(), *(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))]
    cache.check()

    cache, x, table, kv_len, scores, finished = start()
    out_table = torch.empty_like(table)
    args = (hq, hkv, head, table, kv_len, one_each, rope, scores, finished, out_table)
    x.copy_(xs[0])
    _step(cache, x, *args)                        # what a first call sets up
    fresh = start()
    for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (fresh[0].k, fresh[0].v, fresh[0].k_scale, fresh[0].v_scale)):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(cache, x, *args)

    def replay():
        graph.replay()
        return held

    got = drive(replay, x, table, kv_len, scores, finished, out_table)
    got += [table.clone(), *(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))]
    cache.check()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("new,group,window,sinks", [([4, 2, 3], 16, 70, 3), ([9, 1, 5], 7, 40, 0), ([7], 8, 1, 20)])
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128)])
def test_short_chunks_of_wide_groups(new, group, window, sinks, dtype, d):
    """Several 16-row tiles of one sequence, rows of a tile at different tokens, some keys behind the window of some rows."""
    from vault_b200 import PagedKVCache
    bt = ref.Batch(new, [300, 18, 65][:len(new)], 32, seed=group)
    parts = ref.random_cache(1, bt.n_pages, 2, 32, d, seed=group)
    cache = PagedKVCache.wrap(*(t.cuda() for t in parts))
    q = (1.5 * torch.randn(bt.n, 2 * group, d, generator=torch.Generator().manual_seed(5))).to(dtype)
    out, lse = cache.attention(0, q.cuda(), *bt.cuda(), window=window, n_sink=sinks, return_lse=True, max_q=max(new))
    want, want_lse, tol, tol_lse = ref.attention(q, parts, 0, bt, window, sinks, d ** -0.5)
    assert bool(((out.cpu().double() - want).abs() <= tol + HALF_ULP[dtype] * want.abs() + 2.0 ** -24).all())
    assert bool(((lse.cpu().double() - want_lse).abs() <= tol_lse).all())
