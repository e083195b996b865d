"""GPU: what follows an attention call on its stream, or in a graph, sees its whole output."""
import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


def _prompts_without_a_hint():
    """Two prompts of 100 tokens, 8 heads each way, a table of 512 keys, no max_q: the batch could hold single tokens, so its
    rows have places for shares, but both sequences are the many-row kernel's and none is left for the join."""
    from vault_b200 import PagedKVCache
    bt = ref.Batch([100, 100], [0, 0], 64, seed=1, extra_cols=6)
    parts = ref.random_cache(1, bt.n_pages, 8, 64, 128, seed=2)
    q = torch.randn(bt.n, 8, 128, generator=torch.Generator().manual_seed(3)).half()
    return bt, parts, PagedKVCache.wrap(*(t.cuda() for t in parts)), q


def test_output_is_complete_for_the_next_kernel():
    bt, parts, cache, q = _prompts_without_a_hint()
    dev, qd = bt.cuda(), q.cuda()
    want, _, tol, _ = ref.attention(q, parts, 0, bt, 0, 0, 128 ** -0.5)
    out = torch.empty_like(qd)
    copies = []
    for _ in range(50):
        out.fill_(7.0)
        cache.attention(0, qd, *dev, out=out)
        copies.append(out.clone())
    assert bool(((copies[0].cpu().double() - want).abs() <= tol + 2.0 ** -11 * want.abs() + 2.0 ** -24).all())
    assert all(torch.equal(c, copies[0]) for c in copies)
    cache.check()


def test_output_is_complete_inside_a_graph():
    bt, _, cache, q = _prompts_without_a_hint()
    dev, qd = bt.cuda(), q.cuda()
    want = cache.attention(0, qd, *dev)
    out = torch.empty_like(qd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copies = []
        for _ in range(8):
            out.fill_(7.0)
            cache.attention(0, qd, *dev, out=out)
            copies.append(out.clone())
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c, want) for c in copies)
    cache.check()
