"""GPU: PagedKVCache.check() reports what calls on any stream met."""
import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


def _late_append(cache, bt, stream, table):
    """An append on `stream`, some 20 ms after it is queued."""
    x = torch.randn(bt.n, 1, 64, device="cuda")
    _, kv_len, q_start = bt.cuda()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(40_000_000)
        cache.append(0, x, x, table, kv_len, q_start)
    return x, table, kv_len, q_start   # held by the caller until they have been used


def test_a_call_still_running_on_another_stream_is_waited_for():
    from vault_b200 import PagedKVCache
    bt = ref.Batch([3], [0], 16, seed=1)
    cache = PagedKVCache.wrap(*(t.cuda() for t in ref.random_cache(1, bt.n_pages, 1, 16, 64, seed=2)))
    side, nowhere = torch.cuda.Stream(), torch.full_like(bt.table, -1).cuda()
    held = [_late_append(cache, bt, side, nowhere)]
    with pytest.raises(RuntimeError, match="status"):
        cache.check()
    cache.check()
    held.append(_late_append(cache, bt, side, bt.table.cuda()))
    cache.check()
    with torch.cuda.stream(side):                 # checked from one stream, used on the other
        held.append(_late_append(cache, bt, torch.cuda.Stream(), nowhere))
        with pytest.raises(RuntimeError, match="status"):
            cache.check()
    cache.check()
    torch.cuda.synchronize()
