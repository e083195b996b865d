"""Two Python threads on one stream: each call's kernels are queued together, so none reads another's workspace."""
import threading
import time

import pytest
import torch


def _in_threads(work, n=2):
    """work(i) in n threads that start together; the first exception is raised here."""
    gate, errors = threading.Barrier(n), []

    def body(i):
        try:
            gate.wait()
            work(i)
        except Exception as e:  # noqa: BLE001 - handed to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


def test_calls_that_share_a_workspace_do_not_interleave(monkeypatch):
    """A call of two launches, the interpreter free between them, as an engine call leaves it: what another thread's call
    writes to the workspace never comes between a call's own two launches, growth included."""
    from vault_b200 import _lib, paged
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(paged, "_stream", lambda index: 77)
    monkeypatch.setattr(paged, "_capturing", lambda: False)
    shared, queue = paged._Workspaces(), []

    def work(me):
        for i in range(20):
            need = 4096 << i // 2

            def call(work_ptr, size, stream):
                if size < need:
                    return _lib.V3G_E_SIZE
                queue.append((me, i, work_ptr))
                time.sleep(0.0005)
                queue.append((me, i, work_ptr))
                return 0

            assert shared.run(torch.device("cpu", 0), lambda: need, call) == 0

    _in_threads(work, 3)
    assert len(queue) == 3 * 20 * 2
    assert all(a == b for a, b in zip(queue[::2], queue[1::2]))


def test_a_call_inside_a_call_does_not_wait_for_itself(monkeypatch):
    """A finalizer that runs while a workspace grows may use the same operators."""
    from vault_b200 import paged
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(paged, "_stream", lambda index: 77)
    monkeypatch.setattr(paged, "_capturing", lambda: False)
    shared, cpu = paged._Workspaces(), torch.device("cpu", 0)

    def size():
        assert shared.run(cpu, lambda: 16, lambda *a: 0) == 0
        return 16

    assert shared.run(cpu, size, lambda *a: 0) == 0


@pytest.mark.gpu
def test_beam_select_from_two_threads():
    """The results of each thread are bit for bit what the same calls give alone."""
    from vault_b200 import beam_select
    g = torch.Generator().manual_seed(1)
    cases = [[(torch.randn(1, 4, v, generator=g).cuda(), torch.zeros(1, 4).cuda()) for _ in range(4)] for v in (60000, 61000)]
    want = [[beam_select(*c) for c in mine] for mine in cases]
    got = [[], []]

    def work(me):
        for _ in range(200):
            for c in cases[me]:
                got[me].append(beam_select(*c))

    _in_threads(work)
    for me in range(2):
        for i, r in enumerate(got[me]):
            assert all(torch.equal(a, b) for a, b in zip(r, want[me][i % 4]))


@pytest.mark.gpu
def test_split_attention_from_two_threads():
    from tests import paged_ref as ref
    from vault_b200 import PagedKVCache
    bt = ref.Batch([1], [3000], 64, seed=1)
    cache = PagedKVCache.wrap(*(t.cuda() for t in ref.random_cache(2, bt.n_pages, 2, 64, 128, seed=2)))
    dev = bt.cuda()
    q = [torch.randn(1, 12, 128, generator=torch.Generator().manual_seed(i)).half().cuda() for i in range(2)]
    want = [cache.attention(i, q[i], *dev) for i in range(2)]
    got = [[], []]

    def work(me):
        for _ in range(500):
            got[me].append(cache.attention(me, q[me], *dev))

    _in_threads(work)
    for me in range(2):
        assert all(torch.equal(o, want[me]) for o in got[me])
