"""GPU: the paged 8-bit cache operators against their plain 64-bit forms (tests/paged_ref.py)."""
import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}


def _near(out, want, tol, dtype):
    """Every element within tol and its type's rounding; values past the type's range are infinities of their sign."""
    out = out.cpu().double()
    past = want.abs() > torch.finfo(dtype).max * (1 + HALF_ULP[dtype] / 2)
    near = (out - want).abs() <= tol + HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]
    return bool(torch.where(past, out == math.inf * want.sign(), near).all())


def _wrap(parts):
    from vault_b200 import PagedKVCache
    return PagedKVCache.wrap(*(t.cuda() for t in parts))


def _parts(cache):
    return [t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


# ---------------------------------------------------------------------------------------------------------- append
APPEND = [  # new tokens, cached tokens, page, kv heads, query heads, head dim
    ([1], [0], 16, 1, 1, 64),
    ([1], [15], 16, 2, 12, 128),
    ([1, 1, 1], [0, 16, 4607], 64, 2, 12, 128),
    ([2, 0, 17, 1, 33], [15, 5, 0, 31, 100], 32, 8, 32, 64),
    ([16, 32, 31], [16, 7, 0], 16, 3, 3, 128),
    ([301], [1023], 256, 1, 8, 128),
]


@pytest.mark.parametrize("new,ctx,page,hkv,hq,d", APPEND)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_rounds_by_block(new, ctx, page, hkv, hq, d, dtype):
    """Scales within 2^-21; a code within half a step of the rotated 64-bit value over the scale (plus what fp32 rotation and
    division may move a value near 127 by: 127 x 2^-20); earlier codes within half a step of where the new scale puts them;
    everything outside the touched blocks unchanged; q within its type's rounding of the rotation."""
    from vault_b200 import rope_table
    bt = ref.Batch(new, ctx, page, seed=page + d)
    g = torch.Generator().manual_seed(1)
    before = ref.random_cache(2, bt.n_pages, hkv, page, d, seed=2)
    cache = _wrap(before)
    table, kv_len, q_start = bt.cuda()
    rope = rope_table(max(n + c for n, c in zip(new, ctx)), d)
    qkv = torch.randn(bt.n, hq + 2 * hkv, d, generator=g) * torch.exp(torch.randn(bt.n, 1, 1, generator=g))
    qkv = qkv.to(dtype)
    dev = qkv.cuda()
    q = cache.append(1, dev[:, hq:hq + hkv], dev[:, hq + hkv:], table, kv_len, q_start, rope=rope, q=dev[:, :hq])
    cache.check()
    after = _parts(cache)
    for t0, t1 in zip(before, after):
        assert torch.equal(t0[0], t1[0])   # the other layer
    pos = torch.cat([torch.arange(c, c + n) for n, c in zip(new, ctx)])
    x = qkv.double()
    rot = ref.rotate(x[:, :hq + hkv], pos, rope.cpu())
    size = torch.cat([x[:, :hq, :d // 2].abs() + x[:, :hq, d // 2:].abs()] * 2, -1)
    assert bool(((q.cpu().double() - rot[:, :hq]).abs() <= HALF_ULP[dtype] * rot[:, :hq].abs() + 2.0 ** -22 * size + SMALLEST[dtype]).all())
    touched = torch.zeros(bt.n_pages, page, dtype=torch.bool)
    for b in range(len(new)):
        p, end = ctx[b], ctx[b] + new[b]
        while p < end:
            lo, hi = p - p % 16, min(p - p % 16 + 16, end)
            pg, slot = int(bt.table[b, lo // page]), lo % page
            touched[pg, slot:slot + 16] = True
            r0 = int(bt.q_start[b]) + p - ctx[b]
            for kind, rows in ((0, rot[r0:r0 + hi - p, hq:]), (1, x[r0:r0 + hi - p, hq + hkv:])):
                for h in range(hkv):
                    s_old = float(before[2 + kind][1, pg, h, slot // 16]) if p > lo else 0.0
                    s = max(s_old, float(rows[:, h].abs().max()) / 127)
                    got = float(after[2 + kind][1, pg, h, slot // 16])
                    assert abs(got - s) <= 2.0 ** -21 * s
                    codes = after[kind][1, pg, h].double() - 128
                    assert bool((codes[slot + p - lo:slot + hi - lo] - rows[:, h] / s).abs().max() <= 0.5 + 127 * 2.0 ** -20)
                    if p > lo:
                        old = before[kind][1, pg, h, slot:slot + p - lo].double() - 128
                        assert float((codes[slot:slot + p - lo] - old * (s_old / s)).abs().max()) <= 0.5 + 127 * 2.0 ** -20
            p = hi
    for kind in (0, 1):
        same = (after[kind][1] == before[kind][1]).all(-1).all(1)   # [page, token], every head
        assert bool((same | touched).all())


def test_append_without_rotation_and_single_tokens_in_turn():
    """A sequence appended token by token ends within the accumulated rounding of one appended at once: every code is moved
    at most 15 times, half a step each, at scales that only grow."""
    d, hkv, n = 64, 2, 37
    x = torch.randn(n, 2 * hkv, d, generator=torch.Generator().manual_seed(5))
    bt = ref.Batch([n], [0], 16, seed=1)
    whole, steps = (_wrap(ref.random_cache(1, bt.n_pages, hkv, 16, d, seed=7)) for _ in range(2))
    table, kv_len, q_start = bt.cuda()
    dev = x.cuda()
    assert whole.append(0, dev[:, :hkv], dev[:, hkv:], table, kv_len, q_start) is None
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for i in range(n):
        steps.append(0, dev[i:i + 1, :hkv], dev[i:i + 1, hkv:], table, torch.tensor([i + 1], dtype=torch.int32, device="cuda"), one)
    zero, rows = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for a, b, exact in zip(whole.read(table, zero, kv_len, rows, n), steps.read(table, zero, kv_len, rows, n), (x[:, :hkv], x[:, hkv:])):
        step = exact.abs().reshape(n, -1).max() / 127
        assert float((a[0].cpu() - exact).abs().max()) <= 0.501 * float(step)
        assert float((b[0].cpu() - exact).abs().max()) <= 8.01 * float(step)
    assert torch.equal(whole.k_scale[0, table[0, :2].long()], steps.k_scale[0, table[0, :2].long()])


def test_append_strides_alignment_and_broadcast():
    """Rows at odd element offsets, token strides and a head stride of zero give what contiguous copies give."""
    d, hkv, hq = 128, 2, 3
    bt = ref.Batch([5, 20], [3, 0], 32, seed=3)
    table, kv_len, q_start = bt.cuda()
    from vault_b200 import rope_table
    rope = rope_table(64, d)
    start = ref.random_cache(1, bt.n_pages, hkv, 32, d, seed=4)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        flat = torch.randn(bt.n * 1000 + 64, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
        k = torch.as_strided(flat, (bt.n, hkv, d), (997, 131, 1), 1)
        v = torch.as_strided(flat, (bt.n, hkv, d), (997, 0, 1), 3)
        q = torch.as_strided(flat, (bt.n, hq, d), (991, 129, 1), 7)
        a, b = _wrap(start), _wrap(start)
        qa = a.append(0, k, v, table, kv_len, q_start, rope=rope, q=q)
        qb = b.append(0, k.contiguous(), v.contiguous(), table, kv_len, q_start, rope=rope, q=q.contiguous())
        assert torch.equal(qa, qb)
        for s, t in zip(_parts(a), _parts(b)):
            assert torch.equal(s, t)


def test_append_odd_values():
    """All-zero rows store scale 0; tiny rows too; a NaN or an infinity makes its block (and no other) read as NaN, later
    tokens of the block included; the block's next owner starts anew."""
    d = 64
    bt = ref.Batch([48], [0], 16, seed=1, spare=0)
    cache = _wrap(ref.random_cache(1, bt.n_pages, 1, 16, d, seed=1))
    table, kv_len, q_start = bt.cuda()
    k = torch.randn(48, 1, d, generator=torch.Generator().manual_seed(2))
    v = k.clone()
    k[:16] = 0
    k[16:32] = 1e-39
    v[5, 0, 7], v[40, 0, 1] = math.inf, math.nan
    cache.append(0, k.cuda(), v.cuda(), table, kv_len, q_start)
    rows = torch.tensor([0, 48], dtype=torch.int32, device="cuda")
    kk, vv = (t[0].cpu() for t in cache.read(table, torch.zeros(1, dtype=torch.int32, device="cuda"), kv_len, rows, 48))
    assert bool((kk[:32] == 0).all()) and float((kk[32:] - k[32:]).abs().max()) <= 0.501 * float(k[32:].abs().max()) / 127
    assert bool(vv[:16].isnan().all()) and bool(vv[32:].isnan().all()) and not bool(vv[16:32].isnan().any())
    # the page starts again with another sequence's first token
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    cache.append(0, k[32:33].cuda(), k[32:33].cuda(), table, torch.tensor([1], dtype=torch.int32, device="cuda"), one)
    kk, vv = cache.read(table, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda"), one, 1)
    assert not bool(vv.isnan().any())


def test_append_tokens_without_a_place():
    """Tokens past the page table, on unmapped or impossible pages, before position 0 or past the rotation table are
    dropped, the status says so, and nothing else moves."""
    from vault_b200 import rope_table
    d = 64
    start = ref.random_cache(1, 4, 1, 16, d, seed=1)
    x = torch.randn(40, 1, d, generator=torch.Generator().manual_seed(2)).cuda()

    def run(table, kv_len, n, rope=None):
        cache = _wrap(start)
        t = torch.tensor([table], dtype=torch.int32, device="cuda")
        q = cache.append(0, x[:n], x[:n], t, torch.tensor([kv_len], dtype=torch.int32, device="cuda"),
                         torch.tensor([0, n], dtype=torch.int32, device="cuda"), rope=rope, q=x[:n])
        with pytest.raises(RuntimeError, match="status"):
            cache.check()
        cache.check()
        changed = torch.stack([(a != b).flatten(2).any(-1)[0] for a, b in zip(_parts(cache)[:2], start[:2])]).any(0)
        return changed.tolist(), q

    assert run([0, 1], 40, 40)[0] == [True, True, False, False]      # 8 tokens past the table
    assert run([0, -1, 2], 40, 40)[0] == [True, False, True, False]
    assert run([4, 1, 77], 40, 40)[0] == [False, True, False, False]
    assert run([3], 10, 20)[0] == [False, False, False, True]        # the first ten stand before position 0
    assert run([3], -5, 20)[0] == [False, False, False, False]
    changed, q = run([0, 1, 2], 40, 40, rope=rope_table(20, d))
    assert changed == [True, True, False, False]
    assert bool((q[20:] == 0).all()) and bool((q[:20] != 0).any(-1).all())


def test_read_rows_and_types():
    bt = ref.Batch([0, 0, 0], [70, 0, 33], 16, seed=9)
    parts = ref.random_cache(3, bt.n_pages, 2, 16, 128, seed=3)
    cache = _wrap(parts)
    table, kv_len, _ = bt.cuda()
    first = [60, 0, 0]
    start = torch.tensor([0, 10, 10, 43], dtype=torch.int32, device="cuda")
    f = torch.tensor(first, dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for kind, got in enumerate(cache.read(table, f, kv_len, start, 45, dtype)):
            assert got.shape == (3, 45, 2, 128) and bool((got[:, 43:] == 0).all())
            for layer in range(3):
                for h in range(2):
                    want = torch.cat([ref.values(parts[kind][layer], parts[2 + kind][layer], bt.table[b], h, n)[lo:]
                                      for b, (n, lo) in enumerate(zip((70, 0, 33), first))])
                    assert bool(((got[layer, :43, h].cpu().double() - want).abs() <= HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]).all())


# ------------------------------------------------------------------------------------------------------- attention
ATTEND = [  # new, cached, page, kv heads, query heads, head dim, window, sinks
    ([1], [0], 16, 1, 1, 64, 0, 0),
    ([1], [16], 16, 2, 12, 128, 0, 0),
    ([1, 1, 1], [511, 700, 3], 64, 2, 12, 128, 0, 0),
    ([1, 1], [300, 17], 32, 2, 4, 64, 33, 5),
    ([1], [1500], 16, 1, 1, 128, 100, 40),
    ([4, 0, 1, 9], [100, 7, 0, 63], 64, 4, 8, 128, 0, 0),
    ([70], [0], 16, 2, 6, 64, 0, 0),
    ([130, 1, 40], [5, 250, 0], 64, 2, 12, 128, 64, 4),
    ([129], [128], 128, 1, 16, 128, 0, 0),
    ([257, 3], [31, 400], 32, 3, 3, 64, 200, 130),
    ([33], [0], 256, 1, 7, 128, 1, 0),
    ([64], [300], 64, 2, 8, 128, 70, 1),
]


@pytest.mark.parametrize("new,ctx,page,hkv,hq,d,window,sinks", ATTEND)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hints", [True, False])
def test_attention_matches_64_bit(new, ctx, page, hkv, hq, d, window, sinks, dtype, hints):
    bt = ref.Batch(new, ctx, page, seed=d + page)
    cache_parts = ref.random_cache(2, bt.n_pages, hkv, page, d, seed=len(new))
    cache = _wrap(cache_parts)
    table, kv_len, q_start = bt.cuda()
    q = (1.5 * torch.randn(bt.n, hq, d, generator=torch.Generator().manual_seed(8))).to(dtype)
    kw = dict(max_q=max(new), max_kv=max(n + c for n, c in zip(new, ctx))) if hints else {}
    out, lse = cache.attention(1, q.cuda(), table, kv_len, q_start, window=window, n_sink=sinks, return_lse=True, **kw)
    want, want_lse, tol, tol_lse = ref.attention(q, cache_parts, 1, bt, window, sinks, d ** -0.5)
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol + HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]).all()), float((err - tol).max())
    assert bool(((lse.cpu().double() - want_lse).abs() <= tol_lse).all())
    again = cache.attention(1, q.cuda(), table, kv_len, q_start, window=window, n_sink=sinks, **kw)
    assert torch.equal(out, again)


def _attend(parts, bt, q, window=0, sinks=0, **kw):
    cache = _wrap(parts)
    return cache.attention(0, q.cuda(), *bt.cuda(), window=window, n_sink=sinks, return_lse=True, **kw)


@pytest.mark.parametrize("new", [1, 140])
def test_attention_rows_that_see_nothing(new):
    """Rows before position 0, sequences without a page, and windows whose pages were all given back give zeros and
    lse -inf; the other rows of the batch are not touched by them."""
    d, hq = 128, 4
    bt = ref.Batch([new, new, new], [60, 50, 40], 16, seed=1)
    parts = ref.random_cache(1, bt.n_pages, 2, 16, d, seed=2)
    q = torch.randn(bt.n, hq, d, generator=torch.Generator().manual_seed(3)).half()
    bt.table[0] = -1
    bt.kv_len[1] = new - 1          # the first token stands at -1
    out, lse = (t.cpu() for t in _attend(parts, bt, q, max_q=new))
    want, want_lse, tol, _ = ref.attention(q, parts, 0, bt, 0, 0, d ** -0.5)
    assert bool((out[:new] == 0).all()) and bool((lse[:new] == -math.inf).all())
    assert bool((out[new] == 0).all()) and bool((lse[new] == -math.inf).all())
    assert bool(((out.double() - want).abs() <= tol + 2.0 ** -11 * want.abs() + 2.0 ** -24).all())
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))


@pytest.mark.parametrize("new", [1, 150])
def test_attention_ignores_what_is_hidden(new):
    """Codes and scales of hidden tokens (past the length, behind the window, on foreign pages), NaN scales among them,
    leave every bit of the result as it is."""
    d, window, sinks = 64, 48, 3
    bt = ref.Batch([new, new], [301, 77], 32, seed=4)
    parts = ref.random_cache(1, bt.n_pages, 2, 32, d, seed=5)
    q = torch.randn(bt.n, 4, d, generator=torch.Generator().manual_seed(6)).bfloat16()
    want = _attend(parts, bt, q, window, sinks, max_q=new)
    other = ref.random_cache(1, bt.n_pages, 2, 32, d, seed=99, scale=50.0)
    for b in range(2):
        total, lo = int(bt.kv_len[b]), max(0, int(bt.kv_len[b]) - new - window + 1)
        for i in range(total):
            if i < sinks or i >= lo:
                pg, s = int(bt.table[b, i // 32]), i % 32
                for kind in (0, 1):
                    other[kind][0, pg, :, s] = parts[kind][0, pg, :, s]
                    other[2 + kind][0, pg, :, s // 16] = parts[2 + kind][0, pg, :, s // 16]
    for kind in (2, 3):
        seen = torch.zeros(bt.n_pages, 2, dtype=torch.bool)
        for b in range(2):
            total, lo = int(bt.kv_len[b]), max(0, int(bt.kv_len[b]) - new - window + 1)
            for i in range(total):
                if i < sinks or i >= lo:
                    seen[int(bt.table[b, i // 32]), i % 32 // 16] = True
        other[kind][0].masked_fill_(~seen[:, None, :], math.nan)
    got = _attend(other, bt, q, window, sinks, max_q=new)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("new", [1, 130])
def test_attention_poisoned_blocks_and_queries(new):
    """A NaN scale among the visible blocks makes exactly the rows that see the block NaN; a NaN or infinite query makes its
    own row NaN and no other."""
    d = 64
    bt = ref.Batch([new], [100], 16, seed=4)
    parts = ref.random_cache(1, bt.n_pages, 1, 16, d, seed=5)
    q = torch.randn(bt.n, 2, d, generator=torch.Generator().manual_seed(6)).bfloat16()
    clean = _attend(parts, bt, q, max_q=new)[0]
    bad_q = q.clone()
    bad_q[0, 1, 3], bad_q[-1, 0, 5] = math.nan, math.inf
    got = _attend(parts, bt, bad_q, max_q=new)[0]
    nan = got.isnan().any(-1).cpu()
    want = torch.zeros_like(nan)
    want[0, 1] = want[-1, 0] = True
    assert torch.equal(nan, want) and torch.equal(got[~want.cuda()], clean[~want.cuda()])
    last = 100 + new - 1
    for kind in (2, 3):
        p = [t.clone() for t in parts]
        p[kind][0, int(bt.table[0, last // 16]), 0, 0] = math.nan
        got = _attend(p, bt, q, max_q=new)[0].isnan().any(-1).cpu()
        sees = torch.arange(100, 100 + new) >= last - last % 16
        assert torch.equal(got, sees[:, None].expand(-1, 2))


@pytest.mark.parametrize("new", [1, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_uneven_scales(new, dtype):
    """V scales over nine decades and zero, K scales that make one key dominate, queries of very different size."""
    d = 128
    bt = ref.Batch([new], [400], 64, seed=4)
    parts = ref.random_cache(1, bt.n_pages, 2, 64, d, seed=5)
    g = torch.Generator().manual_seed(1)
    parts[3] *= torch.exp(5 * torch.randn(parts[3].shape, generator=g))
    parts[3][torch.rand(parts[3].shape, generator=g) < 0.2] = 0.0
    parts[2] *= torch.exp(torch.randn(parts[2].shape, generator=g))
    q = (torch.randn(bt.n, 4, d, generator=g) * torch.exp(2 * torch.randn(bt.n, 4, 1, generator=g))).to(dtype)
    out, lse = _attend(parts, bt, q, max_q=new)
    want, want_lse, tol, tol_lse = ref.attention(q, parts, 0, bt, 0, 0, d ** -0.5)
    assert _near(out, want, tol, dtype)
    assert bool(((lse.cpu().double() - want_lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("new", [1, 130])
def test_attention_strides_streams_and_split_invariance(new):
    """Strided and misaligned queries, another stream, an output that the caller holds: same bits as the plain call.  Hints
    on sizes change the split, so only the rounding."""
    d = 128
    bt = ref.Batch([new, 2], [3000, 9], 64, seed=4)
    parts = ref.random_cache(1, bt.n_pages, 2, 64, d, seed=5)
    cache = _wrap(parts)
    dev = bt.cuda()
    flat = torch.randn(bt.n * 700 + 8, generator=torch.Generator().manual_seed(6)).half().cuda()
    q = torch.as_strided(flat, (bt.n, 4, d), (697, 131, 1), 1)
    want = cache.attention(0, q.contiguous(), *dev)
    assert torch.equal(cache.attention(0, q, *dev), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.full_like(want, 7.0)
    with torch.cuda.stream(side):
        got = cache.attention(0, q, *dev, out=out)
    side.synchronize()
    assert got is out and torch.equal(out, want)
    for max_q, max_kv in ((1, 64), (new, 3000 + new), (4096, 1), (1, 1 << 30)):
        other = cache.attention(0, q, *dev, max_q=max_q, max_kv=max_kv)
        assert float((other.float() - want.float()).abs().max()) <= 2.0 ** -8 * float(want.float().abs().max())


@pytest.mark.parametrize("d,new", [(128, 1), (64, 1), (128, 66)])
def test_offsets_past_32_bits(d, new):
    """Pages whose codes lie beyond 2^32 bytes: append, read and attention there."""
    from vault_b200 import PagedKVCache
    page, heads = 256, 8
    n_pages = (1 << 32) // (heads * page * d) + 8
    cache = PagedKVCache(1, n_pages, heads, d, page=page)
    bt = ref.Batch([300], [0], page, seed=0)
    bt.table[0, :2] = torch.tensor([n_pages - 1, n_pages - 3], dtype=torch.int32)
    x = torch.randn(300, heads, d, generator=torch.Generator().manual_seed(6)).cuda()
    table, kv_len, q_start = bt.cuda()
    cache.append(0, x, -x, table, kv_len, q_start)
    k, v = cache.read(table, torch.zeros(1, dtype=torch.int32, device="cuda"), kv_len, q_start, 300)
    assert float((k[0] - x).abs().max()) <= 0.501 * float(x.abs().max()) / 127 and torch.equal(v, -k)
    q = torch.randn(new, heads, d, generator=torch.Generator().manual_seed(7)).half()
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    out = cache.attention(0, q.cuda(), table, kv_len, starts).double().cpu()
    p = torch.arange(300 - new, 300)
    s = torch.einsum("nhd,khd->hnk", q.double(), k[0].double().cpu()) * d ** -0.5
    s.masked_fill_(torch.arange(300)[None, None] > p[None, :, None], -math.inf)
    w = torch.softmax(s, -1)
    want, tol = torch.einsum("hnk,khd->nhd", w, v[0].double().cpu()), torch.einsum("hnk,khd->nhd", w, v[0].double().cpu().abs())
    assert bool(((out - want).abs() <= 2.0 ** -9 * tol + 2.0 ** -11 * want.abs() + 1e-6).all())


def test_empty_batches():
    bt = ref.Batch([0, 0], [5, 0], 16, seed=1)
    cache = _wrap(ref.random_cache(1, bt.n_pages, 2, 16, 64, seed=1))
    table, kv_len, q_start = bt.cuda()
    none = torch.empty(0, 2, 64, device="cuda")
    assert cache.append(0, none, none, table, kv_len, q_start) is None
    out, lse = cache.attention(0, none.half(), table, kv_len, q_start, return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    k, v = cache.read(table, kv_len, kv_len, q_start, 0)
    assert k.shape == v.shape == (1, 0, 2, 64)


# --------------------------------------------------------------------------------------------------------- reorder
@pytest.mark.parametrize("beams,groups,length,page,d", [(1, 2, 5, 16, 64), (3, 2, 37, 16, 128), (4, 1, 64, 32, 128), (8, 3, 95, 64, 64),
                                                        (16, 1, 129, 128, 128), (32, 2, 33, 16, 64), (5, 2, 0, 16, 128), (2, 1, 255, 256, 128)])
@pytest.mark.parametrize("own_pages", [True, False])
def test_reorder_follows_parents(beams, groups, length, page, d, own_pages):
    """Every row's tokens become its parent's, exactly, in every layer; full pages are shared; own_pages: each child's page is
    another child's source."""
    rows = beams * groups
    bt = ref.Batch([0] * rows, [length] * rows, page, seed=beams, spare=rows + 1, extra_cols=2)
    parts = ref.random_cache(3, bt.n_pages, 2, page, d, seed=beams)
    cache = _wrap(parts)
    g = torch.Generator().manual_seed(beams + length)
    parents = torch.randint(0, beams, (groups, beams), generator=g, dtype=torch.int32)
    used = set(bt.table.flatten().tolist())
    spare = [p for p in range(bt.n_pages) if p not in used][:rows]
    dst = None if own_pages else torch.tensor(spare, dtype=torch.int32)
    table = cache.reorder(bt.table.cuda(), bt.kv_len.cuda(), parents.cuda(), None if dst is None else dst.cuda()).cpu()
    cache.check()
    after = _parts(cache)
    full, tail = length // page, length % page
    for r in range(rows):
        parent = r - r % beams + int(parents.flatten()[r])
        want = bt.table[r].clone()
        want[:full] = bt.table[parent, :full]
        if tail and dst is not None:
            want[full] = dst[r]
        assert torch.equal(table[r], want)
        for layer in range(3):
            for h in range(2):
                for kind in (0, 1):
                    a = ref.values(after[kind][layer], after[2 + kind][layer], table[r], h, length)
                    b = ref.values(parts[kind][layer], parts[2 + kind][layer], bt.table[parent], h, length)
                    assert torch.equal(a, b)


def test_reorder_leaves_impossible_rows():
    bt = ref.Batch([0] * 4, [21] * 4, 16, seed=2, spare=5)
    parts = ref.random_cache(1, bt.n_pages, 1, 16, 64, seed=3)
    for parents, table in (([[4, -1, 2, 3]], None), ([[0, 1, 0, 2]], (2, -1))):
        cache = _wrap(parts)
        t = bt.table.clone()
        if table:
            t[table[0], 1] = table[1]      # row 2 has no page to fill, and row 3 none to copy from
        out = cache.reorder(t.cuda(), bt.kv_len.cuda(), torch.tensor(parents, dtype=torch.int32, device="cuda")).cpu()
        with pytest.raises(RuntimeError, match="status"):
            cache.check()
        assert torch.equal(out, t)
        for a, b in zip(_parts(cache), parts):
            assert torch.equal(a, b)


@pytest.mark.parametrize("batch,hkv,hq,d,page,longest,window,sinks", [(20, 16, 16, 128, 64, 2500, 0, 0), (70, 4, 16, 64, 32, 1500, 0, 0),
                                                                     (100, 4, 4, 128, 16, 900, 300, 5), (45, 8, 16, 128, 128, 700, 0, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_uneven_batches(batch, hkv, hq, d, page, longest, window, sinks, dtype):
    """Batches whose key shares follow the sequences' lengths: a few long ones among short ones, some of no token, some that
    see nothing; the same bits at every call, and a hint that is too small changes nothing but the split."""
    g = torch.Generator().manual_seed(batch)
    new = [[1, 1, 0, 3, 2, 1, 1][b % 7] for b in range(batch)]
    ctx = [int(longest * float(torch.rand(1, generator=g)) ** 6) for b in range(batch)]
    ctx[0], ctx[-1], ctx[5] = longest, longest, 0
    bt = ref.Batch(new, ctx, page, seed=batch)
    bt.table[4] = -1
    parts = ref.random_cache(1, bt.n_pages, hkv, page, d, seed=hkv)
    q = torch.randn(bt.n, hq, d, generator=g).to(dtype)
    out, lse = _attend(parts, bt, q, window, sinks, max_q=3, max_kv=longest + 3)
    want, want_lse, tol, tol_lse = ref.attention(q, parts, 0, bt, window, sinks, d ** -0.5)
    for _ in range(2):
        err = (out.cpu().double() - want).abs()
        assert bool((err <= tol + HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]).all()), float((err - tol).max())
        seen = ~torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse.cpu()), ~seen)
        assert bool(((lse.cpu().double() - want_lse).abs()[seen] <= tol_lse[seen]).all())
        again = _attend(parts, bt, q, window, sinks, max_q=3, max_kv=longest + 3)
        assert torch.equal(_attend(parts, bt, q, window, sinks, max_q=3, max_kv=longest + 3)[0], again[0])
        out, lse = _attend(parts, bt, q, window, sinks, max_q=3, max_kv=64)
