"""GPU: attention over blocks whose V scales are far apart.  A row's result is held to what the row itself sees: the largest
term p vs among its own visible keys bounds what rounding may cost it, whatever stands in blocks that other rows see."""
import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def _exact(q, parts, bt, window, sinks):
    """64-bit out [tokens, heads, d] and the bound on each element, of batches of one sequence.

    A probability times its V scale enters the product as fp16 with an offset of the row's own: 2^-11 of itself, and below
    fp16's normal range 2^-25 of a unit that is at most 8 times the row's largest p vs; codes reach 127.  Scores are sums of d
    products in fp32 (2^-19 of the sum of their magnitudes); fp32 sums and the powers cost less than another 2^-11 in all.
    Values below 2^-115 are too near fp32's own smallest normal number to be held to their own size."""
    k8, v8, ks, vs = (t[0] for t in parts)
    n, heads, d = q.shape
    total, group = int(bt.kv_len[0]), heads // k8.shape[1]
    out = torch.full((n, heads, d), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for h in range(heads):
        kk, vv = (ref.values(c, s, bt.table[0], h // group, total) for c, s in ((k8, ks), (v8, vs)))
        scale = torch.stack([vs[int(bt.table[0, j // bt.page]), h // group, j % bt.page // 16] for j in range(total)]).double()
        for i in range(n):
            see = ref.visible(total - n + i, total, window, sinks)
            s = (kk[see] @ q[i, h].double()) * d ** -0.5
            ds = 2.0 ** -19 * float((kk[see].abs() @ q[i, h].double().abs()).max()) * d ** -0.5
            w = torch.softmax(s, 0)
            out[i, h] = w @ vv[see]
            unit = 127 * float((w * scale[see]).max())
            tol[i, h] = (2.0 ** -10 + 4 * ds) * (w @ vv[see].abs()) + int(see.sum()) * 2.0 ** -22 * unit + 2.0 ** -115
    return out, tol


def _attend(parts, bt, q, window, sinks):
    from vault_b200 import PagedKVCache
    cache = PagedKVCache.wrap(*(t.cuda() for t in parts))
    out, lse = cache.attention(0, q.cuda(), *bt.cuda(), window=window, n_sink=sinks, return_lse=True, max_q=q.shape[0])
    return out.cpu().double(), lse.cpu()


def _near(out, want, tol, dtype):
    past = want.abs() > torch.finfo(dtype).max * (1 + HALF_ULP[dtype] / 2)
    near = (out - want).abs() <= tol + HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]
    return bool(torch.where(past, out == math.inf * want.sign(), near).all())


def _block(bt, j):
    return int(bt.table[0, j // bt.page]), j % bt.page // 16


# tokens in one sequence: few rows (a tile of 8, of 16, several), many rows (one CTA, two), all with a window that the first
# rows' early blocks leave
SHAPES = [(12, 1, 92), (3, 8, 88), (40, 1, 64), (250, 1, 64), (140, 4, 90)]


@pytest.mark.parametrize("new,group,window", SHAPES)
@pytest.mark.parametrize("power", [12, 14, 20, 26, 60])
@pytest.mark.parametrize("sinks", [0, 2])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_large_block_that_only_earlier_rows_see(new, group, window, power, sinks, dtype):
    d, ctx = 64, 150
    bt = ref.Batch([new], [ctx], 32, seed=new)
    parts = ref.random_cache(1, bt.n_pages, 1, 32, d, seed=new + 1, scale=0.01)
    pg, blk = _block(bt, ctx - window + 1)      # behind the window of the rows from a few tokens on
    parts[3][0, pg, :, blk] *= 2.0 ** power
    q = (1.5 * torch.randn(new, group, d, generator=torch.Generator().manual_seed(3))).to(dtype)
    want, tol = _exact(q, parts, bt, window, sinks)
    out, _ = _attend(parts, bt, q, window, sinks)
    assert _near(out, want, tol, dtype)


@pytest.mark.parametrize("new,group,window", SHAPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_poisoned_block_that_only_earlier_rows_see(new, group, window, bad):
    """Rows that do not see it are, to the bit, what they are without it."""
    d, ctx = 64, 150
    bt = ref.Batch([new], [ctx], 32, seed=new)
    parts = ref.random_cache(1, bt.n_pages, 1, 32, d, seed=new + 1, scale=0.01)
    q = torch.randn(new, group, d, generator=torch.Generator().manual_seed(3)).bfloat16()
    clean, _ = _attend(parts, bt, q, window, 0)
    at = ctx - window + 1
    pg, blk = _block(bt, at)
    parts[3][0, pg, :, blk] = bad
    out, _ = _attend(parts, bt, q, window, 0)
    sees = torch.arange(ctx, ctx + new) - window < at - at % 16 + 15
    assert bool(sees.any()) and not bool(sees.all())
    assert torch.equal(out[~sees], clean[~sees]) and not bool(out[sees].isfinite().any())


@pytest.mark.parametrize("new,group", [(1, 2), (5, 2), (40, 1), (150, 2)])
@pytest.mark.parametrize("power", [14, 24, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_large_block_without_weight(new, group, power, dtype):
    """Every row sees the block, and its probabilities are far below the others': what it costs the others is bounded by its
    terms, not by its scale."""
    d, ctx = 128, 200
    bt = ref.Batch([new], [ctx], 64, seed=new)
    parts = ref.random_cache(1, bt.n_pages, 1, 64, d, seed=7, scale=0.004)
    pg, blk = _block(bt, 40)
    parts[3][0, pg, :, blk] *= 2.0 ** power
    parts[0][0, pg, :, 16 * blk:16 * blk + 16] = 1   # codes of -127 in every dim, queries of positive sum: scores near -60
    parts[2][0, pg, :, blk] = 0.06
    q = (0.7 + 0.05 * torch.randn(new, group, d, generator=torch.Generator().manual_seed(3))).to(dtype)
    want, tol = _exact(q, parts, bt, 0, 0)
    out, _ = _attend(parts, bt, q, 0, 0)
    assert _near(out, want, tol, dtype)


@pytest.mark.parametrize("new", [1, 6, 130])
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e20, 1e30])
def test_all_scales_small_or_large(new, size):
    d = 64
    bt = ref.Batch([new], [80], 16, seed=new)
    parts = ref.random_cache(1, bt.n_pages, 1, 16, d, seed=9, scale=1.0)
    parts[2] *= 0.02
    parts[3] *= size
    q = torch.randn(new, 2, d, generator=torch.Generator().manual_seed(3)).bfloat16()
    want, tol = _exact(q, parts, bt, 0, 0)
    out, lse = _attend(parts, bt, q, 0, 0)
    assert _near(out, want, tol, torch.bfloat16)
    parts[3] /= size
    assert float((lse - _attend(parts, bt, q, 0, 0)[1]).abs().max()) <= 2.0 ** -16


@pytest.mark.parametrize("new", [1, 6, 130])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_zero_scales_that_take_the_weight(new, dtype):
    """Blocks of V scale zero, whatever their codes, with nearly all of the probability: the others come out small, not
    lost; a row that sees nothing else is zero; lse counts every key."""
    d, ctx = 64, 160
    bt = ref.Batch([new], [ctx], 16, seed=new)
    parts = ref.random_cache(1, bt.n_pages, 1, 16, d, seed=9, scale=0.02)
    for j in (0, 48):
        pg, blk = _block(bt, j)
        parts[3][0, pg, :, blk] = 0.0
        parts[0][0, pg, :, 16 * blk:16 * blk + 16] = 255
        parts[2][0, pg, :, blk] = 0.012
    q = (0.8 + 0.1 * torch.randn(new, 2, d, generator=torch.Generator().manual_seed(3))).to(dtype)
    want, tol = _exact(q, parts, bt, 0, 0)
    out, lse = _attend(parts, bt, q, 0, 0)
    assert _near(out, want, tol, dtype)
    _, want_lse, _, tol_lse = ref.attention(q, parts, 0, bt, 0, 0, d ** -0.5)
    assert bool(((lse.double() - want_lse).abs() <= tol_lse).all())
    parts[3].zero_()
    out, lse = _attend(parts, bt, q, 0, 0)
    assert bool((out == 0).all()) and bool(((lse.double() - want_lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("new", [1, 40, 140])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_do_not_reach_lse(new, bad, dtype):
    """V scales that are no number: the rows that see them have no output, and the lse they have without them."""
    d = 64
    bt = ref.Batch([new], [100], 16, seed=new)
    parts = ref.random_cache(1, bt.n_pages, 1, 16, d, seed=3, scale=0.02)
    q = torch.randn(new, 2, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    _, want, _, tol = ref.attention(q, parts, 0, bt, 0, 0, d ** -0.5)
    for j in (20, 100 + new - 1):
        pg, blk = _block(bt, j)
        parts[3][0, pg, :, blk] = bad
        out, lse = _attend(parts, bt, q, 0, 0)
        sees = torch.arange(100, 100 + new) >= j - j % 16
        assert bool(((lse.double() - want).abs() <= tol).all()) and not bool(out[sees].isfinite().any())
