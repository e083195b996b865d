"""Plain 64-bit forms of the paged 8-bit cache operators, written from their definitions (include/vault_b200.h), and the
batches the tests share.  Everything here is torch on the CPU, one sequence and one head at a time."""
import math
import random

import torch

BLOCK = 16


class Batch:
    """Sequences with `new` tokens on top of `ctx` cached ones, their pages scattered over a cache with spare pages.
    page_table, kv_len, q_start as the operators take them."""

    def __init__(self, new, ctx, page, seed, spare=3, extra_cols=1):
        rng = random.Random(seed)
        self.new, self.ctx, self.page = list(new), list(ctx), page
        need = [-(-(n + c) // page) for n, c in zip(new, ctx)]
        self.n_pages = sum(need) + spare
        ids = list(range(self.n_pages))
        rng.shuffle(ids)
        cols = max(need + [1]) + extra_cols
        self.table = torch.full((len(new), cols), -1, dtype=torch.int32)
        for b, m in enumerate(need):
            for i in range(m):
                self.table[b, i] = ids.pop()
        self.kv_len = torch.tensor([n + c for n, c in zip(new, ctx)], dtype=torch.int32)
        self.q_start = torch.tensor([sum(self.new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
        self.n = sum(self.new)

    def cuda(self):
        return self.table.cuda(), self.kv_len.cuda(), self.q_start.cuda()


def random_cache(layers, n_pages, heads, page, d, seed, scale=0.03):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, n_pages, heads, page)
    codes = [torch.randint(1, 256, (*shape, d), generator=g, dtype=torch.uint8) for _ in range(2)]
    scales = [scale * torch.exp(0.5 * torch.randn(*shape[:3], page // BLOCK, generator=g)) for _ in range(2)]
    return [*codes, *scales]


def values(codes, scales, table_row, head, n):
    """Tokens 0 .. n - 1 of one sequence and head as 64-bit values [n, d]; rows without a page are NaN."""
    page, d = codes.shape[2], codes.shape[3]
    out = torch.full((n, d), math.nan, dtype=torch.float64)
    for i in range(0, n, page):
        col = i // page
        pg = int(table_row[col]) if col < table_row.numel() else -1
        if 0 <= pg < codes.shape[0]:
            v = (codes[pg, head].double() - 128) * scales[pg, head].double().repeat_interleave(BLOCK)[:, None]
            out[i:i + page] = v[:n - i]
    return out


def rotate(x, pos, theta_table):
    """x [tokens, heads, d] at positions pos, in 64 bits, with the table's own cosines and sines."""
    cs = theta_table.double()[pos]
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(cs[:, :half], cs[:, half:])[:, None]
    return torch.cat([z.real, z.imag], -1)


def visible(p, n_keys, window, n_sink):
    j = torch.arange(n_keys)
    see = j <= p
    if window:
        see &= (j > p - window) | (j < n_sink)
    return see


def attention(q, cache, layer, batch, window, n_sink, scale):
    """64-bit out [tokens, heads, d], lse [tokens, heads], and the element-wise bound on what the kernels may be off.

    The kernels hold scores, sums and accumulators in fp32 and round each probability (times its V scale) to fp16, 11
    bits or an absolute 2^-25 of the largest V scale below fp16's normal range; scores are sums of d products accumulated
    in fp32 (bounded by 2^-19 of the sum of their magnitudes)."""
    k8, v8, ks, vs = (t[layer] for t in cache)
    n, heads, d = q.shape
    group = heads // k8.shape[1]
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.full((n, heads), 2.0 ** -16, dtype=torch.float64)
    for b in range(len(batch.new)):
        total = int(batch.kv_len[b])
        for h in range(heads):
            kk, vv = (values(c, s, batch.table[b], h // group, max(total, 0)) for c, s in ((k8, ks), (v8, vs)))
            held = ~torch.isnan(kk).any(1)
            kk, vv = kk.nan_to_num(0.0), vv.nan_to_num(0.0)
            big_vs = float(vv.abs().max()) / 1.0 if vv.numel() else 0.0
            for i in range(batch.new[b]):
                p = total - batch.new[b] + i
                r = int(batch.q_start[b]) + i
                see = visible(p, max(total, 0), window, n_sink) & held
                if not bool(see.any()):
                    continue
                qq = q[r, h].double()
                s = (kk[see] @ qq) * scale
                mag = float(((kk[see].abs() @ qq.abs()) * abs(scale)).max())
                m = s.max()
                w = torch.exp(s - m)
                l = w.sum()
                out[r, h] = (w @ vv[see]) / l
                lse[r, h] = m + torch.log(l)
                ds = 2.0 ** -19 * mag
                mean_abs = (w @ vv[see].abs()) / l
                tol[r, h] = (2.0 ** -10 + 4 * ds) * mean_abs + int(see.sum()) * 2.0 ** -23 * big_vs / l
                tol_lse[r, h] += 2 * ds + 2.0 ** -20 * abs(float(lse[r, h]))
    return out, lse, tol, tol_lse
