"""The paged 8-bit KV cache operators and beam selection as measured cases: inputs, plain torch forms, exact values.

A cache block is 16 consecutive tokens of one KV head; its codes are bytes biased by 128 and share one fp32 scale.
Layout: codes [layers, pages, kv heads, page, head dim], scales [layers, pages, kv heads, page / 16]."""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
TINY = 2.0 ** -120   # scales below this are stored as zero
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EOS = 2


def listed():
    return [
        # one decode step of 16 conversations: one token each, rotated and appended, fp32 projections
        dict(name="append_step", op="append", batch=16, new=1, ctx=4608, hq=12, hkv=2, d=128, page=64, dtype="f32", ragged=True),
        # prompts of uneven length arriving together at an empty cache
        dict(name="append_prompts", op="append", batch=5, new=6000, ctx=0, hq=32, hkv=8, d=128, page=64, dtype="bf16", ragged=True),
        # a single conversation's decode step over a short context: latency
        dict(name="attend_one", op="attend", batch=1, new=1, ctx=1544, hq=12, hkv=2, d=128, page=64, dtype="bf16", ragged=False, window=0, sinks=0),
        # the batched decode step of 64 conversations, uneven contexts
        dict(name="attend_batch", op="attend", batch=64, new=1, ctx=4608, hq=12, hkv=2, d=128, page=64, dtype="bf16", ragged=True, window=0, sinks=0),
        # decode over 100,000-token documents
        dict(name="attend_long", op="attend", batch=4, new=1, ctx=100000, hq=32, hkv=8, d=128, page=64, dtype="f16", ragged=False, window=0, sinks=0),
        # a prompt of 4,608 tokens under a window of 1,024 with four sinks
        dict(name="attend_window_prompt", op="attend", batch=1, new=4608, ctx=0, hq=12, hkv=2, d=128, page=64, dtype="bf16", ragged=False, window=1024, sinks=4),
        # uneven chunks of prompts and single tokens in one batch, on top of cached contexts; as many KV heads as query heads
        dict(name="attend_chunks", op="attend", batch=6, new=700, ctx=6000, hq=16, hkv=16, d=64, page=32, dtype="f16", ragged=True, window=2048, sinks=4),
        # a long prompt, every earlier token visible
        dict(name="attend_prompt", op="attend", batch=1, new=8192, ctx=0, hq=32, hkv=8, d=128, page=64, dtype="bf16", ragged=False, window=0, sinks=0),
        # beam search of one request
        dict(name="beam_one", op="beam", batch=1, beams=4, vocab=151936, dtype="f32", done=False),
        # beam search of 48 requests, some beams finished
        dict(name="beam_batch", op="beam", batch=48, beams=8, vocab=151936, dtype="f32", done=True),
        # the cache of one request follows its four beams
        dict(name="reorder_one", op="reorder", batch=1, beams=4, layers=28, ctx=1543, hkv=2, d=128, page=64),
        # the caches of 24 requests follow their eight beams
        dict(name="reorder_batch", op="reorder", batch=24, beams=8, layers=28, ctx=2047, hkv=2, d=128, page=64),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "beam", "reorder"])
    heads = rng.choice([(12, 2), (32, 8), (16, 16), (8, 1), (4, 2), (28, 4)])
    c = dict(op=op, page=rng.choice([16, 32, 64, 128]), d=rng.choice([64, 128, 128]))
    if op == "beam":
        c = dict(op=op, beams=rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), vocab=_spread(rng, 300, 152000), dtype=rng.choice(["f32", "f32", "f16", "bf16"]),
                 done=rng.random() < 0.5)
        c["batch"] = min(_spread(rng, 1, 48), max(1, 48 * 8 * 151936 // (c["beams"] * c["vocab"])))
        return c
    if op == "reorder":
        c.update(batch=_spread(rng, 1, 24), beams=rng.choice([1, 2, 4, 5, 8]), layers=_spread(rng, 1, 28), ctx=_spread(rng, 1, 2047), hkv=rng.choice([1, 2, 3]))
        return c
    c.update(hq=heads[0], hkv=heads[1], ragged=rng.random() < 0.7)
    if op == "append":
        c.update(dtype=rng.choice(["f32", "f16", "bf16"]), batch=_spread(rng, 1, 64), ctx=rng.choice([0, _spread(rng, 1, 4608)]))
        c["new"] = min(rng.choice([1, _spread(rng, 2, 6000)]), max(1, 5 * 6000 * 8 * 128 // (c["batch"] * c["hkv"] * c["d"])))
        return c
    c.update(dtype=rng.choice(["f16", "bf16"]), window=rng.choice([0, 0, _spread(rng, 16, 4096)]), sinks=rng.choice([0, 1, 4, 40]))
    if rng.random() < 0.5:   # single tokens
        c.update(new=1, batch=_spread(rng, 1, 64))
        c["ctx"] = min(_spread(rng, 1, 100000), max(1, 4 * 100000 * 8 * 128 // (c["batch"] * c["hkv"] * c["d"])))
    else:
        c.update(new=_spread(rng, 2, 6000), batch=_spread(rng, 1, 8), ctx=rng.choice([0, _spread(rng, 1, 8000)]))
        while c["batch"] * c["hq"] * c["new"] * (c["new"] + c["ctx"]) > 32 * 8192 * 8192:
            c.update(new=max(1, c["new"] * 3 // 4), ctx=c["ctx"] * 3 // 4)
    return c


# ------------------------------------------------------------------------------------------------------- lengths
def _lengths(case):
    """New tokens and cached tokens of each sequence: the case's own, uneven where it is ragged."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    b, new, ctx = case["batch"], case["new"], case["ctx"]
    if not case["ragged"]:
        return [new] * b, [ctx] * b
    n = [new if new == 1 else max(1, int(new * rng.uniform(0.0, 1.0) ** 2)) for _ in range(b)]
    if new > 1:
        n[rng.randrange(b)] = new
        if b > 2:
            n[rng.randrange(b)] = 1
    c = [int(ctx * rng.uniform(0.3, 1.0)) for _ in range(b)]
    c[rng.randrange(b)] = ctx
    return n, c


def _visible(case, n, ctx):
    """Of one sequence: (query, key) pairs, and keys that any of its queries sees."""
    w, sinks, total = case["window"], case["sinks"], n + ctx
    if w == 0:
        return sum(range(ctx + 1, total + 1)), total
    first = ctx - w + 1                                    # oldest window key of the first query
    keys = total if first <= sinks else sinks + total - first
    pairs = 0
    for p in range(ctx, total):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(sinks, lo)
    return pairs, keys


def work(case):
    if case["op"] == "beam":
        e = 4 if case["dtype"] == "f32" else 2
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * e + case["batch"] * case["beams"] * 18, "flops": 4 * n}
    if case["op"] == "reorder":
        rows = case["batch"] * case["beams"]
        tail = case["ctx"] % case["page"]
        held = rows * case["layers"] * case["hkv"] * 2 * (tail * case["d"] + 4 * -(-tail // BLOCK))
        values = rows * tail * case["layers"] * case["hkv"] * case["d"] * 2 * 2
        return {"bytes": 3 * held + values + rows * 8 * -(-case["ctx"] // case["page"]), "flops": 0}
    n, ctx = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        e = 4 if case["dtype"] == "f32" else 2
        tokens = sum(n)
        rows = sum(x + y % BLOCK for x, y in zip(n, ctx))
        held = 2 * rows * hkv * d * (1 + 4 / (BLOCK * d))
        return {"bytes": tokens * (2 * hq + 2 * hkv) * d * e + 2 * held + 2 * rows * hkv * d * 2 + tokens * d * 4,
                "flops": tokens * (hq + hkv) * d * 3 + 2 * tokens * hkv * d * 3}
    pairs = keys = 0
    for x, y in zip(n, ctx):
        p, k = _visible(case, x, y)
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * keys * hkv * (d + 4 / BLOCK) + 2 * sum(n) * hq * d * 2 + 4 * sum(-(-(x + y) // case["page"]) for x, y in zip(n, ctx)),
            "flops": 4 * pairs * hq * d}


# -------------------------------------------------------------------------------------------------------- inputs
def _codes(shape, gen):
    """Codes as normal values leave them, the largest of a block near 127."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=gen).mul_(36.0).round_().clamp_(-127, 127).add_(128))
    return out


def _scales(shape, gen):
    return torch.exp(0.3 * torch.randn(shape, device="cuda", generator=gen)) * (3.5 / 127)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    s = {"case": case}
    if case["op"] == "beam":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        s["logits"] = (3.0 * randn(b, k, v)).to(DTYPES[case["dtype"]])
        s["scores"] = (-4.0 + 1.5 * randn(b, k)).sort(dim=1, descending=True).values
        done = torch.zeros(b, k, dtype=torch.uint8)
        if case["done"]:
            for i in range(b):
                for j in range(1, k):
                    done[i, j] = rng.random() < 0.25
        s["finished"] = done.cuda()
        return s
    page, hkv, d = case["page"], case["hkv"], case["d"]
    if case["op"] == "reorder":
        rows, full = case["batch"] * case["beams"], case["ctx"] // case["page"]
        width = full + 2
        pages = rows * 2 + case["batch"] * full            # the requests' shared pages, and two current pages for each beam
        perm = torch.randperm(pages, device="cuda", generator=gen).int()
        table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        shared = perm[2 * rows:].view(case["batch"], full)
        table[:, :full] = shared.repeat_interleave(case["beams"], 0)
        table[:, full] = perm[:rows]
        s["dst"] = perm[rows:2 * rows].contiguous()
        s["kv_len"] = torch.full((rows,), case["ctx"], dtype=torch.int32, device="cuda")
        parents = [sorted(rng.choice(range(case["beams"])) for _ in range(case["beams"])) for _ in range(case["batch"])]
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
        tail = case["ctx"] % page
        s["first"] = torch.full((rows,), case["ctx"] - tail, dtype=torch.int32, device="cuda")
        s["row_start"] = torch.arange(rows + 1, dtype=torch.int32, device="cuda") * tail
        s["rows"] = rows * tail
        layers = case["layers"]
    else:
        n, ctx = _lengths(case)
        dt = DTYPES[case["dtype"]]
        width = max(-(-(x + y) // page) for x, y in zip(n, ctx)) + 1
        used = sum(-(-(x + y) // page) for x, y in zip(n, ctx))
        pages = used + 3
        perm = torch.randperm(pages, device="cuda", generator=gen).int().cpu()
        table = torch.full((case["batch"], width), -1, dtype=torch.int32)
        at = 0
        for b, (x, y) in enumerate(zip(n, ctx)):
            m = -(-(x + y) // page)
            table[b, :m] = perm[at:at + m]
            at += m
            if case["op"] == "attend" and case["window"]:   # pages that no query sees any more are given back
                lo, hi = -(-case["sinks"] // page), max(0, y - case["window"] + 1) // page
                if hi > lo:
                    table[b, lo:hi] = -1
        table = table.cuda()
        s["kv_len"] = torch.tensor([x + y for x, y in zip(n, ctx)], dtype=torch.int32, device="cuda")
        s["q_start"] = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device="cuda")
        s["max_q"], s["max_kv"] = max(n), max(x + y for x, y in zip(n, ctx))
        layers, tokens = 1, sum(n)
        if case["op"] == "append":
            # one projection's output holds q, k and v of a token side by side
            s["qkv"] = randn(tokens, case["hq"] + 2 * hkv, d).to(dt)
            s["qkv"][:, case["hq"]:case["hq"] + hkv] *= (1 + 3 * torch.rand(1, hkv, d, device="cuda", generator=gen)).to(dt)
            angle = torch.arange(s["max_kv"], dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)[None]
            s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
            first = [y - y % BLOCK for y in ctx]
            s["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
            rows = [x + y - f for x, y, f in zip(n, ctx, first)]
            s["row_start"] = torch.tensor(np.cumsum([0] + rows), dtype=torch.int32, device="cuda")
            s["rows"] = sum(rows)
        else:
            s["q"] = (2.0 * randn(tokens, case["hq"], d)).to(dt)
    s["table"] = table
    s["k"], s["v"] = (_codes((layers, pages, hkv, page, d), gen) for _ in range(2))
    s["ks"], s["vs"] = (_scales((layers, pages, hkv, page // BLOCK), gen) for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] != "beam":
        import vault_b200
        s["cache"] = vault_b200.PagedKVCache.wrap(s["k"], s["v"], s["ks"], s["vs"])
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, cs):
    half = x.shape[-1] // 2
    c, sn = cs[:, None, :half], cs[:, None, half:]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _token_places(s, page):
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n)
    i = torch.arange(seq.numel(), device="cuda") - s["q_start"].long()[seq]
    pos = s["kv_len"].long()[seq] - n[seq] + i
    return seq, i, pos, s["table"].long()[seq, pos // page]


def _plain_store(x, codes, scales, pages, pos, lead, page):
    """Rounds the rows x [tokens, heads, d] into their blocks; lead: tokens that come first in their block."""
    blk = pos % page // BLOCK
    block_of = torch.cumsum(lead.long(), 0) - 1
    lp, lb, lslot = pages[lead], blk[lead], pos[lead] % BLOCK
    biggest = torch.zeros(lp.numel(), x.shape[1], device="cuda")
    biggest.index_reduce_(0, block_of, x.abs().amax(-1), "amax")
    old = torch.where(lslot[:, None] > 0, scales[lp, :, lb], 0.0)
    new = torch.maximum(old, biggest / 127)
    new = torch.where(new < TINY, 0.0, new)
    inv = torch.where(new > 0, 1 / new, 0.0)
    rows = lb[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    held = codes[lp[:, None], :, rows].float() - 128                      # [blocks, 16, heads, d]
    ratio = torch.where(new > 0, old / new, 0.0)
    moved = torch.round(held * ratio[:, None, :, None]) + 128
    keep = torch.arange(BLOCK, device="cuda")[None] < lslot[:, None]
    codes[lp[:, None], :, rows] = torch.where(keep[..., None, None], moved, held + 128).to(torch.uint8)
    scales[lp, :, lb] = new
    codes[pages, :, pos % page] = (torch.round(x * inv[block_of][..., None]).clamp(-127, 127) + 128).to(torch.uint8)


def _plain_read(s, dtype):
    """Values of the tokens from `first` on, of every layer."""
    page = s["case"]["page"]
    n = (s["row_start"][1:] - s["row_start"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=s["rows"])
    pos = s["first"].long()[seq] + torch.arange(s["rows"], device="cuda") - s["row_start"].long()[seq]
    pages, slot = s["out_table"].long()[seq, pos // page], pos % page
    return [((codes[:, pages, :, slot].float() - 128) * scales[:, pages, :, slot // BLOCK][..., None]).to(dtype).transpose(0, 1)
            for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"]))]


def _plain_append(s):
    case = s["case"]
    hq, hkv, page, dt = case["hq"], case["hkv"], case["page"], DTYPES[case["dtype"]]
    seq, i, pos, pages = _token_places(s, page)
    x = s["qkv"].float()
    cs = s["rope"][pos]
    lead = (i == 0) | (pos % BLOCK == 0)
    _plain_store(_rotate(x[:, hq:hq + hkv], cs), s["k"][0], s["ks"][0], pages, pos, lead, page)
    _plain_store(x[:, hq + hkv:], s["v"][0], s["vs"][0], pages, pos, lead, page)
    s["out_table"] = s["table"]
    k, v = _plain_read(s, torch.bfloat16)
    return {"q": _rotate(x[:, :hq], cs).to(dt), "k": k, "v": v}


def _plain_attend(s):
    case = s["case"]
    page, hq, hkv, d, w = case["page"], case["hq"], case["hkv"], case["d"], case["window"]
    g, batch, maxq = hq // hkv, case["batch"], s["max_q"]
    used = -(-s["max_kv"] // page)
    table = s["table"][:, :used].long()
    k, v = [((c[0][table.clamp(min=0)].view(batch, used, hkv, page // BLOCK, BLOCK, d).float() - 128) * sc[0][table.clamp(min=0)][..., None, None])
            .permute(0, 2, 1, 3, 4, 5).reshape(batch, hkv, used * page, d) for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"]))]
    seq, i, pos, _ = _token_places(s, page)
    q = torch.zeros(batch, maxq, hq, d, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(batch, maxq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, g * maxq, d)
    x = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(d)).view(batch, hkv, g, maxq, used * page)
    j = torch.arange(used * page, device="cuda")
    at = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1]))[:, None] + torch.arange(maxq, device="cuda")
    see = (j <= at[..., None]) & (j < s["kv_len"][:, None, None]) & (table >= 0).repeat_interleave(page, 1)[:, None]
    if w:
        see &= (j > at[..., None] - w) | (j < case["sinks"])
    x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(batch, hkv, g * maxq, -1) @ v).view(batch, hkv, g, maxq, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, maxq, hq, d)[seq, i].to(s["q"].dtype)


def _plain_beam(s):
    x, b, k, v = s["logits"].float(), s["case"]["batch"], s["case"]["beams"], s["case"]["vocab"]
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    cand = (x - lse) + s["scores"][..., None] + 0.0
    done = s["finished"].bool()
    cand = torch.where(done[..., None], -math.inf, cand)
    cand[..., EOS] = torch.where(done, s["scores"], cand[..., EOS])
    bits = cand.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).view(b, k * v).long() * (1 << 32) + ((1 << 32) - 1 - torch.arange(k * v, device="cuda"))
    best = (1 << 32) - 1 - (key.topk(k, dim=1).values & 0xFFFFFFFF)       # keys are distinct: the lower index wins a tie
    parents, tokens = best // v, best % v
    return {"tokens": tokens.int(), "parents": parents.int(), "scores": cand.view(b, k * v).gather(1, best),
            "finished": (done.gather(1, parents) | (tokens == EOS)).to(torch.uint8)}


def _plain_reorder(s):
    case = s["case"]
    rows, page = case["batch"] * case["beams"], case["page"]
    full, tail = case["ctx"] // page, case["ctx"] % page
    parent = (s["parents"].long() + torch.arange(case["batch"], device="cuda")[:, None] * case["beams"]).view(rows)
    out = s["table"].clone()
    out[:, :full] = s["table"][parent, :full]
    if tail:
        src, dst, blocks = s["table"][parent, full].long(), s["dst"].long(), -(-tail // BLOCK)
        out[:, full] = s["dst"]
        for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            codes[:, dst, :, :tail] = codes[:, src, :, :tail]
            scales[:, dst, :, :blocks] = scales[:, src, :, :blocks]
    s["out_table"] = out
    k, v = _plain_read(s, torch.bfloat16)
    return {"table": out, "k": k, "v": v}


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "beam": _plain_beam, "reorder": _plain_reorder}[op](s)
    import vault_b200
    if op == "beam":
        tokens, parents, scores, finished = vault_b200.beam_select(s["logits"], s["scores"], s["finished"], eos_id=EOS)
        return {"tokens": tokens, "parents": parents, "scores": scores, "finished": finished}
    cache = s["cache"]
    if op == "append":
        hq, hkv = case["hq"], case["hkv"]
        x = s["qkv"]
        q = cache.append(0, x[:, hq:hq + hkv], x[:, hq + hkv:], s["table"], s["kv_len"], s["q_start"], rope=s["rope"], q=x[:, :hq])
        k, v = cache.read(s["table"], s["first"], s["kv_len"], s["row_start"], s["rows"], torch.bfloat16)
        return {"q": q, "k": k, "v": v}
    if op == "attend":
        return cache.attention(0, s["q"], s["table"], s["kv_len"], s["q_start"], window=case["window"], n_sink=case["sinks"],
                               max_q=s["max_q"], max_kv=s["max_kv"])
    table = cache.reorder(s["table"], s["kv_len"], s["parents"], dst_page=s["dst"])
    k, v = cache.read(table, s["first"], s["kv_len"], s["row_start"], s["rows"], torch.bfloat16)
    return {"table": table, "k": k, "v": v}


# --------------------------------------------------------------------------------------------------- exact values
def _exact_block(old, held, rows):
    """One block of one head in 64 bits: earlier values' codes and scale, then the new rows -> codes, scale."""
    s0 = old if held.shape[0] else 0.0
    s1 = max(s0, float(rows.abs().max()) / 127)
    if s1 < TINY:
        return torch.zeros(held.shape[0] + rows.shape[0], rows.shape[1], dtype=torch.float64), 0.0
    return torch.cat([torch.round(held * (s0 / s1)), torch.round(rows / s1).clamp(-127, 127)]), s1


def _exact_append(s):
    case = s["case"]
    hq, hkv, page, d = case["hq"], case["hkv"], case["page"], case["d"]
    n, ctx = _lengths(case)
    if sum(n) * hkv > 400000:   # 20 seconds or so of single blocks
        return None
    x, half = s["qkv"].double().cpu(), d // 2
    table, rope = s["table"].cpu(), s["rope"].double().cpu()
    turn = torch.complex(rope[:, :half], rope[:, half:])
    q, k, v, at = [], [], [], 0
    for b in range(len(n)):
        rows = x[at:at + n[b]]
        at += n[b]
        z = torch.complex(rows[..., :half], rows[..., half:]) * turn[ctx[b]:ctx[b] + n[b], None]
        rows = torch.cat([torch.cat([z.real, z.imag], -1)[:, :hq + hkv], rows[:, hq + hkv:]], 1)
        q.append(rows[:, :hq])
        for codes, scales, first, out in ((s["k"], s["ks"], hq, k), (s["v"], s["vs"], hq + hkv, v)):
            p = ctx[b]
            while p < ctx[b] + n[b]:
                lo, hi = p - p % BLOCK, min(p - p % BLOCK + BLOCK, ctx[b] + n[b])
                pg, slot = int(table[b, lo // page]), lo % page
                held = codes[0, pg, :, slot:slot + p - lo].double().cpu() - 128
                old = scales[0, pg, :, slot // BLOCK].double().cpu()
                heads = []
                for h in range(hkv):
                    c, sc = _exact_block(float(old[h]), held[h], rows[p - ctx[b]:hi - ctx[b], first + h])
                    heads.append(c * sc)
                out.append(torch.stack(heads, 1))
                p = hi
    return {"q": torch.cat(q), "k": torch.cat(k)[None], "v": torch.cat(v)[None]}


def _exact_attend(s):
    case = s["case"]
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    n, ctx = _lengths(case)
    outs, at = [], 0
    for b in range(len(n)):
        total = n[b] + ctx[b]
        t = s["table"][b, :-(-total // page)].long()
        p = torch.arange(ctx[b], total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")[None]
        hidden = (j > p) | (t < 0).repeat_interleave(page)[:total]
        if case["window"]:
            hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
        out = torch.empty(n[b], hq, d, dtype=torch.float64, device="cuda")
        for h in range(hq):
            kv = []
            for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
                val = codes[0][t.clamp(min=0), h // (hq // hkv)].double().sub_(128).view(-1, BLOCK, d)
                kv.append((val * scales[0][t.clamp(min=0), h // (hq // hkv)].double().view(-1, 1, 1)).view(-1, d)[:total])
            x = (s["q"][at:at + n[b], h].double() @ kv[0].T) * d ** -0.5
            out[:, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ kv[1]
            del x, kv
        outs.append(out)
        at += n[b]
    return torch.cat(outs)


def _exact_beam(s):
    b, k, v = s["case"]["batch"], s["case"]["beams"], s["case"]["vocab"]
    cand = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    for i, j in s["finished"].nonzero().tolist():
        cand[i, j] = -math.inf
        cand[i, j, EOS] = s["scores"][i, j].double()
    return {"tokens": None, "parents": None, "scores": cand.view(b, k * v).topk(k, 1).values, "finished": None}


def _exact_reorder(s):
    case = s["case"]
    page, beams = case["page"], case["beams"]
    full, tail = case["ctx"] // page, case["ctx"] % page
    parents, table = s["parents"].view(-1).tolist(), s["table"][:, full].tolist()
    if not tail:
        return None
    out = {"table": None}
    for name, codes, scales in (("k", s["k"], s["ks"]), ("v", s["v"], s["vs"])):
        rows = []
        for r, p in enumerate(parents):
            pg = table[r - r % beams + p]
            val = codes[:, pg, :, :tail].double() - 128                    # [layers, heads, tail, d]
            rows.append((val * scales[:, pg].double().repeat_interleave(BLOCK, -1)[:, :, :tail, None]).permute(0, 2, 1, 3))
        out[name] = torch.cat(rows, 1)
    return out


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "beam": _exact_beam, "reorder": _exact_reorder}[case["op"]](_inputs(case, seed))
