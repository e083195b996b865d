"""Beam search over a VLT3 model with the paged 8-bit KV cache: the operators of vault_b200.paged in the loop they are for.

    python examples/paged_beam_search.py [model.vlt3] [--beams 4] [--steps 24] [--window 0] [--sinks 0]

The projections are the model's own quantized matrices (VAULTv3ForCausalLM.gemm); every layer appends its keys and values to
the cache, rotated on the way, and attends over it; beam_select picks the continuations and reorder lets the caches follow
them.  Prompts of different lengths run as one batch.  Unlike the engine's own decode path this one keeps every token (or,
with --window, each token's own sliding window) and knows no segment memory.  Without a file a small synthetic model with
the real head geometry is used."""

import argparse
import os
import sys
import tempfile
from typing import List, Tuple

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from vault_b200 import PagedKVCache, VAULTv3ForCausalLM, beam_select, read_vlt3, rope_table  # noqa: E402

Q, K, V, O, GATE_UP, DOWN = 2, 4, 6, 8, 10, 12   # tensor kinds of a layer's matrices


class PagedDecoder:
    """A model's layers over a paged cache: forward(tokens, ...) appends packed tokens and returns the logits of each
    sequence's last one."""

    def __init__(self, path: str, n_pages: int, page: int = 64, max_len: int = 4096, window: int = 0, n_sink: int = 0):
        self.m = VAULTv3ForCausalLM(path)
        c, dev, f = self.m.cfg, self.m.device, read_vlt3(path)
        self.cfg, self.window, self.n_sink = c, window, n_sink

        def vec(name: str) -> torch.Tensor:
            return torch.from_numpy(f.tensor(name).copy()).to(dev)

        self.embed = self.m.dequant(1, c.vocab_size, c.d_model)
        self.norm = vec("norm.weight")
        pre = "layers.%d."
        self.vecs = [{k: vec((pre % i) + k) for k in ("input_layernorm.weight", "post_attention_layernorm.weight", "self_attn.q_proj.bias",
                                                      "self_attn.k_proj.bias", "self_attn.v_proj.bias")} for i in range(c.n_layers)]
        self.rope = rope_table(max_len, c.head_dim, c.rope_theta, device=dev)
        self.cache = PagedKVCache(c.n_layers, n_pages, c.n_kv_heads, c.head_dim, page=page, device=dev)

    def _norm(self, x: torch.Tensor, gain: torch.Tensor) -> torch.Tensor:
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.cfg.rms_eps) * gain

    @torch.no_grad()
    def forward(self, tokens: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, q_start: torch.Tensor, max_q: int = 0,
                max_kv: int = 0) -> torch.Tensor:
        c, m = self.cfg, self.m
        n, d, hq, hkv, hd = tokens.numel(), c.d_model, c.n_heads, c.n_kv_heads, c.head_dim
        x = self.embed[tokens.long()]
        for i, w in enumerate(self.vecs):
            tid = (i + 1) << 8
            u = self._norm(x, w["input_layernorm.weight"])
            q, k, v = (((m.gemm(tid | kind, u, h * hd) + w[f"self_attn.{name}_proj.bias"]).half().view(n, h, hd))
                       for kind, name, h in ((Q, "q", hq), (K, "k", hkv), (V, "v", hkv)))
            q = self.cache.append(i, k, v, table, kv_len, q_start, rope=self.rope, q=q)
            o = self.cache.attention(i, q, table, kv_len, q_start, window=self.window, n_sink=self.n_sink, max_q=max_q, max_kv=max_kv)
            x = x + m.gemm(tid | O, o.view(n, hq * hd).float(), d)
            g = m.gemm(tid | GATE_UP, self._norm(x, w["post_attention_layernorm.weight"]), 2 * c.d_ff)
            x = x + m.gemm(tid | DOWN, torch.nn.functional.silu(g[:, :c.d_ff]) * g[:, c.d_ff:], d)
        last = self._norm(x[q_start[1:].long() - 1], self.norm)
        return m.gemm(1, last, c.vocab_size)


def beam_search(dec: PagedDecoder, prompts: List[List[int]], beams: int, steps: int, eos_id: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The best `beams` continuations of every prompt: tokens [prompts, beams, steps] and their log-probabilities
    [prompts, beams], best first.  Each beam owns a column of pages; full pages are shared between the beams that descend
    from the same one."""
    if not prompts or not all(prompts):
        raise ValueError("every prompt needs a token to go on from")
    dev, groups, page = dec.cache.device, len(prompts), dec.cache.page
    rows, longest = groups * beams, max(len(p) for p in prompts)
    cols = -(-(longest + steps) // page)
    if rows * cols > dec.cache.n_pages:
        raise ValueError(f"{rows} beams of {cols} pages need a cache of {rows * cols} pages")
    table = torch.arange(rows * cols, dtype=torch.int32, device=dev).view(rows, cols)
    i32 = dict(dtype=torch.int32, device=dev)
    # the prompts, each in its first beam's pages
    lens = [len(p) for p in prompts]
    starts = torch.tensor([sum(lens[:i]) for i in range(groups + 1)], **i32)
    logits = dec.forward(torch.tensor(sum(prompts, []), device=dev), table[::beams].contiguous(), torch.tensor(lens, **i32), starts,
                         max_q=longest, max_kv=longest)
    # one beam exists at first; all of them continue it
    scores = torch.full((groups, beams), -torch.inf, device=dev)
    scores[:, 0] = 0.0
    logits = logits.view(groups, 1, -1).expand(-1, beams, -1).contiguous()
    kv_len = torch.tensor(lens, **i32).repeat_interleave(beams)
    finished = torch.zeros(groups, beams, dtype=torch.uint8, device=dev)
    one_each = torch.arange(rows + 1, **i32)
    out = torch.empty(groups, beams, 0, **i32)
    for step in range(steps):
        tokens, parents, scores, finished = beam_select(logits, scores, finished, eos_id)
        table = dec.cache.reorder(table, kv_len, parents)
        out = torch.cat([out.gather(1, parents.long()[..., None].expand_as(out)), tokens[..., None]], -1)
        if step + 1 < steps:
            kv_len = kv_len + 1
            logits = dec.forward(tokens.view(-1), table, kv_len, one_each, max_q=1, max_kv=longest + step + 1).view(groups, beams, -1)
    dec.cache.check()
    return out, scores


def synthetic_model(directory: str) -> str:
    """A two-layer model of random weights with 12 query heads on 2 KV heads of 128 dims."""
    from vault_b200 import VAULTv3Config, synth
    cfg = VAULTv3Config(vocab_size=320, n_layers=2, d_ff=512, window=32, max_sink=64, im_start_id=318, im_end_id=319, system_tok_id=300)
    tok, path = os.path.join(directory, "tok"), os.path.join(directory, "model.vlt3")
    synth.make_tokenizer_dir(tok, cfg.vocab_size, synth.SMALL_EXTRA_TOKENS)
    synth.write_synthetic_vlt3(path, cfg, "q8_0", 5, tokenizer_dir=tok, std=0.1)
    return path


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("model", nargs="?")
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    a = ap.parse_args()
    with tempfile.TemporaryDirectory() as td:
        path = a.model or synthetic_model(td)
        dec = PagedDecoder(path, n_pages=256, window=a.window, n_sink=a.sinks)
        g = torch.Generator().manual_seed(0)
        prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (7, 70, 131)]
        out, scores = beam_search(dec, prompts, a.beams, a.steps, eos_id=dec.cfg.im_end_id)
        for p, (o, s) in enumerate(zip(out.tolist(), scores.tolist())):
            for j in range(a.beams):
                print(f"prompt {p} beam {j}: log-probability {s[j]:9.4f}  tokens {o[j]}")
        print(f"cache: {dec.cache.nbytes() / 2**20:.1f} MiB for {dec.cache.n_pages} pages of {dec.cache.page} tokens, "
              f"{dec.cache.n_layers} layers")


if __name__ == "__main__":
    main()
