"""Paged 8-bit KV cache, attention over it, and beam search on the B200 engine.

The operators a serving loop needs around its projections, for batches of sequences of different lengths:

    cache = PagedKVCache(n_layers, n_pages, n_kv_heads, head_dim, page=64)
    rope = rope_table(max_positions, head_dim, theta)
    q = cache.append(layer, k, v, page_table, kv_len, q_start, rope=rope, q=q)      # rotate, round to 8 bits, store
    out = cache.attention(layer, q, page_table, kv_len, q_start, window=1024, n_sink=4)
    tokens, parents, scores, finished = beam_select(logits, scores, finished, eos_id)
    page_table = cache.reorder(page_table, kv_len, parents)

Tokens are packed: rows q_start[b] .. q_start[b + 1] - 1 belong to sequence b and stand at its last positions, kv_len[b]
counting them; rows past q_start[-1] belong to none and come out as zeros.  page_table[b, i] is the page of tokens
i * page .. (i + 1) * page - 1 of sequence b, negative where there is none.  Index tensors are int32 on the cache's device.  Calls run on torch's current stream and read no tensor on the
host; all device work is the C ABI's (include/vault_b200.h).  No result depends on the order in which blocks run.
"""

from __future__ import annotations

import ctypes as C
import threading
from typing import Optional, Tuple

import torch

from . import _lib

BLOCK = 16      # tokens that share a scale
_FAR = 1 << 30  # past every position
_DTYPES = {torch.float32: _lib.V3G_F32, torch.float16: _lib.V3G_F16, torch.bfloat16: _lib.V3G_BF16}


def rope_table(n_positions: int, head_dim: int, theta: float = 1_000_000.0, device=None) -> torch.Tensor:
    """Rotation table [n_positions, head_dim] fp32: head_dim / 2 cosines, then the sines, of position x theta^(-2 i /
    head_dim), from angles in 64 bits (the convention of the model's own rotation: pairs i, i + head_dim / 2)."""
    if n_positions < 1 or head_dim < 2 or head_dim % 2:
        raise ValueError("rope_table needs n_positions >= 1 and an even head_dim")
    inv = float(theta) ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(n_positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device if device is not None else torch.device("cuda"))


def _index(t: torch.Tensor, name: str, device, n: int) -> int:
    if t.dtype is not torch.int32 or t.numel() != n or t.dim() != 1 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on {device}")
    return t.data_ptr()


# The current device, torch's current stream of a device as the C ABI takes it, and whether it is being captured: the calls
# behind torch.cuda's, without the Python objects around them (the stream 0.1 us instead of 2.3).
_current_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream
_capturing = torch._C._cuda_isCurrentStreamCapturing


class _Workspaces:
    """Device workspaces, one for each stream that has used them: a stream runs its kernels in order, so its calls can share
    one.  A call queues several kernels that hand their results on in it and lets other Python threads run meanwhile, so it
    is queued under a lock: no other thread's kernels come between its own.  Workspaces grow and are kept until their owner
    goes.  A captured call has one of its own, in the graph's memory."""

    def __init__(self):
        self.by_stream = {}
        self.lock = threading.RLock()   # a finalizer that runs inside may make a call of its own

    def run(self, device, size, call) -> int:
        """call(workspace, its bytes, stream) on torch's current stream of `device`, which becomes the current device for
        the call.  The workspace that is there is offered as it is: the engine refuses one that is too small before it
        does anything else, and only then is size() asked."""
        index = device.index
        if _current_device() != index:
            with torch.cuda.device(device):
                return self.run(device, size, call)
        stream = _stream(index)
        if _capturing():
            t = torch.empty(size(), dtype=torch.uint8, device=device)
            return call(t.data_ptr(), t.numel(), stream)
        with self.lock:
            held = self.by_stream.get((index, stream))
            if held is not None:
                rc = call(held[0], held[1], stream)
                if rc != _lib.V3G_E_SIZE:
                    return rc
            t = torch.empty(max(size(), 1 << 16), dtype=torch.uint8, device=device)
            self.by_stream[(index, stream)] = (t.data_ptr(), t.numel(), t)
            return call(t.data_ptr(), t.numel(), stream)


_beam_work = _Workspaces()


class PagedKVCache:
    """8-bit keys and values in pages of `page` tokens: k, v uint8 [n_layers, n_pages, n_kv_heads, page, head_dim] (codes
    biased by 128), k_scale, v_scale fp32 [n_layers, n_pages, n_kv_heads, page / 16].  value = (code - 128) * scale."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page: int = 64, device=None):
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if head_dim not in (64, 128) or page not in (16, 32, 64, 128, 256):
            raise ValueError("head_dim must be 64 or 128, page 16, 32, 64, 128 or 256")
        if min(n_layers, n_pages, n_kv_heads) < 1:
            raise ValueError("n_layers, n_pages and n_kv_heads must be positive")
        shape = (n_layers, n_pages, n_kv_heads, page)
        self._bind(*(torch.full((*shape, head_dim), 128, dtype=torch.uint8, device=dev) for _ in range(2)),
                   *(torch.zeros(*shape[:3], page // BLOCK, dtype=torch.float32, device=dev) for _ in range(2)))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "PagedKVCache":
        """A cache over arrays that the caller holds (the layout above)."""
        self = cls.__new__(cls)
        if k.dim() != 5 or k.dtype != torch.uint8 or not k.is_cuda or k.numel() == 0 or k.shape[4] not in (64, 128) or \
                k.shape[3] not in (16, 32, 64, 128, 256):
            raise ValueError("k must be a uint8 CUDA tensor [layers, pages, heads, page, head_dim]")
        scales = (*k.shape[:3], k.shape[3] // BLOCK)
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("v must have the shape and type of k")
        if any(t.shape != scales or t.dtype != torch.float32 for t in (k_scale, v_scale)):
            raise ValueError("scales must be fp32 [layers, pages, heads, page / 16]")
        if any(t.device != k.device or not t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's arrays must be contiguous and on one device")
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_layers, self.n_pages, self.n_kv_heads, self.page, self.head_dim = k.shape
        self.device = k.device
        self._index = k.device.index
        self._scale = self.head_dim ** -0.5
        self.status_word = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._status = self.status_word.data_ptr()
        self._work = _Workspaces()
        self._c = _lib.KVCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        self._ref = C.byref(self._c)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))

    def check(self) -> None:
        """Wait for the device, every stream of it, and raise if a token or a beam had no place (V3G_STATUS_BOUNDS) since the
        last check."""
        torch.cuda.synchronize(self.device)   # the read below waits for the current stream alone
        bits = int(self.status_word.item())
        if bits:
            self.status_word.zero_()
            torch.cuda.synchronize(self.device)   # what other streams run from here on is not wiped
            raise RuntimeError(f"device status bits {bits:#x}: " +
                               ("a token without a page or a rotation row was dropped, or a beam's parent or page does not exist"
                                if bits & _lib.V3G_STATUS_BOUNDS else "a kernel gave up waiting, its output is invalid"))

    # ---- arguments
    def _batch(self, page_table, kv_len, q_start, n_tokens: int) -> _lib.KVBatch:
        dev = self.device
        if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.device != dev:
            raise ValueError("page_table must be int32 [batch, pages] on the cache's device")
        n, cols = page_table.shape
        ld, one = page_table.stride()
        if cols < 1 or (one != 1 and cols > 1) or (n > 1 and ld < cols):
            raise ValueError("page_table needs at least one column and contiguous rows")
        lens = _index(kv_len, "kv_len", dev, n)
        starts = lens if q_start is None else _index(q_start, "q_start", dev, n + 1)
        return _lib.KVBatch(page_table.data_ptr(), ld if ld > cols else cols, lens, starts, n, cols, n_tokens)

    def _rows(self, x: torch.Tensor, name: str, heads: int, n: int, dtype) -> _lib.Rows:
        if x.dim() == 3 and x.dtype is dtype and x.device == self.device:
            shape = x.shape
            tok, head, one = x.stride()
            if one == 1 and shape[0] == n and shape[1] == heads and shape[2] == self.head_dim:
                return _lib.Rows(x.data_ptr(), tok, head)
        raise ValueError(f"{name} must be {dtype} [{n}, {heads}, {self.head_dim}] on the cache's device, its last dimension contiguous")

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        return layer

    def _call(self, fn, what: str, *args) -> None:
        """fn on torch's current stream of the cache's device, which becomes the current device for the call."""
        index = self._index
        if _current_device() == index:
            rc = fn(*args, _stream(index))
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args, _stream(index))
        if rc:
            _lib.check(rc, what)

    # ---- operators
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor,
               q_start: torch.Tensor, rope: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Store the batch's new tokens: k, v [tokens, n_kv_heads, head_dim] (fp32, fp16 or bf16, any token and head
        strides), k rotated at its position when `rope` (rope_table) is given.  With q [tokens, heads, head_dim] of the
        same type, the rotated queries are returned (in q_out, if given).  A block of 16 tokens keeps one scale per
        head: when a later token is larger, the block's earlier codes are rounded again under the larger scale."""
        n, dtype = k.shape[0], k.dtype
        dt = _DTYPES.get(dtype)
        if dt is None:
            raise ValueError("k must be fp32, fp16 or bf16")
        kr = self._rows(k, "k", self.n_kv_heads, n, dtype)
        vr = self._rows(v, "v", self.n_kv_heads, n, dtype)
        batch = self._batch(page_table, kv_len, q_start, n)
        positions = 0
        if rope is not None:
            if rope.dim() != 2 or rope.dtype is not torch.float32 or rope.device != self.device or not rope.is_contiguous() or \
                    rope.shape[1] != self.head_dim or rope.shape[0] < 1:
                raise ValueError("rope must be a contiguous fp32 [positions, head_dim] table on the cache's device")
            positions = rope.shape[0]
        qr, heads = None, 0
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            qr = self._rows(q, "q", heads, n, dtype)
            if heads == 0:
                raise ValueError("q has no heads")
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            elif q_out.shape != q.shape or q_out.dtype is not dtype or q_out.device != self.device or not q_out.is_contiguous():
                raise ValueError("q_out must be a contiguous tensor of q's shape and type")
        elif q_out is not None:
            raise ValueError("q_out without q")
        if n:
            self._call(_lib.lib().v3g_kv_append, "v3g_kv_append", self._ref, self._layer(layer), batch, dt, kr, vr, qr, heads,
                       None if q is None else q_out.data_ptr(), None if rope is None else rope.data_ptr(), positions, self._status)
        return q_out

    def attention(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor, q_start: torch.Tensor,
                  scale: Optional[float] = None, window: int = 0, n_sink: int = 0, max_q: int = 0, max_kv: int = 0,
                  out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Causal attention of q [tokens, heads, head_dim] (fp16 or bf16) over the cached tokens: a token at position p
        sees keys j <= p with j > p - window or j < n_sink (window 0: all).  Returns out of q's shape and type, with
        return_lse also the logarithm of the softmax sum [tokens, heads]; a row that sees no key gives zeros and -inf.
        max_q and max_kv (largest token count and length in the batch, where the host knows them) steer how work is
        split and never what is computed.  scale defaults to head_dim ** -0.5."""
        n, heads, dtype = q.shape[0], q.shape[1] if q.dim() == 3 else 0, q.dtype
        if dtype is not torch.float16 and dtype is not torch.bfloat16:
            raise ValueError("q must be fp16 or bf16")
        if heads == 0 or heads % self.n_kv_heads:
            raise ValueError("the query heads must be a multiple of the KV heads")
        if window < 0 or n_sink < 0 or max_q < 0 or max_kv < 0:
            raise ValueError("window, n_sink, max_q and max_kv must not be negative")
        qr = self._rows(q, "q", heads, n, dtype)
        batch = self._batch(page_table, kv_len, q_start, n)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not dtype or out.device != self.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor of q's shape and type")
        lse = torch.empty(n, heads, dtype=torch.float32, device=self.device) if return_lse else None
        if n:
            if window > _FAR or n_sink > _FAR or max_q > _FAR or max_kv > _FAR:
                window, n_sink, max_q, max_kv = (min(x, _FAR) for x in (window, n_sink, max_q, max_kv))
            L, ref, layer, dt = _lib.lib(), self._ref, self._layer(layer), _DTYPES[dtype]
            scale = self._scale if scale is None else float(scale)
            lse_ptr = None if lse is None else lse.data_ptr()
            rc = self._work.run(
                self.device, lambda: L.v3g_kv_attention_work_size(ref, batch, heads, max_q, max_kv, window, n_sink),
                lambda work, size, stream: L.v3g_kv_attention(ref, layer, batch, dt, qr, heads, scale, window, n_sink, max_q, max_kv,
                                                              out.data_ptr(), lse_ptr, self._status, work, size, stream))
            if rc:
                _lib.check(rc, "v3g_kv_attention")
        return (out, lse) if return_lse else out

    def read(self, page_table: torch.Tensor, first: torch.Tensor, kv_len: torch.Tensor, row_start: torch.Tensor, n_rows: int,
             dtype: torch.dtype = torch.float32, layer: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Cached keys (rotated, as stored) and values of tokens first[b] .. kv_len[b] - 1 of every sequence: two tensors
        [layers, n_rows, n_kv_heads, head_dim] (one layer when `layer` is given), row row_start[b] + i holding token
        first[b] + i.  Rows of no token are zero."""
        dt = _DTYPES.get(dtype)
        if dt is None:
            raise ValueError("dtype must be fp32, fp16 or bf16")
        if n_rows < 0:
            raise ValueError("n_rows must not be negative")
        batch = self._batch(page_table, kv_len, row_start, n_rows)
        f = _index(first, "first", self.device, batch.batch)
        l0, layers = (0, self.n_layers) if layer is None else (self._layer(layer), 1)
        k = torch.empty(layers, n_rows, self.n_kv_heads, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if batch.batch == 0:
            return k.zero_(), v.zero_()
        if n_rows:
            self._call(_lib.lib().v3g_kv_read, "v3g_kv_read", self._ref, l0, layers, batch, f, dt, k.data_ptr(), v.data_ptr())
        return k, v

    def reorder(self, page_table: torch.Tensor, kv_len: torch.Tensor, parents: torch.Tensor,
                dst_page: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The caches of groups of beams follow the chosen parents ([groups, beams] int32, as beam_select returns them):
        returns the new page table, in which row g * beams + j shares the full pages of its parent; the page still being
        filled is copied, in every layer, into dst_page ([rows] int32; default: the row's own entry).  The rows of a
        group have equal kv_len."""
        rows, dev = page_table.shape[0], self.device
        if parents.dtype is not torch.int32 or parents.dim() != 2 or parents.device != dev or not parents.is_contiguous() or \
                parents.numel() != rows or parents.shape[1] < 1:
            raise ValueError("parents must be a contiguous int32 [groups, beams] tensor with one entry for each row")
        batch = self._batch(page_table, kv_len, None, 0)
        dst = None if dst_page is None else _index(dst_page, "dst_page", dev, rows)
        out = torch.empty_like(page_table, memory_format=torch.contiguous_format)
        if rows:
            self._call(_lib.lib().v3g_kv_reorder, "v3g_kv_reorder", self._ref, batch, parents.shape[1], parents.data_ptr(), dst,
                       out.data_ptr(), batch.max_pages, self._status)
        return out


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None,
                eos_id: int = -1) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """One step of beam search: logits [groups, beams, vocab] (fp32, fp16 or bf16), scores [groups, beams] fp32 (-inf: no
    beam yet), finished [groups, beams] uint8.  Of each group's continuations, scored log_softmax(logits) + scores, the
    `beams` best in descending order: (tokens, parents, scores, finished), each [groups, beams].  A finished beam goes on
    with eos_id alone, at its own score; equal (fp32) scores go to the lower (beam, token); continuations at -inf or NaN are
    never chosen, and slots left over come back finished, with score -inf."""
    dt = _DTYPES.get(logits.dtype)
    if dt is None or logits.dim() != 3 or not logits.is_cuda or logits.numel() == 0:
        raise ValueError("logits must be a CUDA tensor [groups, beams, vocab] of fp32, fp16 or bf16")
    b, k, v = logits.shape
    rows = (b, k)
    s0, s1, s2 = logits.stride()
    ld = s1 if k > 1 else (s0 if b > 1 else v)
    if (s2 != 1 and v > 1) or ld < v or (b > 1 and k > 1 and s0 != k * ld):
        raise ValueError("logits must have contiguous rows, evenly spaced")
    dev = logits.device
    if scores.dtype is not torch.float32 or scores.shape != rows or scores.device != dev or not scores.is_contiguous():
        raise ValueError("scores must be a contiguous fp32 [groups, beams] tensor on the logits' device")
    if finished is not None and (finished.dtype not in (torch.uint8, torch.bool) or finished.shape != rows or
                                 finished.device != dev or not finished.is_contiguous()):
        raise ValueError("finished must be a contiguous uint8 [groups, beams] tensor on the logits' device")
    eos_id = min(max(eos_id, -1), 0x7FFFFFFF)   # as 32 bits: none at all, or past every vocabulary, which the engine refuses
    L = _lib.lib()
    best = torch.empty_like(scores)
    tokens = torch.empty_like(scores, dtype=torch.int32)
    parents = torch.empty_like(tokens)
    done = torch.empty_like(scores, dtype=torch.uint8)
    done_ptr = None if finished is None else finished.data_ptr()
    rc = _beam_work.run(
        dev, lambda: L.v3g_beam_select_work_size(b, k, v),
        lambda work, size, stream: L.v3g_beam_select(logits.data_ptr(), dt, b, k, v, ld, scores.data_ptr(), done_ptr, eos_id,
                                                     tokens.data_ptr(), parents.data_ptr(), best.data_ptr(), done.data_ptr(), work, size,
                                                     stream))
    if rc:
        _lib.check(rc, "v3g_beam_select")
    return tokens, parents, best, done


__all__ = ["PagedKVCache", "beam_select", "rope_table"]
