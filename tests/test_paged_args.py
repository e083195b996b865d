"""Refusals of the paged-cache and beam entry points: every check that needs no device, through the C ABI."""
import ctypes as C

import pytest

from vault_b200 import _lib

P = 0x7F0000000000   # an address that no call may reach: each case is refused before anything is launched
E_ARG, E_DTYPE, E_ALIGN, E_LIMIT, E_SIZE, E_UNSUPPORTED = -21, -5, -11, -10, -1, -22


def cache(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, n_layers=2, n_pages=9, n_kv_heads=2, page=64, head_dim=128)
    a.update(kw)
    return _lib.KVCache(**a)


def batch(**kw):
    a = dict(page_table=P, table_ld=4, kv_len=P, q_start=P, batch=2, max_pages=4, n_tokens=2)
    a.update(kw)
    return _lib.KVBatch(**a)


def rows(p=P, t=256, h=128):
    return _lib.Rows(p, t, h)


def refused(code, rc):
    assert rc == code, (rc, _lib.last_error())
    assert _lib.last_error().startswith("v3g_")


def append(c=None, b=None, layer=0, dtype=1, k=None, v=None, q=None, heads=0, q_out=None, rope=None, rope_rows=0):
    return _lib.lib().v3g_kv_append(c or cache(), layer, b or batch(), dtype, k or rows(), v or rows(), q, heads, q_out, rope, rope_rows,
                                    None, None)


def attention(c=None, b=None, layer=0, dtype=1, q=None, heads=4, scale=0.1, out=P, lse=None, work=P, size=1 << 40, max_q=0, max_kv=0):
    return _lib.lib().v3g_kv_attention(c or cache(), layer, b or batch(), dtype, q or rows(), heads, scale, 0, 0, max_q, max_kv, out, lse,
                                       None, work, size, None)


@pytest.mark.parametrize("code,change", [(E_ARG, dict(k=None)), (E_ARG, dict(v_scale=None)), (E_UNSUPPORTED, dict(head_dim=96)),
                                         (E_UNSUPPORTED, dict(page=48)), (E_UNSUPPORTED, dict(page=512)), (E_UNSUPPORTED, dict(page=8)),
                                         (E_ARG, dict(n_pages=0)), (E_ARG, dict(n_layers=0)), (E_ARG, dict(n_kv_heads=0)),
                                         (E_ALIGN, dict(k=P + 8)), (E_ALIGN, dict(k_scale=P + 2))])
def test_caches(code, change):
    c = cache(**change)
    refused(code, append(c=c))
    refused(code, attention(c=c))
    L = _lib.lib()
    refused(code, L.v3g_kv_read(c, 0, 1, batch(), P, 0, P, P, None))
    refused(code, L.v3g_kv_reorder(c, batch(), 2, P, None, P + 4096, 4, None, None))


@pytest.mark.parametrize("code,change", [(E_ARG, dict(page_table=None)), (E_ARG, dict(kv_len=None)), (E_ARG, dict(max_pages=0)),
                                         (E_ARG, dict(table_ld=3)), (E_LIMIT, dict(batch=70000)), (E_ALIGN, dict(kv_len=P + 2))])
def test_batches(code, change):
    b = batch(**change)
    refused(code, append(b=b))
    refused(code, attention(b=b))
    refused(code, _lib.lib().v3g_kv_read(cache(), 0, 1, b, P, 0, P, P, None))


def test_append_arguments():
    refused(E_ARG, append(layer=2))
    refused(E_DTYPE, append(dtype=7))
    refused(E_ARG, append(k=rows(None)))
    refused(E_ARG, append(q=rows(), heads=0, q_out=P))
    refused(E_ARG, append(q=rows(), heads=4, q_out=None))
    refused(E_ARG, append(rope=P, rope_rows=0))
    refused(E_ALIGN, append(k=rows(P + 1)))
    refused(E_ALIGN, append(rope=P + 4, rope_rows=9))
    refused(E_ALIGN, append(q=rows(), heads=4, q_out=P + 2))
    assert append(b=batch(batch=0)) == 0 and append(b=batch(n_tokens=0)) == 0


def test_attention_arguments():
    refused(E_ARG, attention(layer=5))
    refused(E_DTYPE, attention(dtype=0))
    refused(E_ARG, attention(heads=3))
    refused(E_ARG, attention(heads=0))
    refused(E_ARG, attention(scale=float("nan")))
    refused(E_ARG, attention(scale=float("inf")))
    refused(E_ARG, attention(out=None))
    refused(E_ALIGN, attention(out=P + 2))
    refused(E_ALIGN, attention(q=rows(P + 1)))
    need = _lib.lib().v3g_kv_attention_work_size(cache(), batch(max_pages=64, table_ld=64), 4, 1, 4096, 0, 0)
    assert need > 0
    b = batch(max_pages=64, table_ld=64)
    refused(E_SIZE, attention(b=b, size=need - 1, max_q=1, max_kv=4096))
    refused(E_SIZE, attention(b=b, work=None, size=need, max_q=1, max_kv=4096))
    refused(E_ALIGN, attention(b=b, work=P + 16, size=need, max_q=1, max_kv=4096))
    refused(E_LIMIT, attention(b=batch(n_tokens=1 << 24), heads=256))
    assert attention(b=batch(batch=0)) == 0 and attention(b=batch(n_tokens=0)) == 0


def test_read_and_reorder_arguments():
    L = _lib.lib()
    refused(E_DTYPE, L.v3g_kv_read(cache(), 0, 1, batch(), P, 3, P, P, None))
    refused(E_ARG, L.v3g_kv_read(cache(), 0, 1, batch(), None, 0, P, P, None))
    refused(E_ARG, L.v3g_kv_read(cache(), 1, 2, batch(), P, 0, P, P, None))
    refused(E_ARG, L.v3g_kv_read(cache(), 0, 1, batch(), P, 0, None, P, None))
    refused(E_ALIGN, L.v3g_kv_read(cache(), 0, 1, batch(), P, 0, P + 8, P, None))
    refused(E_LIMIT, L.v3g_kv_reorder(cache(), batch(batch=66), 33, P, None, P + 4096, 4, None, None))
    refused(E_LIMIT, L.v3g_kv_reorder(cache(), batch(), 0, P, None, P + 4096, 4, None, None))
    refused(E_ARG, L.v3g_kv_reorder(cache(), batch(batch=3), 2, P, None, P + 4096, 4, None, None))
    refused(E_ARG, L.v3g_kv_reorder(cache(), batch(), 2, None, None, P + 4096, 4, None, None))
    refused(E_ARG, L.v3g_kv_reorder(cache(), batch(), 2, P, None, P, 4, None, None))          # in place
    refused(E_ARG, L.v3g_kv_reorder(cache(), batch(), 2, P, None, P + 4096, 3, None, None))
    refused(E_ALIGN, L.v3g_kv_reorder(cache(), batch(), 2, P + 1, None, P + 4096, 4, None, None))


def test_beam_arguments():
    L = _lib.lib()

    def beam(logits=P, dtype=0, groups=2, beams=4, vocab=1000, ld=1000, scores=P, eos=1, out=P, work=P, size=1 << 40):
        return L.v3g_beam_select(logits, dtype, groups, beams, vocab, ld, scores, None, eos, out, P, P, P, work, size, None)

    refused(E_DTYPE, beam(dtype=9))
    refused(E_LIMIT, beam(beams=33))
    refused(E_LIMIT, beam(beams=0))
    refused(E_ARG, beam(vocab=0))
    refused(E_ARG, beam(ld=999))
    refused(E_ARG, beam(eos=1000))
    refused(E_LIMIT, beam(vocab=1 << 29, ld=1 << 29))
    refused(E_LIMIT, beam(groups=20000))
    refused(E_ARG, beam(logits=None))
    refused(E_ARG, beam(out=None))
    refused(E_ALIGN, beam(logits=P + 2))
    refused(E_SIZE, beam(work=None))
    refused(E_SIZE, beam(size=L.v3g_beam_select_work_size(2, 4, 1000) - 1))
    refused(E_ALIGN, beam(work=P + 128))
    assert beam(groups=0) == 0
    assert L.v3g_beam_select_work_size(1, 33, 5) == 0 and C.sizeof(_lib.Rows) == 24
