"""Refusals of the 8-bit page entry points: a 0 result and a message before
any device work (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest

import inference_c_b200 as P


def _layer(**kw):
    a = dict(key_pool=256, value_pool=256, key_scales=256, value_scales=256, block_size=16,
             block_count=4, kv_heads=2, head_dim=128, dtype=P.PKV_DTYPE_F16)
    a.update(kw)
    return P.PkvQ8Layer(*[a[n] for n, _ in P.PkvQ8Layer._fields_])


def _batch(**kw):
    a = dict(block_tables=256, table_stride=4, seq_lens=256, batch=2)
    a.update(kw)
    return P.PkvBatch(*[a[n] for n, _ in P.PkvBatch._fields_])


BAD = [
    (dict(key_pool=None), {}, "null"), (dict(value_scales=None), {}, "null"),
    ({}, dict(block_tables=None), "null"), ({}, dict(seq_lens=None), "null"),
    (dict(dtype=P.PKV_DTYPE_F32), {}, "dtype"), (dict(dtype=9), {}, "dtype"),
    (dict(block_size=8), {}, "16, 32, 64 or 128"), (dict(block_size=24), {}, "16, 32, 64 or 128"),
    (dict(head_dim=96), {}, "head_dim 64 or 128"), (dict(kv_heads=0), {}, "KV heads"),
    (dict(kv_heads=1025), {}, "KV heads"), (dict(block_count=0), {}, "block count"),
    ({}, dict(batch=0), "batch"), ({}, dict(table_stride=0), "stride"),
    ({}, dict(table_stride=1 << 31), "stride"), (dict(key_pool=264), {}, "16-byte aligned"),
    (dict(key_scales=258), {}, "4-byte aligned"),
]


def _err():
    return ctypes.create_string_buffer(256)


@pytest.mark.parametrize("layer,batch,text", BAD)
def test_layer_and_batch_are_checked(lib, layer, batch, text):
    L, B = _layer(**layer), _batch(**batch)
    for name in ("pkv_q8_append", "pkv_q8_import", "pkv_q8_gather"):
        e = _err()
        assert getattr(lib, name)(ctypes.byref(L), ctypes.byref(B), 256, 256, 256, 2, None, e,
                                  len(e)) == 0
        assert text in e.value.decode() and name in e.value.decode()
    e = _err()
    assert lib.pkv_q8_decode(ctypes.byref(L), ctypes.byref(B), 4, 256, ctypes.c_float(1), 256,
                             P.PKV_DTYPE_F32, 64, 256, 1 << 30, None, e, len(e)) == 0
    assert text in e.value.decode() and "pkv_q8_decode" in e.value.decode()


def test_rows_are_checked(lib):
    L, B = _layer(), _batch()
    for args, text in (((256, None, 256, 2), "null"), ((256, 256, 264, 2), "aligned"),
                       ((None, 256, 256, 3), "total_rows"), ((256, 256, 256, 1 << 30), "rows")):
        e = _err()
        assert lib.pkv_q8_append(ctypes.byref(L), ctypes.byref(B), *args, None, e, len(e)) == 0
        assert text in e.value.decode()
    e = _err()
    assert lib.pkv_q8_append(None, ctypes.byref(B), 256, 256, 256, 2, None, e, len(e)) == 0
    assert lib.pkv_q8_append(ctypes.byref(L), None, 256, 256, 256, 2, None, e, len(e)) == 0
    # no rows: nothing to do, no device touched
    assert lib.pkv_q8_append(ctypes.byref(L), ctypes.byref(B), 256, 256, 256, 0, None, e, len(e)) == 1


def _decode(lib, L, B, q_heads=4, query=256, scale=1.0, out=256, dtype=P.PKV_DTYPE_F32, max_len=64,
            ws=256, ws_bytes=1 << 30):
    e = _err()
    ok = lib.pkv_q8_decode(ctypes.byref(L), ctypes.byref(B), q_heads, query, ctypes.c_float(scale),
                           out, dtype, max_len, ws, ws_bytes, None, e, len(e))
    return ok, e.value.decode()


def test_decode_arguments_are_checked(lib):
    L, B = _layer(), _batch()
    for kw, text in ((dict(query=None), "null"), (dict(out=None), "null"),
                     (dict(dtype=P.PKV_DTYPE_BF16), "output dtype"), (dict(dtype=0), "output dtype"),
                     (dict(q_heads=3), "times kv_heads"), (dict(q_heads=0), "times kv_heads"),
                     (dict(q_heads=34), "times kv_heads")):
        ok, text_got = _decode(lib, L, B, **kw)
        assert ok == 0 and text in text_got, (kw, text_got)


def test_prefill_arguments_are_checked(lib):
    L, B = _layer(), _batch()
    f = ctypes.c_float
    n = lib.pkv_q8_prefill_workspace_bytes(1, 2, 128, 200)
    assert n >= 2 * 256 * 256 * 2 and n < lib.pkv_q8_prefill_workspace_bytes(2, 2, 128, 200)

    def call(L=L, q_heads=4, offs=256, query=256, rows=2, scale=1.0, causal=1, out=256,
             dtype=P.PKV_DTYPE_F16, max_len=200, ws=256, ws_bytes=1 << 30):
        e = _err()
        ok = lib.pkv_q8_prefill(ctypes.byref(L), ctypes.byref(B), q_heads, offs, query, rows, 1,
                                f(scale), causal, out, dtype, max_len, ws, ws_bytes, None, e, len(e))
        return ok, e.value.decode()
    for kw, text in ((dict(L=_layer(block_size=8)), "16, 32, 64 or 128"), (dict(offs=None), "null"),
                     (dict(query=None), "null"), (dict(out=None), "null"),
                     (dict(max_len=0), "max_seq_len"), (dict(ws=None), "workspace"),
                     (dict(ws_bytes=n - 1), "workspace"), (dict(ws=264), "workspace"),
                     (dict(dtype=P.PKV_DTYPE_BF16), "output dtype"), (dict(q_heads=3), "multiple"),
                     (dict(causal=2), "invalid"), (dict(scale=float("nan")), "invalid")):
        ok, got = call(**kw)
        assert ok == 0 and text in got and "pkv_q8_prefill" in got, (kw, got)


def test_mass_and_evict_arguments_are_checked(lib):
    f = ctypes.c_float
    L, B = _layer(), _batch()
    H = P.PkvPagedLayer(256, 256, 16, 4, 2, 128, P.PKV_DTYPE_F16)

    def mass(name, layer, mass=256, q_heads=4, ws_bytes=1 << 40, max_len=64):
        e = _err()
        ok = getattr(lib, name)(ctypes.byref(layer), ctypes.byref(B), q_heads, 256, f(1), 256,
                                P.PKV_DTYPE_F32, max_len, mass, 256, ws_bytes, None, e, len(e))
        return ok, e.value.decode()
    for name, layer in (("pkv_q8_decode_mass", L), ("pkv_paged_decode_mass", H)):
        for kw, text in ((dict(mass=None), "mass"), (dict(mass=260), "mass"),
                         (dict(ws_bytes=1 << 12), "workspace"), (dict(q_heads=3), "kv_heads")):
            ok, got = mass(name, layer, **kw)
            assert ok == 0 and text in got and name in got, (name, kw, got)
    ok, got = mass("pkv_paged_decode_mass", P.PkvPagedLayer(256, 256, 12, 4, 2, 128, 1))
    assert ok == 0 and "pages of 16, 32, 64 or 128" in got

    def evict(name, layer, batch=B, mass=256, keep=8, recent=2, dst=None, stride=0, kept=256,
              max_len=64):
        e = _err()
        ok = getattr(lib, name)(ctypes.byref(layer), ctypes.byref(batch), mass, keep, recent, dst,
                                stride, kept, max_len, None, e, len(e))
        return ok, e.value.decode()
    for name, layer in (("pkv_q8_evict", L), ("pkv_kv_evict", H)):
        for kw, text in ((dict(mass=None), "mass"), (dict(mass=264), "mass"),
                         (dict(kept=None), "kept"), (dict(keep=0), "keep"),
                         (dict(recent=9), "recent"), (dict(dst=512, stride=0), "stride"),
                         (dict(batch=_batch(batch=0)), "batch"),
                         (dict(batch=_batch(batch=65536)), "65535"),
                         (dict(batch=_batch(seq_lens=None)), "null")):
            ok, got = evict(name, layer, **kw)
            assert ok == 0 and text in got and name in got, (name, kw, got)
    ok, got = evict("pkv_kv_evict", P.PkvPagedLayer(256, 256, 16, 4, 2, 96, 1))
    assert ok == 0 and "head_dim" in got
    e = _err()
    assert lib.pkv_mass_clear(16, 4, 2, ctypes.byref(B), None, None, None, e, len(e)) == 0
    assert b"null" in e.value
    assert lib.pkv_mass_clear(0, 4, 2, ctypes.byref(B), None, 256, None, e, len(e)) == 0
    assert b"shape" in e.value


def test_workspaces_grow_with_what_they_hold(lib):
    a = lib.pkv_q8_decode_workspace_bytes(1, 32, 8, 128, 4096)
    b = lib.pkv_q8_decode_workspace_bytes(64, 32, 8, 128, 4096)
    assert 0 < a < b and a % 256 == 0 and b % 256 == 0
    m = lib.pkv_decode_mass_workspace_bytes(64, 32, 8, 128, 4096)
    # every score of every query head, and the decode's own scratch
    assert m >= b + 64 * 32 * 4096 * 4
    assert lib.pkv_q8_decode_workspace_bytes(1, 3, 2, 128, 64) == 0


def test_q8_pool_shapes_are_checked(lib):
    for bs, hd, kv, dtype in ((12, 128, 2, P.PKV_DTYPE_F16), (16, 96, 2, P.PKV_DTYPE_F16),
                              (16, 128, 2000, P.PKV_DTYPE_F16), (16, 128, 2, P.PKV_DTYPE_F32)):
        cache = P.PagedKVCache(bs, 4, 1)
        with pytest.raises(P.PkvError, match="8|pages"):
            P.PagedPool.q8(cache, 0, dtype, 1, kv, hd, 1, 4)
        cache.free()


def test_python_calls_check_their_tensors(lib):
    """Types, shapes and devices of mass, kept and dst_tables: a ValueError
    before the library is called (which would refuse these addresses too)."""
    import torch
    L, B = _layer(key_pool=None), _batch()
    mass = torch.zeros(4, 2, 16)
    for bad in (mass, mass.to(torch.int32), mass.half(), mass[:, :1],
                mass.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(ValueError, match="mass is a contiguous float32"):
            P.mass_clear(L, B, bad)
        with pytest.raises(ValueError, match="mass is a contiguous float32"):
            P.q8_decode_mass(L, B, torch.zeros(2, 4, 128).half(), torch.zeros(2, 4, 128), 1.0, 64,
                             bad, mass)
    kept = torch.zeros(2, 2, 8, dtype=torch.int32)
    for bad in (kept, kept.float(), kept.long(), kept[:, :, :7]):
        with pytest.raises(ValueError, match="kept is a contiguous int32"):
            P.kv_evict(L, B, 256, 8, 2, bad, 64)
