"""Paged key-value cache operators, what needs no GPU: refusals of the C ABI and of the Python layer, the rotation table."""
import ctypes
import math

import pytest
import torch

from wush_b200 import _lib, paged_kv

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _pages(p, **kw):
    """A bf16 pool of 4 pages of 16 rows, 2 heads of 64 channels."""
    d = dict(k=p, v=p, k_page=2048, k_row=128, k_head=64, v_page=2048, v_row=128, v_head=64, k_scale=None, v_scale=None,
             bounds=p, num_pages=4, page_size=16, heads=2, dim=64, type=0, bounds_type=0)
    d.update(kw)
    return _lib.KVPages(**d)


@pytest.fixture()
def ptr():
    buf = (ctypes.c_uint8 * 4096)()
    yield (ctypes.addressof(buf) + 15) // 16 * 16
    del buf


def _append(lib, pages, table, p, typ=0, q_heads=4, rotary=64, rope_rows=100, rows=1, k=None, q=None, q_out=None, ids=True):
    h = lambda **kw: _lib.Heads(**{**dict(data=p, row=512, head=64), **kw})
    k, q, q_out = k or h(), q or h(), q_out or h()
    r = ctypes.byref
    return lib.wush_kv_append(r(pages), r(table), typ, r(q), q_heads, r(q_out), r(k), r(h()), None, p, rope_rows, rotary, 0,
                              p if ids else None, p, rows, None, None)


def test_c_abi_refusals(ptr):
    lib, p = _lib.load(), ptr
    table = _lib.KVTable(p, 8, 3, 8)
    r = ctypes.byref
    lens = p
    assert _append(lib, _pages(p), table, p, rows=0) == 0
    assert _append(lib, _pages(None), table, p) == -1
    assert _append(lib, _pages(p), table, p, ids=False) == -1
    assert _append(lib, _pages(p), table, p, q_out=_lib.Heads(None, 512, 64)) == -1
    assert _append(lib, _pages(p), table, p, typ=2) == -4                 # queries have 16 bits
    assert _append(lib, _pages(p), table, p, typ=1) == -4                 # fp16 queries, bf16 pages
    assert _append(lib, _pages(p, type=3), table, p) == -4
    assert _append(lib, _pages(p, dim=264), table, p) == -2               # more than 256 channels
    assert _append(lib, _pages(p, dim=60), table, p) == -2                # no whole 16 bytes
    assert _append(lib, _pages(p, type=2, dim=72, k_scale=p, v_scale=p), table, p) == -2
    assert _append(lib, _pages(p, type=2), table, p) == -1                # 8-bit pages without scales
    assert _append(lib, _pages(p, k_scale=p, v_scale=p), table, p) == -1  # scales without 8-bit pages
    assert _append(lib, _pages(p, k_row=130), table, p) == -3
    assert _append(lib, _pages(p, v_page=-2048), table, p) == -2
    assert _append(lib, _pages(p + 8), table, p) == -3
    assert _append(lib, _pages(p, page_size=0), table, p) == -2
    assert _append(lib, _pages(p, num_pages=1 << 31), table, p) == -2
    assert _append(lib, _pages(p), _lib.KVTable(p, 8, 3, 0), p) == -2
    assert _append(lib, _pages(p), _lib.KVTable(p, 8, 3, 1 << 27), p) == -8   # 2^31 tokens
    assert _append(lib, _pages(p), table, p, rotary=24) == -2
    assert _append(lib, _pages(p), table, p, rotary=80) == -2             # more than the head
    assert _append(lib, _pages(p), table, p, rope_rows=0) == -2
    assert _append(lib, _pages(p), table, p, q_heads=0) == -2
    assert _append(lib, _pages(p), table, p, k=_lib.Heads(p + 2, 512, 64)) == -3
    assert _append(lib, _pages(p), table, p, k=_lib.Heads(p, 516, 64)) == -3
    assert _append(lib, _pages(p), table, p, rows=-1) == -2

    assert lib.wush_kv_bounds(r(_pages(p, bounds=None)), r(table), lens, 1, None, None) == -1
    assert lib.wush_kv_bounds(r(_pages(p, bounds_type=1)), r(table), lens, 1, None, None) == -4
    assert lib.wush_kv_bounds(r(_pages(p)), r(table), None, 1, None, None) == -1
    assert lib.wush_kv_bounds(r(_pages(p)), r(table), lens, -1, None, None) == -2
    assert lib.wush_kv_bounds(r(_pages(p)), r(table), lens, 0, None, None) == 0

    h = _lib.Heads(p, 512, 64)
    select = lambda pages=None, heads=4, top=4, sink=1, recent=1, work=p, nbytes=4096, q=h: lib.wush_kv_select_pages(
        r(pages or _pages(p)), r(table), 0, r(q), heads, lens, top, sink, recent, p, p, work, nbytes, None, None)
    need = lib.wush_kv_select_workspace_bytes(3, 2, 8)
    assert need >= 3 * 2 * 8 * 8
    assert select(heads=3) == -2                                          # not a multiple of the key heads
    assert select(top=0, sink=0, recent=0) == -2 and select(top=1) == -2 and select(sink=-1) == -2
    assert select(pages=_pages(p, bounds=None)) == -1 and select(work=None) == -1
    assert select(nbytes=need - 1) == -5
    assert select(q=_lib.Heads(p, 512, 60)) == -3

    nbytes = lib.wush_kv_attention_workspace_bytes(r(_pages(p)), 4)
    attend = lambda heads=4, window=0, pages=None, counts=None, top=0, out=h, q=h, lens=p, work=p, nbytes=1 << 40: \
        lib.wush_kv_attention(r(_pages(p)), r(table), 0, r(q), heads, r(out), None, lens, 0.125, window, pages, counts, top, work,
                              nbytes, None, None)
    assert attend(heads=5) == -2 and attend(window=-1) == -2
    assert attend(pages=p) == -1 and attend(counts=p) == -1               # they go together
    assert attend(pages=p, counts=p, top=0) == -2 and attend(pages=p, counts=p, top=1 << 28) == -2
    assert attend(pages=p, counts=p, top=4, window=5) == -4
    assert attend(out=_lib.Heads(None, 512, 64)) == -1 and attend(lens=None) == -1
    assert attend(q=_lib.Heads(p + 4, 512, 64)) == -3
    if nbytes:
        assert attend(nbytes=nbytes - 1) == -5
    empty = _lib.KVTable(None, 8, 0, 8)
    assert lib.wush_kv_attention(r(_pages(p)), r(empty), 0, r(h), 4, r(h), None, None, 1.0, 0, None, None, 0, None, 0, None, None) == 0


def test_cpu_tensors_are_refused():
    k = torch.zeros(4, 16, 2, 64, dtype=BF)
    with pytest.raises(_lib.WushB200Error, match="no CPU fallback"):
        paged_kv.PagedKVCache(k, k.clone())
    with pytest.raises(_lib.WushB200Error, match="no CPU fallback"):
        paged_kv.PagedKVCache.allocate(4, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="layout"):
        paged_kv.PagedKVCache.allocate(4, 16, 2, 64, device="cpu", layout="dhn")
    with pytest.raises(ValueError, match="dtype"):
        paged_kv.PagedKVCache.allocate(4, 16, 2, 64, dtype=torch.float32, device="cpu")


def test_pool_checks():
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)
    ok = lambda k, v=None, **kw: paged_kv._check_pool(k, k.clone() if v is None else v, kw.get("ks"), kw.get("vs"), kw.get("b"))
    ok(z(4, 16, 2, 64))
    ok(z(4, 2, 16, 64).transpose(1, 2))
    ok(z(4, 16, 2, 2, 64)[:, :, 0], z(4, 16, 2, 2, 64)[:, :, 1])
    ok(z(4, 16, 2, 64, dt=F8), ks=torch.ones(2), vs=torch.ones(2), b=z(4, 2, 2, 64, dt=HF))
    bad = [
        (z(4, 16, 128), {}), (z(0, 16, 2, 64), {}), (z(4, 16, 2, 64, dt=torch.float32), {}),
        (z(4, 16, 2, 264), {}), (z(4, 16, 2, 60), {}), (z(4, 16, 2, 72, dt=F8), dict(ks=torch.ones(2), vs=torch.ones(2))),
        (z(4, 16, 64, 2).transpose(2, 3), {}), (z(4, 16, 2, 68)[..., 4:], {}), (z(4, 16, 2, 68)[..., :64], {}),
        (z(4, 16, 2, 64, dt=F8), {}), (z(4, 16, 2, 64), dict(ks=torch.ones(2), vs=torch.ones(2))),
        (z(4, 16, 2, 64, dt=F8), dict(ks=torch.ones(3), vs=torch.ones(2))),
        (z(4, 16, 2, 64), dict(b=z(4, 2, 2, 64, dt=HF))), (z(4, 16, 2, 64), dict(b=z(4, 2, 64))),
    ]
    for k, kw in bad:
        with pytest.raises(ValueError):
            ok(k, **kw)
    with pytest.raises(ValueError):
        ok(z(4, 16, 2, 64), z(4, 16, 2, 64, dt=HF))
    with pytest.raises(ValueError):
        ok(z(4, 16, 2, 64), z(4, 16, 2, 32))


def test_rope_table():
    t = paged_kv.rope_table(50000, 64, base=10000.0)
    assert t.shape == (50000, 64) and t.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (49999, 0), (49999, 31), (777, 13)):
        a = p * 10000.0 ** (-2 * i / 64)
        # one rounding to fp32, on top of a float64 angle that is off by p 2^-52
        assert abs(float(t[p, i]) - math.cos(a)) <= 2.0 ** -24 and abs(float(t[p, 32 + i]) - math.sin(a)) <= 2.0 ** -24
    for bad in ((10, 0), (10, 3), (0, 16)):
        with pytest.raises(ValueError):
            paged_kv.rope_table(*bad)
