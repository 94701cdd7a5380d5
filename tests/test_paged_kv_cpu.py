"""Paged key-value cache operators, what needs no GPU: refusals of the C ABI and of the Python layer, the rotation table."""
import ctypes
import math

import pytest
import torch

from wush_b200 import _lib, paged_kv

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


P, Q, I, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float
fields = lambda names, t: [(n, t) for n in names.split()]


class Pages(ctypes.Structure):
    _fields_ = fields("k v", P) + fields("k_page k_row k_head v_page v_row v_head", Q) + fields("k_scale v_scale bounds", P) \
        + fields("num_pages", Q) + fields("page_size heads dim type bounds_type", I)


class Table(ctypes.Structure):
    _fields_ = fields("block_table", P) + fields("stride seqs width", Q)


class Heads(ctypes.Structure):
    _fields_ = fields("data", P) + fields("row head", Q)


POOL = [("kv", Pages), ("table", Table)]


class Append(ctypes.Structure):
    _fields_ = POOL + fields("q q_out k v k_out", Heads) + fields("rope seq_ids positions status stream", P) \
        + fields("rows rope_rows", Q) + fields("type q_heads rotary interleaved", I)


class Bounds(ctypes.Structure):
    _fields_ = POOL + fields("seq_lens status stream", P) + fields("new_tokens", Q)


class Select(ctypes.Structure):
    _fields_ = POOL + fields("q", Heads) + fields("seq_lens pages counts workspace", P) + fields("workspace_bytes", ctypes.c_uint64) \
        + fields("status stream", P) + fields("type q_heads top sink recent", I)


class Attention(ctypes.Structure):
    _fields_ = POOL + fields("q out", Heads) + fields("lse seq_lens pages counts workspace", P) \
        + fields("workspace_bytes", ctypes.c_uint64) + fields("status stream", P) + fields("window", Q) + fields("type q_heads top", I) \
        + fields("scale", F)


def test_packed_structs_have_the_layout_of_the_header():
    for cls, packed in ((Append, paged_kv._APPEND), (Bounds, paged_kv._BOUNDS), (Select, paged_kv._SELECT), (Attention, paged_kv._ATTENTION)):
        assert paged_kv._PAGES.size == ctypes.sizeof(Pages) and ctypes.sizeof(cls) == ctypes.sizeof(Pages) + packed.size
        values = list(range(1, len(packed.unpack(bytes(packed.size))) + 1))
        got, flat = cls.from_buffer_copy(bytes(ctypes.sizeof(Pages)) + packed.pack(*values)), []
        for name, t in cls._fields_[1:]:
            v = getattr(got, name)
            flat += [getattr(v, n) for n, _ in t._fields_] if isinstance(v, ctypes.Structure) else [v]
        assert flat == values


def _pages(p, **kw):
    """A bf16 pool of 4 pages of 16 rows, 2 heads of 64 channels."""
    d = dict(k=p, v=p, k_page=2048, k_row=128, k_head=64, v_page=2048, v_row=128, v_head=64, k_scale=None, v_scale=None,
             bounds=p, num_pages=4, page_size=16, heads=2, dim=64, type=0, bounds_type=0)
    d.update(kw)
    return Pages(**d)


@pytest.fixture()
def ptr():
    buf = (ctypes.c_uint8 * 4096)()
    yield (ctypes.addressof(buf) + 15) // 16 * 16
    del buf


def test_c_abi_refusals(ptr):
    lib, p = _lib.load(), ptr
    h = lambda **kw: Heads(**{**dict(data=p, row=512, head=64), **kw})

    def call(fn, cls, base, kw):
        return getattr(lib, fn)(bytes(cls(**{**dict(kv=_pages(p), table=Table(p, 8, 3, 8)), **base, **kw})))
    append = lambda **kw: call("wush_kv_append", Append, dict(q=h(), q_out=h(), k=h(), v=h(), rope=p, seq_ids=p, positions=p, rows=1,
                                                             rope_rows=100, q_heads=4, rotary=64), kw)
    assert append(rows=0) == 0
    assert append(kv=_pages(None)) == -1 and append(seq_ids=None) == -1 and append(q_out=h(data=None)) == -1
    assert append(type=2) == -4                                            # queries have 16 bits
    assert append(type=1) == -4                                            # fp16 queries, bf16 pages
    assert append(kv=_pages(p, type=3)) == -4
    assert append(kv=_pages(p, dim=264)) == -2                             # more than 256 channels
    assert append(kv=_pages(p, dim=60)) == -2                              # no whole 16 bytes
    assert append(kv=_pages(p, type=2, dim=72, k_scale=p, v_scale=p)) == -2
    assert append(kv=_pages(p, type=2)) == -1                              # 8-bit pages without scales
    assert append(kv=_pages(p, k_scale=p, v_scale=p)) == -1                # scales without 8-bit pages
    assert append(kv=_pages(p, k_row=130)) == -3 and append(kv=_pages(p + 8)) == -3
    assert append(kv=_pages(p, v_page=-2048)) == -2 and append(kv=_pages(p, page_size=0)) == -2
    assert append(kv=_pages(p, num_pages=1 << 31)) == -2
    assert append(table=Table(p, 8, 3, 0)) == -2
    assert append(table=Table(p, 8, 3, 1 << 27)) == -8                     # 2^31 tokens
    assert append(rotary=24) == -2 and append(rotary=80) == -2 and append(rope_rows=0) == -2
    assert append(q_heads=0) == -2 and append(rows=-1) == -2
    assert append(k=h(data=p + 2)) == -3 and append(k=h(row=516)) == -3 and append(k_out=h(head=4)) == -3

    bounds = lambda **kw: call("wush_kv_bounds", Bounds, dict(seq_lens=p, new_tokens=1), kw)
    assert bounds(kv=_pages(p, bounds=None)) == -1 and bounds(kv=_pages(p, bounds_type=1)) == -4
    assert bounds(seq_lens=None) == -1 and bounds(new_tokens=-1) == -2 and bounds(new_tokens=0) == 0

    need = lib.wush_kv_select_workspace_bytes(3, 2, 8)
    assert need >= 3 * 2 * 8 * 8
    select = lambda **kw: call("wush_kv_select_pages", Select, dict(q=h(), q_heads=4, seq_lens=p, top=4, sink=1, recent=1, pages=p,
                                                                    counts=p, workspace=p, workspace_bytes=4096), kw)
    assert select(q_heads=3) == -2                                         # not a multiple of the key heads
    assert select(top=0, sink=0, recent=0) == -2 and select(top=1) == -2 and select(sink=-1) == -2
    assert select(kv=_pages(p, bounds=None)) == -1 and select(workspace=None) == -1 and select(counts=None) == -1
    assert select(workspace_bytes=need - 1) == -5 and select(q=h(head=60)) == -3

    nbytes = lib.wush_kv_attention_workspace_bytes(bytes(_pages(p)), 4)
    attend = lambda **kw: call("wush_kv_attention", Attention, dict(q=h(), out=h(), q_heads=4, seq_lens=p, scale=0.125, workspace=p,
                                                                    workspace_bytes=1 << 40), kw)
    assert attend(q_heads=5) == -2 and attend(window=-1) == -2
    assert attend(pages=p) == -1 and attend(counts=p) == -1                # they go together
    assert attend(pages=p, counts=p, top=0) == -2 and attend(pages=p, counts=p, top=1 << 28) == -2
    assert attend(pages=p, counts=p, top=4, window=5) == -4
    assert attend(out=h(data=None)) == -1 and attend(seq_lens=None) == -1 and attend(workspace=None) == -1
    assert attend(q=h(data=p + 4)) == -3 and attend(workspace=p + 4) == -3 and attend(workspace_bytes=nbytes - 1) == -5
    assert attend(table=Table(None, 8, 0, 8)) == 0
    for fn in ("wush_kv_append", "wush_kv_bounds", "wush_kv_select_pages", "wush_kv_attention"):
        assert getattr(lib, fn)(None) == -1


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
