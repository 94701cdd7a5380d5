"""Paged key-value cache operators over pools, tables and batches of other shapes than the usual: keys and values interleaved
in one tensor, rows and heads with gaps between them, pools that begin inside a larger one, batches without a token, thousands
of sequences, rows of more heads than a block loads at once."""
import pytest
import torch

from tests import paged_reference as ref
from tests.test_paged_attention_cut_gpu import Long
from tests.test_paged_kv_gpu import BF, F8, HF, _dev, _gen, _randn, _status_clear

pytestmark = pytest.mark.gpu


def _pools(kind, total, page, kv, dim, dtype):
    """Two zeroed pools [total, page, kv, dim] of one kind, and the tensor they lie in (filled with a value of its own)."""
    size = {"pages": (total, 2, page, kv, dim), "rows": (total, page, 2, kv, dim), "heads": (total, page, kv, 2, dim),
            "halves": (total, page, kv, 2 * dim), "gaps": (2, total + 2, page + 1, kv + 3, dim + 16),
            "heads first": (2, kv, total, page, dim), "rows first": (2, page, kv, total, dim)}[kind]
    whole = torch.full(size, 5.0, dtype=torch.float32, device=_dev()).to(dtype)
    k, v = {"pages": lambda t: (t[:, 0], t[:, 1]), "rows": lambda t: (t[:, :, 0], t[:, :, 1]),
            "heads": lambda t: (t[:, :, :, 0], t[:, :, :, 1]), "halves": lambda t: (t[..., :dim], t[..., dim:]),
            "gaps": lambda t: tuple(x[1:1 + total, :page, 2:2 + kv, 16:] for x in t),
            "heads first": lambda t: tuple(x.permute(1, 2, 0, 3) for x in t),
            "rows first": lambda t: tuple(x.permute(2, 0, 1, 3) for x in t)}[kind](whole)
    return k, v, whole


@pytest.mark.parametrize("kind", ["pages", "rows", "heads", "halves", "gaps", "heads first", "rows first"])
@pytest.mark.parametrize("cache,page,dim", [(BF, 16, 128), (F8, 32, 64), (HF, 24, 80), (F8, 16, 256)])
def test_pools_of_any_strides(kind, cache, page, dim):
    """The same calls on a pool of this kind and on a contiguous one: the same results, and nothing between is touched."""
    from wush_b200 import paged_kv
    typ = HF if cache == HF else BF
    lens = [1300, 0, 3, page, 2 * page + 1]
    s = Long(lens, page=page, kv=3, dim=dim, cache=cache, seed=dim + page, bounds=True)
    bits = torch.uint8 if cache == F8 else torch.int16
    k, v, whole = _pools(kind, s.cache.num_pages, page, 3, dim, cache)
    k.view(bits).copy_(s.cache.k.view(bits))
    v.view(bits).copy_(s.cache.v.view(bits))
    other = paged_kv.PagedKVCache(k, v, s.cache.k_scale, s.cache.v_scale, torch.zeros_like(s.cache.bounds))
    x = _randn(s.g, 5, 12 + 6, dim).to(typ)
    ids = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=_dev())
    pos = s.seq_lens - 1
    rope = paged_kv.rope_table(2048, dim // 16 * 16 // 2 // 16 * 16 or 16, device=_dev())
    results = []
    for c in (s.cache, other):
        q = paged_kv.paged_kv_append(c, x[:, 12:15], x[:, 15:], s.table, ids, pos, q=x[:, :12], rope=rope)
        paged_kv.paged_kv_bounds(c, s.table, s.seq_lens, 2000)
        out, lse = paged_kv.paged_decode_attention(q, c, s.table, s.seq_lens, return_lse=True)
        near = paged_kv.paged_decode_attention(q, c, s.table, s.seq_lens, window=50)
        pages, counts = paged_kv.paged_select_pages(q, c, s.table, s.seq_lens, 7)
        few = paged_kv.paged_decode_attention(q, c, s.table, s.seq_lens, pages=pages, counts=counts)
        results.append((q, out, lse, near, pages, counts, few, c.bounds.view(torch.int16), c.k.view(bits), c.v.view(bits)))
    _status_clear()
    for a, b in zip(*results):
        assert torch.equal(a, b)
    s.check(results[1][0], results[1][1], results[1][2])
    k.zero_()
    v.zero_()
    if kind == "gaps":                                        # what lies between is as it was
        assert int((whole.float() == 5.0).sum()) == whole.numel() - 2 * k.numel()


def test_batches_without_a_token():
    """All lengths 0 under tables large enough to be cut, and selected pages of which there are none."""
    from wush_b200 import paged_kv
    for seqs in (1, 7, 200):
        s = Long([0] * seqs, page=16, kv=2, dim=64, bounds=True, width=300)
        q = _randn(s.g, seqs, 8, 64).to(BF)
        out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
        assert not out.any() and bool((lse == -float("inf")).all())
        pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 100)
        assert not counts.any() and bool((pages == -1).all())
        out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts, return_lse=True)
        assert not out.any() and bool((lse == -float("inf")).all())
        less = s.seq_lens - 5                                 # a negative length is no token either
        assert not paged_kv.paged_decode_attention(q, s.cache, s.table, less).any()
        paged_kv.paged_kv_bounds(s.cache, s.table, less, 10)
    _status_clear()


@pytest.mark.parametrize("cache,page,width", [(BF, 16, None), (F8, 16, 200), (BF, 8, 200)])
def test_thousands_of_sequences(cache, page, width):
    from wush_b200 import paged_kv
    lens = [(i * 37) % 50 for i in range(3000)]
    lens[1234], lens[2999] = 700, 333
    s = Long(lens, page=page, kv=2, dim=64, cache=cache, seed=5, bounds=True, width=width)
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, max(lens))
    q = (2.0 * _randn(s.g, 3000, 4, 64)).to(BF)
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
    pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 3)
    few, few_lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts, return_lse=True)
    _status_clear()
    assert torch.equal(counts, torch.tensor([min(3, -(-n // page)) for n in lens], dtype=torch.int32, device=_dev())[:, None].expand(3000, 2))
    some = [0, 1, 2, 49, 1233, 1234, 1235, 2047, 2048, 2998, 2999]
    chosen = [[pages[b, h, : int(counts[b, h])].tolist() for h in range(2)] for b in some]
    for b, want in zip(some, chosen):
        bounds = s.cache.bounds[s.table[b, : -(-lens[b] // page)].long()].double()
        for h in range(2):
            assert want[h] == ref.select([ref.scores(q[b, 2 * h:2 * h + 2].double(), x[h, 0], x[h, 1]) for x in bounds], 3, 1, 1)
    s.lens, s.table = [lens[b] for b in some], s.table[some]
    s.check(q[some], out[some], lse[some])
    s.check(q[some], few[some], few_lse[some], chosen=chosen)


@pytest.mark.parametrize("typ,cache,dim,rotary,interleaved,heads,kv,rows", [
    (BF, BF, 128, 128, False, 128, 8, 400), (BF, F8, 128, 64, True, 96, 12, 149), (HF, HF, 80, 48, False, 60, 30, 148),
    (HF, F8, 256, 256, True, 40, 5, 700), (BF, BF, 8, 0, False, 301, 7, 200), (BF, BF, 128, 128, True, 128, 8, 147)])
def test_append_of_many_rows_and_heads(typ, cache, dim, rotary, interleaved, heads, kv, rows):
    """More heads than a thread has under way at once, with all heads of a row in one block and with them spread over blocks:
    rotated queries and keys and the stored numbers against float64 (one rounding, and three of fp32 before it)."""
    from wush_b200 import paged_kv
    page, dev, g = 16, _dev(), _gen(rows)
    total = -(-rows // page) + 2
    one = (0.02 + 0.01 * torch.rand(kv, generator=g, device=dev)) if cache == F8 else None
    c = paged_kv.PagedKVCache.allocate(total, page, kv, dim, dtype=cache, device=dev, k_scale=one, v_scale=one, layout="hnd")
    table = torch.randperm(total, generator=g, device=dev)[None].to(torch.int32)
    x = _randn(g, rows, heads + 2 * kv, dim).to(typ)
    at = torch.randperm(rows, generator=g, device=dev).to(torch.int32)
    at[5] = -1                                                # padding
    rope = paged_kv.rope_table(rows, rotary, device=dev) if rotary else None
    q_out, k_out = torch.full_like(x[:, :heads], 9.0), torch.full_like(x[:, heads:heads + kv], 9.0)
    paged_kv.paged_kv_append(c, x[:, heads:heads + kv], x[:, heads + kv:], table, torch.zeros_like(at), at, q=x[:, :heads], rope=rope,
                             interleaved=interleaved, q_out=q_out, k_out=k_out)
    _status_clear()
    turned = x[:, : heads + kv].double().clone()
    if rotary:
        cos, sin = (t.double()[:, None] for t in rope[at.clamp(min=0).long()].split(rotary // 2, dim=1))
        a, b = (turned[..., 0:rotary:2].clone(), turned[..., 1:rotary:2].clone()) if interleaved else \
            (turned[..., : rotary // 2].clone(), turned[..., rotary // 2: rotary].clone())
        na, nb = a * cos - b * sin, b * cos + a * sin
        if interleaved:
            turned[..., 0:rotary:2], turned[..., 1:rotary:2] = na, nb
        else:
            turned[..., : rotary // 2], turned[..., rotary // 2: rotary] = na, nb
    slack = 3 * 2.0 ** -24 * 2 * float(x.double().abs().max()) + (2.0 ** -25 if typ == HF else 0.0)
    real = at >= 0
    got = torch.cat([q_out, k_out], dim=1).double()
    assert bool(((got - turned).abs()[real] <= (ref.HALF[typ] * turned.abs() + slack)[real]).all()) and bool((got[~real] == 9.0).all())
    place = at.clamp(min=0).long()
    where, row = table[0][place // page].long(), place % page
    bits = torch.uint8 if cache == F8 else torch.int16
    for pool, want in ((c.k, turned[:, heads:]), (c.v, x[:, heads + kv:].double())):
        stored = pool.view(bits)[where, row].view(cache).double()
        want, extra = (want / one.double()[:, None], slack / float(one.min()) + 2.0 ** -10) if cache == F8 else (want, slack)
        want = want.clamp(-448, 448) if cache == F8 else want
        assert bool(((stored - want).abs()[real] <= (ref.HALF[cache] * (1 + 2.0 ** -20) * want.abs() + extra)[real]).all())
    hidden = torch.ones(total, page, dtype=torch.bool, device=dev)
    hidden[where[real], row[real]] = False                    # rows that nobody named are as they were
    assert not c.k.view(bits)[hidden].any() and not c.v.view(bits)[hidden].any()
