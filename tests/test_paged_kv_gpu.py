"""Paged key-value cache operators on the GPU against their plain float64 forms (tests/paged_reference.py), at the sizes
and masks where they can go wrong.  Tolerances are derived in paged_reference.py and beside the tests."""
import math

import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _dev():
    return torch.device("cuda:0")


def _gen(seed):
    g = torch.Generator(device=_dev())
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=_dev())


class Setup:
    """A pool whose every free row holds NaN, random tables with unread entries far outside the pool, lengths `lens`."""

    def __init__(self, lens, page=16, kv=2, dim=64, cache=BF, layout="nhd", seed=0, spare=3, width=None, bounds=False):
        from wush_b200.paged_kv import PagedKVCache
        dev, g = _dev(), _gen(seed)
        self.lens, self.page, self.kv, self.dim, self.g = lens, page, kv, dim, g
        need = [-(-n // page) for n in lens]
        width = width or max(1, max(need, default=1))
        total = sum(need) + spare
        ks = vs = None
        if cache == F8:
            ks, vs = 0.02 + 0.02 * torch.rand(kv, generator=g, device=dev), 0.01 + 0.01 * torch.rand(kv, generator=g, device=dev)
        self.cache = PagedKVCache.allocate(total, page, kv, dim, dtype=cache, device=dev, layout=layout, k_scale=ks, v_scale=vs,
                                           bounds=bounds)
        order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        self.table = torch.full((max(1, len(lens)), width), 2 ** 30, dtype=torch.int32, device=dev)[: len(lens)]
        at = 0
        bits = torch.uint8 if cache == F8 else cache
        for pool, scale in ((self.cache.k, ks), (self.cache.v, vs)):
            x = _randn(g, total, page, kv, dim)
            x = x if scale is None else (x / scale[:, None]).clamp(-448, 448)
            pool.copy_(x.to(cache))
        filled = torch.zeros(total, page, dtype=torch.bool, device=dev)
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            for i in range(n):
                filled[order[at + i], : min(page, lens[b] - i * page)] = True
            at += n
        nan = torch.full((1,), math.nan, device=dev).to(cache).view(bits)
        for pool in (self.cache.k, self.cache.v):
            pool.view(bits)[~filled] = nan
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)

    def rows(self, b, head, which):
        pool, scale = (self.cache.k, self.cache.k_scale) if which == "k" else (self.cache.v, self.cache.v_scale)
        return ref.sequence(pool, self.table[b], self.lens[b], self.page, head, scale)

    def check_attention(self, q, out, lse, scale=None, window=0, chosen=None):
        """out / lse against float64; chosen[b][head]: pages of the sparse form."""
        group = q.shape[1] // self.kv
        scale = self.dim ** -0.5 if scale is None else scale
        single = self.cache.dtype == F8 and q.dtype == BF
        for b, n in enumerate(self.lens):
            for hk in range(self.kv):
                k, v = self.rows(b, hk, "k"), self.rows(b, hk, "v")
                if chosen is not None:
                    keep = [p for lp in chosen[b][hk] for p in range(lp * self.page, min(n, (lp + 1) * self.page))]
                    k, v = k[keep], v[keep]
                elif window:
                    k, v = k[max(0, n - window):], v[max(0, n - window):]
                for h in range(hk * group, (hk + 1) * group):
                    want, want_lse, mass = ref.attend(q[b, h].double(), k, v, scale)
                    tol = ref.attention_tolerance(want, len(k), self.dim, mass, float(v.abs().max()) if len(k) else 0.0, q.dtype, single)
                    err = (out[b, h].double() - want).abs()
                    assert bool((err <= tol).all()), (b, h, n, float((err - tol).max()))
                    if lse is not None:
                        if len(k) == 0:
                            assert float(lse[b, h]) == -math.inf
                        else:
                            assert abs(float(lse[b, h]) - want_lse) <= ref.lse_tolerance(want_lse, len(k), self.dim, mass)


def _status_clear():
    from wush_b200 import _lib
    _lib.check_status(_dev())


# ---- append ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", [BF, HF, F8])
@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, False), (64, 64, True), (128, 64, False), (96, 32, True),
                                                    (80, 80, False), (256, 0, False), (16, 16, True), (112, 96, False)])
def test_append_rotates_and_writes(cache, dim, rotary, interleaved):
    from wush_b200 import paged_kv
    typ = HF if cache == HF else BF
    s = Setup([0, 40, 7], page=24, kv=3, dim=dim, cache=cache, seed=dim + rotary, layout="hnd" if interleaved else "nhd")
    s.table[0, 0] = s.table[1, 0]                              # sequence 0 shares no page with rows written below
    g, heads = s.g, 6
    seq = [1, 2, 1, -1, 2, 1, 0]
    pos = [25, 0, 47, 3, 6, 0, -1]                            # rows 3 and 6 are padding
    pages = [int(s.table[a, p // 24]) if a >= 0 and p >= 0 else None for a, p in zip(seq, pos)]
    rows = len(seq)
    qkv = _randn(g, rows, heads + 6, dim).to(typ)             # slices of one fused projection
    qkv[3], qkv[6] = math.nan, math.nan
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + 3], qkv[:, heads + 3:]
    rope = paged_kv.rope_table(64, rotary, device=_dev()) if rotary else None
    before = (s.cache.k.clone(), s.cache.v.clone())
    ids = torch.tensor(seq, dtype=torch.int32, device=_dev())
    at = torch.tensor(pos, dtype=torch.int32, device=_dev())
    k_out = torch.full((rows, 3, dim), 7.0, dtype=typ, device=_dev())
    out = paged_kv.paged_kv_append(s.cache, k, v, s.table, ids, at, q=q, rope=rope, interleaved=interleaved, k_out=k_out)
    inplace = qkv.clone()
    iq, ik = inplace[:, :heads], inplace[:, heads:heads + 3]
    got = paged_kv.paged_kv_append(s.cache, ik, inplace[:, heads + 3:], s.table, ids, at, q=iq, rope=rope, interleaved=interleaved,
                                   q_out=iq, k_out=ik)
    assert got.data_ptr() == iq.data_ptr()
    _status_clear()
    written = torch.zeros(s.cache.num_pages, 24, dtype=torch.bool, device=_dev())
    for r in range(rows):
        if pages[r] is None:
            assert not out[r].any() and bool((k_out[r] == 7).all()) and bool(inplace[r].isnan().all())
            continue
        written[pages[r], pos[r] % 24] = True
        turn = rope[pos[r]].double() if rotary else torch.zeros(0, dtype=torch.float64, device=_dev())
        wq, wk = (ref.rotate(x[r].double(), turn, interleaved) for x in (q, k))
        # two fp32 products and their sum, then one rounding; |a c - b s| may cancel: 3 fp32 roundings of at most |a| + |b|
        slack = 3 * 2.0 ** -24 * 2 * float(qkv[r].double().abs().max())
        for got_, want in ((out[r], wq), (iq[r], wq), (k_out[r], wk), (ik[r], wk)):
            assert bool(((got_.double() - want).abs() <= ref.HALF[typ] * want.abs() + slack).all())
        stored_k, stored_v = s.cache.k[pages[r], pos[r] % 24].double(), s.cache.v[pages[r], pos[r] % 24].double()
        wv = v[r].double()
        if cache == F8:
            wk, wv = wk / s.cache.k_scale.double()[:, None], wv / s.cache.v_scale.double()[:, None]
            slack = slack / float(s.cache.k_scale.min()) + 2.0 ** -10                       # half the smallest e4m3 step, 2^-9
            wk, wv = wk.clamp(-448, 448), wv.clamp(-448, 448)
        elif typ == HF:
            slack += 2.0 ** -25
        for got_, want in ((stored_k, wk), (stored_v, wv)):
            assert bool(((got_ - want).abs() <= ref.HALF[cache] * (1 + 2.0 ** -20) * want.abs() + slack).all())
    bits = torch.uint8 if cache == F8 else torch.int16
    for now, then in zip((s.cache.k, s.cache.v), before):     # nothing else of the pool changed
        assert torch.equal(now.view(bits)[~written], then.view(bits)[~written])


def test_append_saturates_and_keeps_nan():
    from wush_b200 import paged_kv
    s = Setup([1], page=16, kv=1, dim=64, cache=F8)
    s.cache.k_scale.fill_(1.0)
    s.cache.v_scale.fill_(0.5)
    k = torch.zeros(1, 1, 64, dtype=BF, device=_dev())
    k[0, 0, :5] = torch.tensor([1e6, -1e6, math.inf, math.nan, 2.0 ** -9])
    zero = torch.zeros(1, dtype=torch.int32, device=_dev())
    paged_kv.paged_kv_append(s.cache, k, k, s.table, zero, zero)
    got = s.cache.k[int(s.table[0, 0]), 0, 0].float()
    assert got[:3].tolist() == [448, -448, 448] and bool(got[3].isnan()) and float(got[4]) == 2.0 ** -9
    assert float(s.cache.v[int(s.table[0, 0]), 0, 0, 4].float()) == 2.0 ** -8


def test_append_bad_indices_are_skipped_and_reported():
    from wush_b200 import _lib, paged_kv
    s = Setup([20, 20], page=16, kv=2, dim=64)
    rope = paged_kv.rope_table(24, 64, device=_dev())
    k = _randn(s.g, 1, 2, 64).to(BF)
    before = s.cache.k.clone()
    t = lambda x: torch.tensor([x], dtype=torch.int32, device=_dev())
    bad_table = s.table.clone()
    bad_table[1, 0] = s.cache.num_pages
    bad_table[0, 0] = -1
    for table, seq, pos in ((s.table, 2, 0), (s.table, 0, 32), (s.table, 0, 24), (bad_table, 1, 3), (bad_table, 0, 3)):
        q_out = torch.full((1, 2, 64), 5.0, dtype=BF, device=_dev())
        paged_kv.paged_kv_append(s.cache, k, k, table, t(seq), t(pos), q=k, q_out=q_out, rope=rope)
        with pytest.raises(_lib.WushB200Error, match="outside its table"):
            _lib.check_status(_dev())
        _status_clear()
        assert torch.equal(before.view(torch.int16), s.cache.k.view(torch.int16)) and bool((q_out == 5).all())


def test_append_many_rows_and_no_rows():
    from wush_b200 import paged_kv
    n = 3001
    s = Setup([n], page=8, kv=2, dim=128, seed=5)
    k, v = _randn(s.g, n, 2, 128).to(BF), _randn(s.g, n, 2, 128).to(BF)
    pos = torch.randperm(n, generator=s.g, device=_dev()).to(torch.int32)
    paged_kv.paged_kv_append(s.cache, k, v, s.table, torch.zeros_like(pos), pos)
    where = s.table[0][pos.long() // 8].long()
    assert torch.equal(s.cache.k[where, pos.long() % 8], k) and torch.equal(s.cache.v[where, pos.long() % 8], v)
    none = torch.zeros(0, dtype=torch.int32, device=_dev())
    assert paged_kv.paged_kv_append(s.cache, k[:0], v[:0], s.table, none, none, q=k[:0]).shape == (0, 2, 128)
    _status_clear()


# ---- bounds ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache,dim,page,new", [(BF, 64, 16, 1), (HF, 96, 24, 30), (F8, 128, 64, 1000), (F8, 256, 1, 3), (BF, 8, 128, 17),
                                                (HF, 256, 16, 2 ** 31 - 1)])
def test_bounds(cache, dim, page, new):
    from wush_b200 import paged_kv
    s = Setup([1, 0, 130, 48, page, page + 1], page=page, kv=3, dim=dim, cache=cache, bounds=True, seed=dim)
    s.cache.bounds.fill_(77.0)
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, new)
    _status_clear()
    want = torch.full_like(s.cache.bounds, 77.0)
    for b, n in enumerate(s.lens):
        for lp in range(max(0, n - new) // page, -(-n // page)):
            keys = s.cache.k[int(s.table[b, lp]), : min(page, n - lp * page)].float()
            want[int(s.table[b, lp])] = torch.stack([keys.amin(0), keys.amax(0)], dim=1).to(want.dtype)
    assert torch.equal(s.cache.bounds, want)                   # stored numbers: no rounding at all


def test_bounds_keep_nan_and_infinity():
    from wush_b200 import paged_kv
    s = Setup([10], page=16, kv=1, dim=64, bounds=True)
    p = int(s.table[0, 0])
    s.cache.k[p, 3, 0, 5], s.cache.k[p, 4, 0, 6], s.cache.k[p, 9, 0, 7] = math.nan, math.inf, -math.inf
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, 1)
    b = s.cache.bounds[p, 0].float()
    assert bool(b[:, 5].isnan().all()) and float(b[1, 6]) == math.inf and float(b[0, 7]) == -math.inf
    assert int(b.isnan().sum()) == 2


# ---- attention ---------------------------------------------------------------------------------------------------------

CASES = [   # (queries, cache, dim, page, kv, heads, lens, window, layout)
    (BF, BF, 128, 64, 2, 16, [1, 63, 64, 65, 0, 200], 0, "nhd"),
    (BF, BF, 128, 16, 1, 1, [17, 1, 2], 0, "hnd"),
    (HF, HF, 64, 16, 4, 4, [37, 500], 0, "nhd"),
    (HF, HF, 96, 24, 2, 12, [301, 24, 23, 25], 100, "nhd"),
    (BF, BF, 80, 8, 1, 7, [129, 8, 9], 1, "hnd"),
    (BF, BF, 256, 32, 2, 6, [77, 33], 0, "nhd"),
    (HF, HF, 256, 1, 1, 16, [50], 33, "nhd"),
    (BF, F8, 128, 64, 2, 16, [1000, 1, 15, 16, 31], 0, "nhd"),
    (HF, F8, 64, 32, 3, 9, [255, 256, 257], 64, "hnd"),
    (BF, F8, 256, 16, 1, 8, [95], 0, "nhd"),
    (BF, F8, 48, 5, 2, 4, [61, 4], 7, "nhd"),
    (BF, BF, 128, 16, 1, 40, [90, 3], 0, "nhd"),              # more queries of a key head than a tile has rows
    (BF, F8, 112, 128, 1, 24, [300], 0, "hnd"),
    (BF, BF, 8, 16, 2, 2, [19], 0, "nhd"),
    (HF, F8, 16, 16, 2, 34, [40, 41], 0, "nhd"),
    (BF, BF, 192, 48, 2, 10, [150, 49], 0, "nhd"),
    (BF, BF, 128, 64, 1, 8, [7000], 0, "nhd"),                # split over the length
    (BF, F8, 128, 16, 1, 16, [9001, 3], 0, "nhd"),
]


@pytest.mark.parametrize("typ,cache,dim,page,kv,heads,lens,window,layout", CASES)
def test_attention(typ, cache, dim, page, kv, heads, lens, window, layout):
    from wush_b200 import paged_kv
    s = Setup(lens, page=page, kv=kv, dim=dim, cache=cache, layout=layout, seed=dim + page + heads)
    q = (2.0 * _randn(s.g, len(lens), heads, dim)).to(typ)
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, window=window, return_lse=True)
    _status_clear()
    assert out.dtype == typ and out.shape == q.shape and lse.dtype == torch.float32
    s.check_attention(q, out, lse, window=window)
    again = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, window=window)
    assert torch.equal(out, again)                            # the same bits every time


@pytest.mark.parametrize("scale", [0.0, -0.25, 30.0])
def test_attention_scales(scale):
    from wush_b200 import paged_kv
    s = Setup([100, 5], page=16, kv=1, dim=64, seed=3)
    q = _randn(s.g, 2, 8, 64).to(BF)
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, scale=scale, return_lse=True)
    s.check_attention(q, out, lse, scale=scale)


@pytest.mark.parametrize("cache", [BF, F8])
def test_attention_strided_queries_and_outputs_in_place(cache):
    from wush_b200 import paged_kv
    s = Setup([90, 0, 300], page=16, kv=2, dim=64, cache=cache, seed=9)
    wide = _randn(s.g, 3, 12, 64).to(BF)
    q = wide[:, 2:10]
    keep, rest = q.clone(), wide.clone()
    out = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, out=q)
    assert out.data_ptr() == q.data_ptr()
    s.check_attention(keep, out, None)
    assert torch.equal(wide[:, :2], rest[:, :2]) and torch.equal(wide[:, 10:], rest[:, 10:])
    table = torch.full((3, s.table.shape[1] + 5), 2 ** 30, dtype=torch.int32, device=_dev())
    table[:, : s.table.shape[1]] = s.table
    other = paged_kv.paged_decode_attention(keep, s.cache, table[:, : s.table.shape[1]], s.seq_lens)
    assert torch.equal(other, out)


def test_attention_with_infinities_and_nan():
    """A masked NaN or infinity has no effect; a visible NaN key makes its head NaN and no other; a logit of -inf weighs
    nothing; only -inf logits leave an empty row."""
    from wush_b200 import paged_kv
    s = Setup([40, 40], page=16, kv=2, dim=64, seed=4)
    q = _randn(s.g, 2, 4, 64).to(BF)
    q[0] = q[0].abs() + 0.1
    s.cache.k[int(s.table[0, 1]), 3, 0] = -math.inf           # token 19 of sequence 0, head 0: logit -inf
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
    k, v = s.rows(0, 0, "k"), s.rows(0, 0, "v")
    keep = [i for i in range(40) if i != 19]
    want, _, mass = ref.attend(q[0, 1].double(), k[keep], v[keep], 64 ** -0.5)
    tol = ref.attention_tolerance(want, 40, 64, mass, float(v.abs().max()), BF, False)
    assert bool(((out[0, 1].double() - want).abs() <= tol).all())
    s.cache.k[int(s.table[1, 0]), 2, 1, 7] = math.nan
    out2 = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens)
    assert bool(out2[1, 2:].isnan().all()) and torch.equal(out2[1, :2], out[1, :2]) and torch.equal(out2[0], out[0])
    for lp in range(3):
        s.cache.k[int(s.table[0, lp]), :, 0] = -math.inf
    out3, lse3 = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
    assert not out3[0, :2].any() and bool((lse3[0, :2] == -math.inf).all()) and torch.equal(out3[0, 2:], out[0, 2:])


def test_attention_bad_pages_are_left_out_and_reported():
    from wush_b200 import _lib, paged_kv
    s = Setup([48, 48], page=16, kv=1, dim=64, seed=6)
    q = _randn(s.g, 2, 2, 64).to(BF)
    s.table[0, 1] = s.cache.num_pages + 7
    out = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens)
    with pytest.raises(_lib.WushB200Error, match="outside its table"):
        _lib.check_status(_dev())
    _status_clear()
    s.lens, s.table = [48, 48], s.table.clone()
    keep = list(range(16)) + list(range(32, 48))
    s.table[0, 1] = 0
    k, v = s.rows(0, 0, "k")[keep], s.rows(0, 0, "v")[keep]
    want, _, mass = ref.attend(q[0, 1].double(), k, v, 64 ** -0.5)
    tol = ref.attention_tolerance(want, 32, 64, mass, float(v.abs().max()), BF, False)
    assert bool(((out[0, 1].double() - want).abs() <= tol).all())
    # a length beyond the table is cut at it
    long = torch.tensor([48, 49], dtype=torch.int32, device=_dev())
    cut = paged_kv.paged_decode_attention(q, s.cache, s.table, long)
    with pytest.raises(_lib.WushB200Error, match="outside its table"):
        _lib.check_status(_dev())
    assert torch.equal(cut[1], out[1])


def test_attention_offsets_beyond_32_bits():
    """Pages whose first element lies beyond 2^32 elements and bytes."""
    from wush_b200.paged_kv import PagedKVCache, paged_decode_attention, paged_kv_append, paged_kv_bounds
    dev, page, kv, d = _dev(), 64, 8, 128
    total = (2 ** 32) // (page * kv * d) + 40                  # 8.6 GB of keys, and the same of values
    k = torch.empty(total, page, kv, d, dtype=BF, device=dev)
    v = torch.empty(total, page, kv, d, dtype=BF, device=dev)
    bounds = torch.empty(total, kv, 2, d, dtype=BF, device=dev)
    cache = PagedKVCache(k, v, bounds=bounds)
    s = Setup([1], page=page, kv=kv, dim=d, seed=8)
    s.cache, s.lens = cache, [130]
    s.table = torch.tensor([[total - 1, 5, total - 30]], dtype=torch.int32, device=dev)
    s.seq_lens = torch.tensor([130], dtype=torch.int32, device=dev)
    new = _randn(s.g, 130, 2 * kv, d).to(BF)
    pos = torch.arange(130, dtype=torch.int32, device=dev)
    paged_kv_append(cache, new[:, :kv], new[:, kv:], s.table, torch.zeros_like(pos), pos)
    paged_kv_bounds(cache, s.table, s.seq_lens, 130)
    assert torch.equal(k[total - 1], new[:64, :kv]) and torch.equal(v[5], new[64:128, kv:])
    assert torch.equal(bounds[total - 1, :, 1], new[:64, :kv].amax(0))
    q = _randn(s.g, 1, kv, d).to(BF)
    out, lse = paged_decode_attention(q, cache, s.table, s.seq_lens, return_lse=True)
    _status_clear()
    s.check_attention(q, out, lse)


def test_a_page_of_nearly_2_31_rows():
    """One page that is a whole table: its rows and a length's, added up, pass 2^31 (34 GB; keys and values share it)."""
    from wush_b200.paged_kv import PagedKVCache, paged_decode_attention, paged_kv_bounds, paged_select_pages
    dev, rows, n, d = _dev(), 2 ** 31 - 2 ** 16 - 16, 70000, 16
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 34 GB")
    s = Setup([1], page=16, kv=1, dim=d, cache=F8, seed=9)
    pool = torch.empty(1, rows, 1, d, dtype=torch.uint8, device=dev).view(F8)
    pool[0, :n] = _randn(s.g, n, 1, d).mul(8).clamp(-448, 448).to(F8)
    one = torch.full((1,), 0.125, device=dev)
    s.cache = PagedKVCache(pool, pool, k_scale=one, v_scale=one, bounds=torch.empty(1, 1, 2, d, dtype=BF, device=dev))
    s.lens = [n]
    s.table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    s.seq_lens = torch.tensor([n], dtype=torch.int32, device=dev)
    paged_kv_bounds(s.cache, s.table, s.seq_lens)
    stored = pool[0, :n, 0].float() * 0.125                    # (exact)
    s.rows = lambda b, head, which: stored.double()
    assert torch.equal(s.cache.bounds[0, 0].float() * 0.125, torch.stack([stored.amin(0), stored.amax(0)]))
    q = _randn(s.g, 1, 2, d).to(BF)
    pages, counts = paged_select_pages(q, s.cache, s.table, s.seq_lens, 2)
    assert pages.tolist() == [[[0, -1]]] and counts.tolist() == [[1]]
    out, lse = paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
    _status_clear()
    s.check_attention(q, out, lse)
    out, lse = paged_decode_attention(q, s.cache, s.table, s.seq_lens, window=1000, return_lse=True)
    _status_clear()
    s.check_attention(q, out, lse, window=1000)


# ---- selection ---------------------------------------------------------------------------------------------------------

def _expected_pages(s, q, top, sink, recent):
    group = q.shape[1] // s.kv
    out = []
    for b, n in enumerate(s.lens):
        count = -(-n // s.page)
        low_high = s.cache.bounds[s.table[b, :count].long()].double()
        out.append([ref.select([ref.scores(q[b, h * group:(h + 1) * group].double(), x[h, 0], x[h, 1]) for x in low_high], top, sink,
                               recent) for h in range(s.kv)])
    return out


@pytest.mark.parametrize("typ,cache,dim,page,heads,top,sink,recent", [
    (BF, BF, 128, 16, 16, 8, 1, 1), (HF, HF, 64, 8, 2, 5, 0, 0), (BF, F8, 96, 4, 10, 16, 2, 3), (HF, F8, 256, 16, 6, 3, 1, 2),
    (BF, BF, 80, 1, 4, 64, 1, 1), (BF, BF, 16, 2, 24, 1, 0, 1), (BF, F8, 192, 32, 2, 2, 1, 1), (BF, BF, 8, 16, 2, 4, 2, 2)])
def test_selection_and_sparse_attention(typ, cache, dim, page, heads, top, sink, recent):
    from wush_b200 import paged_kv
    lens = [page * 40 + 3, 0, 1, page * top, page * top + 1, page * 9]
    s = Setup(lens, page=page, kv=2, dim=dim, cache=cache, seed=dim + top, bounds=True)
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, max(lens))
    q = (2.0 * _randn(s.g, len(lens), heads, dim)).to(typ)
    pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, top, sink=sink, recent=recent)
    _status_clear()
    want = _expected_pages(s, q, top, sink, recent)
    for b in range(len(lens)):
        for h in range(2):
            assert int(counts[b, h]) == len(want[b][h])
            assert pages[b, h].tolist() == want[b][h] + [-1] * (top - len(want[b][h])), (b, h)
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts, return_lse=True)
    _status_clear()
    s.check_attention(q, out, lse, chosen=want)


def test_selection_takes_the_lowest_page_among_equals_and_nan_first():
    from wush_b200 import paged_kv
    s = Setup([16 * 2000], page=16, kv=1, dim=64, seed=2, bounds=True)
    q = torch.ones(1, 1, 64, dtype=BF, device=_dev())
    s.cache.bounds.zero_()
    for lp, x in ((1500, 2.0), (700, 2.0), (1999, -5.0), (1998, math.nan)):
        s.cache.bounds[int(s.table[0, lp])] = x
    s.cache.bounds[int(s.table[0, 3])] = -0.0
    s.cache.bounds[int(s.table[0, 1997]), 0, 0, 5] = -math.inf      # only the lower bound, which a positive query does not use
    pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 6, sink=0, recent=0)
    assert pages[0, 0].tolist() == [0, 1, 700, 1500, 1997, 1998] and int(counts[0, 0]) == 6
    pages, _ = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 6, sink=2, recent=1)
    assert pages[0, 0].tolist() == [0, 1, 700, 1997, 1998, 1999]
    pages, _ = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 5, sink=2, recent=3)
    assert pages[0, 0].tolist() == [0, 1, 1997, 1998, 1999]
    pages, _ = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 1999, sink=0, recent=0)
    assert pages[0, 0].tolist() == list(range(1999))
    pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 2100)
    assert pages[0, 0].tolist() == list(range(2000)) + [-1] * 100 and int(counts[0, 0]) == 2000


@pytest.mark.parametrize("width", [1000, 1025, 3000, 8192, 8193, 20000])
def test_selection_over_many_pages(width):
    """Widths around the sizes at which the kernel changes its block, with many equal scores across the border."""
    from wush_b200 import paged_kv
    from wush_b200.paged_kv import PagedKVCache
    g, dev = _gen(width), _dev()
    lens = [width, width - 7, width // 2]
    pool = PagedKVCache.allocate(width, 1, 1, 8, device=dev, bounds=True)
    pool.bounds.copy_(torch.randint(-3, 4, pool.bounds.shape, generator=g, device=dev).sort(dim=2).values.to(BF))
    table = torch.stack([torch.randperm(width, generator=g, device=dev) for _ in lens]).to(torch.int32)
    q = torch.randint(-2, 3, (3, 2, 8), generator=g, device=dev).to(BF)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    for top, sink, recent in ((1, 0, 0), (77, 1, 1), (width // 3, 5, 0)):
        pages, counts = paged_kv.paged_select_pages(q, pool, table, seq_lens, top, sink=sink, recent=recent)
        for b, n in enumerate(lens):
            bound = pool.bounds[table[b, :n].long(), 0].double()
            score = torch.maximum(q[b].double()[:, None] * bound[:, 0], q[b].double()[:, None] * bound[:, 1]).sum(2).amax(0)
            want = ref.select(score.tolist(), top, sink, recent)
            assert int(counts[b, 0]) == len(want) and pages[b, 0, : len(want)].tolist() == want, (b, top)
    _status_clear()


@pytest.mark.parametrize("typ,bounds", [(BF, BF), (HF, HF), (HF, BF), (BF, HF)])
@pytest.mark.parametrize("crowd,width", [(3, 900), (200, 900), (900, 900), (900, 9000)])
def test_selection_where_fp32_scores_cannot_decide(typ, bounds, crowd, width):
    """`crowd` pages of `width` are equal but for terms of 2^12 and -2^12 in other channels and one of -2^-14 to 2^-14: fp32
    sums lose it.  The border runs through them; bounds of the other 16-bit type than the queries' go with 8-bit pages."""
    from wush_b200 import paged_kv
    from wush_b200.paged_kv import PagedKVCache
    g, dev = _gen(crowd + width), _dev()
    one = torch.ones(2, device=dev)
    cache = F8 if typ != bounds else typ
    data = torch.zeros(width, 16, 2, 128, dtype=cache, device=dev)
    pool = PagedKVCache(data, data, k_scale=one if cache == F8 else None, v_scale=one if cache == F8 else None,
                        bounds=torch.zeros(width, 2, 2, 128, dtype=bounds, device=dev))
    low = torch.randn(width, 2, 128, generator=g, device=dev) - 4
    who = torch.randperm(width, generator=g, device=dev)[:crowd]
    low[who] = 0.0
    for h in range(2):
        at = torch.randint(0, 63, (crowd,), generator=g, device=dev)
        low[who, h, at], low[who, h, at + 64] = 2.0 ** 12, -2.0 ** 12
        low[who, h, 63] = 2.0 ** -14 * torch.randint(-1, 2, (crowd,), generator=g, device=dev).float()
    pool.bounds[:, :, 0] = low.to(bounds)
    pool.bounds[:, :, 1] = pool.bounds[:, :, 0]
    q = torch.ones(1, 6, 128, dtype=typ, device=dev)
    q[0, 4] = 0.5
    table = torch.randperm(width, generator=g, device=dev).to(torch.int32)[None]
    lens = torch.tensor([16 * width], dtype=torch.int32, device=dev)
    for top, sink, recent in ((max(2, crowd // 2), 0, 0), (crowd // 3 + 3, 1, 1), (1, 0, 0)):
        pages, counts = paged_kv.paged_select_pages(q, pool, table, lens, top, sink=sink, recent=recent)
        for h in range(2):
            b = pool.bounds[table[0].long(), h].double()
            score = torch.stack([torch.maximum(q[0, x].double() * b[:, 0], q[0, x].double() * b[:, 1]).sum(1) for x in range(3 * h, 3 * h + 3)])
            assert pages[0, h].tolist() == ref.select(score.amax(0).tolist(), top, sink, recent), (top, h)
    # one page that is not finite: every score is computed again
    pool.bounds[int(table[0, width // 2]), 0, 1, 7] = math.inf
    pages, _ = paged_kv.paged_select_pages(q, pool, table, lens, 2, sink=0, recent=0)
    assert width // 2 in pages[0, 0].tolist()
    _status_clear()


def test_selection_of_scores_below_the_smallest_fp32_number():
    """Queries of 2^-70 and keys of 2^-70: fp32 products vanish, 64-bit ones do not."""
    from wush_b200 import paged_kv
    s = Setup([16 * 300], page=16, kv=1, dim=64, seed=2, bounds=True)
    s.cache.bounds.copy_((_randn(s.g, 303, 1, 2, 64).sort(dim=2).values * 2.0 ** -70).to(BF))
    q = (_randn(s.g, 1, 3, 64) * 2.0 ** -70).to(BF)
    pages, _ = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 40, sink=1, recent=1)
    assert pages[0, 0].tolist() == _expected_pages(s, q, 40, 1, 1)[0][0]
    _status_clear()


def test_selection_close_scores_do_not_depend_on_the_order_of_the_sum():
    """Pages whose scores differ only in the 40th bit: terms of 2^20 and -2^20 around one of 2^-20."""
    from wush_b200 import paged_kv
    s = Setup([16 * 64], page=16, kv=1, dim=64, seed=2, bounds=True)
    q = torch.ones(1, 1, 64, dtype=BF, device=_dev())
    s.cache.bounds.zero_()
    for lp in range(64):
        row = s.cache.bounds[int(s.table[0, lp]), 0]
        row[:, lp] = 2.0 ** 20
        row[:, (lp + 17) % 64] = -2.0 ** 20
        if lp in (9, 33, 60):
            row[:, (lp + 5) % 64] = 2.0 ** -20
    pages, _ = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 3, sink=0, recent=0)
    assert pages[0, 0].tolist() == [9, 33, 60]


def test_sparse_attention_over_given_pages():
    """Lists of the caller: any order, a page twice, an empty list; negative or too large entries are left out and reported."""
    from wush_b200 import _lib, paged_kv
    s = Setup([70, 33], page=16, kv=2, dim=64, seed=11)
    q = _randn(s.g, 2, 8, 64).to(BF)
    pages = torch.tensor([[[4, 0, 2], [3, 3, 7]], [[1, 9, 9], [2, 0, 1]]], dtype=torch.int32, device=_dev())
    counts = torch.tensor([[3, 2], [0, 3]], dtype=torch.int32, device=_dev())
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts, return_lse=True)
    _status_clear()
    s.check_attention(q, out, lse, chosen=[[[4, 0, 2], [3, 3]], [[], [2, 0, 1]]])
    counts[0, 1] = 3                                           # entry 7: outside the table
    bad = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts)
    with pytest.raises(_lib.WushB200Error, match="outside its table"):
        _lib.check_status(_dev())
    assert torch.equal(bad, out)
    pages[0, 1, 2] = -1
    assert torch.equal(paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts), out)
    with pytest.raises(_lib.WushB200Error, match="outside its table"):
        _lib.check_status(_dev())


# ---- together, streams, graphs -----------------------------------------------------------------------------------------

def _steps(s, rope, tokens, heads, stream_of=None):
    """A prompt, then tokens one by one; returns the outputs of every step."""
    from wush_b200 import paged_kv
    outs = []
    for t in tokens:
        q = paged_kv.paged_kv_append(s.cache, t["k"], t["v"], s.table, t["ids"], t["pos"], q=t["q"], rope=rope)
        paged_kv.paged_kv_bounds(s.cache, s.table, t["lens"], t["new"])
        if t["new"] == 1:
            pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, t["lens"], 4)
            outs.append(paged_kv.paged_decode_attention(q, s.cache, s.table, t["lens"]))
            outs.append(paged_kv.paged_decode_attention(q, s.cache, s.table, t["lens"], pages=pages, counts=counts))
    return outs


def _token_plan(g, prompt, steps, heads, kv, dim):
    dev, n = _dev(), len(prompt)
    plan = []
    ids = torch.cat([torch.full((p,), b, dtype=torch.int32, device=dev) for b, p in enumerate(prompt)])
    pos = torch.cat([torch.arange(p, dtype=torch.int32, device=dev) for p in prompt])
    for step in range(steps + 1):
        rows = len(ids) if step == 0 else n
        lens = torch.tensor([p + step for p in prompt], dtype=torch.int32, device=dev)
        x = _randn(g, rows, heads + 2 * kv, dim).to(BF)
        plan.append({"q": x[:, :heads], "k": x[:, heads:heads + kv], "v": x[:, heads + kv:], "lens": lens,
                     "ids": ids if step == 0 else torch.arange(n, dtype=torch.int32, device=dev),
                     "pos": pos if step == 0 else lens - 1, "new": max(prompt) if step == 0 else 1})
    return plan


@pytest.mark.parametrize("cache", [BF, F8])
def test_prompt_and_tokens_together(cache):
    """Append, bounds, selection and attention as a generation loop uses them, against float64 attention over the
    contiguous history of rotated keys and values (the pool's own rounding taken from the pool)."""
    from wush_b200 import paged_kv
    heads, kv, dim, page, prompt, steps = 8, 2, 64, 16, [37, 90, 1], 5
    s = Setup([p + steps for p in prompt], page=page, kv=kv, dim=dim, cache=cache, bounds=True, seed=21)
    rope = paged_kv.rope_table(256, dim, device=_dev())
    plan = _token_plan(s.g, prompt, steps, heads, kv, dim)
    outs = _steps(s, rope, plan, heads)
    _status_clear()
    for step in range(1, steps + 1):
        t = plan[step]
        s.lens = [p + step for p in prompt]
        q = torch.stack([ref.rotate(t["q"][b].double(), rope[s.lens[b] - 1].double(), False) for b in range(3)]).to(BF)
        # the queries' own rounding may differ by one step in the rare tie: compare with what the kernel was given
        got_q = paged_kv.paged_kv_append(s.cache, t["k"], t["v"], s.table, t["ids"], t["pos"], q=t["q"], rope=rope)
        assert float((got_q.float() - q.float()).abs().max()) <= 2.0 ** -7 * float(q.float().abs().max())
        s.check_attention(got_q, outs[2 * step - 2], None)
        paged_kv.paged_kv_bounds(s.cache, s.table, t["lens"], 1)


def test_another_stream_and_captured_graphs():
    """The loop on a side stream, captured into two graphs (which do not share scratch with each other or with eager
    calls) and replayed with new inputs, gives the bits of the eager loop."""
    from wush_b200 import paged_kv
    heads, kv, dim = 16, 2, 128
    s = Setup([3000, 17], page=16, kv=kv, dim=dim, bounds=True, seed=31)
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, 3000)
    qa, qb = (_randn(s.g, 2, heads, dim).to(BF) for _ in range(2))

    def both(q):
        pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 12)
        return (paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens), pages,
                paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts))
    want_a, want_b = both(qa), both(qb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = both(qa)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(on_side, want_a))
    held, graphs, results = [qa.clone(), qb.clone()], [], []
    for q in held:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            results.append(both(q))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        eager = both(qb)
        torch.cuda.synchronize()
        for got, want in zip(results + [eager], (want_a, want_b, want_b)):
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        held[0].copy_(qa)
    held[0].copy_(qb)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(results[0], want_b))
    _status_clear()


def test_operators_captured_behind_copies_and_fills():
    """The kernels may start while the one before them ends; in a graph that one can also be a copy or a memset."""
    from wush_b200 import paged_kv
    heads, kv, dim = 8, 2, 64
    s = Setup([700, 33, 5], page=16, kv=kv, dim=dim, bounds=True, seed=41)
    rope = paged_kv.rope_table(1024, dim, device=_dev())
    ids = torch.arange(3, dtype=torch.int32, device=_dev())
    src = [_randn(s.g, 3, heads + 2 * kv, dim).to(BF) for _ in range(3)]
    x = torch.empty_like(src[0])
    lens = s.seq_lens.clone()

    def step():
        y = torch.empty_like(x)
        y.copy_(x)                                             # a device-to-device copy in front of the append's fill
        q = paged_kv.paged_kv_append(s.cache, y[:, heads:heads + kv], y[:, heads + kv:], s.table, ids, lens - 1, q=y[:, :heads], rope=rope)
        s.cache.bounds[int(0)].copy_(s.cache.bounds[int(0)].clone())
        paged_kv.paged_kv_bounds(s.cache, s.table, lens)
        z = torch.zeros(3, heads, dim, dtype=BF, device=_dev())
        out = paged_kv.paged_decode_attention(q, s.cache, s.table, lens, out=z)
        w = torch.zeros(4096, device=_dev())
        pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, lens, 5)
        w.zero_()
        return out, pages, counts, paged_kv.paged_decode_attention(q, s.cache, s.table, lens, pages=pages, counts=counts)
    want = []
    for v in src:
        x.copy_(v)
        want.append([t.clone() for t in step()])
    x.copy_(src[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for v, w in zip(src, want):
            x.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w))
    _status_clear()


def test_operators_captured_on_forked_streams():
    """The first kernel of a forked stream waits for another stream's work, and for two streams' after a join."""
    from wush_b200 import paged_kv
    s = Setup([900, 40], page=16, kv=2, dim=64, bounds=True, seed=43)
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, 900)
    x = _randn(s.g, 2, 8, 64).to(BF)
    src = [x.clone(), _randn(s.g, 2, 8, 64).to(BF)]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]

    def step():
        main = torch.cuda.current_stream()
        q = x * 2
        outs = []
        for st in sides:
            st.wait_stream(main)
            with torch.cuda.stream(st):
                outs.append(paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens))
                outs += paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 9)
        for st in sides:
            main.wait_stream(st)
        outs.append(paged_kv.paged_decode_attention(outs[0], s.cache, s.table, s.seq_lens, pages=outs[4], counts=outs[5]))
        return outs
    want = []
    for v in src:
        x.copy_(v)
        want.append([t.clone() for t in step()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for v, w in zip(src, want):
            x.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w))
    _status_clear()


def test_threads_on_one_stream():
    """Two threads call on the default stream, and so with one workspace: the kernels of a call stay together."""
    import threading
    from wush_b200 import paged_kv
    calls, want = [], []
    for seed, lens, heads in ((51, [3000, 5, 700], 8), (52, [90, 2048, 0, 4000, 333], 16)):
        s = Setup(lens, page=16, kv=2, dim=128, bounds=True, seed=seed)
        paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, max(lens))
        q = _randn(s.g, len(lens), heads, 128).to(BF)

        def call(s=s, q=q):
            pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, 60)
            return (pages, counts, paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts),
                    paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens))
        calls.append(call)
        want.append(call())
    got = [[], []]
    start = threading.Barrier(2)

    def work(i):
        start.wait(30)
        for _ in range(200):
            got[i].append(calls[i]())
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 200
        for result in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i]))
    _status_clear()


def test_refusals():
    from wush_b200 import paged_kv
    s = Setup([40, 20], page=16, kv=2, dim=64, bounds=True)
    dev = _dev()
    q = _randn(s.g, 2, 4, 64).to(BF)
    k = _randn(s.g, 2, 2, 64).to(BF)
    ids = torch.zeros(2, dtype=torch.int32, device=dev)
    attend = lambda **kw: paged_kv.paged_decode_attention(**{**dict(q=q, cache=s.cache, block_table=s.table, seq_lens=s.seq_lens), **kw})
    append = lambda **kw: paged_kv.paged_kv_append(**{**dict(cache=s.cache, k=k, v=k, block_table=s.table, seq_ids=ids, positions=ids), **kw})
    select = lambda **kw: paged_kv.paged_select_pages(**{**dict(q=q, cache=s.cache, block_table=s.table, seq_lens=s.seq_lens, top=4), **kw})
    pages = torch.zeros(2, 2, 3, dtype=torch.int32, device=dev)
    counts = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    rope = paged_kv.rope_table(64, 64, device=dev)
    for bad in (lambda: attend(q=q.float()), lambda: attend(q=q.to(HF)), lambda: attend(q=q[:, :3]), lambda: attend(q=q[:1]),
                lambda: attend(q=q[:, :, :32]), lambda: attend(q=q.transpose(1, 2)), lambda: attend(seq_lens=s.seq_lens.long()),
                lambda: attend(seq_lens=s.seq_lens[:1]), lambda: attend(block_table=s.table.long()), lambda: attend(block_table=s.table[0]),
                lambda: attend(window=-1), lambda: attend(pages=pages), lambda: attend(counts=counts),
                lambda: attend(pages=pages, counts=counts, window=3), lambda: attend(pages=pages[:1], counts=counts),
                lambda: attend(out=q[:, :2]), lambda: attend(out=q.float()), lambda: attend(q=q[:, :, 4:].contiguous()),
                lambda: append(k=k.float()), lambda: append(v=k[:1]), lambda: append(seq_ids=ids.long()), lambda: append(q_out=q),
                lambda: append(q=q[:1]), lambda: append(rope=rope.double()), lambda: append(rope=rope[:, :24].contiguous()),
                lambda: append(rope=paged_kv.rope_table(64, 96, device=dev)), lambda: append(rope=rope[:, :32]),
                lambda: append(k_out=k[:1]), lambda: append(positions=ids[:1]),
                lambda: select(top=1), lambda: select(top=0, sink=0, recent=0), lambda: select(sink=-1), lambda: select(q=q.to(HF)),
                lambda: paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, -1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(Exception):
        attend(q=q.cpu())
    plain = Setup([5], page=16, kv=2, dim=64)
    with pytest.raises(ValueError):
        paged_kv.paged_kv_bounds(plain.cache, plain.table, plain.seq_lens)
    with pytest.raises(ValueError):
        paged_kv.paged_select_pages(q[:1], plain.cache, plain.table, plain.seq_lens, 4)
    empty = attend(q=q[:0], block_table=s.table[:0], seq_lens=s.seq_lens[:0])
    assert empty.shape == (0, 4, 64)
    _status_clear()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_on_a_device_that_is_not_the_current_one():
    from wush_b200 import paged_kv
    s = Setup([100], page=16, kv=2, dim=64, bounds=True)
    dev = torch.device("cuda:1")
    cache = paged_kv.PagedKVCache(s.cache.k.to(dev), s.cache.v.to(dev), bounds=s.cache.bounds.to(dev))
    q = _randn(s.g, 1, 4, 64).to(BF)
    want = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens)
    got = paged_kv.paged_decode_attention(q.to(dev), cache, s.table.to(dev), s.seq_lens.to(dev))
    assert torch.equal(got.cpu(), want.cpu())
