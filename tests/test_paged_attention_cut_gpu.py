"""Attention of a new token where items are cut: their tokens are walked by several blocks, teams of blocks walk the same
tokens for neighbouring key heads, and the parts are joined by a second kernel.  Against float64 (tests/paged_reference.py,
where the tolerances are derived), with several key heads, ragged lengths, windows, selected pages and chunks of queries."""
import pytest
import torch

from tests import paged_reference as ref
from tests.test_paged_kv_gpu import BF, F8, HF, Setup, _dev, _randn, _status_clear

pytestmark = pytest.mark.gpu


class Long(Setup):
    """Setup whose sequences are gathered page by page instead of row by row."""

    def rows(self, b, head, which):
        pool, scale = (self.cache.k, self.cache.k_scale) if which == "k" else (self.cache.v, self.cache.v_scale)
        pages = self.table[b, : -(-self.lens[b] // self.page)].long()
        x = pool.view(torch.uint8)[pages].view(pool.dtype)[:, :, head] if pool.dtype == F8 else pool[pages][:, :, head]
        x = x.reshape(-1, self.dim)[: self.lens[b]].double()
        return x if scale is None else x * scale[head].double()

    def check(self, q, out, lse, window=0, chosen=None):
        """All queries of a key head at once; chosen[b][head]: selected pages."""
        group = q.shape[1] // self.kv
        for b, n in enumerate(self.lens):
            for hk in range(self.kv):
                k, v = self.rows(b, hk, "k"), self.rows(b, hk, "v")
                if chosen is not None:
                    keep = [p for lp in chosen[b][hk] for p in range(lp * self.page, min(n, (lp + 1) * self.page))]
                    k, v = k[keep], v[keep]
                elif window:
                    k, v = k[max(0, n - window):], v[max(0, n - window):]
                for h in range(hk * group, (hk + 1) * group):
                    want, want_lse, mass = ref.attend(q[b, h].double(), k, v, self.dim ** -0.5)
                    v_max = float(v.abs().max()) if len(k) else 0.0
                    tol = ref.attention_tolerance(want, len(k), self.dim, mass, v_max, q.dtype, False)
                    err = (out[b, h].double() - want).abs()
                    assert bool((err <= tol).all()), (b, h, n, float((err - tol).max()))
                    if len(k) == 0:
                        assert float(lse[b, h]) == -float("inf")
                    else:
                        assert abs(float(lse[b, h]) - want_lse) <= ref.lse_tolerance(want_lse, len(k), self.dim, mass), (b, h, n)


RAGGED = [4096, 1, 0, 2900, 700]
CASES = [   # (queries, cache, dim, page, kv, heads, lens, window, layout)
    (BF, BF, 128, 64, 8, 64, RAGGED, 0, "nhd"),               # a team of eight blocks
    (BF, F8, 128, 64, 8, 64, RAGGED, 0, "nhd"),
    (HF, F8, 128, 16, 8, 32, RAGGED, 0, "hnd"),
    (HF, HF, 64, 32, 3, 12, [5003, 31, 2049], 0, "nhd"),      # of three
    (BF, BF, 96, 16, 6, 6, [3000, 2999, 0, 4100], 0, "nhd"),  # of six
    (HF, HF, 128, 16, 5, 10, [1, 6000], 0, "hnd"),
    (BF, BF, 128, 16, 11, 22, [2500, 40], 0, "nhd"),          # eleven heads have no team
    (BF, BF, 128, 64, 2, 80, [2500, 3, 1999], 0, "nhd"),      # 40 queries a key head: three chunks
    (BF, F8, 64, 64, 3, 60, [3333, 128], 0, "nhd"),           # 20 queries a key head: two
    (BF, BF, 256, 32, 4, 24, [3000, 0, 1200], 0, "nhd"),
    (BF, F8, 256, 16, 2, 20, [2600, 15], 0, "hnd"),
    (HF, HF, 80, 24, 2, 8, [2501, 23, 25], 0, "nhd"),         # pages of 24: rows copied piece by piece
    (BF, F8, 128, 24, 4, 32, [4001, 700], 0, "hnd"),
    (BF, BF, 128, 1, 2, 2, [1500, 900], 0, "nhd"),
    (BF, BF, 128, 16, 4, 32, [4000, 2500, 10, 2499], 2500, "nhd"),
    (HF, HF, 96, 24, 4, 24, [9001, 17, 2101], 2100, "nhd"),
    (BF, F8, 128, 32, 8, 64, [5000, 2304, 2303], 2303, "nhd"),
    (BF, BF, 64, 16, 2, 16, [40000, 3], 0, "nhd"),            # more than 32 parts
    (BF, F8, 128, 16, 1, 4, [70001], 0, "nhd"),
]


@pytest.mark.parametrize("typ,cache,dim,page,kv,heads,lens,window,layout", CASES)
def test_cut_items(typ, cache, dim, page, kv, heads, lens, window, layout):
    from wush_b200 import paged_kv
    s = Long(lens, page=page, kv=kv, dim=dim, cache=cache, layout=layout, seed=dim + page + heads)
    q = (2.0 * _randn(s.g, len(lens), heads, dim)).to(typ)
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, window=window, return_lse=True)
    _status_clear()
    s.check(q, out, lse, window=window)
    in_place = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, window=window, out=q)
    assert torch.equal(out, in_place)                         # the same bits every time


def test_cut_items_of_many_sequences():
    """More items than SMs, most of them short, so that a block has ends and beginnings of several."""
    from wush_b200 import paged_kv
    lens = [(37 * i * i) % 300 for i in range(60)] + [3000, 1, 0, 4096, 1500]
    for cache in (BF, F8):
        s = Long(lens, page=16, kv=4, dim=64, cache=cache, seed=77)
        q = (2.0 * _randn(s.g, len(lens), 8, 64)).to(BF)
        out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
        _status_clear()
        s.check(q, out, lse)


@pytest.mark.parametrize("typ,cache,dim,page,kv,heads,top", [
    (BF, BF, 128, 16, 2, 16, 128), (BF, F8, 128, 16, 8, 64, 128), (HF, HF, 64, 64, 5, 20, 40), (BF, BF, 96, 24, 2, 40, 70),
    (HF, F8, 256, 32, 3, 6, 64)])
def test_cut_selected_pages(typ, cache, dim, page, kv, heads, top):
    from wush_b200 import paged_kv
    lens = [page * top * 2 + 5, 3, 0, page * top - 1, page * top + 1]
    s = Long(lens, page=page, kv=kv, dim=dim, cache=cache, seed=dim + top, bounds=True)
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, max(lens))
    q = (2.0 * _randn(s.g, len(lens), heads, dim)).to(typ)
    pages, counts = paged_kv.paged_select_pages(q, s.cache, s.table, s.seq_lens, top)
    chosen = [[pages[b, h, : int(counts[b, h])].tolist() for h in range(kv)] for b in range(len(lens))]
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts, return_lse=True)
    _status_clear()
    s.check(q, out, lse, chosen=chosen)
