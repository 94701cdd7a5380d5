"""What the paged key-value cache operators promise beyond their formulas: precision of the weights, copies of a cache,
lengths that the caller writes, reports of what is left out, refusals."""
import copy
import math
import pickle

import pytest
import torch

from tests import paged_reference as ref
from tests.test_paged_kv_gpu import BF, F8, HF, Setup, _dev, _gen, _randn, _status_clear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,cache", [(BF, F8), (HF, F8), (BF, BF), (HF, HF)])
@pytest.mark.parametrize("n", [2, 34])
def test_weights_enter_the_product_with_more_than_16_bits(typ, cache, n):
    """Values a, -a, a, ... under nearly equal weights: the result is a small difference, whose own rounding is small, and
    shows what the weights lost.  A weight of one fp16 term is off by up to 2^-11 of itself; allowed are the 2^-16 of two
    terms (n + 64 additions and the exponentials come on top, see paged_reference.attention_tolerance)."""
    from wush_b200 import paged_kv
    s = Setup([n] * 8, page=16, kv=2, dim=64, cache=cache, seed=n)
    v = torch.ones(64, device=_dev())
    for b in range(8):
        for p in range(n):
            s.cache.v[int(s.table[b, p // 16]), p % 16] = ((1 - 2 * (p % 2)) * v).to(cache)
    q = (0.005 * _randn(s.g, 8, 16, 64)).to(typ)
    out = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens)
    _status_clear()
    for b in range(8):
        for h in range(16):
            k, values = s.rows(b, h // 8, "k"), s.rows(b, h // 8, "v")
            want, _, mass = ref.attend(q[b, h].double(), k, values, 64 ** -0.5)
            tol = ref.attention_tolerance(want, n, 64, mass, float(values.abs().max()), typ, False)
            err = (out[b, h].double() - want).abs()
            assert bool((err <= tol).all()), (b, h, float((err / tol).max()))


@pytest.mark.parametrize("typ", [BF, HF])
@pytest.mark.parametrize("big,small", [(1.0, 2.0 ** -18), (1.0, 2.0 ** -13), (0.0, 2.0 ** -14), (49152.0, 0.25), (2.0 ** -12, 2.0 ** -14)])
def test_small_elements_of_a_query_over_8_bit_pages_keep_their_bits(typ, big, small):
    """One element of every query is large where all keys are zero; the others, far below it, make the logits.  They are
    held to the tolerance of 16-bit pages: every product is exact, and only the sum is rounded."""
    from wush_b200 import paged_kv
    s = Setup([40, 7], page=16, kv=1, dim=64, cache=F8, seed=7)
    for b in range(2):
        for p in range(s.lens[b]):
            s.cache.k[int(s.table[b, p // 16]), p % 16, 0, 5] = 0.0
    q = (small * (1 + 0.5 * _randn(s.g, 2, 4, 64))).to(typ)
    q[:, :, 5] = big
    used = q.double().clone()
    scale = 64 ** -0.5 / small / 0.03                         # (float32, as the call takes it)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, scale=scale, return_lse=True)
    _status_clear()
    for b, n in enumerate(s.lens):
        k, v = s.rows(b, 0, "k"), s.rows(b, 0, "v")
        for h in range(4):
            want, want_lse, mass = ref.attend(used[b, h], k, v, scale)
            assert abs(float(lse[b, h]) - want_lse) <= ref.lse_tolerance(want_lse, n, 64, mass), (b, h)
            tol = ref.attention_tolerance(want, n, 64, mass, float(v.abs().max()), typ, False)
            assert bool(((out[b, h].double() - want).abs() <= tol).all()), (b, h)


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "copy"])
@pytest.mark.parametrize("cache", [BF, F8])
def test_copies_of_a_cache(how, cache):
    """A copied cache names the copy's pages, not those of the original (copy.copy: the same pages, as of any object)."""
    from wush_b200 import paged_kv
    s = Setup([20], page=16, kv=2, dim=64, cache=cache, bounds=True, seed=3, layout="hnd")
    paged_kv.paged_kv_bounds(s.cache, s.table, s.seq_lens, 20)
    other = {"deepcopy": copy.deepcopy, "pickle": lambda c: pickle.loads(pickle.dumps(c)), "copy": copy.copy}[how](s.cache)
    bits = torch.uint8 if cache == F8 else torch.int16
    before = [t.clone() for t in (s.cache.k.view(bits), s.cache.v.view(bits), s.cache.bounds.view(torch.int16))]
    x = torch.full((1, 2, 64), 3.0, dtype=BF, device=_dev())
    at = torch.tensor([19], dtype=torch.int32, device=_dev())
    ids = torch.zeros_like(at)
    paged_kv.paged_kv_append(other, x, x, s.table, ids, at)
    paged_kv.paged_kv_bounds(other, s.table, s.seq_lens, 20)
    q = _randn(s.g, 1, 4, 64).to(BF)
    out = paged_kv.paged_decode_attention(q, other, s.table, s.seq_lens)
    _status_clear()
    now = (s.cache.k.view(bits), s.cache.v.view(bits), s.cache.bounds.view(torch.int16))
    if how == "copy":
        assert not torch.equal(now[0], before[0])
        return
    assert all(torch.equal(a, b) for a, b in zip(now, before))
    page = int(s.table[0, 1])
    assert not torch.equal(other.k[page, 3].float(), s.cache.k[page, 3].float())
    paged_kv.paged_kv_append(s.cache, x, x, s.table, ids, at)            # the same token: then both give the same
    assert torch.equal(paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens), out)


def test_copies_of_a_cache_keep_their_shape_and_what_hangs_on_them():
    from wush_b200 import paged_kv
    dev = _dev()
    pool = torch.zeros(4, 2, 16, 2, 64, dtype=BF, device=dev)
    cache = paged_kv.PagedKVCache(pool[:, 0], pool[:, 1])     # keys and values interleaved
    cache.layer = 7
    twin = copy.deepcopy(cache)
    again = pickle.loads(pickle.dumps(cache))
    assert twin.v.data_ptr() - twin.k.data_ptr() == cache.v.data_ptr() - cache.k.data_ptr()      # still interleaved
    for c in (twin, again):
        assert c.layer == 7 and c.k.stride() == cache.k.stride() and c.v.stride() == cache.v.stride()
        assert c.k.data_ptr() != cache.k.data_ptr() and c._packed[:8] == c.k.data_ptr().to_bytes(8, "little")


@pytest.mark.parametrize("captured", [False, True])
def test_decode_step_follows_lengths_written_by_the_caller(captured):
    """A serving loop puts another sequence into a row by writing seq_lens in place; the token goes where the new length
    says, in a captured step as well."""
    from wush_b200 import paged_kv
    s = Setup([40, 33, 20], page=16, kv=2, dim=64, seed=5)
    step = paged_kv.DecodeStep(s.table, s.seq_lens.clone())
    x = [_randn(s.g, 3, n, 64).to(BF) for n in (4, 2, 2)]
    held = [t.clone() for t in x]
    graph = None
    if captured:
        step.attend(s.cache, *held)                           # warm-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step.attend(s.cache, *held)
    for lens in ([40, 33, 20], [7, 0, 20], [38, 1, 0]):
        step.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32, device=_dev()))
        for t, v in zip(held, x):
            t.copy_(v)
        want = [(s.cache.k.clone(), s.cache.v.clone())]
        for b, n in enumerate(lens):
            if n > 0:
                page, row = int(s.table[b, (n - 1) // 16]), (n - 1) % 16
                want[0][0][page, row], want[0][1][page, row] = x[1][b], x[2][b]
        if graph is not None:
            graph.replay()
        else:
            step.attend(s.cache, *held)
        _status_clear()
        for got, w in zip((s.cache.k, s.cache.v), want[0]):
            assert torch.equal(got.view(torch.int16), w.view(torch.int16)), lens
        assert step.positions.tolist() == [n - 1 for n in lens]
    step.advance()
    assert step.seq_lens.tolist() == [39, 2, 0] and step.positions.tolist() == [38, 1, -1]


def test_counts_beyond_the_list_are_reported():
    """More selected pages than the list holds: the whole list is attended to, and the count is reported."""
    from wush_b200 import _lib, paged_kv
    for page, top in ((16, 3), (16, 90), (24, 3)):            # whole items, cut ones, odd pages
        s = Setup([page * top + 5, 33], page=page, kv=2, dim=64, seed=11)
        q = _randn(s.g, 2, 8, 64).to(BF)
        pages = torch.arange(top, dtype=torch.int32, device=_dev()).flip(0).expand(2, 2, top).contiguous()
        counts = torch.full((2, 2), top, dtype=torch.int32, device=_dev())
        counts[1] = 1
        pages[1] = 0
        want = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts)
        _status_clear()
        counts[0, 1] = top + 1
        got = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, pages=pages, counts=counts)
        with pytest.raises(_lib.WushB200Error, match="outside its table"):
            _lib.check_status(_dev())
        assert torch.equal(got, want)


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("entry", [-2 ** 31, -1, 2 ** 31 - 1])
def test_every_table_entry_outside_the_pool_is_reported(page, entry):
    from wush_b200 import _lib, paged_kv
    s = Setup([3 * page], page=page, kv=2, dim=64, seed=6)
    q = _randn(s.g, 1, 4, 64).to(BF)
    good = s.table.clone()
    s.table[0, 1] = entry
    out = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens)
    with pytest.raises(_lib.WushB200Error, match="outside its table"):
        _lib.check_status(_dev())
    pages = torch.tensor([[[0, 2]] * 2], dtype=torch.int32, device=_dev())
    counts = torch.full((1, 2), 2, dtype=torch.int32, device=_dev())
    want = paged_kv.paged_decode_attention(q, s.cache, good, s.seq_lens, pages=pages, counts=counts)
    _status_clear()
    # the same 2 * page tokens, in tiles that start elsewhere: both within the tolerance of the float64 result
    assert float((out.float() - want.float()).abs().max()) <= 2 * 2.0 ** -8 * float(want.float().abs().max()) + 1e-4


def test_outputs_whose_rows_or_heads_share_memory_are_refused():
    from wush_b200 import paged_kv
    s = Setup([40, 20], page=16, kv=2, dim=64)
    q, k = _randn(s.g, 2, 4, 64).to(BF), _randn(s.g, 2, 2, 64).to(BF)
    ids = torch.arange(2, dtype=torch.int32, device=_dev())
    for bad in (q[:1].expand(2, 4, 64), q[:, :1].expand(2, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, out=bad)
        with pytest.raises(ValueError, match="overlap"):
            paged_kv.paged_kv_append(s.cache, k, k, s.table, ids, ids, q=q, q_out=bad)
    for bad in (k[:1].expand(2, 2, 64), k[:, :1].expand(2, 2, 64)):
        with pytest.raises(ValueError, match="overlap"):
            paged_kv.paged_kv_append(s.cache, k, k, s.table, ids, ids, k_out=bad)
    # inputs may: one key for all heads, one query for all sequences
    same = k[:, :1].expand(2, 2, 64)
    paged_kv.paged_kv_append(s.cache, same, same, s.table, ids, ids)
    got = paged_kv.paged_decode_attention(q[:1].expand(2, 4, 64), s.cache, s.table, s.seq_lens)
    _status_clear()
    want = paged_kv.paged_decode_attention(q[:1].expand(2, 4, 64).contiguous(), s.cache, s.table, s.seq_lens)
    assert torch.equal(got, want) and torch.equal(s.cache.k[int(s.table[1, 0]), 1, 1], k[1, 0])


def _fp32_scores(q, cache, table, lens, top):
    """(value, magnitude) float32 [sequences, key heads, pages]: what the scoring kernel leaves in the call's workspace."""
    from wush_b200 import _lib, paged_kv
    lib = _lib.load()
    seqs, width, kv = table.shape[0], table.shape[1], cache.n_kv_heads
    work = torch.zeros(lib.wush_kv_select_workspace_bytes(seqs, kv, width), dtype=torch.uint8, device=_dev())
    pages = torch.empty(seqs, kv, top, dtype=torch.int32, device=_dev())
    counts = torch.empty(seqs, kv, dtype=torch.int32, device=_dev())
    rc = lib.wush_kv_select_pages(cache._packed + paged_kv._SELECT.pack(
        table.data_ptr(), table.stride(0), seqs, width, q.data_ptr(), q.stride(0), q.stride(1), lens.data_ptr(), pages.data_ptr(),
        counts.data_ptr(), work.data_ptr(), work.numel(), cache._status, torch.cuda.current_stream().cuda_stream,
        paged_kv.TYPES[q.dtype], q.shape[1], top, 0, 0))
    assert rc == 0
    torch.cuda.synchronize()
    return work.view(torch.float32).view(seqs, kv, width, 2).unbind(-1)


@pytest.mark.parametrize("typ,bounds", [(BF, BF), (HF, HF), (HF, BF), (BF, HF)])
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 80, 128, 208, 256])
def test_fp32_scores_stay_within_the_bound_that_the_selection_uses(typ, bounds, dim):
    """The selection trusts fp32 scores up to a bound: each product of 16 terms is off by at most 17 * 2^-23 of its terms'
    magnitude, and 4 * ceil(dim / 32) products are added with 2^-24 of the magnitude each.  Terms of very mixed size: every
    addend's own cut counts.  (1 + 2^-10: errors of errors.)"""
    from wush_b200.paged_kv import PagedKVCache
    width, kv, group = 400, 2, 3
    g, dev = _gen(dim), _dev()
    cache = typ if typ == bounds else F8
    dim = -(-dim // 16) * 16 if cache == F8 else dim
    one = torch.ones(kv, device=dev)
    data = torch.zeros(width, 1, kv, dim, dtype=cache, device=dev)
    pool = PagedKVCache(data, data, k_scale=one if cache == F8 else None, v_scale=one if cache == F8 else None,
                        bounds=torch.zeros(width, kv, 2, dim, dtype=bounds, device=dev))
    spread = lambda *shape: torch.exp2(torch.randint(-13, 1, shape, generator=g, device=dev).float())
    x = _randn(g, width, kv, 2, dim) * spread(width, kv, 1, dim)
    # a third of the pages: one large term a product, the others around the last bit of it and of one sign
    some = torch.arange(width, device=dev) % 3 == 0
    small = (1 + torch.rand(width, kv, 1, dim, generator=g, device=dev)) * 2.0 ** -11
    small[..., ::16] = 1.0 + torch.rand(width, kv, 1, dim, generator=g, device=dev)[..., ::16]
    x[some] = small.expand(width, kv, 2, dim)[some]
    if cache == F8:                                           # bounds of 8-bit keys are 8-bit numbers
        x = (x * 128).clamp(-448, 448).to(F8).float()
    low, high = x.amin(2).to(bounds), x.amax(2).to(bounds)
    pool.bounds[:, :, 0], pool.bounds[:, :, 1] = low, high
    table = torch.randperm(width, generator=g, device=dev).to(torch.int32)[None]
    lens = torch.tensor([width], dtype=torch.int32, device=dev)
    q = (_randn(g, 1, kv * group, dim) * spread(1, kv * group, dim)).to(typ)
    q[0, 0] = 2.0 ** -12 * (1 + torch.rand(dim, generator=g, device=dev)).to(typ)
    q[0, 0, ::16] = 1.5
    value, magnitude = _fp32_scores(q, pool, table, lens, 5)
    _status_clear()
    rel = (17 + 2 * -(-dim // 32)) * 2.0 ** -23 * (1 + 2.0 ** -10)
    at = table[0].long()
    worst = 0.0
    for h in range(kv):
        qs = q[0, h * group:(h + 1) * group].double()
        lo, hi = low[at, h].double(), high[at, h].double()
        exact = torch.maximum(qs[:, None] * lo, qs[:, None] * hi).sum(2).amax(0)
        most = (qs.abs()[:, None] * torch.maximum(lo.abs(), hi.abs())).sum(2).amax(0)
        err = (value[0, h].double() - exact).abs()
        worst = max(worst, float((err / (rel * most)).max()))
        assert bool((err <= rel * most + 2.0 ** -120).all()), float((err / (rel * most)).max())
        assert bool((magnitude[0, h].double() >= most * (1 - 1 / 32)).all())
    print(f"dim {dim}: worst error {worst:.3f} of the bound")


@pytest.mark.parametrize("span", [20, 40, 100])
def test_choice_of_scores_that_64_bits_cannot_hold(span):
    """Terms of 2^span and -2^span around small ones.  What is chosen has the largest exact scores, up to the rounding of 64-bit
    sums: 64 additions (and as many products, exact) of 2^-53 of the magnitude each, on either side."""
    from wush_b200.paged_kv import PagedKVCache, paged_select_pages
    width, dim = 500, 64
    g, dev = _gen(span), _dev()
    pool = PagedKVCache.allocate(width, 1, 1, dim, device=dev, bounds=True)
    x = _randn(g, width, dim) * torch.exp2(torch.randint(-span, span // 2, (width, dim), generator=g, device=dev).float())
    at = torch.randint(0, dim // 2, (width,), generator=g, device=dev)
    rows = torch.arange(width, device=dev)
    x[rows, at], x[rows, at + dim // 2] = 2.0 ** span, -2.0 ** span
    pool.bounds[:, 0] = x.to(BF)[:, None]
    q = torch.ones(1, 1, dim, dtype=BF, device=dev)
    table = torch.arange(width, dtype=torch.int32, device=dev)[None]
    lens = torch.tensor([width], dtype=torch.int32, device=dev)
    terms = x.to(BF).double().tolist()
    exact = [math.fsum(t) for t in terms]
    slack = 2 * dim * 2.0 ** -53 * max(sum(abs(y) for y in t) for t in terms)
    for top in (1, 60, 300):
        pages, counts = paged_select_pages(q, pool, table, lens, top, sink=0, recent=0)
        chosen = set(pages[0, 0].tolist())
        assert len(chosen) == top == int(counts[0, 0])
        worst, best = min(exact[i] for i in chosen), max(exact[i] for i in range(width) if i not in chosen)
        assert worst >= best - slack, (top, worst, best, slack)
    _status_clear()


@pytest.mark.parametrize("width", [34, 130, 700, 2100, 9000])
def test_selection_among_pages_that_are_all_equal(width):
    from wush_b200.paged_kv import PagedKVCache, paged_select_pages
    dev, seqs = _dev(), 40
    pool = PagedKVCache.allocate(width, 1, 2, 16, device=dev, bounds=True)
    table = torch.arange(width, dtype=torch.int32, device=dev).expand(seqs, width)
    lens = torch.full((seqs,), width, dtype=torch.int32, device=dev)
    q = torch.ones(seqs, 4, 16, dtype=BF, device=dev)
    for value in (0.0, 3.0):                                  # bounds not filled yet, and filled alike
        pool.bounds.fill_(value)
        for top, sink, recent in ((33, 0, 0), (width // 2, 1, 3), (1, 0, 1)):
            pages, counts = paged_select_pages(q, pool, table, lens, top, sink=sink, recent=recent)
            want = list(range(top - recent)) + list(range(width - recent, width))
            assert bool((counts == top).all()) and bool((pages == torch.tensor(want, dtype=torch.int32, device=dev)).all())
    _status_clear()


@pytest.mark.parametrize("width,odd", [(300, 1), (300, 40), (300, 290), (2047, 3), (2047, 700), (9000, 5), (9000, 300)])
@pytest.mark.parametrize("typ,bounds", [(BF, BF), (HF, HF), (BF, HF)])
def test_pages_with_a_bound_that_is_not_finite_do_not_hide_the_others(typ, bounds, width, odd):
    """Such a page counts as +infinity; the fp32 scores of all others stand, and the choice is that of exact scores."""
    from wush_b200.paged_kv import PagedKVCache, paged_select_pages
    g, dev, dim, kv = _gen(width + odd), _dev(), 48, 2
    cache = typ if typ == bounds else F8
    one = torch.ones(kv, device=dev)
    data = torch.zeros(width, 1, kv, dim, dtype=cache, device=dev)
    pool = PagedKVCache(data, data, k_scale=one if cache == F8 else None, v_scale=one if cache == F8 else None,
                        bounds=torch.zeros(width, kv, 2, dim, dtype=bounds, device=dev))
    pool.bounds.copy_(_randn(g, width, kv, 2, dim).sort(dim=2).values.to(F8).to(bounds) if cache == F8 else
                      _randn(g, width, kv, 2, dim).sort(dim=2).values.to(bounds))
    table = torch.randperm(width, generator=g, device=dev).to(torch.int32)[None]
    who = torch.randperm(width, generator=g, device=dev)[:odd]          # logical pages
    channel = torch.randint(0, dim, (odd,), generator=g, device=dev)
    kinds = torch.tensor([math.inf, -math.inf, math.nan], device=dev)[torch.arange(odd, device=dev) % 3].to(bounds)
    pool.bounds[table[0][who].long(), 0, torch.arange(odd, device=dev) % 2, channel] = kinds      # key head 0 only
    q = _randn(g, 1, 6, dim).to(typ)
    q[0, 1, channel[0]] = 0.0
    lens = torch.tensor([width], dtype=torch.int32, device=dev)
    _, magnitude = _fp32_scores(q, pool, table, lens, min(odd + 5, width - 1))       # (fewer: hundreds of equal ones at the border)
    at = table[0].long()
    low, high = pool.bounds[at, :, 0].double(), pool.bounds[at, :, 1].double()
    strange = torch.zeros(width, dtype=torch.bool, device=dev)
    strange[who] = True
    assert bool(magnitude.isfinite().all())
    for top, sink, recent in ((max(1, odd // 2), 0, 0), (min(odd, width - 1), 0, 0), (min(odd + 20, width - 1), 1, 1)):
        pages, counts = paged_select_pages(q, pool, table, lens, top, sink=sink, recent=recent)
        for h in range(kv):
            qs = q[0, 3 * h:3 * h + 3].double()
            score = torch.maximum(qs[:, None] * low[:, h], qs[:, None] * high[:, h]).sum(2).amax(0)
            if h == 0:
                score[strange] = math.inf
            assert pages[0, h].tolist() == ref.select(score.tolist(), top, sink, recent), (top, h)
    _status_clear()


@pytest.mark.parametrize("cache", [BF, F8])
def test_results_carry_no_gradient(cache):
    from wush_b200 import paged_kv
    s = Setup([40], page=16, kv=2, dim=64, cache=cache, bounds=True)
    q = _randn(s.g, 1, 4, 64).to(BF).requires_grad_()
    out, lse = paged_kv.paged_decode_attention(q, s.cache, s.table, s.seq_lens, return_lse=True)
    assert not out.requires_grad and not lse.requires_grad
