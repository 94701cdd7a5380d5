"""Prompt and single-token passes of the decoder block over a paged key-value cache (ShardedDecoderBlock.prefill and
decode), against the block's own whole-sequence pass: causal attention makes row t of a sequence the same whether the
rows behind it are there or not, so a token decoded at position t must reproduce row t of one pass over everything.

With the weights of tests/test_block_gpu.py all logits are nearly 0 and the attention is a mean that moves the output by
little; here queries, keys and values are larger (64, 64 and 8 times: powers of two, so only the scales of their weights
change), and the attention's results and the cache's contents are compared as well.  The two ways run the same quantizer and the same W4A4 products on
the same rows; they differ in the attention kernel (results rounded to bf16, and the weights of the prompt's attention
too: each 2^-9 / sqrt(3) = 1.1e-3 relative in the Frobenius norm) and in the GEMM kernel that the row count selects (order
of fp32 sums, which moves few bf16 roundings of q, k and v by one step).  Tolerance: 1e-2 relative Frobenius, under which
tests/test_block_gpu.py compares two computations of the block that differ in just that.  8-bit pages round keys and
values by at most half a step, which is checked on the cache; for the block's output the bound is that rounding, as if all
of it came from them: 2^-4 / sqrt(3) + 1e-2 < 5e-2."""
import pytest
import torch

from oracle import synth
from tests.test_block_gpu import SEQ, TOKENS, _setup

pytestmark = pytest.mark.gpu


def _block(fmt="mx"):
    from wush_b200.block import ShardedDecoderBlock, quantize_block_weights
    dev = torch.device("cuda:0")
    cfg, qw, transforms, gammas, h = _setup(fmt, dev)
    kv = cfg.n_kv_heads * cfg.head_dim
    strong = {n: synth.weights(rows, 1024, seed=100 + i) * f for i, (n, rows, f) in enumerate((("q", 1024, 64), ("k", kv, 64), ("v", kv, 8)))}
    qw |= quantize_block_weights(cfg, strong, transforms, dev)
    return cfg, ShardedDecoderBlock(cfg, qw, transforms, gammas, SEQ, TOKENS, dev, micro_batches=2), h.to(dev)


def _cache(cfg, page, dtype=torch.bfloat16, bounds=False, pages=40):
    from wush_b200.paged_kv import PagedKVCache
    scale = torch.full((cfg.n_kv_heads,), 0.01, device="cuda") if dtype != torch.bfloat16 else None
    return PagedKVCache.allocate(pages, page, cfg.n_kv_heads, cfg.head_dim, dtype=dtype, device="cuda", k_scale=scale, v_scale=scale,
                                 bounds=bounds)


def _tables(seqs, page, pages):
    per = -(-SEQ // page)
    return torch.randperm(pages, generator=torch.Generator().manual_seed(3))[: seqs * per].view(seqs, per).to(torch.int32).cuda()


def _rel(got, want):
    return float((got.float() - want.float()).norm() / want.float().norm())


@pytest.mark.parametrize("fmt,page,dtype,tol", [("mx", 16, torch.bfloat16, 1e-2), ("nv", 24, torch.bfloat16, 1e-2),
                                                ("mx", 64, torch.float8_e4m3fn, 5e-2)])
def test_decoded_tokens_match_one_pass_over_everything(fmt, page, dtype, tol):
    from wush_b200 import _lib
    from wush_b200.paged_kv import DecodeStep, rope_table
    cfg, block, h = _block(fmt)
    seqs = TOKENS // SEQ
    rope = rope_table(SEQ, cfg.head_dim, device="cuda")
    table = _tables(seqs, page, 40)
    full = torch.full((seqs,), SEQ, dtype=torch.int32, device="cuda")
    seen, attention = [], block._attention
    block._attention = lambda qkv, prompt=None: seen.append(attention(qkv, prompt)) or seen[-1]
    whole = _cache(cfg, page)
    want = block.prefill(h.clone(), whole, table, full, rope=rope).view(seqs, SEQ, -1)
    turned = torch.cat(seen).view(seqs, SEQ, -1)                  # attention of every token
    seen.clear()
    block.forward(h.clone())
    plain = torch.cat(seen).view(seqs, SEQ, -1)
    block._attention = attention
    # a query sees the keys before it turned by their distances: the first two tokens see (nearly) the same with and without
    assert torch.equal(turned[:, 0], plain[:, 0]) and _rel(turned[:, 8:], plain[:, 8:]) > 3e-2
    cache = _cache(cfg, page, dtype)
    start = torch.tensor([SEQ - 6, 1, 77, SEQ - 6], dtype=torch.int32, device="cuda")
    noisy = h.clone().view(seqs, SEQ, -1)
    for b in range(seqs):
        noisy[b, int(start[b]):] = 3.0                            # what lies behind a prompt does not matter
    out = block.prefill(noisy.view(TOKENS, -1), cache, table, start, rope=rope).view(seqs, SEQ, -1)
    for b in range(seqs):
        assert _rel(out[b, : int(start[b])], want[b, : int(start[b])]) <= tol
    step = DecodeStep(table, start + 1, rope=rope)
    step.seq_lens[3] = 0                                          # a padded row from here on
    step.positions[3] = -1
    attended, attend = [], step.attend
    step.attend = lambda *a: attended.append(attend(*a)) or attended[-1]
    for i in range(6):
        rows = torch.stack([h.view(seqs, SEQ, -1)[b, min(int(start[b]) + i, SEQ - 1)] for b in range(seqs)])
        got = block.decode(rows.clone(), cache, step)
        target = torch.stack([want[b, min(int(start[b]) + i, SEQ - 1)] for b in range(seqs)])
        assert _rel(got[:3], target[:3]) <= tol, i
        if dtype == torch.bfloat16:
            target = torch.stack([turned[b, int(start[b]) + i] for b in range(3)])
            assert _rel(attended[i][:3].flatten(1), target) <= 1e-2, i
        assert not attended[i][3].any()
        step.advance()
        assert step.seq_lens.tolist() == [SEQ - 6 + i + 2, i + 3, 77 + i + 2, 0]
    _lib.check_status("cuda")
    for b, n in enumerate([SEQ, 7, 83]):                          # the caches: rotated keys and values of every token
        for p in range(n):
            at = int(table[b, p // page]), p % page
            for mine, theirs in ((cache.k, whole.k), (cache.v, whole.v)):
                x, y = mine[at].double() * (1 if dtype == torch.bfloat16 else 0.01), theirs[at].double()
                if dtype == torch.bfloat16:
                    assert _rel(x, y) <= 1e-2
                else:       # one bf16 step of a few, half an e4m3 step of all (2^-10 is half the smallest step, times the scale)
                    assert _rel(x, y) <= 2.0 ** -4 and bool(((x - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * 0.01 + 2.0 ** -7 * y.abs()).all())


def test_selected_pages_and_windows_in_the_block():
    """All pages selected, or a window over everything, is the whole attention; fewer pages change the result."""
    from wush_b200.paged_kv import DecodeStep
    cfg, block, h = _block()
    seqs, page = TOKENS // SEQ, 8
    table = _tables(seqs, page, 80)
    cache = _cache(cfg, page, bounds=True, pages=80)
    lengths = torch.tensor([100, 127, 64, 33], dtype=torch.int32, device="cuda")
    block.prefill(h.clone(), cache, table, lengths)
    rows = h.view(seqs, SEQ, -1)[:, 5].contiguous()
    dense = block.decode(rows.clone(), cache, DecodeStep(table, lengths + 1))
    every = block.decode(rows.clone(), cache, DecodeStep(table, lengths + 1, top_pages=16))
    window = block.decode(rows.clone(), cache, DecodeStep(table, lengths + 1, window=SEQ))
    few = block.decode(rows.clone(), cache, DecodeStep(table, lengths + 1, top_pages=3))
    assert _rel(every, dense) <= 1e-2 and _rel(window, dense) <= 1e-6 and _rel(few, dense) > 0
    assert bool(few.isfinite().all())


def test_captured_decode_replays_over_several_tokens():
    from wush_b200.paged_kv import DecodeStep
    cfg, block, h = _block()
    seqs, page = TOKENS // SEQ, 16
    table = _tables(seqs, page, 40)
    lengths = torch.tensor([100, 3, 64, 33], dtype=torch.int32, device="cuda")
    eager_cache, graph_cache = _cache(cfg, page, bounds=True), _cache(cfg, page, bounds=True)
    for cache in (eager_cache, graph_cache):
        block.prefill(h.clone(), cache, table, lengths)
    eager, captured = DecodeStep(table, lengths + 1, top_pages=4), DecodeStep(table, lengths + 1, top_pages=4)
    rows = h.view(seqs, SEQ, -1)[:, :8].contiguous()
    x = torch.empty_like(rows[:, 0])
    x.copy_(rows[:, 0])
    block.decode(x, graph_cache, captured)                        # warm-up: writes the token that the first replay writes again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.decode(x, graph_cache, captured)
        captured.advance()
    for i in range(8):
        want = block.decode(rows[:, i].clone(), eager_cache, eager)
        eager.advance()
        x.copy_(rows[:, i])
        graph.replay()
        assert torch.equal(x, want), i
    assert torch.equal(captured.seq_lens, lengths + 9) and torch.equal(eager_cache.k, graph_cache.k)


def test_refusals():
    from wush_b200.paged_kv import DecodeStep
    cfg, block, h = _block()
    seqs = TOKENS // SEQ
    table, cache = _tables(seqs, 16, 40), _cache(cfg, 16)
    lengths = torch.full((seqs,), 5, dtype=torch.int32, device="cuda")
    from wush_b200.paged_kv import PagedKVCache
    wrong = PagedKVCache.allocate(4, 16, cfg.n_kv_heads + 1, cfg.head_dim, device="cuda")
    half = PagedKVCache.allocate(4, 16, cfg.n_kv_heads, cfg.head_dim, dtype=torch.float16, device="cuda")
    step = DecodeStep(table, lengths)
    rows = h[:seqs].contiguous()
    for bad in (lambda: block.prefill(h.clone(), wrong, table, lengths), lambda: block.prefill(h.clone(), half, table, lengths),
                lambda: block.prefill(h.clone(), cache, table, lengths.long()), lambda: block.prefill(h.clone(), cache, table[:2], lengths),
                lambda: block.decode(rows[:2], cache, step), lambda: block.decode(rows.float(), cache, step),
                lambda: block.decode(rows, wrong, step), lambda: block.decode(rows, half, step),
                lambda: DecodeStep(table, lengths, window=4, top_pages=4), lambda: DecodeStep(table, lengths.long()),
                lambda: block.decode(rows, cache, DecodeStep(table, lengths, top_pages=4))):
        with pytest.raises(ValueError):
            bad()
    assert block.decode(h[:0], cache, DecodeStep(table[:0], lengths[:0])).shape[0] == 0
