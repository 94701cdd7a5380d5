"""Exchange of a GEMM operand between the ranks of the sharded decoder block (wush_b200/block.py), on the CPU: two ranks'
buffers in one process, symmetric memory and the quantize kernel replaced by plain ones."""
import pytest
import torch

from wush_b200 import block

ROWS, SHARD, GROUP, WORLD, UNTOUCHED = 300, 512, 32, 2, 0xEE


@pytest.fixture()
def ranks(monkeypatch):
    import torch.distributed._symmetric_memory as symm
    flats, log = [], []

    class Handle:
        def get_buffer(self, peer, shape, dtype):
            while len(flats) <= peer:
                flats.append(torch.full(shape, UNTOUCHED, dtype=dtype))
            return flats[peer]

        def barrier(self, channel):
            log.append("barrier")
    made = iter(range(WORLD))
    handle = Handle()
    monkeypatch.setattr(symm, "empty", lambda n, dtype, device: handle.get_buffer(next(made), (n,), dtype))
    monkeypatch.setattr(symm, "rendezvous", lambda flat, group: handle)

    def quantize(x, matrix, fmt, gs, codes, scales, col0, sf_layout, row_scale, col_scale):
        codes.copy_(x[:, : codes.shape[1]])
        n = (x.shape[0] + 127) // 128 * 128 * (SHARD // GROUP)
        scales[:n] = (torch.arange(n) % 100 + x[0, 0]).to(torch.uint8)
    monkeypatch.setattr(block.ops, "fused_quantize_into", quantize)
    sent = []
    plain = block._broadcast

    def broadcast(flat, handle, peers, rank, world, lo, hi, table):
        assert lo % 16 == 0 and hi % 16 == 0 and rank * len(flat) // world <= lo < hi <= (rank + 1) * len(flat) // world
        sent.append(hi - lo)
        log.append("copy")
        plain(flat, handle, peers, rank, world, lo, hi, table)
    monkeypatch.setattr(block, "_broadcast", broadcast)
    monkeypatch.delenv("WUSH_B200_BLOCK_BROADCAST", raising=False)
    return [block._Exchange(ROWS, SHARD, GROUP, WORLD, r, "cpu", None) for r in range(WORLD)], flats, sent, log


@pytest.mark.parametrize("m", [1, 4, 127, 128, 129, 299, 300])
def test_put_sends_the_rows_in_use(ranks, m):
    exchanges, flats, sent, log = ranks
    assert len(flats) == WORLD and not torch.equal(exchanges[0].my_codes, torch.zeros_like(exchanges[0].my_codes))
    used = (m + 127) // 128 * 128 * (SHARD // GROUP)
    for r, e in enumerate(exchanges):
        x = ((torch.arange(m * SHARD).view(m, SHARD) * 7 + 3 * r + 1) % 200).to(torch.uint8)
        e.put(x, None, "mx", None)
        assert log[-1] == "barrier" and sum(sent) == m * SHARD // 2 + used        # nothing but codes and scales of m rows
        sent.clear()
        other = flats[1 - r][r * e.slot:(r + 1) * e.slot]
        mine = flats[r][r * e.slot:(r + 1) * e.slot]
        codes, scales = other[: e.code_bytes].view(ROWS, SHARD // 2), other[e.code_bytes:]
        assert torch.equal(codes[:m], x[:, : SHARD // 2]) and torch.equal(scales[:used], mine[e.code_bytes:][:used])
        assert bool((codes[m:] == UNTOUCHED).all()) and bool((scales[used:] == UNTOUCHED).all())
    # what the GEMM reads: rank s's rows in slot s, the same on every rank
    for e in exchanges:
        assert torch.equal(e.codes[:, :m], torch.stack([x.codes[s, :m] for s, x in enumerate(exchanges)]))
