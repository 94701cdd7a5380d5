"""Prompt and single-token passes of the decoder block with its weights, heads and cache sharded over two GPUs, against the
same block on one.  Tolerance: 1e-2 relative Frobenius, as for the whole-sequence pass in tests/test_block_gpu.py; the two
differ in the order in which row norms are summed and in the bf16 roundings that follow from it."""
import os
import sys

import numpy as np
import pytest
import torch

from oracle import synth
from tests.test_block_gpu import ROOT, SEQ, TOKENS, _setup

pytestmark = pytest.mark.gpu


def _passes(dev, rank, world):
    """This rank's columns of the results of a prompt pass, of three steps of four sequences and of two of one."""
    from wush_b200.block import ShardedDecoderBlock, quantize_block_weights
    from wush_b200.paged_kv import DecodeStep, PagedKVCache, rope_table
    cfg, qw, transforms, gammas, h = _setup("mx", dev)
    kv = cfg.n_kv_heads * cfg.head_dim
    strong = {n: synth.weights(rows, 1024, seed=100 + i) * f for i, (n, rows, f) in enumerate((("q", 1024, 64), ("k", kv, 64), ("v", kv, 8)))}
    qw |= quantize_block_weights(cfg, strong, transforms, dev)
    block = ShardedDecoderBlock(cfg, qw, transforms, gammas, SEQ, TOKENS, dev, micro_batches=2)
    assert block.world == world
    hs = cfg.hidden // world
    mine = h[:, rank * hs:(rank + 1) * hs].contiguous().to(dev)
    seqs, page = TOKENS // SEQ, 16
    table = torch.randperm(40, generator=torch.Generator().manual_seed(3))[: seqs * 8].view(seqs, 8).to(torch.int32).to(dev)
    cache = PagedKVCache.allocate(40, page, block.hkv, cfg.head_dim, device=dev, bounds=True)
    rope = rope_table(SEQ, cfg.head_dim, device=dev)
    lengths = torch.tensor([100, 3, 64, 33], dtype=torch.int32, device=dev)
    outs = [block.prefill(mine.clone(), cache, table, lengths, rope=rope)]
    step = DecodeStep(table, lengths + 1, rope=rope)
    for i in range(3):
        outs.append(block.decode(mine.view(seqs, SEQ, -1)[:, 5 + i].contiguous(), cache, step))
        step.advance()
    one = DecodeStep(table[:1], lengths[:1] + 4, rope=rope)
    for i in range(2):
        outs.append(block.decode(mine[9 + i:10 + i].clone(), cache, one))
        one.advance()
    torch.cuda.synchronize()
    return outs


def _worker(rank, world, port, out):
    sys.path.insert(0, ROOT)
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
    torch.cuda.set_device(rank)
    dev = torch.device("cuda", rank)
    dist.init_process_group("nccl", rank=rank, world_size=world, device_id=dev)
    gathered = []
    for x in _passes(dev, rank, world):
        parts = [torch.empty_like(x) for _ in range(world)]
        dist.all_gather(parts, x.contiguous())
        gathered.append(torch.cat(parts, dim=1).float().cpu().numpy())
    if rank == 0:
        np.savez(out, *gathered)
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_two_gpu_decoding_matches_one_gpu(tmp_path):
    import torch.multiprocessing as mp
    out = str(tmp_path / "h.npz")
    mp.spawn(_worker, args=(2, 29650 + os.getpid() % 300, out), nprocs=2, join=True)
    with np.load(out) as got:
        results = [got[n] for n in got.files]
    want = _passes(torch.device("cuda:0"), 0, 1)              # (no process group in the test process)
    assert len(results) == len(want)
    for i, (a, b) in enumerate(zip(results, want)):
        b = b.float().cpu().numpy()
        assert np.linalg.norm(a - b) <= 1e-2 * np.linalg.norm(b), i
