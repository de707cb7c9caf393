"""GPU: 4-bit blocks through the tiers: the TransferEngine with files behind the
host pool, and tensor-parallel ranks that share a block by heads."""
import numpy as np
import pytest
import torch

import fp4_model as M
from flexkv_b200 import fp4_cache
from flexkv_b200.engine import TransferEngine, TransferType
from flexkv_b200.layout import KVCacheLayout, KVCacheLayoutType
from flexkv_b200.ssd import allocate_ssd_files
from test_engine_gpu import dev, one_op_graph
from test_engine_ssd_gpu import read_graph, wait_graphs, write_graph

pytestmark = pytest.mark.gpu


def engine_cache(lay, seed):
    """The engine's 16-bit layers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(lay.kv_shape[1:], generator=g, device="cuda").bfloat16() for _ in range(lay.num_layer)]


@pytest.mark.parametrize("pool", ["BLOCKWISE", "LAYERWISE"])
@pytest.mark.parametrize("use_mla,heads,dim,tpb", [(False, 4, 128, 16), (False, 2, 64, 32), (True, 1, 576, 64)])
def test_engine_and_files(tmp_path, pool, use_mla, heads, dim, tpb):
    """Blocks of a 16-bit cache: packed, to the host pool and its files, the pool and the staging cleared, back into
    other staging blocks and unpacked into other blocks of the cache: the quantised values, bit for bit."""
    layers, n, blocks = 3, 7, 12
    lay = KVCacheLayout(KVCacheLayoutType.LAYERWISE, layers, blocks, tpb, heads, dim, use_mla)
    host = KVCacheLayout(KVCacheLayoutType[pool], layers, 16, tpb, heads, dim, use_mla).fp4()
    disk = KVCacheLayout(KVCacheLayoutType[pool], layers, 24, tpb, heads, dim, use_mla).fp4()
    kv, staging = engine_cache(lay, 1), fp4_cache.allocate_fp4_layers(lay, "cuda")
    cpu = torch.zeros(host.get_total_elements(), dtype=torch.uint8).pin_memory()
    files, per_file = allocate_ssd_files(disk, 2, str(tmp_path / "ssd"), max_blocks_per_file=24)
    eng = TransferEngine([staging], cpu, lay.fp4(), host, ssd_files=files, ssd_layout=disk, ssd_num_blocks_per_file=per_file)
    r = np.random.RandomState(2)
    src, at, back, dst = (r.permutation(blocks)[:n] for _ in range(4))
    cpu_ids, ssd_ids = r.permutation(16)[:n], r.permutation(24)[:n]
    t = torch.from_numpy
    try:
        fp4_cache.fp4_pack_blocks(kv, staging, t(src), t(at))
        torch.cuda.synchronize()  # the engine copies on streams of its own
        held = [x[:, at].cpu() for x in staging]
        g = write_graph(at, cpu_ids, ssd_ids, layers)
        eng.submit_transfer_graph(g)
        wait_graphs(eng, [g.graph_id])
        for x in staging:
            x.fill_(255)
        cpu.zero_()
        torch.cuda.synchronize()
        g = read_graph(back, cpu_ids, ssd_ids, layers)
        eng.submit_transfer_graph(g)
        wait_graphs(eng, [g.graph_id])
        assert not eng.failed_ops
        torch.cuda.synchronize()
        out = [torch.zeros_like(x) for x in kv]
        fp4_cache.fp4_unpack_blocks(staging, out, t(back), t(dst))
        for x, h, y, z in zip(staging, held, out, kv):
            assert torch.equal(x[:, back].cpu(), h)
            assert np.array_equal(y[:, dst].double().cpu().numpy(), M.dequantise(*M.quantise(z[:, src].double().cpu().numpy())))
    finally:
        eng.shutdown()


@pytest.mark.parametrize("tp", [2, 4])
def test_ranks_share_a_block_by_heads(tp):
    """Each rank's 4-bit layers hold its heads; what the ranks put into the pool is what one rank with all heads reads,
    and the other way round."""
    layers, heads, dim, tpb, blocks, n = 2, 8, 64, 16, 20, 9
    lay = KVCacheLayout(KVCacheLayoutType.LAYERWISE, layers, blocks, tpb, heads, dim)
    host = KVCacheLayout(KVCacheLayoutType.BLOCKWISE, layers, 16, tpb, heads, dim).fp4()
    kv = engine_cache(lay, 3)
    whole = fp4_cache.allocate_fp4_layers(lay, "cuda")
    every = torch.arange(blocks)
    fp4_cache.fp4_pack_blocks(kv, whole, every, every)
    hp = heads // tp
    ranks = [[x[:, :, r * hp:(r + 1) * hp].contiguous().to(dev(r)) for x in whole] for r in range(tp)]
    # a rank that packs its own heads of the 16-bit cache has the same bytes
    own = fp4_cache.allocate_fp4_layers(lay.div_head(tp), "cuda")
    fp4_cache.fp4_pack_blocks([x[:, :, :, hp:2 * hp].contiguous() for x in kv], own, every, every)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(own, ranks[1]))
    cpu = torch.zeros(host.get_total_elements(), dtype=torch.uint8)
    one = [torch.full_like(x, 255) for x in whole]
    many = TransferEngine(ranks, cpu, lay.fp4().div_head(tp), host, tp, 1)
    single = TransferEngine([one], cpu, lay.fp4(), host)
    r = np.random.RandomState(4)
    a, b, c, pool = r.permutation(blocks)[:n], r.permutation(blocks)[:n], r.permutation(blocks)[:n], r.permutation(16)[:n]

    def move(eng, kind, gpu_ids):
        torch.cuda.synchronize()
        g, _ = one_op_graph(kind, gpu_ids, pool)
        eng.submit_transfer_graph(g)
        wait_graphs(eng, [g.graph_id])
        assert not eng.failed_ops
        torch.cuda.synchronize()
    try:
        move(many, TransferType.D2H, a)
        move(single, TransferType.H2D, b)
        for x, y in zip(one, whole):
            assert torch.equal(x[:, b], y[:, a])
        cpu.zero_()
        move(single, TransferType.D2H, b)
        for rank in ranks:
            for x in rank:
                x.fill_(255)
        move(many, TransferType.H2D, c)
        for i, rank in enumerate(ranks):
            for x, y in zip(rank, whole):
                assert torch.equal(x[:, c].cpu(), y[:, a, i * hp:(i + 1) * hp].cpu())
    finally:
        many.shutdown()
        single.shutdown()
