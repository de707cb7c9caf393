"""The 4-bit cache's calls: what they accept and refuse, and that they only
enqueue work (CPU where no device is needed, else GPU)."""
import ctypes

import numpy as np
import pytest
import torch

import fp4_model as M
from flexkv_b200 import _lib, fp4_cache
from test_fp4_cache import BASE, block_args

INV = _lib.FKV_ERR_INVALID_ARG


# ---- block ids on the host ------------------------------------------------------------------------------------


@pytest.mark.parametrize("name", ["fkv_fp4_pack_blocks_listed", "fkv_fp4_unpack_blocks_listed"])
def test_listed_block_calls_refuse(name):
    call = getattr(_lib.load(), name)

    def args(lists, **kw):
        a = block_args(**kw)
        return a[:-1] + [lists] + a[-1:]
    for lists in (4, -1, 7):
        assert call(*args(lists)) == INV and b"host_lists" in _lib.load().fkv_last_error()
    for kw in (dict(ids1=None), dict(ids2=None), dict(first=None), dict(n=-1), dict(kv=0)):
        assert call(*args(3, **kw)) == INV
    assert call(*args(3, n=0)) == 0 and call(*args(3, layers=0)) == 0
    assert ctypes.addressof(ctypes.c_char.from_address(BASE)) == BASE


def converted(n, layers=2, pool=None, tpb=16, heads=2, dim=64, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = pool or n + 5
    src = [torch.randn(2, pool, tpb, heads, dim, generator=g, device="cuda").bfloat16() for _ in range(layers)]
    packed = [torch.full((2, pool + 1, heads, tpb // 16, 9 * dim), 255, dtype=torch.uint8, device="cuda") for _ in range(layers)]
    dst = [torch.full_like(x, 5.0) for x in src]
    ids = [torch.randperm(pool, generator=g, device="cuda")[:n] for _ in range(3)]
    return src, packed, dst, ids


@pytest.mark.gpu
@pytest.mark.parametrize("n,layers", [(1, 2), (9, 28), (255, 2), (256, 1), (257, 1), (1000, 1), (3, 130)])
def test_host_ids_are_as_device_ids(n, layers):
    """Either list or both on the host, more pairs than one launch takes: bit for bit what ids on the device give."""
    src, packed, dst, (a, b, c) = converted(n, layers)
    fp4_cache.fp4_pack_blocks(src, packed, a, b)
    fp4_cache.fp4_unpack_blocks(packed, dst, b, c)
    host = lambda x, on: x.cpu() if on else x  # noqa: E731
    for lists in (1, 2, 3):
        p, d = [torch.full_like(x, 255) for x in packed], [torch.full_like(x, 5.0) for x in dst]
        fp4_cache.fp4_pack_blocks(src, p, host(a, lists & 1), host(b, lists & 2))
        fp4_cache.fp4_unpack_blocks(p, d, host(b, lists & 2), host(c, lists & 1))
        assert all(torch.equal(x, y) for x, y in zip(packed + dst, p + d))
    want = M.dequantise(*M.quantise(src[-1].double().cpu().numpy()[:, a.cpu().numpy()]))
    assert np.array_equal(dst[-1].double().cpu().numpy()[:, c.cpu().numpy()], want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [9, 600])
def test_host_ids_wait_for_nothing(n):
    """The calls return while what is before them on the stream still runs; the ids may change as soon as they do."""
    src, packed, dst, (a, b, c) = converted(n)
    fp4_cache.fp4_pack_blocks(src, packed, a, b)
    fp4_cache.fp4_unpack_blocks(packed, dst, b, c)
    p, d = [torch.full_like(x, 255) for x in packed], [torch.full_like(x, 5.0) for x in dst]
    ids = [torch.empty(n, dtype=torch.int64, pin_memory=pin) for pin in (False, True, False)]
    for x, y in zip(ids, (a, b, c)):
        x.copy_(y)
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)  # half a second and more
    event = torch.cuda.Event()
    event.record()
    fp4_cache.fp4_pack_blocks(src, p, ids[0], ids[1])
    fp4_cache.fp4_unpack_blocks(p, d, ids[1], ids[2])
    assert not event.query(), "the calls waited for the stream"
    for x in ids:
        x.zero_()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(packed + dst, p + d))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [9, 600])
def test_host_ids_in_a_graph(n):
    """A captured call keeps its ids, whatever becomes of the tensors that held them."""
    src, packed, dst, (a, b, c) = converted(n)
    ids = [x.cpu() for x in (a, b, c)]
    fp4_cache.fp4_pack_blocks(src, packed, *ids[:2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp4_cache.fp4_pack_blocks(src, packed, ids[0], b)
        fp4_cache.fp4_unpack_blocks(packed, dst, ids[1], ids[2])
    for x in ids:
        x.fill_(-7)
    for turn in range(3):
        for x in src:
            x.normal_()
        graph.replay()
        p, d = [torch.full_like(x, 255) for x in packed], [torch.full_like(x, 5.0) for x in dst]
        fp4_cache.fp4_pack_blocks(src, p, a, b)
        fp4_cache.fp4_unpack_blocks(p, d, b, c)
        assert all(torch.equal(x, y) for x, y in zip(packed + dst, p + d))
