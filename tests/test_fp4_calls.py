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


# ---- outputs that share memory --------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def share_memory(tmp_path_factory):
    """rows_share_memory of csrc/fp4_overlap.h, on plain numbers."""
    import os
    import subprocess
    from flexkv_b200.build import CSRC
    d = tmp_path_factory.mktemp("overlap")
    (d / "o.cpp").write_text('#include "fp4_overlap.h"\nextern "C" int share(const int64_t *a, const int64_t *b) {\n'
                             '  auto s = [](const int64_t *x) { return fkv::RowSet{(uintptr_t)x[0], x[1], x[2], x[3], x[4], x[5]}; };\n'
                             '  return fkv::rows_share_memory(s(a), s(b));\n}\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "o.so"), str(d / "o.cpp")], check=True)
    f = ctypes.CDLL(os.path.join(d, "o.so")).share
    return lambda a, b: bool(f((ctypes.c_int64 * 6)(*a), (ctypes.c_int64 * 6)(*b)))


def pieces(base, tokens, heads, token, head, nbytes):
    at = base + np.arange(tokens)[:, None] * token + np.arange(heads) * head
    return set((at.reshape(-1, 1) + np.arange(nbytes)).reshape(-1).tolist())


def test_rows_that_share_memory(share_memory):
    """Against every byte of both sets: equal and unlike strides, interleaved, self-overlapping, single rows."""
    r = np.random.RandomState(0)
    seen = [0, 0, 0, 0]
    for _ in range(6000):
        tokens, heads, nbytes = r.randint(0, 6), r.randint(1, 5), r.choice([4, 8])
        strides = lambda: (int(r.randint(0, 12)) * 4 if tokens > 1 else 0, int(r.randint(0, 12)) * 4 if heads > 1 else 0)  # noqa: E731
        (ta, ha), (tb, hb) = strides(), strides()
        alike = r.rand() < 0.6
        if alike:
            tb, hb = ta, ha
        a = (1000, tokens, heads, ta, ha, nbytes)
        b = (1000 + int(r.randint(-20, 21)) * 4, tokens, heads, tb, hb, nbytes)
        want = bool(pieces(*a) & pieces(*b))
        assert share_memory(a, b) == want and share_memory(b, a) == want, (a, b, want)
        seen[2 * want + alike] += 1
    assert min(seen) > 100
    far = 1 << 45  # no product passes 64 bits at real sizes
    assert not share_memory((far, 32768, 8, 12288, 256, 256), (far + 2048, 32768, 8, 12288, 256, 256))
    assert share_memory((far, 32768, 8, 12288, 256, 256), (far + 12288 * 32767 + 1792, 32768, 8, 12288, 256, 256))
    assert not share_memory((far, 32768, 8, 12288, 256, 256), (far + 12288 * 32768 + 1792, 32768, 8, 12288, 256, 256))
    assert share_memory((far, 1 << 25, 2, 256, 128, 128), (far, 1 << 25, 2, 128, 1 << 32, 128))


@pytest.mark.gpu
def test_strided_outputs_that_share_memory_are_refused():
    layer, slots = torch.zeros(2, 4, 4, 1, 9 * 64, dtype=torch.uint8, device="cuda"), torch.arange(5, device="cuda")
    buf = torch.zeros(6, 8, 64, dtype=torch.bfloat16, device="cuda")
    tables, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")

    def attend(q, out):
        return fp4_cache.fp4_attention(layer, q, tables, lens, out=out)
    for q, out in ((buf[:5, :4], buf[1:, :4]), (buf[:5, :4], buf[:5, 2:6]), (buf[:5, ::2], buf[:5, :4]),
                   (buf[:1, :4], buf[:1, 3:7]), (buf[:4, :4].transpose(0, 1), buf[:4, :4])):
        with pytest.raises(RuntimeError, match="out may be q"):
            attend(q, out)
        with pytest.raises(RuntimeError, match="k and v overlap"):
            fp4_cache.fp4_read(layer, slots[:q.shape[0]], out=(q, out))
    with pytest.raises(RuntimeError, match="k and v overlap"):
        fp4_cache.fp4_read(layer, slots, out=(buf[:5, :4], buf[:5, :4]))
    # side by side, interleaved, far apart, the same place
    for q, out in ((buf[:5, :4], buf[:5, 4:]), (buf[:5, ::2], buf[:5, 1::2]), (buf[:2, :4], buf[2:4, :4])):
        attend(q, out)
        fp4_cache.fp4_read(layer, slots[:q.shape[0]], out=(q, out))
    attend(buf[:5, :4], buf[:5, :4])


@pytest.mark.gpu
def test_a_layer_is_written_once():
    """The same tensor twice among the layers to write to is refused; to read from it is fine."""
    src, packed, dst, (a, b, _) = converted(4, 3)
    for lists in ([packed[0], packed[1], packed[0]], [packed[0], packed[0].view(packed[0].shape), packed[1]]):
        with pytest.raises(RuntimeError, match="fp4_layers: a layer to write to appears twice"):
            fp4_cache.fp4_pack_blocks(src, lists, a, b)
    with pytest.raises(RuntimeError, match="kv_layers: a layer to write to appears twice"):
        fp4_cache.fp4_unpack_blocks(packed, [dst[2], dst[1], dst[2]], b, a)
    assert all(bool((x == 255).all()) for x in packed) and all(bool((x == 5.0).all()) for x in dst)
    fp4_cache.fp4_pack_blocks([src[0], src[0], src[1]], packed, a, b)
    assert torch.equal(packed[0], packed[1]) and not torch.equal(packed[0], packed[2])
    fp4_cache.fp4_unpack_blocks([packed[0], packed[0], packed[2]], dst, b, a)
    assert torch.equal(dst[0], dst[1])
    empty = [x[:, :0] for x in packed]
    fp4_cache.fp4_pack_blocks(src, empty, a[:0], b[:0])


# ---- the module they are in -----------------------------------------------------------------------------------


def test_the_module_belongs_to_one_torch_and_python(monkeypatch):
    """Another version of either is not served by what was built for this one."""
    import sysconfig
    from flexkv_b200 import build
    path = build.binding_path()
    assert torch.__version__ in path and sysconfig.get_config_var("SOABI") in path
    assert not build._binding_stale()
    monkeypatch.setattr(torch, "__version__", "2.99.0+cu999")
    assert build.binding_path() != path and build._binding_stale()
    monkeypatch.setattr(fp4_cache, "_module", None)
    with pytest.raises(ImportError, match="2.99.0.cu999.*flexkv_b200.build"):
        fp4_cache._native()


def test_the_library_is_built_without_torchs_headers(monkeypatch, tmp_path):
    from flexkv_b200 import build
    assert build._binding_lacks() == ""
    monkeypatch.setattr(build, "_binding_stale", lambda: True)
    monkeypatch.setattr(build, "_binding_includes", lambda: [str(tmp_path)])
    monkeypatch.setattr(build, "_build_binding", lambda verbose: pytest.fail("built without its headers"))
    with pytest.warns(UserWarning, match="fp4_cache is not built: Python.h not found"):
        assert build.build() == build.LIB_PATH
    (tmp_path / "Python.h").write_text("")
    with pytest.warns(UserWarning, match="python_variable.h not found"):
        build.build()


# ---- beside autograd ------------------------------------------------------------------------------------------


def small():
    layer = torch.zeros(2, 4, 2, 1, 9 * 64, dtype=torch.uint8, device="cuda")
    x = torch.randn(5, 2, 64, device="cuda").bfloat16()
    return layer, x, torch.arange(5, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), \
        torch.full((1,), 5, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
def test_what_is_written_gets_a_new_version():
    """A backward pass that kept a tensor which a call has since written is refused by autograd."""
    layer, x, slots, tables, lens = small()
    kv, ids = [torch.zeros(2, 4, 16, 2, 64, dtype=x.dtype, device="cuda")], torch.arange(2)

    def writes(t, call):
        w = torch.ones((), device="cuda", requires_grad=True)
        y = (w * t).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    out, other = torch.zeros_like(x), torch.zeros_like(x)
    writes(layer, lambda: fp4_cache.fp4_write(layer, x, x, slots))
    writes(out, lambda: fp4_cache.fp4_read(layer, slots, out=(out, other)))
    writes(other, lambda: fp4_cache.fp4_read(layer, slots, out=(out, other)))
    writes(out, lambda: fp4_cache.fp4_attention(layer, x, tables, lens, out=out))
    writes(layer, lambda: fp4_cache.fp4_pack_blocks(kv, [layer], ids, ids))
    writes(kv[0], lambda: fp4_cache.fp4_unpack_blocks([layer], kv, ids, ids))
    # what is only read stays as it was, and tensors of inference mode have no version
    w = torch.ones((), device="cuda", requires_grad=True)
    y = (w * x).sum() + (w * layer).sum()
    fp4_cache.fp4_read(layer, slots)
    fp4_cache.fp4_attention(layer, x, tables, lens)
    y.backward()
    with torch.inference_mode():
        layer2, x2, *rest = small()
        fp4_cache.fp4_write(layer2, x2, x2, rest[0])
        fp4_cache.fp4_read(layer2, rest[0], out=(x2, torch.zeros_like(x2)))


@pytest.mark.gpu
def test_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    layer, x, slots, tables, lens = small()
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        with torch.no_grad():
            for call in (lambda: fp4_cache.fp4_write(layer, d, x, slots), lambda: fp4_cache.fp4_write(layer, x, d, slots),
                         lambda: fp4_cache.fp4_attention(layer, d, tables, lens),
                         lambda: fp4_cache.fp4_pack_blocks([fw.make_dual(torch.zeros(2, 4, 16, 2, 64, device="cuda").bfloat16(),
                                                                         torch.ones(2, 4, 16, 2, 64, device="cuda").bfloat16())],
                                                           [layer], slots[:1], slots[:1])):
                with pytest.raises(RuntimeError, match="tangent"):
                    call()
        fp4_cache.fp4_write(layer, x, x, slots)
    assert not bool((layer == 0).all())


# ---- several threads ------------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_threads():
    """Every operator from several threads at once, each on a stream of its own: what one thread alone gets."""
    import threading

    def work(seed, stream, turns, out):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.cuda.stream(stream):
            layer = torch.zeros(2, 70, 2, 1, 9 * 64, dtype=torch.uint8, device="cuda")
            kv = torch.zeros(2, 70, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
            tables = torch.randperm(70, generator=g, device="cuda")[:66].view(2, 33).int()
            lens = torch.tensor([500, 177 + seed], dtype=torch.int32, device="cuda")
            rows = torch.randn(1120, 2, 64, generator=g, device="cuda").bfloat16()
            slots = torch.randperm(1120, generator=g, device="cuda")
            ids = torch.arange(40)
            for turn in range(turns):
                fp4_cache.fp4_write(layer, rows, rows, slots)
                got = [fp4_cache.fp4_attention(layer, torch.randn(2 * n, 4, 64, generator=g, device="cuda").bfloat16(), tables, lens)
                       for n in (1, 3, 40)]
                fp4_cache.fp4_unpack_blocks([layer], [kv], ids + turn, ids)
                fp4_cache.fp4_pack_blocks([kv], [layer], ids.cuda(), ids + turn)
                got += [*fp4_cache.fp4_read(layer, slots), kv.clone()]
                out.append(got)
        stream.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    want = [[] for _ in streams]
    for i, s in enumerate(streams):
        work(i, s, 6, want[i])
    got = [[] for _ in streams]
    threads = [threading.Thread(target=work, args=(i, s, 6, got[i])) for i, s in enumerate(streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, g in zip(want, got):
        assert len(w) == len(g) == 6
        assert all(torch.equal(x, y) for a, b in zip(w, g) for x, y in zip(a, b))
