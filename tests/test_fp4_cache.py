"""CPU: the 4-bit cache's format, byte layout and argument checks (every
refusal comes before any device work)."""
import ctypes

import numpy as np
import pytest
import torch

import fp4_model as M
from flexkv_b200 import _lib, fp4_cache
from flexkv_b200.layout import KVCacheLayout, KVCacheLayoutType, cpu_byte_strides, gpu_byte_strides

INV, MIS, UNS = _lib.FKV_ERR_INVALID_ARG, _lib.FKV_ERR_MISALIGNED, _lib.FKV_ERR_UNSUPPORTED


def test_model_format():
    """The scale grid is the upper byte of non-negative halves without their sign, and stored values
    are exact in bfloat16 and half."""
    codes = np.arange(227, dtype=np.uint16)
    assert np.array_equal((codes << 7).view(np.float16).astype(np.float64), M.SCALES)
    v = torch.tensor(np.outer(M.SCALES, M.E2M1))
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(v.to(t).double(), v)
    # ties go to the even code on both grids
    assert M.nearest_code(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]), M.E2M1).tolist() == [0, 2, 2, 4, 4, 6, 6]
    x = np.random.RandomState(0).randn(3, 16, 64)
    c, s = M.quantise(x)
    u = M.unit_bytes(c, s)
    assert u.shape == (3, 9 * 64)
    c2, s2 = M.unit_codes(u)
    assert np.array_equal(c, c2) and np.array_equal(s, s2)
    err = np.abs(M.dequantise(c, s) - x).reshape(3, 16, 4, 16)
    amax = np.abs(x).reshape(3, 16, 4, 16).max(-1, keepdims=True)
    assert (err <= amax / 6 * (1 + 2 ** -4) + 1e-12).all()  # half a step (1) of the largest values' spacing 2


def test_layout_bytes():
    lay = KVCacheLayout(KVCacheLayoutType.LAYERWISE, 3, 10, 32, 4, 128)
    b = lay.fp4()
    assert b.get_chunk_size() == 32 * 4 * 128 * 9 // 16
    g = gpu_byte_strides(b, 1)
    t = fp4_cache.allocate_fp4_layers(lay, "cpu")
    assert len(t) == 3 and t[0].shape == (2, 10, 4, 2, 9 * 128)
    assert (g["kv"], g["block"]) == (t[0].stride(0), t[0].stride(1))
    assert g["chunk"] == t[0][0, 0].numel()
    blk = KVCacheLayout(KVCacheLayoutType.BLOCKWISE, 3, 10, 32, 4, 128).fp4()
    assert cpu_byte_strides(blk, 1)["block"] == 3 * 2 * g["chunk"]
    mla = KVCacheLayout(KVCacheLayoutType.LAYERWISE, 1, 5, 64, 1, 576, is_mla=True)
    assert fp4_cache.allocate_fp4_layers(mla, "cpu")[0].shape == (1, 5, 1, 4, 9 * 576)
    for bad in (KVCacheLayout(KVCacheLayoutType.LAYERWISE, 1, 5, 8, 1, 64),
                KVCacheLayout(KVCacheLayoutType.LAYERWISE, 1, 5, 16, 1, 40)):
        with pytest.raises(ValueError):
            bad.fp4()
    with pytest.raises(ValueError):
        fp4_cache.allocate_fp4_layers(KVCacheLayout(KVCacheLayoutType.BLOCKWISE, 1, 5, 16, 1, 64), "cpu")


BUF = (ctypes.c_char * 4096)()
BASE = (ctypes.addressof(BUF) + 63) // 64 * 64


def tokens_args(**kw):
    a = dict(layer=BASE, kv=2, blocks=4, tpb=16, heads=2, dim=64, kvs=1 << 14, bs=1 << 10, k=BASE, v=BASE,
             kt=256, kh=128, vt=256, vh=128, dtype=0, slots=BASE, n=3, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(kv=3), INV), (dict(tpb=8), INV), (dict(tpb=0), INV), (dict(dim=40), INV), (dict(dim=0), INV),
    (dict(heads=0), INV), (dict(blocks=-1), INV), (dict(n=-1), INV), (dict(k=None), INV), (dict(v=None), INV),
    (dict(slots=None), INV), (dict(layer=None), INV), (dict(kv=1), INV), (dict(dtype=2), UNS),
    (dict(blocks=1 << 62), INV), (dict(heads=65536, dim=65536), INV),
    (dict(layer=BASE + 8), MIS), (dict(kvs=8), MIS), (dict(bs=24), MIS), (dict(k=BASE + 2), MIS),
    (dict(kt=130), MIS), (dict(vh=8), MIS), (dict(n=1 << 62), INV)])
def test_token_calls_refuse(kw, code):
    for name in ("fkv_fp4_write", "fkv_fp4_read"):
        assert getattr(_lib.load(), name)(*tokens_args(**kw)) == code
        assert name.encode() in _lib.load().fkv_last_error() or "n" in kw


def test_token_calls_of_nothing():
    for name in ("fkv_fp4_write", "fkv_fp4_read"):
        assert getattr(_lib.load(), name)(*tokens_args(n=0)) == 0


def block_args(**kw):
    ptrs = (ctypes.c_void_p * 2)(BASE, BASE)
    a = dict(layers=2, first=ptrs, second=ptrs, kv=2, tpb=16, heads=2, dim=64, nb1=4, kvs1=1 << 14, bs1=1 << 10,
             nb2=4, kvs2=1 << 14, bs2=1 << 10, dtype=0, ids1=BASE, ids2=BASE, n=3, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(kv=0), INV), (dict(tpb=24), INV), (dict(dim=72), INV), (dict(layers=-1), INV), (dict(n=-2), INV),
    (dict(first=None), INV), (dict(second=None), INV), (dict(ids1=None), INV), (dict(ids2=None), INV),
    (dict(first=(ctypes.c_void_p * 2)(BASE, None)), INV), (dict(second=(ctypes.c_void_p * 2)(BASE + 8, BASE)), MIS),
    (dict(kvs1=24), MIS), (dict(bs2=8), MIS), (dict(dtype=5), UNS), (dict(nb1=-1), INV), (dict(nb2=-1), INV)])
def test_block_calls_refuse(kw, code):
    for name in ("fkv_fp4_pack_blocks", "fkv_fp4_unpack_blocks"):
        assert getattr(_lib.load(), name)(*block_args(**kw)) == code


def test_block_calls_of_nothing():
    for name in ("fkv_fp4_pack_blocks", "fkv_fp4_unpack_blocks"):
        assert getattr(_lib.load(), name)(*block_args(n=0)) == 0
        assert getattr(_lib.load(), name)(*block_args(layers=0)) == 0


def attention_args(**kw):
    a = dict(layer=BASE, blocks=4, tpb=16, heads=2, dim=64, kvs=1 << 14, bs=1 << 10, q=BASE, out=BASE, lse=None,
             qt=512, qh=128, ot=512, oh=128, dtype=0, n=4, q_heads=4, tables=BASE, ts=4, max_blocks=4, lens=BASE,
             cu=None, seqs=2, max_q=2, scale=0.1, causal=1, ws=BASE, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(tpb=8), INV), (dict(dim=96), UNS), (dict(dim=576), UNS), (dict(dtype=7), UNS), (dict(q_heads=3), INV),
    (dict(heads=0), INV), (dict(q_heads=0), INV), (dict(blocks=-1), INV), (dict(n=-1), INV), (dict(seqs=-1), INV),
    (dict(max_blocks=-1), INV), (dict(scale=float("nan")), INV), (dict(scale=float("inf")), INV), (dict(q=None), INV),
    (dict(out=None), INV), (dict(lens=None), INV), (dict(tables=None), INV), (dict(layer=None), INV),
    (dict(n=5), INV), (dict(layer=BASE + 4), MIS), (dict(q=BASE + 8), MIS), (dict(out=BASE + 2), MIS),
    (dict(qt=130), MIS), (dict(qh=72), MIS), (dict(ot=8), MIS), (dict(oh=24), MIS), (dict(kvs=8), MIS), (dict(bs=8), MIS)])
def test_attention_refuses(kw, code):
    assert _lib.load().fkv_fp4_attention(*attention_args(**kw)) == code
    assert b"fkv_fp4_attention" in _lib.load().fkv_last_error()


def test_attention_of_nothing():
    assert _lib.load().fkv_fp4_attention(*attention_args(n=0)) == 0
    assert _lib.load().fkv_fp4_attention(*attention_args(n=0, seqs=0)) == 0


def test_python_refuses_host_tensors():
    layer = torch.zeros(2, 4, 2, 1, 9 * 64, dtype=torch.uint8)
    x, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp4_cache.fp4_write(layer, x, x, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp4_cache.fp4_read(layer, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp4_cache.fp4_attention(layer, x, slots, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp4_cache.fp4_pack_blocks([x], [layer], slots, slots)
    with pytest.raises(RuntimeError, match="at least one"):
        fp4_cache.fp4_pack_blocks([], [], slots, slots)
    with pytest.raises(RuntimeError, match="uint8"):
        fp4_cache.fp4_read(layer.float(), slots)
    with pytest.raises(RuntimeError, match=r"got \[2, 4, 2, 1, 540\]"):
        fp4_cache.fp4_read(layer[..., :540], slots)
    with pytest.raises(RuntimeError, match="contiguous"):
        fp4_cache.fp4_read(layer[:, :, :, :, ::1].transpose(1, 2), slots)
    for args in ((layer,), (layer, x, x, slots, slots)):
        with pytest.raises(TypeError):
            fp4_cache._native().write(*args)
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        fp4_cache.fp4_write([layer], x, x, slots)


@pytest.mark.parametrize("flags", [4, -1, 7])
def test_attention_refuses_unknown_flags(flags):
    assert _lib.load().fkv_fp4_attention(*attention_args(causal=flags)) == INV
    assert b"flags" in _lib.load().fkv_last_error()
