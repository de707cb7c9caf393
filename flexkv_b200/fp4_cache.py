"""The paged KV cache in 4 bits: operators over ``fkv_fp4_*`` (csrc/fp4_cache.cu,
csrc/fp4_attention.cu), for the GPU of the tensors and its current stream.

A layer is a uint8 tensor [kv, num_blocks, num_heads, tokens_per_block / 16,
9 * head_size] (``allocate_fp4_layers``); the last axis is a unit, 16 tokens
of one head: 16 rows of head_size / 2 bytes (two e2m1 values a byte, the even
channel in the low four bits), then 16 rows of head_size / 16 scale bytes, one
for each 16 channels.  A scale byte c stands for the half-precision number
with the bits c << 7.  4.5 bits a value, 3.56 times the blocks of a 16-bit
cache in the same memory, and in each transfer.

  * ``fp4_write`` quantises new tokens into their slots, ``fp4_read`` gives
    tokens back in 16 bits;
  * ``fp4_pack_blocks`` / ``fp4_unpack_blocks`` convert blocks of every layer
    between a 16-bit cache and a 4-bit one, before a D2H and after an H2D copy;
  * ``fp4_attention`` reads the 4-bit cache: one new token a sequence
    (decoding), a few, or chunks of prompts behind a cached prefix.

A 4-bit block is an ordinary chunk of bytes: ``KVCacheLayout.fp4()`` gives
the layout whose strides ``transfer_kv_blocks``, ``TransferEngine``,
``CpuCacheIndex`` and the SSD tier take, and those move it unchanged.

Every operator only enqueues work (nothing waits), so it can be captured into
a CUDA graph.  Wrong shapes, types, devices or alignments raise RuntimeError
before anything is launched.  Slots, ids, tables and lengths in device memory
are checked on the device: entries that point outside a pool are skipped (see
each operator).  Inference only: an input that requires a gradient is refused
while gradients are recorded.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import FKV_DTYPE_BF16, FKV_DTYPE_FP16, check
from .layout import KVCacheLayout, KVCacheLayoutType

__all__ = ["allocate_fp4_layers", "fp4_write", "fp4_read", "fp4_pack_blocks", "fp4_unpack_blocks",
           "fp4_attention"]

_DTYPES = {torch.bfloat16: FKV_DTYPE_BF16, torch.float16: FKV_DTYPE_FP16}
UNIT_TOKENS = 16


def allocate_fp4_layers(layout: KVCacheLayout, device) -> List[torch.Tensor]:
    """Zeroed 4-bit layers for the cache that ``layout`` (LAYERWISE, the
    16-bit cache's geometry) describes: one tensor per layer."""
    if layout.type != KVCacheLayoutType.LAYERWISE:
        raise ValueError("GPU layers are LAYERWISE")
    b = layout.fp4()
    return [torch.zeros(b.kv_dim, b.num_block, b.num_head, b.tokens_per_block // UNIT_TOKENS,
                        UNIT_TOKENS * b.head_size, dtype=torch.uint8, device=device)
            for _ in range(b.num_layer)]


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise RuntimeError(message)


def _geometry(layer: torch.Tensor, name: str = "layer") -> Tuple[int, int, int, int, int, int, int]:
    """(kv, blocks, tokens per block, heads, head size, kv stride, block stride)."""
    _require(isinstance(layer, torch.Tensor) and layer.dtype == torch.uint8 and layer.dim() == 5,
             f"{name} must be a uint8 tensor [kv, blocks, heads, tokens_per_block / 16, 9 * head_size]")
    _require(layer.is_cuda, f"{name} must be a CUDA tensor")
    kv, blocks, heads, units, nbytes = layer.shape
    _require(kv in (1, 2) and heads > 0 and units > 0 and nbytes > 0 and nbytes % 144 == 0,
             f"{name} must be [kv, blocks, heads, tokens_per_block / 16, 9 * head_size] with kv 1 or 2 and "
             f"head_size a multiple of 16, got {tuple(layer.shape)}")
    s = layer.stride()
    _require(s[4] == 1 and (units == 1 or s[3] == nbytes) and (heads == 1 or s[2] == units * nbytes),
             f"{name}: a block must be contiguous")
    return kv, blocks, units * UNIT_TOKENS, heads, nbytes // 9, s[0], s[1]


def _ids(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device, dim: int = 1) -> None:
    _require(isinstance(t, torch.Tensor) and t.dtype == dtype and t.dim() == dim,
             f"{name} must be a {dim}-D {dtype} tensor")
    _require(t.device == device, f"{name} must be on {device}, got {t.device}")


def _rows(t: torch.Tensor, name: str, tokens: int, heads: int, dim: int, dtype: torch.dtype,
          device: torch.device) -> Tuple[int, int]:
    """Token and head stride in bytes of rows [tokens, heads, dim]."""
    _require(isinstance(t, torch.Tensor) and t.dtype == dtype and tuple(t.shape) == (tokens, heads, dim),
             f"{name} must be a {dtype} tensor of shape {(tokens, heads, dim)}")
    _require(t.device == device, f"{name} must be on {device}, got {t.device}")
    s = t.stride()
    _require(s[2] == 1, f"{name}: the channels of a head must be contiguous")
    # an axis of one entry is never stepped along: its stride says nothing
    return (2 * s[0] if tokens > 1 else 0), (2 * s[1] if heads > 1 else 0)


def _no_grad(*tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            _require(t is None or not t.requires_grad, "the 4-bit cache has no gradient: call under torch.no_grad()")


class _On:
    """Make `device` current for the call (nothing to do when it is)."""

    __slots__ = ("guard",)

    def __init__(self, device: torch.device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _stream(device: torch.device) -> int:
    return int(torch.cuda.current_stream(device).cuda_stream)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dtype(dtype: torch.dtype, name: str) -> int:
    _require(dtype in _DTYPES, f"{name} must be bfloat16 or half, got {dtype}")
    return _DTYPES[dtype]


def fp4_write(layer: torch.Tensor, k: torch.Tensor, v: Optional[torch.Tensor],
              slot_mapping: torch.Tensor) -> None:
    """Quantise the rows of ``k`` and ``v`` [tokens, num_heads, head_size]
    (bfloat16 or half; slices of a larger projection are fine while rows start
    on 16-byte boundaries) into slots ``slot_mapping`` [tokens] (int64, slot =
    block * tokens_per_block + offset) of ``layer``.  A negative slot, or one
    past the pool, drops its row (padding).  The other slots must differ from
    one another.  ``v`` is None for a latent layer (kv = 1)."""
    kv, blocks, tpb, heads, dim, kv_stride, block_stride = _geometry(layer)
    _no_grad(k, v)
    dev = layer.device
    _ids(slot_mapping, "slot_mapping", torch.int64, dev)
    n = slot_mapping.shape[0]
    _require((v is None) == (kv == 1), "v must be given for a layer of keys and values, and None for a latent layer")
    dt = _dtype(k.dtype, "k")
    kt, kh = _rows(k, "k", n, heads, dim, k.dtype, dev)
    vt, vh = _rows(v, "v", n, heads, dim, k.dtype, dev) if v is not None else (0, 0)
    slots = slot_mapping.contiguous()
    with _On(dev):
        check(_lib.load().fkv_fp4_write(layer.data_ptr(), kv, blocks, tpb, heads, dim, kv_stride, block_stride,
                                        k.data_ptr(), _ptr(v), kt, kh, vt, vh, dt, slots.data_ptr(), n,
                                        _stream(dev)), "fp4_write")


def fp4_read(layer: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
             out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The tokens in slots ``slot_mapping`` [tokens] as (k, v) [tokens,
    num_heads, head_size] of ``dtype`` (bfloat16 or half; stored values are
    exact in both), v None for a latent layer.  A negative slot, or one past
    the pool, reads as zeros.  ``out``: the tensors to fill, of that shape and
    type (rows on 16-byte boundaries)."""
    kv, blocks, tpb, heads, dim, kv_stride, block_stride = _geometry(layer)
    dev = layer.device
    _ids(slot_mapping, "slot_mapping", torch.int64, dev)
    n = slot_mapping.shape[0]
    dt = _dtype(dtype, "dtype")
    if out is None:
        k = torch.empty(n, heads, dim, dtype=dtype, device=dev)
        v = torch.empty(n, heads, dim, dtype=dtype, device=dev) if kv == 2 else None
    else:
        k, v = out
        _require((v is None) == (kv == 1), "out must hold v for a layer of keys and values, and None for a latent layer")
        _no_grad(k, v)
    kt, kh = _rows(k, "k", n, heads, dim, dtype, dev)
    vt, vh = _rows(v, "v", n, heads, dim, dtype, dev) if v is not None else (0, 0)
    slots = slot_mapping.contiguous()
    with _On(dev):
        check(_lib.load().fkv_fp4_read(layer.data_ptr(), kv, blocks, tpb, heads, dim, kv_stride, block_stride,
                                       k.data_ptr(), _ptr(v), kt, kh, vt, vh, dt, slots.data_ptr(), n,
                                       _stream(dev)), "fp4_read")
    return k, v


def _block_ids(t: torch.Tensor, name: str, pool: int, device: torch.device, distinct: bool) -> torch.Tensor:
    """Block ids on the device; host ids are checked first."""
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int64 and t.dim() == 1,
             f"{name} must be a 1-D torch.int64 tensor")
    if t.is_cuda:
        _require(t.device == device, f"{name} must be on {device} or on the host, got {t.device}")
        return t.contiguous()
    if t.numel():
        _require(int(t.min()) >= 0 and int(t.max()) < pool, f"{name}: a block id is outside [0, {pool})")
        _require(not distinct or t.unique().numel() == t.numel(), f"{name}: a block id appears twice")
    return t.to(device)


def _convert(call, where: str, kv_layers: Sequence[torch.Tensor], fp4_layers: Sequence[torch.Tensor],
             kv_block_ids: torch.Tensor, fp4_block_ids: torch.Tensor, pack: bool) -> None:
    _require(len(kv_layers) == len(fp4_layers) and len(kv_layers) > 0,
             "kv_layers and fp4_layers must hold the same layers, at least one")
    first = fp4_layers[0]
    kv, blocks, tpb, heads, dim, kv_stride, block_stride = _geometry(first, "fp4_layers[0]")
    dev = first.device
    shape, strides = first.shape, first.stride()
    for i, t in enumerate(fp4_layers):
        _require(t.dtype == torch.uint8 and t.shape == shape and t.stride() == strides and t.device == dev,
                 f"fp4_layers[{i}] must have the shape, strides and device of fp4_layers[0]")
    one = kv_layers[0]
    _require(isinstance(one, torch.Tensor) and one.dim() == 5 and one.shape[0] == kv
             and tuple(one.shape[2:]) == (tpb, heads, dim),
             f"a 16-bit layer must be [{kv}, blocks, {tpb}, {heads}, {dim}]")
    dt = _dtype(one.dtype, "a 16-bit layer")
    kshape, kstrides, kdtype = one.shape, one.stride(), one.dtype
    _require(kstrides[4] == 1 and (heads == 1 or kstrides[3] == dim) and kstrides[2] == heads * dim,
             "a block of a 16-bit layer must be contiguous")
    for i, t in enumerate(kv_layers):
        _require(t.dtype == kdtype and t.shape == kshape and t.stride() == kstrides and t.device == dev,
                 f"kv_layers[{i}] must have the type, shape and strides of kv_layers[0] and be on {dev}")
    _no_grad(*kv_layers)
    _require(kv_block_ids.numel() == fp4_block_ids.numel(), "kv_block_ids and fp4_block_ids differ in length")
    with _On(dev):
        a = _block_ids(kv_block_ids, "kv_block_ids", kshape[1], dev, not pack)
        b = _block_ids(fp4_block_ids, "fp4_block_ids", blocks, dev, pack)
        n = len(kv_layers)
        kp = (ctypes.c_void_p * n)(*[t.data_ptr() for t in kv_layers])
        fp = (ctypes.c_void_p * n)(*[t.data_ptr() for t in fp4_layers])
        kside = (kshape[1], 2 * kstrides[0], 2 * kstrides[1])
        fside = (blocks, kv_stride, block_stride)
        if pack:
            rc = call(n, kp, fp, kv, tpb, heads, dim, *kside, *fside, dt, a.data_ptr(), b.data_ptr(), a.numel(),
                      _stream(dev))
        else:
            rc = call(n, fp, kp, kv, tpb, heads, dim, *fside, *kside, dt, b.data_ptr(), a.data_ptr(), a.numel(),
                      _stream(dev))
        check(rc, where)


def fp4_pack_blocks(kv_layers: Sequence[torch.Tensor], fp4_layers: Sequence[torch.Tensor],
                    kv_block_ids: torch.Tensor, fp4_block_ids: torch.Tensor) -> None:
    """Quantise blocks ``kv_block_ids[i]`` of a 16-bit cache (one tensor [kv,
    blocks, tokens_per_block, num_heads, head_size] per layer) into blocks
    ``fp4_block_ids[i]`` of ``fp4_layers``, all layers in one launch.  Ids
    (int64) may be host tensors, which are checked, or device tensors, where a
    pair with an id outside its pool is skipped.  No destination may repeat."""
    _convert(_lib.load().fkv_fp4_pack_blocks, "fp4_pack_blocks", kv_layers, fp4_layers, kv_block_ids,
             fp4_block_ids, True)


def fp4_unpack_blocks(fp4_layers: Sequence[torch.Tensor], kv_layers: Sequence[torch.Tensor],
                      fp4_block_ids: torch.Tensor, kv_block_ids: torch.Tensor) -> None:
    """The other way: blocks ``fp4_block_ids[i]`` of ``fp4_layers`` into
    blocks ``kv_block_ids[i]`` of the 16-bit cache ``kv_layers``."""
    _convert(_lib.load().fkv_fp4_unpack_blocks, "fp4_unpack_blocks", kv_layers, fp4_layers, kv_block_ids,
             fp4_block_ids, False)


def fp4_attention(layer: torch.Tensor, q: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  cu_seqlens_q: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                  softmax_scale: Optional[float] = None, causal: bool = True,
                  out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of the new tokens ``q`` [tokens, num_q_heads, head_size]
    (bfloat16 or half) over the 4-bit ``layer``, to which their own keys and
    values have been written already.

    ``block_tables`` [sequences, max_blocks], ``seq_lens`` [sequences] (tokens
    in the cache, the new ones among them) and ``cu_seqlens_q`` [sequences + 1]
    (the first row of each sequence in q; None: the same number of rows each)
    are int32 tensors on the device.  ``max_q_len``, the most new tokens of a
    sequence, only chooses the kernel.  Row i of a sequence of n new tokens sees
    the keys up to position seq_len - n + i (``causal``) or all.  A row that
    sees nothing gives zeros; tokens past the table's width or in a block
    outside the pool count as hidden.  num_q_heads is a multiple of the layer's
    heads, head_size 64 or 128, ``softmax_scale`` 1 / sqrt(head_size) unless
    given.

    Returns ``out`` [tokens, num_q_heads, head_size] of q's type, with
    ``return_lse`` also the natural logarithm of each row's sum of exponentials,
    float32 [tokens, num_q_heads], -inf where it sees nothing.  Rows that belong
    to no sequence are left as they were in a given ``out``, and are zeros
    (lse: -inf) in a new one."""
    kv, blocks, tpb, heads, dim, kv_stride, block_stride = _geometry(layer)
    dev = layer.device
    _require(kv == 2, "attention reads a layer of keys and values (kv = 2)")
    _require(isinstance(q, torch.Tensor) and q.dim() == 3, "q must be [tokens, num_q_heads, head_size]")
    n, q_heads, _ = q.shape
    dt = _dtype(q.dtype, "q")
    qt, qh = _rows(q, "q", n, q_heads, dim, q.dtype, dev)
    _no_grad(q, out)
    _require(q_heads > 0 and q_heads % heads == 0, f"num_q_heads ({q_heads}) must be a multiple of the layer's heads ({heads})")
    _ids(seq_lens, "seq_lens", torch.int32, dev)
    _ids(block_tables, "block_tables", torch.int32, dev, 2)
    seqs = seq_lens.shape[0]
    _require(block_tables.shape[0] == seqs, "block_tables and seq_lens differ in their number of sequences")
    if cu_seqlens_q is None:
        _require(n % seqs == 0 if seqs else n == 0, "without cu_seqlens_q every sequence has the same number of rows")
        longest = n // seqs if seqs else 0
    else:
        _ids(cu_seqlens_q, "cu_seqlens_q", torch.int32, dev)
        _require(cu_seqlens_q.shape[0] == seqs + 1, "cu_seqlens_q must have one entry more than seq_lens")
        _require(max_q_len is None or max_q_len >= 0, "max_q_len must be non-negative")
        longest = n if max_q_len is None else min(int(max_q_len), n)
        cu_seqlens_q = cu_seqlens_q.contiguous()
    scale = dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    _require(math.isfinite(scale), "softmax_scale must be finite")
    if out is None:
        # a sequence owns every row when their numbers are the same
        out = (torch.empty if cu_seqlens_q is None else torch.zeros)(n, q_heads, dim, dtype=q.dtype, device=dev)
    ot, oh = _rows(out, "out", n, q_heads, dim, q.dtype, dev)
    lse = None
    if return_lse:
        lse = torch.full((n, q_heads), -math.inf, dtype=torch.float32, device=dev)
    if seq_lens.stride(0) != 1:
        seq_lens = seq_lens.contiguous()
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    lib = _lib.load()
    with _On(dev):
        nbytes = lib.fkv_fp4_attention_workspace(n, q_heads, heads, dim, seqs, longest)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        check(lib.fkv_fp4_attention(layer.data_ptr(), blocks, tpb, heads, dim, kv_stride, block_stride, q.data_ptr(),
                                    out.data_ptr(), _ptr(lse), qt, qh, ot, oh, dt, n, q_heads,
                                    block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1],
                                    seq_lens.data_ptr(), _ptr(cu_seqlens_q), seqs, longest, scale,
                                    int(bool(causal)), _ptr(workspace), nbytes, _stream(dev)), "fp4_attention")
    return (out, lse) if return_lse else out
