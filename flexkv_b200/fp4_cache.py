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

Every operator only enqueues work (nothing waits; ``fp4_wait_timeouts``, which
is no operator, does), so it can be captured into a CUDA graph.  Wrong shapes, types, devices or alignments raise RuntimeError
before anything is launched.  Slots, ids, tables and lengths in device memory
are checked on the device: entries that point outside a pool are skipped (see
each operator).  Inference only: an input that requires a gradient is refused
while gradients are recorded, one with a forward-mode tangent always.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import threading
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .build import binding_path
from .layout import KVCacheLayout, KVCacheLayoutType

__all__ = ["allocate_fp4_layers", "fp4_write", "fp4_read", "fp4_pack_blocks", "fp4_unpack_blocks",
           "fp4_attention", "fp4_wait_timeouts"]

UNIT_TOKENS = 16

_ENTRY_POINTS = ("fkv_last_error", "fkv_fp4_write", "fkv_fp4_read", "fkv_fp4_pack_blocks",
                 "fkv_fp4_unpack_blocks", "fkv_fp4_pack_blocks_listed", "fkv_fp4_unpack_blocks_listed",
                 "fkv_fp4_attention_workspace", "fkv_fp4_attention")
_lock = threading.Lock()
_module = None


def _native():
    """The binding (csrc/fp4_binding.cpp), loaded once; there is no other path."""
    global _module
    if _module is None:
        with _lock:
            if _module is None:
                path = binding_path()
                if not os.path.exists(path):
                    raise ImportError(f"{path} not found; build it with `python -m flexkv_b200.build`")
                loader = importlib.machinery.ExtensionFileLoader("flexkv_b200._fp4", path)
                spec = importlib.util.spec_from_file_location("flexkv_b200._fp4", path, loader=loader)
                module = importlib.util.module_from_spec(spec)
                loader.exec_module(module)
                lib = _lib.load()
                module.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in _ENTRY_POINTS))
                _module = module
    return _module


def allocate_fp4_layers(layout: KVCacheLayout, device) -> List[torch.Tensor]:
    """Zeroed 4-bit layers for the cache that ``layout`` (LAYERWISE, the
    16-bit cache's geometry) describes: one tensor per layer."""
    if layout.type != KVCacheLayoutType.LAYERWISE:
        raise ValueError("GPU layers are LAYERWISE")
    b = layout.fp4()
    return [torch.zeros(b.kv_dim, b.num_block, b.num_head, b.tokens_per_block // UNIT_TOKENS,
                        UNIT_TOKENS * b.head_size, dtype=torch.uint8, device=device)
            for _ in range(b.num_layer)]


def fp4_write(layer: torch.Tensor, k: torch.Tensor, v: Optional[torch.Tensor],
              slot_mapping: torch.Tensor) -> None:
    """Quantise the rows of ``k`` and ``v`` [tokens, num_heads, head_size]
    (bfloat16 or half; slices of a larger projection are fine while rows start
    on 16-byte boundaries) into slots ``slot_mapping`` [tokens] (int64, slot =
    block * tokens_per_block + offset) of ``layer``.  A negative slot, or one
    past the pool, drops its row (padding).  The other slots must differ from
    one another.  ``v`` is None for a latent layer (kv = 1)."""
    _native().write(layer, k, v, slot_mapping)


def fp4_read(layer: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
             out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The tokens in slots ``slot_mapping`` [tokens] as (k, v) [tokens,
    num_heads, head_size] of ``dtype`` (bfloat16 or half; stored values are
    exact in both), v None for a latent layer.  A negative slot, or one past
    the pool, reads as zeros.  ``out``: the tensors to fill, of that shape and
    type (rows on 16-byte boundaries), which must not overlap."""
    k, v = (None, None) if out is None else out
    return _native().read(layer, slot_mapping, dtype, k, v)


def fp4_pack_blocks(kv_layers: Sequence[torch.Tensor], fp4_layers: Sequence[torch.Tensor],
                    kv_block_ids: torch.Tensor, fp4_block_ids: torch.Tensor) -> None:
    """Quantise blocks ``kv_block_ids[i]`` of a 16-bit cache (one tensor [kv,
    blocks, tokens_per_block, num_heads, head_size] per layer) into blocks
    ``fp4_block_ids[i]`` of ``fp4_layers``, all layers in one launch (128 of
    them, and with ids on the host 256 blocks).  Ids (int64) may be host
    tensors, which are checked and read before the call returns (a captured
    graph keeps them), or device tensors, where a pair with an id outside its
    pool is skipped.  No destination may repeat, neither a block nor a layer."""
    _native().convert(True, kv_layers, fp4_layers, kv_block_ids, fp4_block_ids)


def fp4_unpack_blocks(fp4_layers: Sequence[torch.Tensor], kv_layers: Sequence[torch.Tensor],
                      fp4_block_ids: torch.Tensor, kv_block_ids: torch.Tensor) -> None:
    """The other way: blocks ``fp4_block_ids[i]`` of ``fp4_layers`` into
    blocks ``kv_block_ids[i]`` of the 16-bit cache ``kv_layers``."""
    _native().convert(False, kv_layers, fp4_layers, kv_block_ids, fp4_block_ids)


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
    sequence, only chooses the kernel; without it all rows count as one
    sequence's, so give it where many sequences have few rows each (64 sequences
    of 4000 tokens, one new token each: 73 us with it, 230 without).  Row i of a sequence of n new tokens sees
    the keys up to position seq_len - n + i (``causal``) or all.  A row that
    sees nothing gives zeros; tokens past the table's width or in a block
    outside the pool count as hidden.  num_q_heads is a multiple of the layer's
    heads, ``softmax_scale`` 1 / sqrt(head_size) unless given.  Only layers of
    keys and values with heads of 64 or 128 are attended to: latent layers and
    other head sizes can be written, read, converted and moved, and are refused
    here.

    Returns ``out`` [tokens, num_q_heads, head_size] of q's type (a given one
    may be q itself, and must not overlap it otherwise), with ``return_lse``
    also the natural logarithm of each row's sum of exponentials, float32
    [tokens, num_q_heads], -inf where it sees nothing.  Rows that belong
    to no sequence are left as they were in a given ``out``, and are zeros
    (lse: -inf) in a new one.  Waits inside the kernel have a limit;
    ``fp4_wait_timeouts`` tells whether one ran out."""
    return _native().attention(layer, q, block_tables, seq_lens, cu_seqlens_q, max_q_len, softmax_scale, causal, out,
                               return_lse)


def fp4_wait_timeouts(device=None) -> int:
    """How many waits between the warps of ``fp4_attention``'s kernels ran out
    of their limit (about a second) on ``device`` (the current one unless given)
    since the process began: 0 unless something is wrong.  A kernel whose wait
    runs out ends all the same, and what it wrote is not to be used.  Waits for
    the device; not for capturing."""
    n = ctypes.c_int64()
    with torch.cuda.device(device):
        _lib.check(_lib.load().fkv_fp4_wait_timeouts(ctypes.byref(n)), "fp4_wait_timeouts")
    return n.value
