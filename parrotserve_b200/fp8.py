"""The paged KV cache in 8 bits: fill, gather and attention.

Keys and values are e4m3 codes in the framework's paged layout (``x = 16``) with one fp32 scale for each block and kv head:

* K ``[num_blocks, num_kv_heads, head_size/16, block_size, 16]``, V ``[num_blocks, num_kv_heads, head_size, block_size]``,
  ``torch.float8_e4m3fn``; key and value scales ``[num_blocks, num_kv_heads]`` float32. An element is code * scale.
* block sizes 16 and 32, head sizes 64, 80, 96, 112, 128, 256; queries and rows in fp16, bf16 or fp32.

The operators stand beside those of ``ops`` and take the four cache tensors where those take two. What is filled with
``fp8_reshape_and_cache`` has powers of two as scales; attention and gather take others too (a tile with scale 0 is zero and holds no
NaN; attention of 16-bit queries counts value scales below 2^-100 as 0 and is inexact above 2^100). Nothing here falls back
to torch: the operators fail without the library or a GPU.

Beside the reference's ``vllm_reshape_and_cache`` (kernels/vllm/reshape_and_cache.py:9-22) and ``flash_paged_attention``
(kernels/shared_flash_decoding.py:285-329); the reference has no 8-bit cache.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import PbFp8Cache, check, lib
from .ops import _DTYPES, AttentionCall, Workspace, _dtype_code, _flat_slots, _kv_geometry, _ptr, _require_cuda, _single_group_meta

CACHE_DTYPE = torch.float8_e4m3fn
_NOTHING = contextlib.nullcontext()


def fp8_kv_cache(num_blocks: int, num_kv_heads: int, head_size: int, block_size: int, device) -> Tuple[torch.Tensor, ...]:
    """An empty cache: (key_cache, value_cache, key_scale, value_scale), all zero."""
    if head_size % 16:
        raise RuntimeError("head_size must be a multiple of 16")
    return (torch.zeros((num_blocks, num_kv_heads, head_size // 16, block_size, 16), dtype=CACHE_DTYPE, device=device),
            torch.zeros((num_blocks, num_kv_heads, head_size, block_size), dtype=CACHE_DTYPE, device=device),
            torch.zeros((num_blocks, num_kv_heads), dtype=torch.float32, device=device),
            torch.zeros((num_blocks, num_kv_heads), dtype=torch.float32, device=device))


def _describe(c: PbFp8Cache, key_cache, value_cache, key_scale, value_scale):
    """Fills `c` with the four tensors' addresses and strides; returns (num_kv_heads, head_size, block_size)."""
    if key_cache.dtype != CACHE_DTYPE or value_cache.dtype != CACHE_DTYPE:
        raise RuntimeError("key_cache and value_cache must be torch.float8_e4m3fn")
    nb, hkv, d, b, kbs, khs = _kv_geometry(key_cache, value_cache)
    if key_scale.dtype != torch.float32 or value_scale.dtype != torch.float32:
        raise RuntimeError("key_scale and value_scale must be float32")
    shape = (nb, hkv)
    if key_scale.shape != shape or value_scale.shape != shape:
        raise RuntimeError("key_scale and value_scale must be [num_blocks, num_kv_heads]")
    ss = key_scale.stride()
    if value_scale.stride() != ss:
        raise RuntimeError("key_scale and value_scale must share strides")
    c.key_cache, c.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    c.key_scale, c.value_scale = key_scale.data_ptr(), value_scale.data_ptr()
    c.kv_block_stride, c.kv_head_stride = kbs, khs
    c.scale_block_stride, c.scale_head_stride = ss
    c.num_blocks, c.num_kv_heads, c.head_size, c.block_size = nb, hkv, d, b
    return hkv, d, b


def _on(index: Optional[int]):
    """Makes the tensors' device the current one for a library call (nothing to do when it is)."""
    return _NOTHING if index is None or index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _one_device(*tensors) -> int:
    """The index of the one GPU that all tensors are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or index < 0:  # (-1: the CPU)
            _require_cuda(*tensors)
            raise RuntimeError("all tensors of a call must be on one device")
    return index


def _rows(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping):
    index = _one_device(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping)
    shape = key.shape
    if shape != value.shape or len(shape) != 3:
        raise RuntimeError("key and value must both be [num_tokens, num_heads, head_size]")
    if key.dtype != value.dtype:
        raise RuntimeError("key and value must share a dtype")
    c = PbFp8Cache()
    hkv, d, _ = _describe(c, key_cache, value_cache, key_scale, value_scale)
    t, h, hd = shape
    if h != hkv or hd != d:
        raise RuntimeError("cache heads/head_size differ from key's")
    ks, vs = key.stride(), value.stride()
    if t and (ks[2] != 1 or ks[1] != d or vs[2] != 1 or vs[1] != d):
        raise RuntimeError("key/value must be dense over (head, dim)")
    slots = _flat_slots(slot_mapping, t)
    # what both entry points take behind the cache
    return c, t, index, (slots, key.data_ptr(), value.data_ptr(), slots.data_ptr(), 1 if slots.dtype == torch.int64 else 0, t, ks[0], vs[0],
                         _dtype_code(key))


def fp8_reshape_and_cache(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping) -> None:
    """KV fill: quantises new rows ``[num_tokens, num_kv_heads, head_size]`` into the cache at ``slot_mapping`` (one int32 or
    int64 slot per token, negative: none) and updates the scales.

    The scale of a (block, head) becomes the largest of what it was and the smallest power of two with which the new
    tokens' largest element fits (448 codes); when it grows the tokens that the block holds already are re-quantised (under a scale
    of 0 they were zeros and stay so). A
    call that brings the token at offset 0 of a block begins the block anew: what it held, its scale included, is void. Tokens of
    a block may stand in any order; of tokens with one slot the last counts. NaN and infinities are cached as NaN, under a scale of at least
    2^-100."""
    c, t, index, (_slots, *args) = _rows(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping)
    if t == 0:
        return
    with _on(index):
        nbytes = lib().pb_fp8_fill_workspace_bytes(t, c.num_blocks, c.block_size)
        ws = Workspace.get(key.device, nbytes) if nbytes else None  # (a small call needs none)
        rc = lib().pb_fp8_reshape_and_cache(C.byref(c), *args, _ptr(ws), nbytes, torch._C._cuda_getCurrentRawStream(index))
    check(rc, "pb_fp8_reshape_and_cache")


def fp8_gather_cached_kv(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping) -> None:
    """Rows out of the cache: ``key[t], value[t]`` = code * scale of slot ``slot_mapping[t]``, rounded once to the rows' type.
    Rows with a negative slot stay as they were."""
    c, t, index, (_slots, *args) = _rows(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping)
    if t == 0:
        return
    with _on(index):
        rc = lib().pb_fp8_gather_cached_kv(C.byref(c), *args, torch._C._cuda_getCurrentRawStream(index))
    check(rc, "pb_fp8_gather_cached_kv")


class Fp8AttentionCall(AttentionCall):
    """``AttentionCall`` over the 8-bit cache: the same constructor (without ``slot_mapping``: the fill is a call of its own),
    ``plan()`` and ``run()`` take the four cache tensors. Decode rows, shared prefixes, outer prefixes, causal segments,
    head mappings and statistics mean what they mean there."""

    def __init__(self, *, slot_mapping=None, **kwargs):
        if slot_mapping is not None:
            raise RuntimeError("the 8-bit attention call performs no fill: call fp8_reshape_and_cache before it")
        if kwargs["dtype"] not in _DTYPES:
            raise RuntimeError(f"unsupported dtype {kwargs['dtype']}")
        if kwargs["block_size"] not in (16, 32):
            raise _lib.PbError(_lib.PB_ERR_UNSUPPORTED, "Fp8AttentionCall", f"block_size={kwargs['block_size']}")
        with _on(torch.device(kwargs["device"]).index):
            super().__init__(**kwargs)
        self._index = _one_device(*self._keep) if self._keep else None  # where the lengths and tables are
        self._cache = PbFp8Cache()
        self._cache_ref = C.byref(self._cache)

    def _take_workspace(self, workspace, shared_workspace) -> None:
        # its size depends on the number of kv heads, which the cache brings: taken when the first one is bound
        self._workspace_args = (workspace, shared_workspace)
        self._sized_for = None

    def _size_for(self, num_kv_heads: int) -> None:
        self.params.num_kv_heads = num_kv_heads
        nbytes = lib().pb_fp8_attn_workspace_bytes(self._params_ref)
        if nbytes == 0:
            raise _lib.PbError(_lib.PB_ERR_UNSUPPORTED, "pb_fp8_attn_workspace_bytes",
                               f"head_size={self.params.head_size} block_size={self.params.block_size} dtype={self.dtype}")
        self._use_workspace(nbytes, *self._workspace_args)
        self._sized_for = num_kv_heads
        self._planned = False

    def _bind_fp8(self, query, out, key_cache, value_cache, key_scale, value_scale, qk_max=None, exp_sum=None,
                  stats_mode=_lib.PB_STATS_NONE):
        p = self.params
        index = _one_device(query, out, key_cache, value_cache, key_scale, value_scale)
        if self._index is not None and index != self._index:
            raise RuntimeError("all tensors of a call must be on one device")
        hkv, d, b = _describe(self._cache, key_cache, value_cache, key_scale, value_scale)
        if query.dtype != self.dtype or out.dtype != self.dtype:
            raise RuntimeError("query and out must have the dtype of the call")
        if query.shape != self._q_shape or out.shape != self._q_shape:
            raise RuntimeError(f"query and out must be [{p.num_rows}, {p.num_heads}, {p.head_size}]")
        if d != self._q_shape[2] or b != p.block_size:
            raise RuntimeError("cache head_size/block_size differ from the call's")
        qs, os = query.stride(), out.stride()
        if p.num_rows and (qs[2] != 1 or qs[1] != d or os[2] != 1 or os[1] != d):
            raise RuntimeError("query/out must be dense over (head, dim)")
        if hkv != self._sized_for:
            self._size_for(hkv)
        if stats_mode != _lib.PB_STATS_NONE:
            for x in (qk_max, exp_sum):
                if (x is None or x.dtype != torch.float32 or x.shape != self._q_shape[:2] or not x.is_contiguous()
                        or x.get_device() != index):
                    raise RuntimeError(f"qk_max and exp_sum must be float32 [{p.num_rows}, {p.num_heads}], contiguous, on the call's device")
        p.out, p.query = out.data_ptr(), query.data_ptr()
        p.q_stride, p.out_stride = qs[0], os[0]
        p.qk_max, p.exp_sum, p.stats_mode = _ptr(qk_max), _ptr(exp_sum), stats_mode
        return index

    def plan(self, query, out, key_cache, value_cache, key_scale, value_scale) -> None:
        index = self._bind_fp8(query, out, key_cache, value_cache, key_scale, value_scale)
        with _on(index):
            rc = lib().pb_fp8_attn_plan(self._params_ref, self._cache_ref, torch._C._cuda_getCurrentRawStream(index))
        check(rc, "pb_fp8_attn_plan")
        self._planned = True

    def run(self, query, out, key_cache, value_cache, key_scale, value_scale, qk_max=None, exp_sum=None,
            stats_mode=_lib.PB_STATS_NONE):
        """One layer: attention of ``query`` over the cache into ``out``."""
        index = self._bind_fp8(query, out, key_cache, value_cache, key_scale, value_scale, qk_max, exp_sum, stats_mode)
        fn = lib().pb_fp8_attention_planned if self._planned else lib().pb_fp8_attention
        with _on(index):
            rc = fn(self._params_ref, self._cache_ref, torch._C._cuda_getCurrentRawStream(index))
        if rc != _lib.PB_OK:
            check(rc, "pb_fp8_attention")
        return out


def _one_shot(query, cache, head_mapping, suffix_lens, suffix_tables, out=None, **kwargs):
    num_rows, num_heads, head_size = query.shape
    if out is None:
        out = query.new_empty((num_rows, num_heads, head_size))
    if num_rows == 0:
        return out
    call = Fp8AttentionCall(
        num_rows=num_rows, num_heads=num_heads, head_size=head_size, block_size=cache[1].shape[3], dtype=query.dtype,
        device=query.device, suffix_lens=suffix_lens, suffix_tables=suffix_tables, head_mapping=head_mapping,
        shared_workspace=True, **kwargs)
    return call.run(query, out, *cache)


def fp8_paged_attention(query, key_cache, value_cache, key_scale, value_scale, head_mapping: Optional[torch.Tensor],
                        context_lens: torch.Tensor, block_tables: torch.Tensor) -> torch.Tensor:
    """Unshared decode attention over the 8-bit cache (``vllm_paged_attention`` with scales)."""
    return _one_shot(query, (key_cache, value_cache, key_scale, value_scale), head_mapping, context_lens, block_tables)


def fp8_flash_paged_attention_grouped(query, key_cache, value_cache, key_scale, value_scale,
                                      head_mapping: Optional[torch.Tensor], group_prefix_lens: torch.Tensor,
                                      group_block_tables: torch.Tensor, group_row_offsets: torch.Tensor,
                                      paged_context_lens: torch.Tensor, paged_block_tables: torch.Tensor,
                                      out: Optional[torch.Tensor] = None, **tuning) -> torch.Tensor:
    """Shared-prefix decode attention for G prefix groups (``flash_paged_attention_grouped`` with scales)."""
    return _one_shot(query, (key_cache, value_cache, key_scale, value_scale), head_mapping, paged_context_lens, paged_block_tables,
                     out, group_row_offsets=group_row_offsets, group_prefix_lens=group_prefix_lens, group_tables=group_block_tables,
                     **tuning)


def fp8_flash_paged_attention(query, key_cache, value_cache, key_scale, value_scale, head_mapping: Optional[torch.Tensor],
                              flash_context_len: int, flash_block_table: torch.Tensor, paged_context_lens: torch.Tensor,
                              paged_block_tables: torch.Tensor, **tuning) -> torch.Tensor:
    """Decode attention over one shared prefix and private contexts (``flash_paged_attention`` with scales)."""
    offs, plen = _single_group_meta(query.device, int(flash_context_len), query.shape[0])
    return fp8_flash_paged_attention_grouped(query, key_cache, value_cache, key_scale, value_scale, head_mapping, plen,
                                             flash_block_table.reshape(1, -1), offs, paged_context_lens, paged_block_tables, **tuning)
