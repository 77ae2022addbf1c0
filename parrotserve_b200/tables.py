"""Block tables, slot maps and row lengths of an iteration, built on the GPU from the requests' lengths.

The host loops this stands beside are those of ``attn_func.IterationMetadata`` (and of the reference's
``init_iteration_state``, parrot/engine/builtin/attn_func.py:461-599): an engine whose lengths, tables and free blocks live
on the GPU gets what ``AttentionCall``, ``Fp8AttentionCall`` and the fills read without a transfer or a synchronisation.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import check, lib
from .fp8 import _on, _one_device
from .ops import Workspace, _ptr


class BlockTables(NamedTuple):
    """What ``build_block_tables`` returns. With P prefills among the requests, ``row_offsets[:P + 1]``, ``kv_lens[:P]`` and
    ``block_tables[:P]`` are an attention call's causal segments."""

    slot_mapping: torch.Tensor   # [num_tokens] int64, -1: no slot
    positions: torch.Tensor      # [num_tokens] int64
    row_offsets: torch.Tensor    # [num_requests + 1] int32
    kv_lens: torch.Tensor        # [num_requests] int32, tokens held afterwards
    suffix_lens: torch.Tensor    # [num_tokens] int32, 0 for the rows of prefills
    suffix_tables: Optional[torch.Tensor]  # [num_tokens, table width] int32, 0-padded
    free_head: torch.Tensor      # [1] int32, entries of free_blocks taken so far
    num_failed: torch.Tensor     # [1] int32, requests that did not get their blocks


def build_block_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor,
                       free_head: torch.Tensor, *, block_size: int, num_tokens: int, num_prefills: int = 0,
                       prefix_lens: Optional[torch.Tensor] = None, with_suffix_tables: bool = True) -> BlockTables:
    """Gives every request the blocks its new tokens need and returns the iteration's slots, positions and lengths.

    ``context_lens``, ``new_lens`` [R] int32: tokens a request holds and adds. ``block_tables`` [R, W] int32: changed in place,
    row r's first ceil(context / block_size) entries are its blocks and the new ones are appended, taken from ``free_blocks``
    (int32) from entry ``free_head[0]`` on in the order of the requests. ``num_tokens``: rows to write, at least the sum of
    ``new_lens`` (rows behind the last token get slot -1 and length 0, so that a captured iteration can be padded). The first
    ``num_prefills`` requests are prefills. ``prefix_lens`` [R] int32 is added to the positions (a shared prefix in front of the
    request's own context).

    A request whose tokens do not fit its table row, or for which the free blocks run out, gets none: its slots are -1, its
    ``kv_lens`` entry stays, ``num_failed`` counts it. Only ``block_tables`` is changed; the next iteration passes
    ``kv_lens`` and ``free_head`` of this one."""
    tensors = (context_lens, new_lens, block_tables, free_blocks, free_head) + (() if prefix_lens is None else (prefix_lens,))
    index = _one_device(*tensors)
    for t in tensors:
        if t.dtype != torch.int32:
            raise RuntimeError("lengths, tables and free blocks must be int32 tensors")
    shape, table_shape = context_lens.shape, block_tables.shape
    if len(shape) != 1 or new_lens.shape != shape or (prefix_lens is not None and prefix_lens.shape != shape):
        raise RuntimeError("context_lens, new_lens and prefix_lens must be [num_requests]")
    r = shape[0]
    if len(table_shape) != 2 or table_shape[0] != r or free_blocks.dim() != 1 or free_head.numel() != 1:
        raise RuntimeError("block_tables must be [num_requests, width], free_blocks [n], free_head one number")
    width, (table_stride, entry_stride) = table_shape[1], block_tables.stride()
    if r and width > 1 and entry_stride != 1:
        raise RuntimeError("the rows of block_tables must be dense")
    if not (context_lens.is_contiguous() and new_lens.is_contiguous() and free_blocks.is_contiguous()
            and (prefix_lens is None or prefix_lens.is_contiguous())):
        raise RuntimeError("lengths and free blocks must be contiguous")
    if not 0 <= num_prefills <= r or num_tokens < 0:
        raise RuntimeError("num_prefills must be at most the number of requests, num_tokens not negative")
    # two allocations: the 64-bit and the 32-bit results
    dev = context_lens.device
    longs = torch.empty((2, num_tokens), dtype=torch.int64, device=dev)
    sizes = (r + 1, r, 1, 1, num_tokens, num_tokens * width if with_suffix_tables else 0)
    ints = torch.empty(sum(sizes), dtype=torch.int32, device=dev)
    row_offsets, kv_lens, head_out, failed, suffix_lens, flat = ints.split_with_sizes(sizes)
    slot_mapping, positions = longs.unbind()
    at64, at = longs.data_ptr(), ints.data_ptr()
    with _on(index):
        nbytes = lib().pb_block_tables_workspace_bytes(r)
        ws = Workspace.get(dev, nbytes) if nbytes else None  # (up to some number of requests the call needs none)
        rc = lib().pb_build_block_tables(
            context_lens.data_ptr(), new_lens.data_ptr(), r, block_tables.data_ptr(), width, table_stride, free_blocks.data_ptr(),
            free_blocks.shape[0], free_head.data_ptr(), _ptr(prefix_lens), block_size, num_prefills, num_tokens, at64, at64 + 8 * num_tokens,
            at, at + 4 * (r + 1), at + 4 * (2 * r + 3), at + 4 * (2 * r + 3 + num_tokens) if with_suffix_tables else None,
            at + 4 * (2 * r + 1), at + 4 * (2 * r + 2), _ptr(ws), nbytes, torch._C._cuda_getCurrentRawStream(index))
    check(rc, "pb_build_block_tables")
    return BlockTables(slot_mapping, positions, row_offsets, kv_lens, suffix_lens,
                       flat.view(num_tokens, width) if with_suffix_tables else None, head_out, failed)
