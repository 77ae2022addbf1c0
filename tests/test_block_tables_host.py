"""Refusals of the block tables' entry point that need no GPU: results that share memory with inputs or with each other."""
import pytest

from parrotserve_b200 import _lib

STEP = 1 << 20  # every array has a megabyte to itself; the addresses are never dereferenced: each call is refused before a launch


def arguments(**over):
    names = ["context_lens", "new_lens", "num_requests", "block_tables", "table_width", "table_stride", "free_blocks", "num_free", "free_head",
             "prefix_lens", "block_size", "num_prefills", "num_tokens", "slot_mapping", "positions", "row_offsets", "kv_lens", "suffix_lens",
             "suffix_tables", "free_head_out", "num_failed", "workspace", "workspace_bytes"]
    a = {n: (i + 1) * STEP for i, n in enumerate(names)}
    a.update(num_requests=3, table_width=4, table_stride=6, num_free=5, block_size=16, num_prefills=1, num_tokens=7, workspace_bytes=1 << 18)
    return {**a, **over}


@pytest.mark.parametrize("result, other, off", [
    ("kv_lens", "context_lens", 0), ("kv_lens", "new_lens", 0), ("free_head_out", "free_head", 0), ("free_head_out", "free_blocks", 16),
    ("kv_lens", "context_lens", 8), ("kv_lens", "context_lens", -8), ("row_offsets", "prefix_lens", -12), ("num_failed", "free_head_out", 0),
    ("suffix_tables", "block_tables", 60), ("suffix_tables", "suffix_lens", -108), ("slot_mapping", "positions", -48),
    ("num_failed", "block_tables", 60), ("positions", "free_blocks", 16)])
@pytest.mark.parametrize("requests", [3, 1025])
def test_results_may_not_share_memory(result, other, off, requests):
    a = arguments(num_requests=requests)
    a[result] = a[other] + off
    assert _lib.lib().pb_build_block_tables(*a.values(), None) == _lib.PB_ERR_INVALID_ARG


def test_workspace_may_not_be_an_input():
    a = arguments(num_requests=1025)
    a["workspace"] = a["context_lens"]
    assert _lib.lib().pb_build_block_tables(*a.values(), None) == _lib.PB_ERR_INVALID_ARG
