"""Which strides of an 8-bit cache the fill refuses: those under which blocks or heads share memory."""
import ctypes as C

import pytest

from parrotserve_b200 import _lib
from tests.test_fp8_host import FAKE, cache

TILE = 128 * 16


@pytest.mark.parametrize("over", [
    dict(kv_block_stride=TILE, kv_head_stride=TILE),               # block i + 1, head j is block i, head j + 1
    dict(kv_block_stride=3 * TILE),                                # four heads in the room of three
    dict(kv_block_stride=4 * TILE - 16),
    dict(kv_block_stride=TILE - 16, kv_head_stride=8 * TILE),      # heads outside, blocks that overlap
    dict(kv_block_stride=TILE, kv_head_stride=7 * TILE),           # eight blocks in the room of seven
    dict(scale_block_stride=1, scale_head_stride=1), dict(scale_block_stride=3), dict(scale_block_stride=1, scale_head_stride=7),
    dict(num_kv_heads=1, kv_block_stride=TILE - 16), dict(num_kv_heads=1, scale_block_stride=0), dict(num_blocks=1, scale_head_stride=0),
])
def test_overlapping_tiles_or_scales_are_refused(over):
    c = cache(**over)
    rc = _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), FAKE, FAKE, FAKE, 1, 3, 512, 512, _lib.PB_F16, None, 0, None)
    assert rc == _lib.PB_ERR_INVALID_ARG


@pytest.mark.parametrize("over", [
    {}, dict(kv_block_stride=TILE, kv_head_stride=8 * TILE), dict(scale_block_stride=1, scale_head_stride=8),
    dict(kv_block_stride=12 * TILE, kv_head_stride=2 * TILE, scale_block_stride=2, scale_head_stride=16),
    dict(num_blocks=1, kv_block_stride=0, scale_block_stride=0), dict(num_kv_heads=1, scale_head_stride=0)])
def test_strides_of_views_pass(over):
    """Dense, transposed and sliced caches get past the strides (and are refused for their missing workspace, before a launch)."""
    c = cache(**over)
    rc = _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), FAKE, FAKE, FAKE, 1, 1025, 512, 512, _lib.PB_F16, None, 0, None)
    assert rc == _lib.PB_ERR_WORKSPACE
