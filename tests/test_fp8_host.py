"""Refusals of the 8-bit cache's and the block tables' entry points, and the oracle against torch's e4m3, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from oracle import fp8_oracle as orc
from parrotserve_b200 import _lib, fp8

FAKE = 1 << 20  # an address that is never dereferenced: every call below is refused before a launch


def cache(**over):
    c = _lib.PbFp8Cache(key_cache=FAKE, value_cache=FAKE, key_scale=FAKE, value_scale=FAKE, kv_block_stride=4 * 2048, kv_head_stride=2048,
                        scale_block_stride=4, scale_head_stride=1, num_blocks=8, num_kv_heads=4, head_size=128, block_size=16)
    for k, v in over.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [
    (dict(key_cache=None), _lib.PB_ERR_INVALID_ARG),
    (dict(value_scale=None), _lib.PB_ERR_INVALID_ARG),
    (dict(key_cache=FAKE + 8), _lib.PB_ERR_INVALID_ARG),
    (dict(key_scale=FAKE + 2), _lib.PB_ERR_INVALID_ARG),
    (dict(kv_block_stride=4 * 2048 + 8), _lib.PB_ERR_INVALID_ARG),
    (dict(kv_head_stride=1024), _lib.PB_ERR_INVALID_ARG),
    (dict(num_blocks=0), _lib.PB_ERR_INVALID_ARG),
    (dict(num_kv_heads=0), _lib.PB_ERR_INVALID_ARG),
    (dict(scale_block_stride=-1), _lib.PB_ERR_INVALID_ARG),
    (dict(block_size=8), _lib.PB_ERR_UNSUPPORTED),
    (dict(head_size=48), _lib.PB_ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("over, code", BAD_CACHES)
def test_fill_and_gather_refuse_a_bad_cache(over, code):
    c = cache(**over)
    args = (FAKE, FAKE, FAKE, 1, 3, 512, 512, _lib.PB_F16)
    assert _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), *args, FAKE, 1 << 30, None) == code
    assert _lib.lib().pb_fp8_gather_cached_kv(C.byref(c), *args, None) == code


@pytest.mark.parametrize("args, code", [
    ((None, FAKE, FAKE, 1, 3, 512, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE, FAKE, None, 1, 3, 512, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE + 2, FAKE, FAKE, 1, 3, 512, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE, FAKE, FAKE, 1, -1, 512, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE, FAKE, FAKE, 1, 1 << 31, 512, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE, FAKE, FAKE, 1, 3, 516, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE, FAKE, FAKE, 1, 3, 256, 512, _lib.PB_F16), _lib.PB_ERR_INVALID_ARG),
    ((FAKE, FAKE, FAKE, 1, 3, 512, 512, 7), _lib.PB_ERR_UNSUPPORTED),
])
def test_fill_and_gather_refuse_bad_rows(args, code):
    c = cache()
    assert _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), *args, FAKE, 1 << 30, None) == code
    assert _lib.lib().pb_fp8_gather_cached_kv(C.byref(c), *args, None) == code


def test_fill_needs_its_workspace():
    c = cache()
    assert _lib.lib().pb_fp8_fill_workspace_bytes(1024, 8, 16) == 0  # (the fill of few tokens reads the whole list)
    need = _lib.lib().pb_fp8_fill_workspace_bytes(1025, 8, 16)
    assert need > 0
    args = (FAKE, FAKE, FAKE, 1, 1025, 512, 512, _lib.PB_F16)
    for ws, n in ((None, need), (FAKE, need - 1), (FAKE + 4, need)):
        assert _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), *args, ws, n, None) == _lib.PB_ERR_WORKSPACE
    assert _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), FAKE, FAKE, FAKE, 1, 0, 512, 512, _lib.PB_F16, None, 0, None) == _lib.PB_OK


@pytest.mark.parametrize("over", [dict(kv_block_stride=0), dict(scale_block_stride=0), dict(scale_head_stride=0)])
def test_fill_refuses_blocks_or_heads_that_share_memory(over):
    c = cache(**over)
    assert _lib.lib().pb_fp8_reshape_and_cache(C.byref(c), FAKE, FAKE, FAKE, 1, 3, 512, 512, _lib.PB_F16, None, 0, None) == _lib.PB_ERR_INVALID_ARG


def attn_params(**over):
    p = _lib.PbAttnParams(out=FAKE, query=FAKE, scale=0.1, dtype=_lib.PB_F16, num_rows=2, num_heads=4, num_kv_heads=4, head_size=128,
                          block_size=16, q_stride=512, out_stride=512, suffix_lens=FAKE, suffix_tables=FAKE, suffix_table_stride=2)
    for k, v in over.items():
        setattr(p, k, v)
    p.workspace, p.workspace_bytes = FAKE, 1 << 30
    return p


@pytest.mark.parametrize("over, cache_over, code", [
    ({}, dict(block_size=8), _lib.PB_ERR_INVALID_ARG),          # not the call's block size
    (dict(block_size=8), dict(block_size=8), _lib.PB_ERR_UNSUPPORTED),
    ({}, dict(head_size=64), _lib.PB_ERR_INVALID_ARG),
    ({}, dict(num_kv_heads=2), _lib.PB_ERR_INVALID_ARG),
    (dict(num_heads=8, q_stride=1024, out_stride=1024), {}, _lib.PB_ERR_INVALID_ARG),  # more heads than kv heads and no mapping
    (dict(slot_mapping=FAKE), {}, _lib.PB_ERR_INVALID_ARG),
    (dict(key_new=FAKE, value_new=FAKE), {}, _lib.PB_ERR_INVALID_ARG),
    (dict(query=None), {}, _lib.PB_ERR_INVALID_ARG),
    (dict(query=FAKE + 2), {}, _lib.PB_ERR_INVALID_ARG),
    (dict(q_stride=256), {}, _lib.PB_ERR_INVALID_ARG),
    (dict(dtype=5), {}, _lib.PB_ERR_UNSUPPORTED),
    ({}, dict(key_scale=None), _lib.PB_ERR_INVALID_ARG),
])
def test_attention_refusals(over, cache_over, code):
    p, c = attn_params(**over), cache(**cache_over)
    for fn in ("pb_fp8_attn_plan", "pb_fp8_attention_planned", "pb_fp8_attention"):
        assert getattr(_lib.lib(), fn)(C.byref(p), C.byref(c), None) == code


def test_attention_needs_its_workspace():
    p, c = attn_params(), cache()
    p.workspace_bytes = 64
    assert _lib.lib().pb_fp8_attention(C.byref(p), C.byref(c), None) == _lib.PB_ERR_WORKSPACE


GOOD_TABLES = dict(context_lens=FAKE, new_lens=FAKE, num_requests=3, block_tables=FAKE, table_width=4, table_stride=4, free_blocks=FAKE,
                   num_free=5, free_head=FAKE, prefix_lens=None, block_size=16, num_prefills=1, num_tokens=7, slot_mapping=FAKE,
                   positions=FAKE, row_offsets=FAKE, kv_lens=FAKE, suffix_lens=FAKE, suffix_tables=FAKE, free_head_out=FAKE,
                   num_failed=FAKE, workspace=FAKE, workspace_bytes=1 << 20)


@pytest.mark.parametrize("over, code", [
    (dict(context_lens=None), _lib.PB_ERR_INVALID_ARG),
    (dict(free_head=None), _lib.PB_ERR_INVALID_ARG),
    (dict(free_blocks=None), _lib.PB_ERR_INVALID_ARG),
    (dict(slot_mapping=None), _lib.PB_ERR_INVALID_ARG),
    (dict(num_prefills=4), _lib.PB_ERR_INVALID_ARG),
    (dict(num_tokens=-1), _lib.PB_ERR_INVALID_ARG),
    (dict(block_size=0), _lib.PB_ERR_INVALID_ARG),
    (dict(table_stride=3), _lib.PB_ERR_INVALID_ARG),
    (dict(num_requests=1025, workspace=None), _lib.PB_ERR_WORKSPACE),
    (dict(num_requests=1025, workspace_bytes=8), _lib.PB_ERR_WORKSPACE),
    (dict(num_requests=1025, workspace=FAKE + 4), _lib.PB_ERR_WORKSPACE),
])
def test_block_table_refusals(over, code):
    a = {**GOOD_TABLES, **over}
    assert _lib.lib().pb_build_block_tables(*a.values(), None) == code


def test_python_operators_refuse_cpu_tensors():
    kc, vc, ks, vs = fp8.fp8_kv_cache(2, 1, 64, 16, "cpu")
    row = torch.zeros(1, 1, 64, dtype=torch.float16)
    slot = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        pb.fp8_reshape_and_cache(row, row, kc, vc, ks, vs, slot)
    with pytest.raises(RuntimeError, match="CUDA"):
        pb.fp8_gather_cached_kv(row, row, kc, vc, ks, vs, slot)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pb.build_block_tables(i32, i32, i32.view(1, 1), i32, i32, block_size=16, num_tokens=0)


def test_call_refuses_what_the_cache_does_not_have():
    kw = dict(num_rows=1, num_heads=1, head_size=64, dtype=torch.float16, device=torch.device("cpu"), suffix_lens=None, suffix_tables=None)
    with pytest.raises(RuntimeError, match="no fill"):
        pb.Fp8AttentionCall(block_size=16, slot_mapping=torch.zeros(1, dtype=torch.int64), **kw)
    with pytest.raises(_lib.PbError):
        pb.Fp8AttentionCall(block_size=8, **kw)


def test_oracle_codes_are_torch_codes():
    x = np.concatenate([np.linspace(-460, 460, 20001), np.ldexp(1.0, np.arange(-14, 9)), orc.VALUES[:127], [0.0, -0.0],
                        (orc.VALUES[:126] + orc.VALUES[1:127]) / 2])
    mine = orc.to_codes(x)
    theirs = torch.from_numpy(x).float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(mine, theirs)
    values = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(orc.VALUES, values, equal_nan=True)
