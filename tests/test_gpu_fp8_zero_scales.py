"""Tiles of the 8-bit cache with scale 0: they are zero, whatever their codes, and stay so when their scale grows."""
import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from oracle import fp8_oracle as orc
from tests.test_gpu_fp8 import DEV, TYPES, fill_both, i32, on_gpu, rand_rows, random_cache, same_cache, to_host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d, b, heads", [(128, 16, 4), (64, 32, 5), (80, 16, 2), (256, 32, 3)])
@pytest.mark.parametrize("per_block", [1, 3])
def test_cells_under_a_scale_of_zero_stay_zero(dtype, d, b, heads, per_block):
    """New tokens behind others in blocks some of whose heads have scale 0 and codes of any value, NaN among them: one token for each
    block, and several."""
    rng = np.random.default_rng(d + heads + per_block)
    blocks = 12
    cache = random_cache(rng, blocks, heads, d, b)
    cache[2][::2, ::2] = 0.0
    cache[3][1::2] = 0.0
    cache[0][:, :, :, 3, 5] = 0x7F
    cache[1][:, :, 7, 2] = 0xFF
    slots = np.concatenate([i * b + 4 + i % (b - 7) + np.arange(per_block) for i in range(blocks)])
    key, value = rand_rows(rng, len(slots), heads, d, dtype), rand_rows(rng, len(slots), heads, d, dtype)
    key[3 * per_block], value[5 * per_block, 0] = 0, 0  # (a token of zeros grows nothing)
    zero_k, zero_v = cache[2] == 0, cache[3] == 0
    got, want = fill_both(cache, key, value, slots)
    same_cache(got, want)
    # and by the definition: what stood for 0 before stands for 0 now
    new = np.zeros(blocks * b, dtype=bool)
    new[slots] = True
    every = np.arange(blocks * b)
    for value_side, zero in ((0, zero_k), (1, zero_v)):
        rows = orc.token_rows(*[np.where(np.isin(c, (0x7F, 0xFF)), 0, c) if c.dtype == np.uint8 else c for c in got], every)[value_side]
        old = np.repeat(zero, b, axis=0) & ~new[:, None]
        assert not rows[old].any()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_tokens_of_zeros_then_others(dtype):
    """A block that was used before begins anew with zeros and goes on with other tokens, one call each: attention and gather see what
    was filled."""
    rng = np.random.default_rng(4)
    heads, d, b = 2, 128, 16
    cache = random_cache(rng, 3, heads, d, b)
    dev = on_gpu(cache)
    want = tuple(x.copy() for x in cache)
    rows = [rand_rows(rng, 5, heads, d, dtype) for _ in range(2)]
    for x in rows:
        x[:2] = 0
    slots = [16 + i for i in range(5)]
    for i in range(5):
        key, value = rows[0][i:i + 1].contiguous(), rows[1][i:i + 1].contiguous()
        pb.fp8_reshape_and_cache(key, value, *dev, torch.tensor(slots[i:i + 1], device=DEV))
        orc.fill(*want, key.double().cpu().numpy(), value.double().cpu().numpy(), slots[i:i + 1])
        same_cache(to_host(dev), want)
    key, value = torch.empty_like(rows[0]), torch.empty_like(rows[1])
    pb.fp8_gather_cached_kv(key, value, *dev, torch.tensor(slots, device=DEV))
    assert not key[:2].any() and not value[:2].any() and key[2:].any() and value[2:].any()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 3])
def test_nan_beside_zeros_has_a_scale(dtype, tokens):
    """A tile whose only finite elements are zeros, with a NaN or an infinity among them: gather, decode and a shared prefix all see
    NaN where it stands, and zeros elsewhere."""
    heads, d, b, rows = 2, 128, 16, 5
    cache = tuple(np.zeros_like(x) for x in random_cache(np.random.default_rng(1), 4, heads, d, b))
    key = torch.zeros(tokens, heads, d, dtype=TYPES[dtype], device=DEV)
    value = torch.zeros_like(key)
    value[tokens - 1, 0, 9], value[0, 1, 100], key[0, 1, 3] = float("inf"), float("nan"), float("nan")
    slots = [2 * b + i for i in range(tokens)]
    got, want = fill_both(cache, key, value, slots)
    same_cache(got, want)
    assert got[3][2].tolist() == [2.0 ** -100] * 2 and got[2][2].tolist() == [0.0, 2.0 ** -100]
    dev = on_gpu(got)
    k, v = torch.ones_like(key), torch.ones_like(value)
    pb.fp8_gather_cached_kv(k, v, *dev, torch.tensor(slots, device=DEV))
    for x, rows_in in ((k, key), (v, value)):
        assert torch.equal(x.isnan(), ~rows_in.isfinite()) and not torch.nan_to_num(x, nan=0).any()
    q = rand_rows(np.random.default_rng(2), rows, heads, d, dtype)
    lens, tables = i32([tokens] * rows), i32([[2]] * rows)
    for out in (pb.fp8_paged_attention(q, *dev, None, lens, tables),
                pb.fp8_flash_paged_attention(q, *dev, None, tokens, i32([2]), i32([0] * rows), i32([[0]] * rows))):
        assert torch.equal(out[:, 0].isnan(), torch.arange(d, device=DEV).eq(9).expand(rows, d))
        assert not torch.nan_to_num(out[:, 0], nan=0).any() and out[:, 1].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_nan_beside_tiny_values_has_a_scale(dtype):
    """NaN that joins tiny values, with them and after them, is not read as zero either."""
    heads, d, b, rows = 1, 128, 16, 5
    rng = np.random.default_rng(6)
    cache = tuple(np.zeros_like(x) for x in random_cache(rng, 4, heads, d, b))
    tiny = rand_rows(rng, 4, heads, d, dtype, 2.0 ** -120)
    tiny[1, 0, 5] = float("nan")
    late = tiny[1:2].clone()
    for steps in ([(0, 4)], [(0, 1), (2, 2), (3, 1)]):
        dev, want = on_gpu(cache), tuple(x.copy() for x in cache)
        at = 0
        for first, n in steps:
            new = late if (first, n) == (3, 1) else tiny[first:first + n].contiguous()
            slots = list(range(2 * b + at, 2 * b + at + len(new)))
            at += len(new)
            pb.fp8_reshape_and_cache(tiny[:len(new)].abs().nan_to_num().contiguous(), new, *dev, torch.tensor(slots, device=DEV))
            orc.fill(*want, tiny[:len(new)].abs().nan_to_num().double().cpu().numpy(), new.double().cpu().numpy(), slots)
            same_cache(to_host(dev), want)
        assert want[3][2, 0] == 2.0 ** -100
        q = rand_rows(rng, rows, heads, d, dtype)
        for out in (pb.fp8_paged_attention(q, *dev, None, i32([at] * rows), i32([[2]] * rows)),
                    pb.fp8_flash_paged_attention(q, *dev, None, at, i32([2]), i32([0] * rows), i32([[0]] * rows))):
            assert torch.equal(out[:, 0].isnan(), torch.arange(d, device=DEV).eq(5).expand(rows, d))
