"""NaN and infinities in queries and caches of the 8-bit calls: they reach the outputs that the formula says, and no others."""
import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from parrotserve_b200 import _lib
from tests.test_gpu_fp8 import DEV, TYPES, i32, layer_problem, on_gpu, paged_problem

pytestmark = pytest.mark.gpu

# decode on tcgen05 (one head an item, and four and eight of them), the other single-query kernel (fp32, blocks of 32, odd head sizes)
SHAPES = [("f16", 128, 16, 2, 2), ("bf16", 64, 16, 8, 2), ("f16", 96, 16, 8, 1), ("f32", 128, 16, 2, 2), ("f32", 80, 32, 6, 2),
          ("f16", 128, 32, 3, 3), ("bf16", 112, 16, 4, 1), ("bf16", 256, 16, 1, 1)]
BAD = [float("nan"), float("inf"), -float("inf")]


def same_but(got, clean, bad):
    """NaN where `bad` [rows, heads] (or [rows, heads, d]) says, everything else as in the clean run, bit for bit."""
    bad = torch.as_tensor(bad, device=got.device)
    bad = (bad if bad.dim() == 3 else bad[..., None]).expand(got.shape)
    assert got[bad].isnan().all(), f"{(~got[bad].isnan()).sum().item()} of {bad.sum().item()} are no NaN"
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dtype, d, b, heads, kv", SHAPES)
def test_queries_of_decodes(dtype, d, b, heads, kv, bad):
    rng = np.random.default_rng(1)
    lens = [1, 17, 0, 300, 40, 700]
    cache, tables, q, mapping, _ = paged_problem(rng, lens, heads, kv, d, b, dtype)
    args = (*on_gpu(cache), None if mapping is None else i32(mapping), i32(lens), i32(tables))
    clean = pb.fp8_paged_attention(q, *args)
    where = np.zeros((len(lens), heads), dtype=bool)
    for row, head, at in ((0, 0, 0), (1, heads - 1, d - 1), (2, 0, 3), (3, heads // 2, d // 2)):
        q[row, head, at] = bad
        where[row, head] = lens[row] > 0  # (an empty context stays zero)
    same_but(pb.fp8_paged_attention(q, *args), clean, where)


@pytest.mark.parametrize("dtype, d, b, heads, kv", SHAPES)
def test_codes_of_decodes(dtype, d, b, heads, kv):
    """NaN codes in K make a row NaN under every query head of that kv head; NaN in V the elements that they stand at."""
    rng = np.random.default_rng(2)
    lens = [1, 17, 300, 40, 700]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    args = (None if mapping is None else i32(mapping), i32(lens), i32(tables))
    clean = pb.fp8_paged_attention(q, *on_gpu(cache), *args)
    where = np.zeros((len(lens), heads, d), dtype=bool)
    share = heads // kv
    for row, at in ((0, 0), (2, 250)):
        s = int(contexts[row][at])
        cache[0][s // b, kv - 1, 1, s % b, 3] = 0xFF
        where[row, (kv - 1) * share:] = True
    for row, at in ((1, 16), (3, 2)):
        s = int(contexts[row][at])
        cache[1][s // b, 0, d - 5, s % b] = 0x7F
        where[row, :share, d - 5] = True
    same_but(pb.fp8_paged_attention(q, *on_gpu(cache), *args), clean, where)


@pytest.mark.parametrize("bad", BAD[:2])
@pytest.mark.parametrize("dtype, d, b, heads, kv", [("f16", 64, 16, 8, 1), ("bf16", 128, 16, 2, 2), ("f32", 96, 16, 3, 3), ("f16", 128, 32, 2, 2)])
def test_few_rows_with_many_partials_and_statistics(dtype, d, b, heads, kv, bad):
    """Long contexts in chunks of 128 tokens: the partials of a row are joined by a CTA of its own. A NaN that a call leaves behind
    survives the call that goes on from its statistics."""
    rng = np.random.default_rng(3)
    lens = [9001, 0, 5, 4096]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    call = pb.Fp8AttentionCall(num_rows=len(lens), num_heads=heads, head_size=d, block_size=b, dtype=TYPES[dtype], device=torch.device(DEV),
                               suffix_lens=i32(lens), suffix_tables=i32(tables), head_mapping=None if mapping is None else i32(mapping),
                               suffix_chunk_blocks=128 // b)
    dev = on_gpu(cache)
    m, l = torch.zeros(len(lens), heads, device=DEV), torch.zeros(len(lens), heads, device=DEV)
    clean = call.run(q, torch.empty_like(q), *dev, m, l, _lib.PB_STATS_SAVE).clone()
    more = call.run(q, clean.clone(), *dev, m, l, _lib.PB_STATS_LOAD)
    where = np.zeros((len(lens), heads), dtype=bool)
    odd = q.clone()
    odd[0, heads - 1, 7] = bad
    where[0, heads - 1] = True
    s = int(contexts[3][4000])
    cache[0][s // b, 0, 0, s % b, 0] = 0x7F
    where[3, :heads // kv] = True
    got = call.run(odd, torch.empty_like(q), *on_gpu(cache), m, l, _lib.PB_STATS_SAVE).clone()
    same_but(got, clean, where)
    assert call.status() == 0
    same_but(call.run(q, got.clone(), *dev, m, l, _lib.PB_STATS_LOAD), more, where)


# a shared prefix whose rows have partials to be merged; several prefixes; prompts finished by the prefix kernel itself and such as
# are not; both; an outer prefix; fp32 and other shapes, which take the single-query kernel
LAYERS = [
    ("f16", dict(heads=2, kv=2, prefixes=(515,), group_rows=(70,), suffixes=tuple(range(1, 71)))),
    ("bf16", dict(heads=4, kv=2, prefixes=(130, 16, 1, 700), group_rows=(3, 9, 1, 40), suffixes=tuple([7] * 53))),
    ("bf16", dict(heads=2, kv=2, segments=((130, 0), (300, 5), (20, 0)))),
    ("f16", dict(heads=1, kv=1, segments=((700, 0), (600, 100)))),
    ("f16", dict(heads=1, kv=1, prefixes=(260,), group_rows=(183,), segments=((150, 0), (20, 33)), suffixes=(0, 1, 31, 32, 33, 200, 3, 4, 5, 6, 7, 8, 9))),
    ("bf16", dict(heads=2, kv=2, prefixes=(48, 90), group_rows=(6, 5), suffixes=tuple([20] * 11), outer=200)),
    ("bf16", dict(heads=2, kv=2, prefixes=(4000,), group_rows=(6,), suffixes=(0, 0, 0, 0, 0, 0))),
    ("f32", dict(heads=2, kv=2, prefixes=(100,), group_rows=(5,), suffixes=(1, 16, 17, 40, 300))),
    ("f16", dict(heads=2, kv=2, d=64, b=32, prefixes=(100,), group_rows=(7,), segments=((3, 10),), suffixes=(5, 40, 41, 1))),
]


@pytest.mark.parametrize("bad", BAD[:2])
@pytest.mark.parametrize("case", range(len(LAYERS)))
def test_queries_of_layers(case, bad):
    dtype, spec = LAYERS[case]
    rng = np.random.default_rng(50 + case)
    call, q, cache, contexts, _ = layer_problem(rng, dtype=dtype, **spec)
    dev = on_gpu(cache)
    rows, heads, d = q.shape
    clean = call.run(q, torch.empty_like(q), *dev).clone()
    where = np.zeros((rows, heads), dtype=bool)
    for row in {0, rows // 3, rows - 1}:
        q[row, row % heads, (5 * row) % d] = bad
        where[row, row % heads] = len(contexts[row]) > 0
    same_but(call.run(q, torch.empty_like(q), *dev), clean, where)
    assert call.status() == 0


@pytest.mark.parametrize("case", range(len(LAYERS)))
def test_key_codes_of_layers(case):
    """A NaN code in K: NaN for the rows that see the token, in a prefix all of its rows, in a prompt those from it on."""
    dtype, spec = LAYERS[case]
    rng = np.random.default_rng(70 + case)
    call, q, cache, contexts, _ = layer_problem(rng, dtype=dtype, **spec)
    rows, heads, d = q.shape
    b, kv = cache[1].shape[3], cache[1].shape[1]
    clean = call.run(q, torch.empty_like(q), *on_gpu(cache)).clone()
    where = np.zeros((rows, heads), dtype=bool)
    for row in (0, rows - 1):
        s = int(contexts[row][-1])
        cache[0][s // b, 0, d // 16 - 1, s % b, 15] = 0x7F
        for r in range(rows):
            where[r, :heads // kv] |= s in contexts[r]
    same_but(call.run(q, torch.empty_like(q), *on_gpu(cache)), clean, where)


@pytest.mark.parametrize("case", range(len(LAYERS)))
@pytest.mark.parametrize("where_in", [0.0, 0.4, 1.0])
def test_value_codes_of_layers(case, where_in):
    """A NaN code in V: NaN in its element for the rows that see the token. The tensor cores take 256 rows of a prompt with 128 tokens at a
    time: earlier rows of the prompt may get NaN in that element too, if a row of their 256 sees one of the token's 128 (0 times NaN).
    Nothing else changes."""
    dtype, spec = LAYERS[case]
    rng = np.random.default_rng(90 + case)
    call, q, cache, contexts, _ = layer_problem(rng, dtype=dtype, **spec)
    rows, heads, d = q.shape
    b, kv = cache[1].shape[3], cache[1].shape[1]
    clean = call.run(q, torch.empty_like(q), *on_gpu(cache)).clone()
    where, may = np.zeros((rows, heads, d), dtype=bool), np.zeros((rows, heads, d), dtype=bool)
    at = np.concatenate([[0], np.cumsum([n for n, _ in spec.get("segments", ())])])
    for row, element, head in ((rows // 2, d - 3, 0), (rows - 1, 34, kv - 1)):
        s = int(contexts[row][int(where_in * (len(contexts[row]) - 1))])
        cache[1][s // b, head, element, s % b] = 0xFF
        under = slice(head * (heads // kv), (head + 1) * (heads // kv))
        for r in range(rows):
            if s in contexts[r]:
                where[r, under, element] = True
        for lo, hi, (n, past) in zip(at, at[1:], spec.get("segments", ())):
            own = contexts[hi - 1][-(n + past):]  # the prompt's own tokens, behind a prefix
            if s in own:
                tile = int(np.flatnonzero(own == s)[0]) // 128 * 128
                for first in range(0, n, 256):
                    last = min(n, first + 256)
                    if tile < past + last:
                        may[lo + first:lo + last, under, element] = True
    got = call.run(q, torch.empty_like(q), *on_gpu(cache))
    assert call.status() == 0
    leaked = torch.as_tensor(may & ~where, device=DEV) & got.isnan()
    same_but(torch.where(leaked, clean, got), clean, where)
