"""build_block_tables on the GPU against a walk over the requests, and an engine's loop on top of it."""
import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from oracle import fp8_oracle as orc
from tests.test_gpu_fp8 import check_attention, i32, rand_rows, to_host

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def problem(rng, requests, ctx_hi, new_hi, width, block, free_extra=10, zero_new=0.2):
    ctx = rng.integers(0, ctx_hi + 1, size=requests)
    new = np.where(rng.random(requests) < zero_new, 0, rng.integers(1, new_hi + 1, size=requests))
    tables = rng.integers(1000, 2000, size=(requests, width)).astype(np.int32)
    need = int(sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(ctx, new)))
    free = rng.permutation(need + free_extra).astype(np.int32)
    return ctx, new, tables, free


def both(ctx, new, tables, free, head, block, tokens, prefills=0, prefix=None, with_suffix=True):
    want = orc.block_tables(ctx, new, tables, free, head, block, tokens, prefills, prefix)
    dev_tables = i32(tables)
    got = pb.build_block_tables(i32(ctx), i32(new), dev_tables, i32(free), i32([head]), block_size=block, num_tokens=tokens,
                                num_prefills=prefills, prefix_lens=None if prefix is None else i32(prefix), with_suffix_tables=with_suffix)
    for name, w in want.items():
        g = dev_tables if name == "block_tables" else getattr(got, name)
        if name == "suffix_tables" and not with_suffix:
            assert g is None
            continue
        assert np.array_equal(g.cpu().numpy(), w), name
    return got, want


@pytest.mark.parametrize("block", [16, 32, 8, 1, 24])
@pytest.mark.parametrize("requests, ctx_hi, new_hi", [(1, 0, 1), (1, 40, 300), (7, 100, 1), (33, 60, 90), (300, 500, 3), (1025, 70, 2), (2500, 30, 40)])
def test_tables(requests, ctx_hi, new_hi, block):
    rng = np.random.default_rng(requests + block)
    width = -(-(ctx_hi + new_hi) // block) + 1
    ctx, new, tables, free = problem(rng, requests, ctx_hi, new_hi, width, block)
    total = int(new.sum())
    prefix = rng.integers(0, 5000, size=requests)
    for prefills in {0, requests // 2, requests}:
        both(ctx, new, tables, free, 0, block, total, prefills, prefix)
    both(ctx, new, tables, free, 3, block, total + 37)            # padded rows
    both(ctx, new, tables, free, 0, block, max(total - 5, 0))     # fewer rows than tokens
    both(ctx, new, tables, free, 0, block, total, with_suffix=False)


@pytest.mark.parametrize("short", [0, 1, 2, 5, 1000])
def test_free_blocks_run_out(short):
    rng = np.random.default_rng(short)
    ctx, new, tables, free = problem(rng, 60, 100, 40, 12, 16, free_extra=0, zero_new=0.1)
    free = free[:max(len(free) - short, 0)]
    got, want = both(ctx, new, tables, free, 0, 16, int(new.sum()))
    assert (int(got.num_failed) > 0) == (short > 0)


def test_requests_that_do_not_fit_their_row():
    rng = np.random.default_rng(5)
    ctx, new, tables, free = problem(rng, 40, 100, 40, 6, 16, free_extra=100)
    got, want = both(ctx, new, tables, free, 0, 16, int(new.sum()))
    assert int(got.num_failed) > 0


def test_no_requests_no_tokens():
    both(np.zeros(0, int), np.zeros(0, int), np.zeros((0, 4), np.int32), np.arange(4), 1, 16, 0)
    both(np.zeros(0, int), np.zeros(0, int), np.zeros((0, 4), np.int32), np.arange(4), 1, 16, 9)
    both(np.array([5, 16]), np.array([0, 0]), np.zeros((2, 2), np.int32), np.arange(4), 1, 16, 3)


def test_rows_of_a_larger_table_and_untouched_entries():
    big = torch.full((5, 40), -9, dtype=torch.int32, device=DEV)
    view = big[:, 3:13]
    ctx, new, free = [0, 16, 17, 40, 3], [33, 1, 1, 0, 13], np.arange(100, 120)
    for r, c in enumerate(ctx):
        view[r, :-(-c // 16)] = 50 + r
    before = big.clone()
    want = orc.block_tables(ctx, new, view.cpu().numpy(), free, 2, 16, sum(new), 1)
    got = pb.build_block_tables(i32(ctx), i32(new), view, i32(free), i32([2]), block_size=16, num_tokens=sum(new), num_prefills=1)
    assert np.array_equal(view.cpu().numpy(), want["block_tables"]) and np.array_equal(got.slot_mapping.cpu().numpy(), want["slot_mapping"])
    before[:, 3:13] = big[:, 3:13]
    assert torch.equal(before, big)


def test_refusals():
    ok = dict(context_lens=i32([1]), new_lens=i32([1]), block_tables=i32([[0]]), free_blocks=i32([0]), free_head=i32([0]))
    for bad in (dict(context_lens=i32([1]).long()), dict(new_lens=i32([1, 2])), dict(block_tables=i32([0])), dict(free_head=i32([0, 0])),
                dict(block_tables=i32([[0], [1]])), dict(block_tables=i32([[0, 1]]).t())):
        with pytest.raises(RuntimeError):
            pb.build_block_tables(**{**ok, **bad}, block_size=16, num_tokens=1)
    for kw in (dict(num_prefills=2, num_tokens=1), dict(num_tokens=-1)):
        with pytest.raises(RuntimeError):
            pb.build_block_tables(**ok, block_size=16, **kw)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_an_engine_loop(dtype):
    """Prompts, then decode steps, one captured and replayed: tables from lengths, fill, attention, all on the GPU; the cache and
    every step's output against the oracle's."""
    rng = np.random.default_rng(31)
    heads, d, b, blocks, width = 2, 128, 16, 64, 12
    prompts = [70, 5, 16, 130]
    r = len(prompts)
    cache = pb.fp8_kv_cache(blocks, heads, d, b, DEV)
    mirror = tuple(x.copy() for x in to_host(cache))
    ctx, free = np.zeros(r, int), rng.permutation(blocks).astype(np.int32)
    host_tables, head = np.zeros((r, width), np.int32), 0
    context_lens, tables, free_head, free_dev = i32(ctx), i32(host_tables), i32([0]), i32(free)

    def step(new_dev, rows, prefills, k, v, q):
        t = pb.build_block_tables(context_lens, new_dev, tables, free_dev, free_head, block_size=b, num_tokens=rows, num_prefills=prefills)
        pb.fp8_reshape_and_cache(k, v, *cache, t.slot_mapping)
        seg = dict(seg_row_offsets=t.row_offsets[:prefills + 1], seg_kv_lens=t.kv_lens[:prefills], seg_tables=tables[:prefills]) if prefills else {}
        call = pb.Fp8AttentionCall(num_rows=rows, num_heads=heads, head_size=d, block_size=b, dtype=q.dtype, device=q.device,
                                   suffix_lens=t.suffix_lens, suffix_tables=t.suffix_tables, **seg)
        out = call.run(q, torch.empty_like(q), *cache)
        context_lens.copy_(t.kv_lens)
        free_head.copy_(t.free_head)
        return out, t

    def check(out, new, prefills, k, v, q):
        nonlocal host_tables, head, ctx
        want = orc.block_tables(ctx, new, host_tables, free, head, b, q.shape[0], prefills)
        orc.fill(*mirror, k.double().cpu().numpy(), v.double().cpu().numpy(), want["slot_mapping"])
        host_tables, head = want["block_tables"], int(want["free_head"][0])
        contexts = [orc.context_slots(host_tables[i], ctx[i] + j + 1, b) for i in range(r) for j in range(new[i])]
        ctx = want["kv_lens"].astype(int)
        for g, w in zip(to_host(cache), mirror):
            assert np.array_equal(g, w)
        want = orc.attention(q.double().cpu().numpy(), mirror, contexts, d ** -0.5)
        check_attention(out, want, dtype)

    rows = lambda n: [rand_rows(rng, n, heads, d, dtype) for _ in range(3)]  # noqa: E731
    k, v, q = rows(sum(prompts))
    out, _ = step(i32(prompts), sum(prompts), r, k, v, q)
    check(out, prompts, r, k, v, q)
    one = [1] * r
    new_dev = i32(one)
    k, v, q = rows(r)
    out, _ = step(new_dev, r, 0, k, v, q)
    check(out, one, 0, k, v, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = step(new_dev, r, 0, k, v, q)
    for _ in range(20):
        nk, nv, nq = rows(r)
        k.copy_(nk), v.copy_(nv), q.copy_(nq)
        graph.replay()
        check(out, one, 0, k, v, q)
