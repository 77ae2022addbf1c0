"""Value and key scales of the 8-bit cache over the range that a fill can make, from 2^-126 on, and their spread inside a row."""
import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from oracle import fp8_oracle as orc
from tests.test_gpu_fp8 import DEV, TYPES, i32, layer_problem, on_gpu, paged_problem

pytestmark = pytest.mark.gpu


def counted(cache, dtype, d, b):
    """The cache as attention reads it: on the tensor cores (16-bit queries, blocks of 16) value scales below 2^-100 are 0."""
    tensor_cores = dtype != "f32" and b == 16 and d in (64, 96, 128)
    return (*cache[:3], np.where(cache[3] < 2.0 ** -100, 0, cache[3]) if tensor_cores else cache[3])


def check(out, want, dtype, unit=0, far=False):
    """The tolerance of check_attention (its derivation is there) without its absolute terms, of an output multiplied by 2^-unit. Instead:
    * what falls below the normal numbers: half the smallest step of the output's type (bf16 2^-134, fp32 2^-150), and of fp32 for each
      of at most 128 partials of a row before they are divided by their sum (>= 1);
    * far: exponents of value scales beyond 2^6 are fp32 numbers below 2^8. The kernel for fp32 queries adds three of them in a row (half
      steps of 2^-17) and takes a logarithm with an error of 2^-22 of itself, 2^-15: together less than 2^-14 of a weight."""
    e = torch.finfo(TYPES[dtype]).eps / 2
    weights, logits = (2.0 ** -22, 2.0 ** -19) if dtype == "f32" else (2.0 ** -11, 2.0 ** -17 + 2.0 ** -19)
    small = (128 + (1 if dtype == "f32" else 2.0 ** 16)) * np.ldexp(1.0, -150 - unit)
    got = np.ldexp(out.detach().double().cpu().numpy(), -unit)
    assert np.isfinite(got).all()
    more = 2.0 ** -14 if far and dtype == "f32" else 0.0
    tol = e * np.abs(want.out) + (2 * weights + 2 * logits * want.reach[..., None] + 2.0 ** -20 + more) * want.absolute + 2.0 ** -30 * want.loud + small
    worst = (np.abs(got - want.out) / tol)[want.absolute > 0].max(initial=0.0)
    assert worst <= 1.0, f"{worst:.3g} of the tolerance"
    assert not got[want.absolute == 0].any()


SHAPES = [("bf16", 128, 16, 2, 2), ("bf16", 64, 16, 8, 2), ("bf16", 96, 16, 8, 1), ("f32", 128, 16, 2, 2), ("f32", 80, 32, 6, 2), ("bf16", 128, 32, 3, 3)]


@pytest.mark.parametrize("shift", [-115, -100, -92, -70, -25, 40, 100])
@pytest.mark.parametrize("dtype, d, b, heads, kv", SHAPES)
def test_decodes_with_value_scales_of_any_size(dtype, d, b, heads, kv, shift):
    rng = np.random.default_rng(d + heads)
    lens = [1, 17, 0, 300, 700]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    cache[3][:] = np.ldexp(cache[3], shift)
    scales = np.ldexp(counted(cache, dtype, d, b)[3], -shift)
    want = orc.attention(q.double().cpu().numpy(), (*cache[:3], scales), contexts, d ** -0.5, mapping)
    out = pb.fp8_paged_attention(q, *on_gpu(cache), None if mapping is None else i32(mapping), i32(lens), i32(tables))
    check(out, want, dtype, shift, far=True)


@pytest.mark.parametrize("shift", [-110, -92, -70, 40, 100])
@pytest.mark.parametrize("dtype, spec", [
    ("bf16", dict(heads=2, kv=2, prefixes=(515,), group_rows=(70,), suffixes=tuple(range(1, 71)))),            # a lone row tile
    ("bf16", dict(heads=3, kv=3, prefixes=(1500, 3000, 130), group_rows=(7, 140, 5), suffixes=tuple([3] * 152))),  # and pairs
    ("bf16", dict(heads=2, kv=2, segments=((130, 0), (300, 5), (20, 0)))),                                      # finished rows
    ("bf16", dict(heads=4, kv=1, segments=((300, 500), (140, 900)), suffixes=(30, 0))),
    ("f32", dict(heads=2, kv=2, prefixes=(100,), group_rows=(5,), suffixes=(1, 16, 17, 40, 300))),
])
def test_layers_with_value_scales_of_any_size(dtype, spec, shift):
    rng = np.random.default_rng(7)
    call, q, cache, contexts, mapping = layer_problem(rng, dtype=dtype, **spec)
    cache[3][:] = np.ldexp(cache[3], shift)
    scales = np.ldexp(counted(cache, dtype, 128, 16)[3], -shift)
    want = orc.attention(q.double().cpu().numpy(), (*cache[:3], scales), contexts, q.shape[2] ** -0.5, mapping)
    check(call.run(q, torch.empty_like(q), *on_gpu(cache)), want, dtype, shift, far=True)
    assert call.status() == 0


@pytest.mark.parametrize("first, then", [(-126, -60), (-60, -126), (-10, 60), (60, -10), (-100, -30), (100, 30), (-80, -80), (0, -75)])
@pytest.mark.parametrize("dtype, d, b, heads, kv", SHAPES)
def test_value_scales_that_differ_inside_a_row(dtype, d, b, heads, kv, first, then):
    """Scales near 2^first in the first 40 blocks of a context and near 2^then behind them, in one item of 64 blocks."""
    rng = np.random.default_rng((d + heads + first) % 1000)
    lens = [700 * b // 16, 1000 * b // 16]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    lift = np.full(cache[3].shape[0], then)
    lift[tables[:, :40].ravel()] = first
    cache[3][:] = np.ldexp(np.ones(cache[3].shape), np.maximum(lift[:, None] + rng.integers(-3, 4, size=cache[3].shape), -126)).astype(np.float32)
    want = orc.attention(q.double().cpu().numpy(), counted(cache, dtype, d, b), contexts, d ** -0.5, mapping)
    call = pb.Fp8AttentionCall(num_rows=2, num_heads=heads, head_size=d, block_size=b, dtype=TYPES[dtype], device=torch.device(DEV),
                               suffix_lens=i32(lens), suffix_tables=i32(tables), head_mapping=None if mapping is None else i32(mapping),
                               suffix_chunk_blocks=64)
    out = call.run(q, torch.empty_like(q), *on_gpu(cache))
    assert call.status() == 0
    check(out, want, dtype, far=True)


@pytest.mark.parametrize("first, then", [(-120, -60), (-60, -110), (-10, 60), (60, -10), (0, -75)])
def test_value_scales_that_differ_under_a_prefix(first, then):
    """The same for a prefix and its rows' own contexts: shares of the prefix begin anywhere in it."""
    rng = np.random.default_rng(9)
    call, q, cache, contexts, mapping = layer_problem(rng, dtype="bf16", heads=2, kv=2, prefixes=(3000,), group_rows=(9,), suffixes=tuple([40] * 9))
    lift = np.full(cache[3].shape[0], then)
    lift[contexts[0][:1500] // 16] = first
    cache[3][:] = np.ldexp(np.ones(cache[3].shape), np.maximum(lift[:, None] + rng.integers(-3, 4, size=cache[3].shape), -126)).astype(np.float32)
    want = orc.attention(q.double().cpu().numpy(), counted(cache, "bf16", 128, 16), contexts, 128 ** -0.5, mapping)
    check(call.run(q, torch.empty_like(q), *on_gpu(cache)), want, "bf16", far=True)


@pytest.mark.parametrize("dtype, d, b, heads, kv", SHAPES)
def test_a_key_scale_of_zero_is_zero(dtype, d, b, heads, kv):
    """Logits of exactly 0 under key scales of 0, whatever the codes and however large the queries: the mean of the values."""
    rng = np.random.default_rng(d)
    lens = [40, 300]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    cache[2][:] = 0.0
    want = orc.attention(np.zeros(q.shape), cache, contexts, d ** -0.5, mapping)
    out = pb.fp8_paged_attention(q * 1e30, *on_gpu(cache), None if mapping is None else i32(mapping), i32(lens), i32(tables))
    check(out, want, dtype)
    if dtype == "bf16" and b == 16 and d == 128:
        rows = [lens[0]] * 70  # and by the prefix kernel
        big = q[:1].expand(70, -1, -1).contiguous() * 1e30
        call = pb.Fp8AttentionCall(num_rows=70, num_heads=heads, head_size=d, block_size=b, dtype=TYPES[dtype], device=torch.device(DEV),
                                   group_row_offsets=i32([0, 70]), group_prefix_lens=i32([lens[1]]), group_tables=i32(tables[1:]),
                                   suffix_lens=i32([0] * 70), suffix_tables=i32(np.zeros((70, 1))))
        got = call.run(big, torch.empty_like(big), *on_gpu(cache))
        many = orc.attention(np.zeros(big.shape), cache, [contexts[1]] * len(rows), d ** -0.5, mapping)
        check(got, many, dtype)
