"""The bounds of the single-query kernel on tcgen05 by themselves: four e4m3 parts of every weight, not only what a 16-bit output shows."""
import math

import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from oracle import fp8_oracle as orc
from tests.test_gpu_fp8 import TYPES, i32, on_gpu, paged_problem


def cancelling(rng, cache, contexts, q, mapping, b):
    """Changes the V codes of every context's last four tokens so that the outputs nearly cancel: then half a step of the output's type says
    little, and the weights' own errors, relative to the same sum over |V|, are seen. Heads that share V take the elements in turn."""
    rows, heads, d = q.shape
    kv = cache[1].shape[1]
    share = heads // kv
    codes = rng.integers(0, 254, size=(4000, 4), dtype=np.uint8)
    codes = np.where(codes >= 127, codes + 1, codes).astype(np.uint8)
    for r in range(rows):
        slots = np.asarray(contexts[r])
        k, v = orc.token_rows(*cache, slots)
        scale = cache[3].astype(np.float64)[slots // b]
        for h in range(heads):
            at = h if mapping is None else mapping[h]
            s = (k[:, at] @ q[r, h]) * d ** -0.5
            p = np.exp(s - s.max())
            p /= p.sum()
            tries = orc.VALUES[codes] @ (p[-4:] * scale[-4:, at])
            for e in range(h % share, d, share):
                best = codes[np.argmin(np.abs(tries + p[:-4] @ v[:-4, at, e]))]
                for c, slot in zip(best, slots[-4:]):
                    cache[1][slot // b, at, e, slot % b] = c


def tolerance(want, dtype):
    """* the output's rounding: half a step of its type, or of its smallest numbers;
    * a weight: four parts, each the rounded remainder of those before it. A part is off by 2^-4 of itself at most, so four leave 2^-16 of the
      weight, or half the last one's smallest step, 2^-10 / 16^3 with a largest weight of 2^8: 2^-30 of that (`loud`). Its exponent,
      numbers below 2^4, is rounded three times to fp32 (half steps of 2^-21), and 2^x is off by 2^-22 in numerator and sum: below 2^-19;
    * a logit: at most 16 instructions of the tensor cores (four of 32 elements for each part of q) and the sum of the parts in fp32, and
      two rounded factors: 2^-19 of what it can reach. It changes its weight by as much; both enter numerator and denominator;
    * the sums: 2^-20."""
    e = torch.finfo(TYPES[dtype]).eps / 2
    weight = 2.0 ** -16 + 2.0 ** -19
    tiny = 2.0 ** -25 if dtype == "f16" else 2.0 ** -134
    return e * np.abs(want.out) + (weight + 2 * 2.0 ** -19 * want.reach[..., None] + 2.0 ** -20) * want.absolute + 2.0 ** -30 * want.loud + tiny


def problem(dtype, d, heads, kv):
    rng = np.random.default_rng(d + heads)
    lens, b = [4, 5, 16, 21, 40, 130], 16
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    q = q * 2.0 ** -6  # (exact: logits reach little, so that the weights' errors lead)
    cancelling(rng, cache, contexts, q.double().cpu().numpy(), mapping, b)
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, d ** -0.5, mapping)
    return lens, cache, tables, q, mapping, contexts, want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d, heads, kv", [(128, 2, 2), (64, 3, 3), (96, 2, 2), (128, 4, 1), (64, 4, 2), (128, 8, 1), (96, 6, 1)])
def test_weights_are_four_parts(dtype, d, heads, kv):
    lens, cache, tables, q, mapping, contexts, want = problem(dtype, d, heads, kv)
    out = pb.fp8_paged_attention(q, *on_gpu(cache), None if mapping is None else i32(mapping), i32(lens), i32(tables))
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    worst = (np.abs(got - want.out) / tolerance(want, dtype)).max()
    assert worst <= 1.0, f"{worst:.2f} of the tolerance"


def parts(w, n):
    """w as a sum of n e4m3 parts, the way the kernel makes them of the row's largest weight in [2^8, 2^8.75)."""
    total, unit = np.zeros_like(w), 1.0
    for _ in range(n):
        p = orc.VALUES[orc.to_codes(w)]
        total += p * unit
        w, unit = (w - p) * 16.0, unit / 16.0
    return total


def test_the_tolerance_tells_three_parts_from_four():
    """In the oracle: weights of four parts pass, of three do not."""
    rng = np.random.default_rng(5)
    d, b = 64, 16
    k, v = (rng.integers(0, 127, size=s, dtype=np.uint8) for s in ((6, 1, d // 16, b, 16), (6, 1, d, b)))
    scales = np.full((6, 1), 2.0 ** -8, dtype=np.float32)
    cache = (k, v, scales, scales.copy())
    q = rng.standard_normal((3, 1, d)).astype(np.float16).astype(np.float64) * 2.0 ** -6
    contexts = [orc.context_slots([i, i + 3], n, b) for i, n in enumerate((4, 9, 20))]
    cancelling(rng, cache, contexts, q, None, b)
    want = orc.attention(q, cache, contexts, d ** -0.5)
    for n, passes in ((4, True), (3, False)):
        worst = 0.0
        for r, slots in enumerate(contexts):
            kk, vv = orc.token_rows(*cache, slots)
            s = (kk[:, 0] @ q[r, 0]) * d ** -0.5 * math.log2(math.e)
            w = np.exp2(s - s.max())
            out = (parts(w * 2.0 ** 8.3, n) / 2.0 ** 8.3) @ vv[:, 0] / w.sum()
            worst = max(worst, (np.abs(np.float16(out) - want.out[r, 0]) / tolerance(want, "f16")[r, 0]).max())
        assert (worst <= 1.0) == passes, (n, worst)
