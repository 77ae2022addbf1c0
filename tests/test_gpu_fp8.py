"""The 8-bit cache on the GPU against the 64-bit oracle: fill bit for bit, gather exactly, attention within its roundings."""
import numpy as np
import pytest
import torch

import parrotserve_b200 as pb
from oracle import fp8_oracle as orc
from parrotserve_b200 import _lib, fp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------
# helpers
# ---------------------------------------------------------------------------------------------
def random_cache(rng, blocks, heads, d, b, spread=3, pow2=True):
    """Random codes (no NaN) and scales on the host: (key codes, value codes, key scale, value scale)."""
    def codes(shape):
        c = rng.integers(0, 254, size=shape, dtype=np.uint8)
        return np.where(c >= 127, c + 1, c).astype(np.uint8)  # skips 0x7f; 0xff is not drawn
    def scales():
        e = rng.uniform(-spread, spread, size=(blocks, heads)) - 8
        return (np.exp2(np.round(e)) if pow2 else np.exp2(e)).astype(np.float32)
    return codes((blocks, heads, d // 16, b, 16)), codes((blocks, heads, d, b)), scales(), scales()


def on_gpu(cache):
    k, v, ks, vs = cache
    return (torch.from_numpy(k.copy()).to(DEV).view(fp8.CACHE_DTYPE), torch.from_numpy(v.copy()).to(DEV).view(fp8.CACHE_DTYPE),
            torch.from_numpy(ks.copy()).to(DEV), torch.from_numpy(vs.copy()).to(DEV))


def to_host(cache):
    k, v, ks, vs = cache
    return k.view(torch.uint8).cpu().numpy(), v.view(torch.uint8).cpu().numpy(), ks.cpu().numpy(), vs.cpu().numpy()


def same_cache(got, want):
    names = ("key codes", "value codes", "key scale", "value scale")
    for g, w, name in zip(got, want, names):
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), f"{name}: {np.argwhere(g != w)[:5].tolist()}"


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32), device=DEV)


def rand_rows(rng, n, h, d, dtype, size=1.0):
    x = torch.from_numpy(rng.standard_normal((n, h, d)) * size).to(DEV).to(TYPES[dtype])
    return x


def check_attention(out, want, dtype, what="", more=0.0):
    """Roundings that enter, with e the half step of the output's type:
    * the output's own: e |ref|;
    * the weights': 2^-11 of each (rounded to fp16 by the prefix kernel and where several heads share an item; as four e4m3
      parts, each within 2^-4 of what is left, 2^-16), 2^-22 (hi + lo fp16) for fp32 queries; and the smallest step of the format
      they take with the value's scale: parts with a largest weight of at least 2^8 end at half a step of 2^-9 / 16^3, fp16
      with one of at least 2^7 at 2^-25: 2^-30 of the largest weight (times scale) for each token (`loud`);
    * the logits': q . k is summed in fp32 in at most 32 instructions and multiplied by rounded factors: 2^-19 of the
      largest value the sum can reach (`reach`). 16-bit queries go in as e4m3 parts of a row whose largest element is
      at least 2^7: of the prefix kernel the last part's half step is 2^-10, 2^-17 of that element for each of the row's, 2^-17 of
      `reach` for the logit (the single-query kernel's is 2^-22, less than the sum's own). A change x of a logit changes its weight by x;
    * both enter numerator and denominator: twice, relative to the same attention over |V|; sums of weights: 2^-20."""
    e = torch.finfo(TYPES[dtype]).eps / 2
    weights, logits = (2.0 ** -22, 2.0 ** -19) if dtype == "f32" else (2.0 ** -11, 2.0 ** -17 + 2.0 ** -19)
    out = out.detach().double().cpu().numpy()
    assert np.isfinite(out).all(), what
    tol = e * np.abs(want.out) + (2 * weights + 2 * logits * want.reach[..., None] + 2.0 ** -20 + more) * want.absolute + 2.0 ** -30 * want.loud + 1e-30
    if dtype == "f16":
        tol = tol + 2.0 ** -25  # subnormal outputs
    worst = (np.abs(out - want.out) / tol).max() if out.size else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the tolerance"


# ---------------------------------------------------------------------------------------------
# fill and gather
# ---------------------------------------------------------------------------------------------
def fill_both(cache, key, value, slots, slot_type=torch.int64):
    """Runs the fill on the GPU and in the oracle, from the same cache; returns both results."""
    dev = on_gpu(cache)
    pb.fp8_reshape_and_cache(key, value, *dev, torch.as_tensor(np.asarray(slots, dtype=np.int64), device=DEV).to(slot_type))
    want = tuple(x.copy() for x in cache)
    orc.fill(*want, key.double().cpu().numpy(), value.double().cpu().numpy(), slots)
    return to_host(dev), want


def in_order(rng, blocks, b, lens, pasts):
    """Slots of contexts with distinct blocks: tokens past .. past + len of each."""
    ids = iter(rng.permutation(blocks).tolist())
    out = []
    for n, past in zip(lens, pasts):
        table = [next(ids) for _ in range(-(-(n + past) // b))]
        out += [table[p // b] * b + p % b for p in range(past, past + n)]
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d, b, heads", [(128, 16, 4), (64, 32, 3), (80, 16, 1), (96, 32, 2), (112, 16, 5), (256, 16, 2), (256, 32, 1)])
def test_fill_prefills_and_decodes(dtype, d, b, heads):
    rng = np.random.default_rng(d * 31 + b + heads)
    cache = random_cache(rng, 40, heads, d, b)
    lens = [1, 1, 37, 16, 5, 1, 64, 1, 17]
    pasts = [0, 5, 0, 16, 13, 31, 3, 15, 40]
    slots = in_order(rng, 40, b, lens, pasts)
    t = len(slots)
    key, value = rand_rows(rng, t, heads, d, dtype, 3.0), rand_rows(rng, t, heads, d, dtype, 0.01)
    got, want = fill_both(cache, key, value, slots)
    same_cache(got, want)


@pytest.mark.parametrize("b", [16, 32])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 300, 1100])
def test_fill_any_order_duplicates_and_holes(b, tokens):
    rng = np.random.default_rng(tokens + b)
    heads, d, blocks = 2, 64, 20
    cache = random_cache(rng, blocks, heads, d, b)
    slots = rng.integers(-3, blocks * b + 5, size=tokens)  # repeats, negatives, slots behind the cache
    key, value = rand_rows(rng, tokens, heads, d, "f16"), rand_rows(rng, tokens, heads, d, "f16")
    for slot_type in (torch.int64, torch.int32):
        got, want = fill_both(cache, key, value, slots, slot_type)
        same_cache(got, want)


def test_fill_every_token_in_one_slot():
    rng = np.random.default_rng(3)
    cache = random_cache(rng, 3, 1, 64, 16)
    key, value = rand_rows(rng, 700, 1, 64, "bf16"), rand_rows(rng, 700, 1, 64, "bf16")
    got, want = fill_both(cache, key, value, [17] * 700)
    same_cache(got, want)


def test_fill_steps_grow_and_keep_scales():
    """Token after token into the same blocks: the scale grows, stays, and the first token of a block begins anew."""
    rng = np.random.default_rng(5)
    heads, d, b = 3, 128, 16
    cache = tuple(np.zeros_like(x) for x in random_cache(rng, 4, heads, d, b))
    dev, want = on_gpu(cache), tuple(x.copy() for x in cache)
    for step in range(40):
        size = 2.0 ** rng.integers(-6, 7)
        slots = [(step % 32), 32 + (step * 7) % 32]
        key, value = rand_rows(rng, 2, heads, d, "f32", size), rand_rows(rng, 2, heads, d, "f32", 1 / size)
        pb.fp8_reshape_and_cache(key, value, *dev, torch.tensor(slots, device=DEV))
        orc.fill(*want, key.double().cpu().numpy(), value.double().cpu().numpy(), slots)
        same_cache(to_host(dev), want)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("tokens, heads, d, b", [(40, 7, 128, 16), (23, 5, 256, 32), (1030, 6, 64, 16)])
def test_fill_lone_tokens_under_heads_that_differ(dtype, tokens, heads, d, b):
    """One token for each block: some heads keep their scale, some grow it, some bring NaN, infinities or zeros."""
    rng = np.random.default_rng(tokens + heads)
    blocks = tokens + 4
    cache = random_cache(rng, blocks, heads, d, b)
    slots = rng.permutation(blocks)[:tokens] * b + rng.integers(0, b, size=tokens)
    rows = []
    for _ in range(2):
        x = rng.standard_normal((tokens, heads, d)) * np.exp2(rng.integers(-4, 5, size=(tokens, heads, 1)))
        x[rng.random((tokens, heads)) < 0.1] = 0
        x[..., 3] = np.where(rng.random((tokens, heads)) < 0.05, np.nan, x[..., 3])
        x[..., 40] = np.where(rng.random((tokens, heads)) < 0.05, np.inf, x[..., 40])
        rows.append(torch.from_numpy(x).to(DEV).to(TYPES[dtype]))
    got, want = fill_both(cache, *rows, slots)
    same_cache(got, want)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_fill_special_values(dtype):
    """NaN, infinities, zeros, the type's largest and smallest values, values between two codes, borders of a scale."""
    d = 64
    fi = torch.finfo(TYPES[dtype])
    rows = torch.zeros(9, 1, d, dtype=torch.float64)
    rows[0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0], dtype=torch.float64)
    rows[1, 0, :2] = torch.tensor([fi.max, -fi.max], dtype=torch.float64)
    rows[2, 0, :3] = torch.tensor([fi.tiny, fi.smallest_normal, -fi.tiny], dtype=torch.float64)
    rows[4, 0, :] = torch.linspace(-448, 448, d, dtype=torch.float64)
    rows[5, 0, :4] = torch.tensor([448, 17.0, 18.0, -19.0], dtype=torch.float64)
    rows[6, 0, :4] = torch.tensor([450, 0.001, 0.0009765625, -0.0], dtype=torch.float64)
    rows[7, 0, :] = float("nan")
    rows[8, 0, :2] = torch.tensor([float("inf"), 3e-5], dtype=torch.float64)
    rows = rows.to(TYPES[dtype]).to(DEV)
    rng = np.random.default_rng(1)
    cache = random_cache(rng, 12, 1, d, 16)
    for slots in ([16 * i for i in range(9)], [16 * i + 5 for i in range(9)], list(range(9))):
        got, want = fill_both(cache, rows, rows.flip(0).contiguous(), slots)
        same_cache(got, want)


def test_fill_of_strided_rows_and_strided_cache():
    rng = np.random.default_rng(8)
    heads, d, b, blocks = 4, 128, 16, 9
    fused = torch.from_numpy(rng.standard_normal((33, 3, heads, d))).to(DEV).half()  # q, k, v of one projection
    slots = in_order(rng, blocks, b, [20, 13], [0, 9])
    host = random_cache(rng, blocks, heads, d, b)
    # every second block and a slice of the heads of larger caches; scales likewise
    big_k = torch.zeros(2 * blocks, heads + 2, d // 16, b, 16, dtype=torch.uint8, device=DEV)
    big_v = torch.zeros(2 * blocks, heads + 2, d, b, dtype=torch.uint8, device=DEV)
    big_s = torch.zeros(2, heads + 2, 2 * blocks, device=DEV)
    views = (big_k[::2, 1:heads + 1], big_v[::2, 1:heads + 1], big_s[0].t()[::2, 1:heads + 1], big_s[1].t()[::2, 1:heads + 1])
    for view, h in zip(views, host):
        view.copy_(torch.from_numpy(h))
    dev = (views[0].view(fp8.CACHE_DTYPE), views[1].view(fp8.CACHE_DTYPE), views[2], views[3])
    pb.fp8_reshape_and_cache(fused[:, 1], fused[:, 2], *dev, torch.tensor(slots, device=DEV))
    want = tuple(x.copy() for x in host)
    orc.fill(*want, fused[:, 1].double().cpu().numpy(), fused[:, 2].double().cpu().numpy(), slots)
    same_cache(tuple(x.cpu().numpy() for x in (views[0], views[1], views[2], views[3])), want)
    assert not big_k[1::2].any() and not big_k[:, 0].any() and not big_v[:, heads + 1].any() and not big_s[:, :, 1::2].any()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d, b, heads", [(128, 16, 4), (80, 32, 3), (256, 16, 1)])
def test_gather(dtype, d, b, heads):
    rng = np.random.default_rng(d + b)
    blocks = 11
    cache = random_cache(rng, blocks, heads, d, b)
    cache[0][3, 0, 0, 2, 5] = 0x7F  # NaN comes out as NaN
    slots = np.concatenate([np.arange(40), rng.integers(0, blocks * b, size=50), [-1, 3 * b + 2, blocks * b, -7]])
    key = torch.full((len(slots), heads, d), 7.0, device=DEV, dtype=TYPES[dtype])
    value = torch.full_like(key, -7.0)
    pb.fp8_gather_cached_kv(key, value, *on_gpu(cache), torch.as_tensor(slots, device=DEV))
    live = (slots >= 0) & (slots < blocks * b)
    k, v = orc.token_rows(*cache, slots[live])
    for got, want, left in ((key, k, 7.0), (value, v, -7.0)):
        got = got.cpu()
        assert torch.equal(torch.nan_to_num(got[live], nan=-1), torch.nan_to_num(torch.from_numpy(want).to(TYPES[dtype]), nan=-1))
        assert (got[~live] == left).all()


@pytest.mark.parametrize("tokens, heads", [(700, 8), (6000, 8), (10000, 17)])
def test_gather_of_runs(tokens, heads):
    """Runs of consecutive slots of any length from any offset, with holes, up to sizes at which a CTA takes 256 of them."""
    rng = np.random.default_rng(tokens)
    blocks, b, d = 400, 32, 64
    cache = random_cache(rng, blocks, heads, d, b)
    slots = []
    while len(slots) < tokens:
        n, at = int(rng.integers(1, 90)), int(rng.integers(-5, blocks * b))
        slots += [-1] if rng.random() < 0.1 else list(range(at, at + n))
    slots = np.asarray(slots[:tokens])
    key = torch.full((tokens, heads, d), 7.0, device=DEV, dtype=torch.bfloat16)
    value = torch.full_like(key, -7.0)
    pb.fp8_gather_cached_kv(key, value, *on_gpu(cache), torch.as_tensor(slots, device=DEV))
    live = (slots >= 0) & (slots < blocks * b)
    k, v = orc.token_rows(*cache, slots[live])
    for got, want, left in ((key, k, 7.0), (value, v, -7.0)):
        got = got.cpu()
        assert torch.equal(got[live], torch.from_numpy(want).to(torch.bfloat16)) and (got[~live] == left).all()


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def paged_problem(rng, lens, heads, kv, d, b, dtype, **kw):
    width = max(1, max(-(-n // b) for n in lens))
    need = sum(-(-n // b) for n in lens)
    cache = random_cache(rng, need + 3, kv, d, b, **kw)
    ids = iter(rng.permutation(need + 3).tolist())
    tables = np.zeros((len(lens), width), dtype=np.int32)
    for r, n in enumerate(lens):
        tables[r, :-(-n // b)] = [next(ids) for _ in range(-(-n // b))]
    q = rand_rows(rng, len(lens), heads, d, dtype)
    mapping = None if heads == kv else [h // (heads // kv) for h in range(heads)]
    contexts = [orc.context_slots(tables[r], n, b) for r, n in enumerate(lens)]
    return cache, tables, q, mapping, contexts


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d, b, heads, kv", [
    (128, 16, 3, 3), (64, 16, 2, 2), (80, 16, 2, 2), (96, 32, 2, 2), (112, 16, 1, 1), (112, 32, 4, 2), (256, 16, 2, 1), (256, 32, 1, 1),
    (128, 32, 4, 4), (128, 16, 8, 1), (64, 32, 14, 2), (80, 32, 12, 3), (128, 16, 20, 2)])
def test_paged_attention(dtype, d, b, heads, kv):
    rng = np.random.default_rng(d * 7 + b + heads * 3 + kv)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 257, 700]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    out = pb.fp8_paged_attention(q, *on_gpu(cache), None if mapping is None else i32(mapping), i32(lens), i32(tables))
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, d ** -0.5, mapping)
    check_attention(out, want, dtype)
    assert (out[0] == 0).all()  # an empty context


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d, b, heads, kv", [(64, 16, 8, 1), (128, 16, 6, 2), (128, 32, 2, 2), (256, 16, 1, 1), (96, 16, 3, 3)])
def test_few_rows_with_many_partials(dtype, d, b, heads, kv):
    """Long contexts beside short and empty ones, split into chunks over the chip. At most 128 terms of a chunk and 80 partials are
    added one after another: 208 half steps of 2^-24, less than 2^-16, on top of what check_attention counts."""
    rng = np.random.default_rng(d + heads)
    lens = [9001, 0, 5, 4096]
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, heads, kv, d, b, dtype)
    dev = on_gpu(cache)
    m, l = torch.zeros(len(lens), heads, device=DEV), torch.zeros(len(lens), heads, device=DEV)
    call = pb.Fp8AttentionCall(num_rows=len(lens), num_heads=heads, head_size=d, block_size=b, dtype=TYPES[dtype], device=torch.device(DEV),
                               suffix_lens=i32(lens), suffix_tables=i32(tables), head_mapping=None if mapping is None else i32(mapping),
                               suffix_chunk_blocks=128 // b)
    out = torch.full_like(q, float("nan"))
    call.run(q, out, *dev, m, l, _lib.PB_STATS_SAVE)
    assert call.status() == 0
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, d ** -0.5, mapping)
    check_attention(out, want, dtype, more=2.0 ** -16)
    assert (out[1] == 0).all() and (l[1] == 0).all()
    # and joined with what a call has left before: the same once more doubles the sums and keeps the mean
    again = out.clone()
    call.run(q, again, *dev, m, l, _lib.PB_STATS_LOAD_SAVE)
    check_attention(again, want, dtype, more=2.0 ** -16 + torch.finfo(TYPES[dtype]).eps / 2)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_scales_of_any_size(dtype):
    """Scales that are no powers of two, that differ by 2^40 between blocks, that are zero; values of the outputs' range."""
    rng = np.random.default_rng(77)
    lens, d, b, heads = [1, 16, 40, 300, 511], 128, 16, 2
    cache, tables, q, _, contexts = paged_problem(rng, lens, heads, heads, d, b, dtype, pow2=False)
    k, v, ks, vs = cache
    vs[::3] *= np.float32(2.0 ** -20)
    vs[1::5] *= np.float32(2.0 ** 12)
    vs[2::4] = 0.0
    ks[::4] = 0.0
    q = q * 0.25
    out = pb.fp8_paged_attention(q, *on_gpu(cache), None, i32(lens), i32(tables))
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, d ** -0.5)
    check_attention(out, want, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("b, kv", [(16, 2), (32, 1)])
def test_codes_behind_the_context_are_not_looked_at(dtype, b, kv):
    """NaN codes behind a context's end, in its last block and in blocks nobody owns, change nothing."""
    rng = np.random.default_rng(9)
    lens, d = [1, 5, 16, 19, 31, 47], 64
    cache, tables, q, mapping, contexts = paged_problem(rng, lens, 2, kv, d, b, dtype)
    mapping_t = None if mapping is None else i32(mapping)
    clean = pb.fp8_paged_attention(q, *on_gpu(cache), mapping_t, i32(lens), i32(tables))
    used = np.zeros(cache[1].shape[0] * b, dtype=bool)
    for c in contexts:
        used[c] = True
    used = used.reshape(-1, b)
    cache[0][:] = np.where(used[:, None, None, :, None], cache[0], 0x7F)
    cache[1][:] = np.where(used[:, None, None, :], cache[1], 0xFF)
    dirty = pb.fp8_paged_attention(q, *on_gpu(cache), mapping_t, i32(lens), i32(tables))
    assert torch.equal(clean, dirty)


def layer_problem(rng, *, dtype, heads, kv, d=128, b=16, prefixes=(), group_rows=(), segments=(), suffixes=(), outer=0):
    """Rows: the segments' new tokens, then a row per suffix; groups partition the rows in order; `outer`: a context above all."""
    n_seg = sum(n for n, _ in segments)
    rows = n_seg + len(suffixes)
    ctx = [n + past for n, past in segments]
    all_lens = list(prefixes) + ctx + list(suffixes) + [outer]
    need = sum(-(-n // b) for n in all_lens)
    cache = random_cache(rng, need + 2, kv, d, b, spread=2)
    ids = iter(rng.permutation(need + 2).tolist())

    def table(lens):
        t = np.zeros((len(lens), max(1, max(-(-n // b) for n in lens))), dtype=np.int32)
        for i, n in enumerate(lens):
            t[i, :-(-n // b)] = [next(ids) for _ in range(-(-n // b))]
        return t

    kw, contexts = {}, [np.zeros(0, dtype=np.int64) for _ in range(rows)]
    add = lambda r, s: contexts.__setitem__(r, np.concatenate([contexts[r], s]))  # noqa: E731
    if outer:
        t = table([outer])
        kw.update(outer_row_offsets=i32([0, rows]), outer_prefix_lens=i32([outer]), outer_tables=i32(t))
        for r in range(rows):
            add(r, orc.context_slots(t[0], outer, b))
    if prefixes:
        t, offs = table(prefixes), np.concatenate([[0], np.cumsum(group_rows)])
        assert offs[-1] <= rows
        kw.update(group_row_offsets=i32(offs), group_prefix_lens=i32(prefixes), group_tables=i32(t))
        for g, n in enumerate(prefixes):
            for r in range(offs[g], offs[g + 1]):
                add(r, orc.context_slots(t[g], n, b))
    if segments:
        t, offs = table(ctx), np.concatenate([[0], np.cumsum([n for n, _ in segments])])
        kw.update(seg_row_offsets=i32(offs), seg_kv_lens=i32(ctx), seg_tables=i32(t))
        for s, (n, past) in enumerate(segments):
            for i in range(n):
                add(offs[s] + i, orc.context_slots(t[s], past + i + 1, b))
    lens = [0] * n_seg + list(suffixes)
    t = np.zeros((rows, 1), dtype=np.int32)
    if suffixes:
        own = table(suffixes)
        t = np.concatenate([np.zeros((n_seg, own.shape[1]), dtype=np.int32), own])
        for r, n in enumerate(suffixes):
            add(n_seg + r, orc.context_slots(own[r], n, b))
    kw.update(suffix_lens=i32(lens), suffix_tables=i32(t))
    mapping = None if heads == kv else [h // (heads // kv) for h in range(heads)]
    q = rand_rows(rng, rows, heads, d, dtype)
    call = pb.Fp8AttentionCall(num_rows=rows, num_heads=heads, head_size=d, block_size=b, dtype=TYPES[dtype], device=torch.device(DEV),
                               head_mapping=None if mapping is None else i32(mapping), **kw)
    return call, q, cache, contexts, mapping


LAYERS = [
    dict(heads=2, kv=2, prefixes=(100,), group_rows=(5,), suffixes=(1, 16, 17, 40, 300)),
    dict(heads=2, kv=2, prefixes=(515,), group_rows=(70,), suffixes=tuple(range(1, 71))),
    dict(heads=4, kv=2, prefixes=(130, 16, 1, 700), group_rows=(3, 9, 1, 40), suffixes=tuple([7] * 53)),
    dict(heads=2, kv=2, segments=((1, 0), (5, 0), (130, 0), (40, 77), (300, 5))),
    dict(heads=1, kv=1, prefixes=(260,), group_rows=(183,), segments=((150, 0), (20, 33)), suffixes=(0, 1, 31, 32, 33, 200, 3, 4, 5, 6, 7, 8, 9)),
    dict(heads=8, kv=2, prefixes=(260,), group_rows=(52,), segments=((40, 0), (2, 33)), suffixes=(0, 1, 31, 32, 33, 200, 3, 4, 5, 6)),
    dict(heads=2, kv=2, prefixes=(48, 90), group_rows=(6, 5), suffixes=tuple([20] * 11), outer=200),
    dict(heads=2, kv=2, d=64, b=32, prefixes=(100,), group_rows=(7,), segments=((3, 10),), suffixes=(5, 40, 41, 1)),
    # shares of the chip that begin and end inside heads: CTAs with segments of one kv tile, two, and many
    dict(heads=5, kv=5, prefixes=(4000,), group_rows=(6,), suffixes=(1, 2, 3, 4, 5, 6)),
    dict(heads=3, kv=3, prefixes=(1500, 3000, 130, 700), group_rows=(7, 140, 20, 5), suffixes=tuple(range(172))),
    dict(heads=4, kv=1, segments=((300, 500), (20, 0), (140, 900), (1, 700), (260, 0)), suffixes=(30, 0)),
    dict(heads=1, kv=1, segments=((700, 0), (600, 100)), dense_row_tile=256),
    dict(heads=1, kv=1, prefixes=(300,), group_rows=(600,), segments=((250, 0), (349, 20)), suffixes=(50,), dense_row_tile=256),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", range(len(LAYERS)))
def test_layers(dtype, case):
    spec = dict(LAYERS[case])
    tile = spec.pop("dense_row_tile", 0)
    rng = np.random.default_rng(100 + case)
    call, q, cache, contexts, mapping = layer_problem(rng, dtype=dtype, **spec)
    call.params.dense_row_tile = tile
    dev = on_gpu(cache)
    out = torch.full_like(q, float("nan"))
    call.plan(q, out, *dev)
    call.run(q, out, *dev)
    assert call.status() == 0
    first = out.clone()
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, q.shape[2] ** -0.5, mapping)
    check_attention(out, want, dtype, f"layer {case}")
    call.run(q, out, *dev)  # the plan serves every layer
    assert torch.equal(out, first)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_statistics_and_merging_of_two_calls(dtype):
    rng = np.random.default_rng(4)
    lens, d, b, heads = [1, 40, 300], 128, 16, 2
    cache, tables, q, _, contexts = paged_problem(rng, lens, heads, heads, d, b, dtype)
    dev = on_gpu(cache)
    first = [n // 2 // b * b for n in lens]
    skip = np.zeros_like(tables)
    for r, n in enumerate(first):
        skip[r, :tables.shape[1] - n // b] = tables[r, n // b:]
    kw = dict(num_rows=3, num_heads=heads, head_size=d, block_size=b, dtype=TYPES[dtype], device=torch.device(DEV))
    m, l = torch.zeros(3, heads, device=DEV), torch.zeros(3, heads, device=DEV)
    out = torch.zeros_like(q)
    pb.Fp8AttentionCall(suffix_lens=i32(first), suffix_tables=i32(tables), **kw).run(q, out, *dev, m, l, _lib.PB_STATS_SAVE)
    pb.Fp8AttentionCall(suffix_lens=i32(np.asarray(lens) - first), suffix_tables=i32(skip), **kw).run(q, out, *dev, m, l, _lib.PB_STATS_LOAD_SAVE)
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, d ** -0.5)
    # the first call's output is rounded to the type once more on its way
    check_attention(out, want, dtype, more=torch.finfo(TYPES[dtype]).eps / 2)
    slack = 2.0 ** -19 * want.reach * 1.5  # (base-2 logits: log2(e) < 1.5)
    assert (np.abs(m.double().cpu().numpy() - want.top) <= slack).all()
    assert (np.abs(l.double().cpu().numpy() - want.total) <= (2 * slack + 2.0 ** -20) * want.total).all()


def test_bad_tables_give_nan_and_a_status():
    """A block id outside the cache, and a head mapping outside its kv heads: recorded, never dereferenced, NaN everywhere."""
    rng = np.random.default_rng(6)
    cache, tables, q, _, _ = paged_problem(rng, [40, 50], 2, 2, 64, 16, "f16")
    kw = dict(num_rows=2, num_heads=2, head_size=64, block_size=16, dtype=torch.float16, device=torch.device(DEV), suffix_lens=i32([40, 50]))
    bad = tables.copy()
    bad[1, 2] = cache[0].shape[0]
    for args in (dict(suffix_tables=i32(bad)), dict(suffix_tables=i32(tables), head_mapping=i32([0, 2])),
                 dict(suffix_tables=i32(tables), head_mapping=i32([-1, 1]))):
        out = torch.zeros_like(q)
        call = pb.Fp8AttentionCall(**kw, **args)
        call.run(q, out, *on_gpu(cache))
        assert call.status() == 2 and out.isnan().all()


def test_long_cache_offsets_beyond_32_bits():
    """Blocks whose byte offsets in the cache pass 2^31 and 2^32."""
    d, b = 128, 16
    blocks = (1 << 32) // (d * b) + 40
    kc = torch.empty(blocks, 1, d // 16, b, 16, dtype=torch.uint8, device=DEV)
    vc = torch.empty(blocks, 1, d, b, dtype=torch.uint8, device=DEV)
    ks, vs = torch.zeros(blocks, 1, device=DEV), torch.zeros(blocks, 1, device=DEV)
    dev = (kc.view(fp8.CACHE_DTYPE), vc.view(fp8.CACHE_DTYPE), ks, vs)
    rng = np.random.default_rng(2)
    table = [blocks - 1, 5, blocks // 2 + 7, blocks - 30]
    n = 60
    slots = orc.context_slots(table, n, b)
    key, value, q = rand_rows(rng, n, 1, d, "f16"), rand_rows(rng, n, 1, d, "f16"), rand_rows(rng, 1, 1, d, "f16")
    pb.fp8_reshape_and_cache(key, value, *dev, torch.as_tensor(slots, device=DEV))
    k2, v2 = torch.empty_like(key), torch.empty_like(value)
    pb.fp8_gather_cached_kv(k2, v2, *dev, torch.as_tensor(slots, device=DEV))
    for got, rows in ((k2, key), (v2, value)):
        # half a step of e4m3 of the value, or of its smallest step under the block's scale (amax <= 8 -> scale <= 2^-5)
        assert ((got.double() - rows.double()).abs() <= rows.double().abs() * 2.0 ** -4 + 2.0 ** -10 * 2.0 ** -5).all()
    out = pb.fp8_paged_attention(q, *dev, None, i32([n]), i32([table]))
    p = torch.softmax((k2.double()[:, 0] @ q.double()[0, 0]) * d ** -0.5, 0)
    v, reach = v2.double()[:, 0], d ** -0.5 * q.double().abs().max() * k2.double().abs().sum(-1).max()
    two = lambda x: x.cpu().numpy()[None, None]  # noqa: E731
    check_attention(out, orc.Attention(two(p @ v), two(p @ v.abs()), None, None, 0.0, reach.cpu().numpy()[None, None]), "f16")


def test_rows_of_a_wider_tensor_and_into_one():
    rng = np.random.default_rng(12)
    lens, d, heads = [3, 70, 33], 128, 2
    cache, tables, q, _, contexts = paged_problem(rng, lens, heads, heads, d, 16, "bf16")
    fused = torch.zeros(3, 3 * heads * d, dtype=torch.bfloat16, device=DEV)
    fused[:, :heads * d] = q.reshape(3, -1)
    wide = torch.full((3, heads * d + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    call = pb.Fp8AttentionCall(num_rows=3, num_heads=heads, head_size=d, block_size=16, dtype=torch.bfloat16, device=torch.device(DEV),
                               suffix_lens=i32(lens), suffix_tables=i32(tables))
    out = wide[:, 8:].view(3, heads, d)
    call.run(fused[:, :heads * d].view(3, heads, d), out, *on_gpu(cache))
    want = orc.attention(q.double().cpu().numpy(), cache, contexts, d ** -0.5)
    check_attention(out, want, "bf16")
    assert (wide[:, :8] == 5.0).all()


def test_on_a_stream_of_its_own_and_in_graphs():
    """Two captured iterations (fill, one-shot attention) replayed in turn, next to the same calls on a side stream."""
    rng = np.random.default_rng(21)
    d, b, heads, lens = 128, 16, 2, [5, 33, 64]
    problems = [paged_problem(rng, lens, heads, heads, d, b, "f16") for _ in range(2)]
    new_slots = [[int(c[-1]) for c in p[4]] for p in problems]
    rows = [(rand_rows(rng, 3, heads, d, "f16"), rand_rows(rng, 3, heads, d, "f16")) for _ in range(2)]
    args = [(on_gpu(p[0]), i32(lens), i32(p[1]), p[2], torch.tensor(s, device=DEV)) for p, s in zip(problems, new_slots)]

    def step(i):
        dev, ln, tb, q, slots = args[i]
        pb.fp8_reshape_and_cache(*rows[i], *dev, slots)
        return pb.fp8_paged_attention(q, *dev, None, ln, tb)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [step(i).clone() for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)
    for i in range(2):
        want = orc.attention(problems[i][2].double().cpu().numpy(), to_host(args[i][0]), problems[i][4], d ** -0.5)
        check_attention(eager[i], want, "f16")


def test_nothing_to_do():
    kc, vc, ks, vs = fp8.fp8_kv_cache(2, 1, 64, 16, DEV)
    none = torch.zeros(0, 1, 64, dtype=torch.float16, device=DEV)
    slots = torch.zeros(0, dtype=torch.int64, device=DEV)
    pb.fp8_reshape_and_cache(none, none, kc, vc, ks, vs, slots)
    pb.fp8_gather_cached_kv(none, none, kc, vc, ks, vs, slots)
    out = pb.fp8_paged_attention(none, kc, vc, ks, vs, None, i32([]), i32(np.zeros((0, 1))))
    assert out.shape == (0, 1, 64)


def test_operators_refuse():
    kc, vc, ks, vs = fp8.fp8_kv_cache(2, 2, 64, 16, DEV)
    row = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)
    for bad in (dict(key_cache=kc.view(torch.uint8)), dict(key_scale=ks.half()), dict(value_scale=vs[:1]), dict(key=row[:, :1]),
                dict(slot_mapping=slots[:2]), dict(value=row.float()), dict(key=row.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(key_cache=kc[:1])):
        args = {**dict(key=row, value=row, key_cache=kc, value_cache=vc, key_scale=ks, value_scale=vs, slot_mapping=slots), **bad}
        for op in (pb.fp8_reshape_and_cache, pb.fp8_gather_cached_kv):
            with pytest.raises(RuntimeError):
                op(*args.values())
    with pytest.raises(RuntimeError):
        pb.fp8_paged_attention(row.int(), kc, vc, ks, vs, None, i32([1, 1, 1]), i32([[0], [0], [0]]))
    call = pb.Fp8AttentionCall(num_rows=3, num_heads=2, head_size=64, block_size=16, dtype=torch.float16, device=torch.device(DEV),
                               suffix_lens=i32([1, 1, 1]), suffix_tables=i32([[0], [0], [0]]))
    for bad in (dict(query=row.bfloat16()), dict(query=row[:2]), dict(out=row[:, :, :32]), dict(key_cache=kc.view(torch.uint8))):
        args = {**dict(query=row, out=torch.empty_like(row), key_cache=kc, value_cache=vc, key_scale=ks, value_scale=vs), **bad}
        with pytest.raises(RuntimeError):
            call.run(*args.values())


def test_statistics_are_checked():
    kc, vc, ks, vs = fp8.fp8_kv_cache(2, 2, 64, 16, DEV)
    row = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    call = pb.Fp8AttentionCall(num_rows=3, num_heads=2, head_size=64, block_size=16, dtype=torch.float16, device=torch.device(DEV),
                               suffix_lens=i32([1, 1, 1]), suffix_tables=i32([[0], [0], [0]]))
    good = torch.zeros(3, 2, device=DEV)
    for m, l in ((None, good), (good, None), (good.half(), good), (good, good[:2]), (good.cpu(), good), (good.t().contiguous().t(), good)):
        with pytest.raises(RuntimeError):
            call.run(row, torch.empty_like(row), kc, vc, ks, vs, m, l, _lib.PB_STATS_SAVE)
