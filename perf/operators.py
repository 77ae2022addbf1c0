"""The 8-bit paged cache: what fills it, what reads it, and the tables that say where its tokens go.

A case is a dict of plain values; ``op`` says which operators one pass goes through:

* ``tables``  block tables, slots, positions and row lengths of an iteration, from the requests' lengths
  (``build_block_tables``).
* ``fill``    new key / value rows into the 8-bit cache, then the contexts of the touched blocks out of it again
  (``fp8_reshape_and_cache``, ``fp8_gather_cached_kv``).
* ``paged``   decode without sharing, in one shot (``fp8_paged_attention``).
* ``layer``   one layer of an iteration that is already planned: decodes, prefills or both, under shared prefixes
  (``Fp8AttentionCall.run``).

The cache holds e4m3 values, K [blocks, heads, head_size/16, block, 16] and V [blocks, heads, head_size, block], and one
fp32 scale for each block and head. Lengths follow from the case alone (``lens`` seeds them); contents, scales and the
placement of the blocks follow from the seed of ``prepare``.
"""
import random

import numpy as np
import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _layer(dtype, heads, kv_heads, lens, groups=0, prefix_lo=0, prefix_hi=0, seqs=0, skew=0.0, suffix_lo=0, suffix_hi=0,
           prefills=0, new_lo=0, new_hi=0, past_hi=0, **name):
    return dict(name, op="layer", dtype=dtype, heads=heads, kv_heads=kv_heads, head_size=128, block=16, groups=groups,
                prefix_lo=prefix_lo, prefix_hi=prefix_hi, seqs=seqs, skew=skew, suffix_lo=suffix_lo, suffix_hi=suffix_hi,
                prefills=prefills, new_lo=new_lo, new_hi=new_hi, past_hi=past_hi, lens=lens)


def listed():
    return [
        # The tables of a small chat batch: 24 requests that each add a token.
        dict(name="tables_24_decodes", op="tables", requests=24, prefills=0, ctx_lo=1, ctx_hi=900, new_lo=1, new_hi=1, block=16,
             lens=1),
        # Continuous batching: 16 prompts of 256 to 1024 tokens and 240 decodes.
        dict(name="tables_16prefill_240decode", op="tables", requests=256, prefills=16, ctx_lo=0, ctx_hi=1024, new_lo=256,
             new_hi=1024, block=16, lens=2),
        # The fill of a decode step: 64 lone tokens, each at the end of its own block.
        dict(name="fill_64_decodes", op="fill", dtype="f16", heads=32, head_size=128, block=16, prefills=0, new_lo=0, new_hi=0,
             past_hi=500, seqs=64, holes=False, lens=3),
        # A continuous-batching iteration: 16 prefills, some of which go on in a block that is begun, and 240 decodes.
        dict(name="fill_16prefill_240decode", op="fill", dtype="bf16", heads=32, head_size=128, block=16, prefills=16, new_lo=256,
             new_hi=1024, past_hi=300, seqs=240, holes=False, lens=4),
        # fp32 rows of a small model with heads of 80, blocks of 32, and padding tokens without a slot.
        dict(name="fill_fp32_odd", op="fill", dtype="f32", heads=12, head_size=80, block=32, prefills=5, new_lo=1, new_hi=333,
             past_hi=77, seqs=9, holes=True, lens=5),
        # Three requests of a chat: the smallest decode, where launches count.
        dict(name="paged_3seq", op="paged", dtype="f16", heads=32, kv_heads=32, head_size=128, block=16, seqs=3, ctx_lo=1,
             ctx_hi=300, lens=6),
        # Plain paged decode with grouped kv heads.
        dict(name="paged_gqa_128seq", op="paged", dtype="bf16", heads=32, kv_heads=8, head_size=128, block=16, seqs=128, ctx_lo=16,
             ctx_hi=2048, lens=7),
        # One long document: a single query row over 100 thousand tokens.
        dict(name="paged_long_1seq", op="paged", dtype="bf16", heads=64, kv_heads=8, head_size=128, block=16, seqs=1, ctx_lo=100003,
             ctx_hi=100003, lens=8),
        # fp32 queries, heads of 80, blocks of 32.
        dict(name="paged_fp32_odd", op="paged", dtype="f32", heads=12, kv_heads=12, head_size=80, block=32, seqs=57, ctx_lo=1,
             ctx_hi=1777, lens=9),
        # A decode step of a 7B model: 64 sequences over one 4096-token prefix.
        _layer("f16", 32, 32, 10, name="decode_7b_64seq", groups=1, prefix_lo=4096, prefix_hi=4096, seqs=64, suffix_lo=32,
               suffix_hi=512),
        # 13B decode, ragged: 256 sequences spread unevenly over 8 applications with prompts of 1k to 8k.
        _layer("f16", 40, 40, 11, name="decode_13b_8groups", groups=8, prefix_lo=1024, prefix_hi=8192, seqs=256, skew=1.2,
               suffix_lo=1, suffix_hi=2048),
        # Continuous batching: 16 prefills and 240 decodes over a 2048-token prompt.
        _layer("bf16", 32, 32, 12, name="mixed_16prefill_240decode", groups=1, prefix_lo=2048, prefix_hi=2048, seqs=240, suffix_lo=1,
               suffix_hi=1024, prefills=16, new_lo=256, new_hi=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    most = {"bytes": 0.0, "flops": 0.0}
    for c in listed():
        w = work(c)
        most = {k: max(most[k], w[k]) for k in most}
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and w["bytes"] >= 200:
            return case


def _draw(rng):
    lens = rng.randrange(1 << 20)
    op = rng.choice(["tables", "tables", "fill", "fill", "fill", "paged", "paged", "paged", "decode", "groups", "mixed", "prefill"])
    block = rng.choice([16, 16, 32])
    if op == "tables":
        requests = _log_int(rng, 1, 2048)
        prefills = rng.choice([0, min(requests, _log_int(rng, 1, 64))])
        return dict(op="tables", requests=requests, prefills=prefills, ctx_lo=0, ctx_hi=_log_int(rng, 1, 4096), new_lo=1,
                    new_hi=_log_int(rng, 1, 2048) if prefills else 1, block=block, lens=lens)
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    head_size = rng.choice([64, 80, 96, 112, 128, 128, 128, 256])
    if op == "fill":
        prefills = rng.choice([0, _log_int(rng, 1, 32)])
        new = _log_int(rng, 1, 2048) if prefills else 0
        return dict(op="fill", dtype=dtype, heads=rng.choice([1, 4, 8, 12, 32, 40]), head_size=head_size, block=block,
                    prefills=prefills, new_lo=min(new, 1), new_hi=new, past_hi=_log_int(rng, 1, 1000), seqs=_log_int(rng, 1, 512),
                    holes=rng.choice([False, True]), lens=lens)
    if op == "paged":
        heads, kv = rng.choice([(32, 32), (32, 8), (40, 40), (64, 8), (12, 12), (7, 7), (28, 4)])
        return dict(op="paged", dtype=dtype, heads=heads, kv_heads=kv, head_size=head_size, block=block, seqs=_log_int(rng, 1, 256),
                    ctx_lo=rng.choice([0, 1]), ctx_hi=_log_int(rng, 16, 4096), lens=lens)
    half = rng.choice(["f16", "bf16"])
    heads, kv = rng.choice([(8, 8), (32, 32), (40, 40), (12, 12), (32, 8)])
    if op == "decode":
        prefix = _log_int(rng, 64, 8192)
        return _layer(half, heads, kv, lens, groups=1, prefix_lo=prefix, prefix_hi=prefix, seqs=_log_int(rng, 2, 512), suffix_lo=1,
                      suffix_hi=_log_int(rng, 32, 2048))
    if op == "groups":
        prefix = _log_int(rng, 256, 8192)
        return _layer(half, heads, kv, lens, groups=_log_int(rng, 2, 32), prefix_lo=max(16, prefix // rng.choice([1, 4, 8])),
                      prefix_hi=prefix, seqs=_log_int(rng, 32, 1024), skew=rng.choice([0.0, 1.2]), suffix_lo=1,
                      suffix_hi=_log_int(rng, 64, 2048))
    new = _log_int(rng, 16, 2048)
    if op == "mixed":
        prefix = _log_int(rng, 64, 4096)
        return _layer(half, heads, kv, lens, groups=1, prefix_lo=prefix, prefix_hi=prefix, seqs=_log_int(rng, 4, 240), suffix_lo=1,
                      suffix_hi=_log_int(rng, 64, 1024), prefills=_log_int(rng, 1, 16), new_lo=max(1, new // 4), new_hi=new)
    return _layer(half, heads, kv, lens, prefills=_log_int(rng, 1, 16), new_lo=max(1, new // 4), new_hi=new,
                  past_hi=rng.choice([0, 500]))


# ---------------------------------------------------------------------------------------------
# lengths (of the case alone)
# ---------------------------------------------------------------------------------------------
def _spread(r, lo, hi, n):
    return [r.randint(lo, hi) for _ in range(n)]


def _lengths(case):
    """Lengths of a case: prefix tokens and rows of every group, prefill (new, past) and private decode contexts."""
    r = random.Random(case["lens"])
    if case["op"] == "paged":
        return dict(ctx=_spread(r, case["ctx_lo"], case["ctx_hi"], case["seqs"]))
    if case["op"] == "tables":
        n, p = case["requests"], case["prefills"]
        ctx = _spread(r, case["ctx_lo"], case["ctx_hi"], n)
        return dict(ctx=ctx, new=_spread(r, case["new_lo"], case["new_hi"], p) + [1] * (n - p))
    new = _spread(r, case["new_lo"], case["new_hi"], case["prefills"])
    past = _spread(r, 0, case["past_hi"], case["prefills"])
    if case["op"] == "fill":
        return dict(new=new + [1] * case["seqs"], past=past + _spread(r, 0, case["past_hi"], case["seqs"]))
    g = case["groups"]
    steps = [case["prefix_lo"] + (case["prefix_hi"] - case["prefix_lo"]) * i // max(1, g - 1) for i in range(g)]
    weight = [(i + 1) ** -case["skew"] for i in range(g)]
    home = sorted(r.choices(range(g), weights=weight, k=case["seqs"])) if g else [0] * case["seqs"]
    rows = [home.count(i) for i in range(g)]
    return dict(prefix=steps, rows=rows, new=new, past=past, suffix=_spread(r, case["suffix_lo"], case["suffix_hi"], case["seqs"]))


def work(case):
    le = _lengths(case)
    cdiv = lambda a, b: -(-a // b)  # noqa: E731
    if case["op"] == "tables":
        b = case["block"]
        t, n = sum(le["new"]), len(le["new"])
        width = max(cdiv(c + k, b) for c, k in zip(le["ctx"], le["new"]))
        held = sum(cdiv(c + k, b) for c, k in zip(le["ctx"], le["new"]))
        return {"bytes": 4 * (4 * n + held) + t * (8 + 8 + 4 + 4 * width), "flops": 0}
    e = 4 if case["dtype"] == "f32" else 2
    d = case["head_size"]
    if case["op"] == "fill":
        b, h = case["block"], case["heads"]
        t = sum(le["new"])
        out = sum(p % b + k for p, k in zip(le["past"], le["new"]))
        blocks = sum(cdiv(p % b + k, b) for p, k in zip(le["past"], le["new"]))
        return {"bytes": 2 * h * d * (t * (e + 1) + out * (1 + e)) + 16 * blocks * h + 8 * (t + out), "flops": 4 * h * d * (t + out)}
    h, kv, b = case["heads"], case["kv_heads"], case["block"]
    if case["op"] == "paged":
        rows, tokens, pairs = case["seqs"], sum(le["ctx"]), sum(le["ctx"])
    else:
        rows = case["seqs"] + sum(le["new"])
        tokens = sum(le["prefix"]) + sum(le["suffix"]) + sum(le["new"]) + sum(le["past"])
        pairs = sum(le["suffix"]) + sum(k * p + k * (k + 1) // 2 for k, p in zip(le["new"], le["past"]))
        pairs += sum(n * p for n, p in zip(le["rows"], le["prefix"]))
        if le["prefix"]:
            pairs += sum(le["new"]) * le["prefix"][0]  # prefills come under the first group's prefix
    scales = 8 * kv * cdiv(tokens, b)
    return {"bytes": 2 * kv * d * tokens + scales + 2 * rows * h * d * e + 4 * cdiv(tokens, b), "flops": 4 * h * d * pairs}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tables(contexts, block, pool):
    """Block tables [len(contexts), widest] of contexts of the given lengths, blocks taken from `pool` (an iterator)."""
    width = max([-(-c // block) for c in contexts] + [1])
    out = np.zeros((len(contexts), width), dtype=np.int32)
    for i, c in enumerate(contexts):
        n = -(-c // block)
        out[i, :n] = [next(pool) for _ in range(n)]
    return out


def _scale_for(top):
    """The smallest power of two with top <= 448 * scale, 0 for 0 (top >= 0, finite)."""
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    return torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), torch.zeros_like(top))


def _cache(gen, blocks, heads, head_size, block):
    """A cache as fills leave it: normal values, every head with a size of its own, some blocks far larger than others."""
    size = 2.0 ** (3 * torch.rand(heads, device=DEV, generator=gen) - 2)
    made = []
    for shape in ((blocks, heads, head_size // 16, block, 16), (blocks, heads, head_size, block)):
        x = torch.randn(shape, device=DEV, generator=gen)
        loud = 1.0 + 3.0 * (torch.rand(blocks, 1, device=DEV, generator=gen) < 0.02) if len(shape) == 4 else 1.0
        by = (size * loud).expand(blocks, heads)
        x *= by.reshape(blocks, heads, *([1] * (len(shape) - 2)))
        scale = _scale_for(x.abs().flatten(2).amax(2))
        x /= scale.reshape(blocks, heads, *([1] * (len(shape) - 2)))
        made += [x.to(F8), scale]
        del x
    return dict(key_cache=made[0], key_scale=made[1], value_cache=made[2], value_scale=made[3])


def prepare(case, seed):
    le = _lengths(case)
    host = np.random.default_rng([int(seed), case["lens"]])
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 1000003 + case["lens"])
    b = case["block"]
    if case["op"] == "tables":
        n = len(le["ctx"])
        ends = [c + k for c, k in zip(le["ctx"], le["new"])]
        held = sum(-(-c // b) for c in ends)
        ids = host.permutation(2 * held + 64).astype(np.int32)
        pool = iter(ids.tolist())
        have = _tables(le["ctx"], b, pool)
        tables = np.zeros((n, max(-(-e // b) for e in ends)), dtype=np.int32)
        tables[:, :have.shape[1]] = have[:, :tables.shape[1]]
        free = np.fromiter(pool, dtype=np.int32)
        return dict(case=case, context_lens=_i32(le["ctx"]), new_lens=_i32(le["new"]), block_tables=torch.from_numpy(tables).to(DEV),
                    free_blocks=torch.from_numpy(free).to(DEV), free_head=_i32([int(host.integers(0, 8))]),
                    prefix_lens=_i32([int(host.integers(0, 4)) * 256] * n), num_tokens=sum(le["new"]))
    dtype = TYPES[case["dtype"]]
    d = case["head_size"]
    if case["op"] == "fill":
        h = case["heads"]
        ends = [p + k for p, k in zip(le["past"], le["new"])]
        blocks = sum(-(-e // b) for e in ends) + 7
        tables = _tables(ends, b, iter(host.permutation(blocks).tolist()))
        slots, out = [], []
        for i, (p, k) in enumerate(zip(le["past"], le["new"])):
            at = np.arange(p // b * b, p + k)
            s = tables[i][at // b].astype(np.int64) * b + at % b
            out.append(s)
            slots.append(s[p % b:])
        slots, out = np.concatenate(slots), np.concatenate(out)
        if case["holes"]:
            slots = np.concatenate([slots, np.full(5, -1, dtype=np.int64)])
        st = _cache(gen, blocks, h, d, b)
        rows = torch.randn(len(slots), 3, h, d, device=DEV, generator=gen).to(dtype)  # q, k, v of the fused projection
        st.update(case=case, key=rows[:, 1], value=rows[:, 2], slots=torch.from_numpy(slots).to(DEV), out_slots=torch.from_numpy(out).to(DEV),
                  key_out=torch.empty(len(out), h, d, dtype=dtype, device=DEV), value_out=torch.empty(len(out), h, d, dtype=dtype, device=DEV))
        return st
    h, kv = case["heads"], case["kv_heads"]
    mapping = _i32([i // (h // kv) for i in range(h)]) if kv != h else None
    if case["op"] == "paged":
        blocks = sum(-(-c // b) for c in le["ctx"]) + 1
        st = _cache(gen, blocks, kv, d, b)
        st.update(case=case, mapping=mapping, query=torch.randn(case["seqs"], h, d, device=DEV, generator=gen).to(dtype),
                  suffix_lens=_i32(le["ctx"]), suffix_tables=torch.from_numpy(_tables(le["ctx"], b, iter(host.permutation(blocks).tolist()))).to(DEV))
        return st
    # layer: rows are the prefills' tokens, then one row a sequence; the prefills lie under the first group's prefix
    new, past = le["new"], le["past"]
    own_ctx = [k + p for k, p in zip(new, past)]
    blocks = sum(-(-c // b) for c in le["prefix"] + own_ctx + le["suffix"]) + 1
    pool = iter(host.permutation(blocks).tolist())
    st = _cache(gen, blocks, kv, d, b)
    n_new = sum(new)
    rows = n_new + case["seqs"]
    st.update(case=case, mapping=mapping, query=torch.randn(rows, h, d, device=DEV, generator=gen).to(dtype))
    if case["groups"]:
        counts = [c + (n_new if i == 0 else 0) for i, c in enumerate(le["rows"])]
        st.update(group_row_offsets=_i32(np.concatenate([[0], np.cumsum(counts)]).tolist()), group_prefix_lens=_i32(le["prefix"]),
                  group_tables=torch.from_numpy(_tables(le["prefix"], b, pool)).to(DEV))
    if new:
        st.update(seg_row_offsets=_i32(np.concatenate([[0], np.cumsum(new)]).tolist()), seg_kv_lens=_i32(own_ctx),
                  seg_tables=torch.from_numpy(_tables(own_ctx, b, pool)).to(DEV))
    if case["seqs"]:
        tables = np.zeros((rows, max(-(-c // b) for c in le["suffix"])), dtype=np.int32)
        tables[n_new:] = _tables(le["suffix"], b, pool)
        st.update(suffix_lens=_i32([0] * n_new + le["suffix"]), suffix_tables=torch.from_numpy(tables).to(DEV))
    st["out"] = torch.empty_like(st["query"])
    if own:  # the work lists that an iteration builds once and every layer uses
        import parrotserve_b200 as pb

        call = pb.Fp8AttentionCall(num_rows=rows, num_heads=h, head_size=d, block_size=b, dtype=dtype, device=st["query"].device,
                                   suffix_lens=st.get("suffix_lens"), suffix_tables=st.get("suffix_tables"), head_mapping=mapping,
                                   **{k: st.get(k) for k in ("group_row_offsets", "group_prefix_lens", "group_tables", "seg_row_offsets",
                                                             "seg_kv_lens", "seg_tables")})
        call.plan(st["query"], st["out"], st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"])
        st["call"] = call
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    return _own(st) if own else _plain(st)


def _own(st):
    import parrotserve_b200 as pb

    op = st["case"]["op"]
    if op == "tables":
        t = pb.build_block_tables(st["context_lens"], st["new_lens"], st["block_tables"], st["free_blocks"], st["free_head"],
                                  block_size=st["case"]["block"], num_tokens=st["num_tokens"], num_prefills=st["case"]["prefills"],
                                  prefix_lens=st["prefix_lens"])
        return dict(block_tables=st["block_tables"], slot_mapping=t.slot_mapping, positions=t.positions, row_offsets=t.row_offsets,
                    kv_lens=t.kv_lens, suffix_lens=t.suffix_lens, suffix_tables=t.suffix_tables, free_head=t.free_head,
                    num_failed=t.num_failed)
    cache = (st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"])
    if op == "fill":
        pb.fp8_reshape_and_cache(st["key"], st["value"], *cache, st["slots"])
        pb.fp8_gather_cached_kv(st["key_out"], st["value_out"], *cache, st["out_slots"])
        return dict(key=st["key_out"], value=st["value_out"], key_scale=st["key_scale"], value_scale=st["value_scale"])
    if op == "paged":
        return pb.fp8_paged_attention(st["query"], *cache, st["mapping"], st["suffix_lens"], st["suffix_tables"])
    return st["call"].run(st["query"], st["out"], *cache)


# ---- the plain forms ----
def _plain(st):
    op = st["case"]["op"]
    return _plain_tables(st) if op == "tables" else _plain_fill(st) if op == "fill" else _plain_attention(st)


def _plain_tables(st):
    b, p, t = st["case"]["block"], st["case"]["prefills"], st["num_tokens"]
    ctx, new, tables, free = (st[k].long() for k in ("context_lens", "new_lens", "block_tables", "free_blocks"))
    head = st["free_head"].long()
    r, width = tables.shape
    have, want = (ctx + b - 1) // b, (ctx + new + b - 1) // b
    wide = want > width
    need = torch.where(wide, 0, want - have)
    upto = need.cumsum(0)
    failed = wide | ((need > 0) & (head + upto > free.numel()))
    col = torch.arange(width, device=ctx.device)
    take = torch.where(failed, 0, need)
    at = head + (upto - need)[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < (have + take)[:, None])
    tables = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], tables)
    st["block_tables"].copy_(tables)
    offsets = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row = torch.arange(t, device=ctx.device)
    req = torch.searchsorted(offsets, row, right=True) - 1
    behind = req >= r  # rows behind the last token
    req = req.clamp(0, r - 1)
    pos = ctx[req] + row - offsets[req]
    lost = behind | failed[req]
    slot = torch.where(lost, -1, tables[req, (pos // b).clamp(0, width - 1)] * b + pos % b)
    positions = torch.where(behind, 0, pos + st["prefix_lens"].long()[req])
    suffix = torch.where(lost | (req < p), 0, pos + 1)
    row_tables = torch.where(col < ((suffix + b - 1) // b)[:, None], tables[req], 0)
    as32 = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(block_tables=st["block_tables"], slot_mapping=slot, positions=positions, row_offsets=as32(offsets),
                kv_lens=as32(ctx + torch.where(failed, 0, new)), suffix_lens=as32(suffix), suffix_tables=as32(row_tables),
                free_head=as32(head + take.sum()), num_failed=as32(failed.sum().reshape(1)))


def _to_f8(x, inv):
    y = (x * inv).clamp(-F8_MAX, F8_MAX)
    return torch.where(torch.isfinite(x), y, torch.nan).to(F8)


def _plain_fill(st):
    b = st["case"]["block"]
    slots, t = st["slots"], st["slots"].numel()
    blk = torch.where(slots >= 0, slots // b, -1)
    blocks, which = torch.unique(blk, return_inverse=True)
    member = torch.full((blocks.numel() * b,), -1, dtype=torch.int64, device=slots.device)
    member.scatter_reduce_(0, which * b + slots % b, torch.arange(t, device=slots.device), "amax")
    live = blocks >= 0
    blocks, member = blocks[live], member.view(-1, b)[live]
    for name in ("key", "value"):
        cache, scales = st[name + "_cache"], st[name + "_scale"]
        nb, h = scales.shape
        cells = cache[blocks].float()  # key [u, h, d/16, b, 16], value [u, h, d, b]
        cells = cells.permute(0, 3, 1, 2, 4).flatten(3) if name == "key" else cells.permute(0, 3, 1, 2)  # [u, b, h, d]
        rows = st[name].float()[member.clamp(min=0)]
        mine = (member >= 0)[:, :, None, None]
        top = torch.where(mine & torch.isfinite(rows), rows.abs(), 0).amax((1, 3))
        need = _scale_for(top)
        old = torch.where(member[:, :1] >= 0, 0, scales[blocks])
        now = torch.maximum(old, need)
        inv = torch.where(now > 0, 1 / now, 0)[:, None, :, None]
        grown = ((old > 0) & (now > old))[:, None, :, None]
        again = torch.where(grown, _to_f8(cells * old[:, None, :, None], inv).float(), cells)
        cells = torch.where(mine, _to_f8(rows, inv).float(), again).to(F8)
        u, d = cells.shape[0], cells.shape[3]
        cells = cells.view(u, b, h, d // 16, 16).permute(0, 2, 3, 1, 4) if name == "key" else cells.permute(0, 2, 3, 1)
        cache.view(torch.uint8)[blocks] = cells.contiguous().view(torch.uint8)
        scales[blocks] = now
    s = st["out_slots"]
    at, off = s // b, s % b
    key = st["key_cache"].view(torch.uint8)[at, :, :, off].view(F8).float().flatten(2)
    value = st["value_cache"].view(torch.uint8)[at, :, :, off].view(F8).float()
    st["key_out"].copy_(key * st["key_scale"][at][:, :, None])
    st["value_out"].copy_(value * st["value_scale"][at][:, :, None])
    return dict(key=st["key_out"], value=st["value_out"], key_scale=st["key_scale"], value_scale=st["value_scale"])


def _read(st, tables):
    """K and V of the tables' tokens in 32 bits: [n, tokens, kv heads, head_size] each."""
    n, w = tables.shape
    tables = tables.long()
    k = st["key_cache"].view(torch.uint8)[tables].view(F8).float() * st["key_scale"][tables][..., None, None, None]
    v = st["value_cache"].view(torch.uint8)[tables].view(F8).float() * st["value_scale"][tables][..., None, None]
    h, b, d = v.shape[2], v.shape[4], v.shape[3]
    return k.permute(0, 1, 4, 2, 3, 5).reshape(n, w * b, h, d), v.permute(0, 1, 4, 2, 3).reshape(n, w * b, h, d)


def _part(st, rows, tables, seen):
    """Attention of rows [n, m] (row indices, -1: none) over the tables' tokens, of which seen [n, m] are visible: scattered to
    all rows as (maximum, sum, weighted values)."""
    q = st["query"]
    total, h, d = q.shape
    k, v = _read(st, tables)
    kv = k.shape[2]
    n, m = rows.shape
    x = q.float()[rows.clamp(min=0)].view(n, m, kv, h // kv, d)
    s = torch.einsum("nmgsd,ntgd->ngsmt", x, k) * d ** -0.5
    hidden = torch.arange(k.shape[1], device=q.device) >= seen[:, None, None, :, None]
    s.masked_fill_(hidden, -torch.inf)
    top = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(torch.isfinite(top), top, 0))
    sums = s.sum(-1)
    out = torch.einsum("ngsmt,ntgd->nmgsd", s, v).reshape(n, m, h, d)
    live = rows >= 0
    at = rows[live]
    all_top, all_sum = q.new_full((total, h), -torch.inf, dtype=torch.float32), q.new_zeros((total, h), dtype=torch.float32)
    all_out = q.new_zeros((total, h, d), dtype=torch.float32)
    all_top[at] = top.squeeze(-1).permute(0, 3, 1, 2).reshape(n, m, h)[live]
    all_sum[at] = sums.permute(0, 3, 1, 2).reshape(n, m, h)[live]
    all_out[at] = out[live]
    return all_top, all_sum, all_out


def _by_offsets(offsets, widest):
    row = offsets[:-1, None].long() + torch.arange(widest, device=offsets.device)
    return torch.where(row < offsets[1:, None], row, -1)


def _plain_attention(st):
    le, q = _lengths(st["case"]), st["query"]
    parts = []
    if "group_tables" in st:
        widest = max(c + (sum(le["new"]) if i == 0 else 0) for i, c in enumerate(le["rows"]))
        rows = _by_offsets(st["group_row_offsets"], widest)
        parts.append(_part(st, rows, st["group_tables"], st["group_prefix_lens"][:, None].expand(rows.shape)))
    n_new = sum(le.get("new", []))
    if n_new:
        rows = _by_offsets(st["seg_row_offsets"], max(le["new"]))
        count = st["seg_row_offsets"][1:] - st["seg_row_offsets"][:-1]
        seen = (st["seg_kv_lens"] - count)[:, None] + torch.arange(rows.shape[1], device=q.device) + 1
        parts.append(_part(st, rows, st["seg_tables"], seen))
    if "suffix_tables" in st:
        rows = torch.arange(n_new, q.shape[0], device=q.device)[:, None]
        parts.append(_part(st, rows, st["suffix_tables"][n_new:], st["suffix_lens"][n_new:, None]))
    top = torch.stack([p[0] for p in parts]).amax(0)
    weight = [torch.exp(p[0] - torch.where(torch.isfinite(top), top, 0)) for p in parts]
    total = sum(w * p[1] for w, p in zip(weight, parts))
    out = sum(w[..., None] * p[2] for w, p in zip(weight, parts))
    return (out / torch.where(total > 0, total, 1)[..., None]).to(q.dtype)


# ---------------------------------------------------------------------------------------------
# the same in 64 bits, request by request
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None
    st = prepare(case, seed)
    return _exact_fill(st) if case["op"] == "fill" else _exact_attention(st)


def _nearest_f8(x):
    """e4m3 values nearest to x (ties to the even code), |x| <= 448, by the definition of the format."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_fill(st):
    b = st["case"]["block"]
    slots = st["slots"].tolist()
    by_block = {}
    for t, s in enumerate(slots):
        if s >= 0:
            by_block.setdefault(s // b, {})[s % b] = t
    outs = {}
    at, off = st["out_slots"] // b, st["out_slots"] % b
    for name in ("key", "value"):
        cache, scales = st[name + "_cache"], st[name + "_scale"].double()
        vals = {}
        for blk, members in by_block.items():
            cell = cache[blk].double()  # [h, d/16, b, 16] or [h, d, b]
            cell = cell.permute(2, 0, 1, 3).flatten(2) if name == "key" else cell.permute(2, 0, 1)  # [b, h, d]
            offs = list(members)
            rows = st[name][list(members.values())].double()
            top = rows.abs().amax((0, 2))
            old = scales[blk] * (0.0 if 0 in members else 1.0)
            fits = torch.exp2(torch.ceil(torch.log2(top / F8_MAX)))  # off by one where log2 rounds: mended below
            fits = torch.where(top > F8_MAX * fits, fits * 2, fits)
            fits = torch.where(top <= F8_MAX * fits / 2, fits / 2, fits)
            now = torch.maximum(old, torch.where(top > 0, fits, 0))
            div = torch.where(now > 0, now, 1)[:, None]
            grown = (old > 0) & (now > old)
            cell = torch.where(grown[:, None], _nearest_f8(cell * old[:, None] / div), cell)
            cell[offs] = _nearest_f8(rows / div)
            scales[blk] = now
            vals[blk] = cell
        order = {blk: i for i, blk in enumerate(vals)}
        stack = torch.stack(list(vals.values()))
        where = torch.tensor([order[x] for x in at.tolist()], device=stack.device)
        outs[name] = stack[where, off] * scales[at][:, :, None]
        outs[name + "_scale"] = scales
    return {k: outs[k] for k in ("key", "value", "key_scale", "value_scale")}


def _exact_attention(st):
    q = st["query"].double()
    rows, h, d = q.shape
    kv, b = st["case"]["kv_heads"], st["case"]["block"]
    out = torch.zeros_like(q)

    def tokens(table, count):
        ids = table[:-(-count // b)].long()
        k = st["key_cache"].view(torch.uint8)[ids].view(F8).double() * st["key_scale"].double()[ids][:, :, None, None, None]
        v = st["value_cache"].view(torch.uint8)[ids].view(F8).double() * st["value_scale"].double()[ids][:, :, None, None]
        k = k.permute(1, 0, 3, 2, 4).reshape(kv, -1, d)[:, :count]
        v = v.permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :count]
        return k, v

    def attend(lo, hi, pieces, own_len):
        """Rows lo..hi over the pieces' tokens, the last own_len of them causal from the bottom right."""
        if not pieces or hi == lo:
            return
        k, v = torch.cat([p[0] for p in pieces], 1), torch.cat([p[1] for p in pieces], 1)
        if k.shape[1] == 0:
            return
        for g in range(kv):
            x = q[lo:hi, g * (h // kv):(g + 1) * (h // kv)]
            s = (x.reshape(-1, d) @ k[g].T).view(hi - lo, h // kv, -1) * d ** -0.5
            if own_len:
                n = hi - lo
                seen = k.shape[1] - n + torch.arange(n, device=q.device) + 1
                s = s.masked_fill(torch.arange(k.shape[1], device=q.device) >= seen[:, None, None], -torch.inf)
            out[lo:hi, g * (h // kv):(g + 1) * (h // kv)] = torch.softmax(s, -1) @ v[g]

    groups = []
    if "group_tables" in st:
        offs = st["group_row_offsets"].tolist()
        groups = [(offs[i], offs[i + 1], tokens(st["group_tables"][i], n)) for i, n in enumerate(st["group_prefix_lens"].tolist())]

    def prefix_of(row):
        return [g[2] for g in groups if g[0] <= row < g[1]]

    first = 0
    if "seg_tables" in st:
        offs, kvs = st["seg_row_offsets"].tolist(), st["seg_kv_lens"].tolist()
        for i, n in enumerate(kvs):
            attend(offs[i], offs[i + 1], prefix_of(offs[i]) + [tokens(st["seg_tables"][i], n)], n)
        first = offs[-1]
    if "suffix_tables" in st:
        lens = st["suffix_lens"].tolist()
        for r in range(first, rows):
            attend(r, r + 1, prefix_of(r) + [tokens(st["suffix_tables"][r], lens[r])], 0)
    return out
