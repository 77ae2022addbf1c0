"""64-bit oracle of the 8-bit cache's operators and of the block tables: numpy, no code of the package."""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np


def e4m3_values() -> np.ndarray:
    """The 256 codes' values by the definition of the format: 1 sign, 4 exponent (bias 7), 3 mantissa bits; 0x7f and 0xff NaN."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out[c] = math.nan if (c & 0x7F) == 0x7F else (-v if c & 0x80 else v)
    return out


VALUES = e4m3_values()
_POSITIVE = VALUES[:127]  # 0 .. 448, ascending


def to_codes(x: np.ndarray) -> np.ndarray:
    """Nearest code of every value (ties to the even code), saturating; NaN and infinities give 0x7f."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    a = np.minimum(a, 448.0)
    hi = np.searchsorted(_POSITIVE, a)  # first code with value >= a
    lo = np.maximum(hi - 1, 0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    code = code | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isfinite(x), code, 0x7F).astype(np.uint8)


def scale_for(top: float) -> float:
    """The smallest power of two s >= 2^-126 with top <= 448 s; 0 for 0."""
    if not top > 0.0:
        return 0.0
    s = math.ldexp(1.0, -126)
    while top > 448.0 * s:
        s *= 2.0
    return s


def fill(key_codes, value_codes, key_scale, value_scale, key, value, slots) -> None:
    """The quantising fill, in place. codes: K [NB, H, D/16, B, 16], V [NB, H, D, B] uint8; scales [NB, H] float32;
    key / value [T, H, D] float64 (exact values of the rows); slots [T]."""
    nb, h, d, b = value_codes.shape
    blocks = {}
    for t, s in enumerate(slots):
        if 0 <= s < nb * b:
            blocks.setdefault(int(s) // b, {})[int(s) % b] = t  # later tokens replace earlier ones
    for blk, members in blocks.items():
        for codes, scales, rows, is_value in ((key_codes, key_scale, key, False), (value_codes, value_scale, value, True)):
            for head in range(h):
                # view [B, D] of the tile
                tile = codes[blk, head].T if is_value else codes[blk, head].transpose(1, 0, 2).reshape(b, d)
                new = np.stack([rows[t, head] for t in members.values()])
                finite = np.where(np.isfinite(new), np.abs(new), 0.0)
                old = 0.0 if 0 in members else float(scales[blk, head])
                top = float(finite.max())
                if not np.isfinite(new).all():
                    top = max(top, math.ldexp(448.0, -100))  # tiles with smaller scales may be read as zeros, which NaN is not
                now = max(old, scale_for(top))
                inv = np.float32(1.0) / np.float32(now) if now > 0 else np.float32(0.0)
                out = tile.copy()
                if old == 0.0 and now > 0.0 and 0 not in members:
                    out = np.zeros_like(tile)  # a tile with scale 0 is zero, whatever its codes
                elif 0.0 < old < now:
                    with np.errstate(all="ignore"):
                        out = to_codes((VALUES[tile].astype(np.float32) * np.float32(old)) * inv)
                for off, t in members.items():
                    with np.errstate(all="ignore"):
                        out[off] = to_codes(np.where(np.isfinite(rows[t, head]), rows[t, head].astype(np.float32) * inv, np.nan))
                if is_value:
                    codes[blk, head] = out.T
                else:
                    codes[blk, head] = out.reshape(b, d // 16, 16).transpose(1, 0, 2)
                scales[blk, head] = now


def token_rows(key_codes, value_codes, key_scale, value_scale, slots):
    """(key, value) [T, H, D] float64 of the given slots."""
    nb, h, d, b = value_codes.shape
    slots = np.asarray(slots, dtype=np.int64)
    blk, off = slots // b, slots % b
    k = VALUES[key_codes[blk, :, :, off]].reshape(len(slots), h, d) * key_scale.astype(np.float64)[blk][:, :, None]
    v = VALUES[value_codes[blk, :, :, off]] * value_scale.astype(np.float64)[blk][:, :, None]
    return k, v


def context_slots(table, length, block_size):
    p = np.arange(int(length))
    return np.asarray(table, dtype=np.int64)[p // block_size] * block_size + p % block_size


class Attention(NamedTuple):
    out: np.ndarray       # [rows, H, D]; an empty row gives zeros
    absolute: np.ndarray  # the same weights over |V|
    top: np.ndarray       # [rows, H] maximum of the base-2 logits
    total: np.ndarray     # [rows, H] sum of 2^(logit - top)
    loud: np.ndarray      # [rows, H, D] the largest weight * value scale of a token, times sum |code|, over the sum of weights
    reach: np.ndarray     # [rows, H] max over the tokens of scale * max|q| * sum |k|: what the logits of a row could be


def attention(query, cache, contexts, scale, head_mapping=None):
    """query [rows, H, D] float64; cache = (key_codes, value_codes, key_scale, value_scale); contexts[r] = slots that row r
    attends."""
    rows, h, d = query.shape
    out, absolute, loud = np.zeros((rows, h, d)), np.zeros((rows, h, d)), np.zeros((rows, h, d))
    top, total, reach = np.full((rows, h), -np.inf), np.zeros((rows, h)), np.zeros((rows, h))
    mapping = list(range(h)) if head_mapping is None else list(head_mapping)
    for r in range(rows):
        if len(contexts[r]) == 0:
            continue
        k, v = token_rows(*cache, contexts[r])
        for head in range(h):
            s = (k[:, mapping[head]] @ query[r, head]) * scale * math.log2(math.e)
            m = s.max()
            p = np.exp2(s - m)
            top[r, head], total[r, head] = m, p.sum()
            out[r, head] = p @ v[:, mapping[head]] / p.sum()
            absolute[r, head] = p @ np.abs(v[:, mapping[head]]) / p.sum()
            blocks = np.asarray(contexts[r]) // cache[1].shape[3]
            scales = cache[3].astype(np.float64)[blocks, mapping[head]]
            codes = np.abs(VALUES[cache[1][blocks, mapping[head], :, np.asarray(contexts[r]) % cache[1].shape[3]]])
            loud[r, head] = (p * scales).max() * codes.sum(0) / p.sum()
            reach[r, head] = scale * np.abs(query[r, head]).max() * np.abs(k[:, mapping[head]]).sum(-1).max()
    return Attention(out, absolute, top, total, loud, reach)


def block_tables(context_lens, new_lens, tables, free_blocks, free_head, block_size, num_tokens, num_prefills=0, prefix_lens=None):
    """The iteration's tables by a walk over the requests (see build_block_tables): a dict of arrays."""
    b, width = block_size, tables.shape[1]
    tables = tables.copy()
    slots, positions = np.full(num_tokens, -1, dtype=np.int64), np.zeros(num_tokens, dtype=np.int64)
    suffix, rows_tables = np.zeros(num_tokens, dtype=np.int32), np.zeros((num_tokens, width), dtype=np.int32)
    offsets, kv, head, failed, row = [0], [], int(free_head), 0, 0
    short = False  # the list was too short for a request: later ones that need a block fail too
    for r, (c, n) in enumerate(zip(context_lens, new_lens)):
        c, n = int(c), int(n)
        have, want = -(-c // b), -(-(c + n) // b)
        ok = want <= width
        if ok and want > have:
            if short or head + want - have > len(free_blocks):
                ok, short = False, True
            else:
                tables[r, have:want] = free_blocks[head:head + want - have]
                head += want - have
        failed += not ok
        for i in range(n):
            p = c + i
            if row < num_tokens:
                positions[row] = p + (0 if prefix_lens is None else int(prefix_lens[r]))
                if ok:
                    slots[row] = int(tables[r, p // b]) * b + p % b
                    if r >= num_prefills:
                        suffix[row] = p + 1
                        used = -(-(p + 1) // b)
                        rows_tables[row, :used] = tables[r, :used]
            row += 1
        offsets.append(row)
        kv.append(c + n if ok else c)
    i32 = lambda x: np.asarray(x, dtype=np.int32)  # noqa: E731
    return dict(block_tables=tables, slot_mapping=slots, positions=positions, row_offsets=i32(offsets), kv_lens=i32(kv),
                suffix_lens=suffix, suffix_tables=rows_tables, free_head=i32([head]), num_failed=i32([failed]))
