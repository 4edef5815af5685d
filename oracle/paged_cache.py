"""A paged cache of e4m3 codes with a scale for each block and kv head, and what is appended to it, in 64 bits (test
infrastructure; see the package docstring).  Token by token and block by block, as the definition reads.
"""
import math

import torch

from .rotary import turn

E4M3_MAX = 448.0


def round_e4m3(x):
    """float64 -> the nearest e4m3 numbers, ties to the even mantissa: eight steps to a power of two, the least power 2^-6."""
    exponent = torch.frexp(x)[1].double() - 1
    step = torch.exp2(exponent.clamp(min=-6.0) - 3)
    return torch.round(x / step) * step


def least_scale(peak):
    """The least power of two (2^-118 .. 2^120) with peak / scale <= 448."""
    if peak == 0:
        return 2.0 ** -118
    e = math.ceil(math.log2(peak / E4M3_MAX))
    if peak <= E4M3_MAX * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** min(max(e, -118), 120)


def places(context_lens, query_starts, num_rows, block_tables, block_size, num_blocks, table_rows=None):
    """[(row, sequence, position, block, slot)] of the rows that have a place."""
    found = []
    for s, n in enumerate(context_lens.tolist()):
        begin, end = (s, s + 1) if query_starts is None else query_starts[s:s + 2].tolist()
        for row in range(begin, min(end, num_rows)):
            position = n - (end - row)
            if position < 0 or position >= block_tables.shape[1] * block_size or (table_rows is not None and position >= table_rows):
                continue
            block = int(block_tables[s, position // block_size])
            if 0 <= block < num_blocks:
                found.append((row, s, position, block, position % block_size))
    return found


def append(x, cache, scales, found, cos=None, sin=None, interleaved=False):
    """x (rows, heads, D), cache (blocks, heads, block size, D) and scales (blocks, heads) or None -> (cache, scales) in
    float64 after the rows of ``places`` are stored, unrounded in a cache without scales."""
    cache, scales = cache.double().clone(), None if scales is None else scales.double().clone()
    x = x.double()
    new = {}
    for row, s, position, block, slot in found:
        v = x[row]
        if cos is not None:
            v = turn(v, cos[position].double(), sin[position].double(), interleaved)
        new.setdefault((s, block), []).append((slot, v))
    for (s, block), tokens in new.items():
        if scales is None:
            for slot, v in tokens:
                cache[block, :, slot] = v
            continue
        first = min(slot for slot, _ in tokens)
        for h in range(x.shape[1]):
            finite = [v[h][v[h].isfinite()].abs() for _, v in tokens]
            needed = least_scale(max((f.max().item() if f.numel() else 0.0) for f in finite))
            if first > 0 and needed > scales[block, h]:
                cache[block, h, :first] = round_e4m3(cache[block, h, :first] * (scales[block, h] / needed))
            scales[block, h] = max(needed, scales[block, h].item()) if first > 0 else needed
            for slot, v in tokens:
                cache[block, h, slot] = torch.where(v[h].isfinite(), round_e4m3(v[h] / scales[block, h]), torch.nan)
    return cache, scales


def attention_fp8(query, key_cache, value_cache, key_scales, value_scales, context_lens, block_tables, scale):
    """-> (out, spread, reach) in float64: the result, the same sum over |values|, and the largest sum of |products| behind a
    score of the row (what rounding errors are measured by).  Entries outside the cache make their rows NaN."""
    num_seqs, Hq, D = query.shape
    num_blocks, Hkv, block, _ = key_cache.shape
    out = torch.zeros(query.shape, dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros(num_seqs, Hq, 1, dtype=torch.float64)
    q = query.double().cpu()
    kc, vc = (c.double().cpu() * s.double().cpu()[:, :, None, None] for c, s in ((key_cache, key_scales), (value_cache, value_scales)))
    for s, n in enumerate(context_lens.tolist()):
        if n <= 0:
            continue
        columns = -(-n // block)
        ids = block_tables[s, :columns].cpu().long()
        if columns > block_tables.shape[1] or bool(((ids < 0) | (ids >= num_blocks)).any()):
            out[s] = torch.nan
            continue
        for h in range(Hkv):
            k, v = (c[ids, h].reshape(-1, D)[:n] for c in (kc, vc))
            rows = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            p = torch.softmax(q[s, rows] @ k.T * scale, -1)
            out[s, rows], spread[s, rows] = p @ v, p @ v.abs()
            reach[s, rows] = (q[s, rows].abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True)
    return out, spread, reach
