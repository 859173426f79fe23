"""CPU statement of the 4-bit paged cache and its operators in 64 bits; test infrastructure only.

No reference implementation exists for these operators (the reference plans a ``paged_attention`` task and leaves it to the
caller), so this states their definition, step by step and without regard to speed:

  group of 64 channels x: zero = min x, scale = round_T((max x - min x) / 15), code = round_half_even((x - zero) / scale) in
  0..15 (0 where the scale is 0); a group with an infinity or a NaN has NaN for both.  An entry stands for zero + code * scale.

Tables are plain lists, pools numpy arrays of bytes.
"""

import math
from fractions import Fraction

import numpy as np
import torch

TILE, GROUP = 16, 64


def tile_bytes(d, dtype):
    return d * (16 + dtype.itemsize)


def key_place(d, t, c):
    """(byte, low or high half) of the key code of token t, channel c in a tile."""
    u = min(16, d // 8)
    b = c // 64 * 8 + (c % 16) // 8 * 4
    word = ((t // 8) * (d // 8 // u) + b // u) * 32 * u + ((t % 8) * 4 + (c % 64) // 16) * u + b % u
    return word + c % 8 // 2, c % 2


def value_place(d, t, c):
    word = 8 * d + (t % 2 + 2 * (t // 8)) * 2 * d + ((c % 64) // 8 * 4 + (t % 8) // 2) * (d // 16) + c // 64 * 4
    return word + c % 8 // 2, c % 2


_PLACES = {}


def places(d):
    if d not in _PLACES:
        found = []
        for place in (key_place, value_place):
            both = [[place(d, t, c) for c in range(d)] for t in range(TILE)]
            found.append((np.array([[b for b, _ in row] for row in both]), np.array([[4 * h for _, h in row] for row in both])))
        _PLACES[d] = found
    return _PLACES[d]


def quantise(x):
    """x torch ``[..., d]`` -> codes uint8 ``[..., d]``, scale and zero ``[..., d / 64]`` in x's type."""
    g = x.reshape(-1, GROUP)
    wide = g.double()
    fine = torch.isfinite(wide).all(1)
    low, high = wide.amin(1), wide.amax(1)
    nan = torch.full_like(low, math.nan)
    scale, zero = torch.where(fine, (high - low) / 15, nan).to(x.dtype), torch.where(fine, low, nan).to(x.dtype) + 0.0
    step = scale.double()[:, None]
    n = torch.floor((wide - zero.double()[:, None]) / step)
    rest = (wide - zero.double()[:, None]) - (n + 0.5) * step
    n = n + ((rest > 0) | ((rest == 0) & (n % 2 == 1)))
    code = torch.where(step > 0, n, torch.zeros_like(n)).nan_to_num(0.0).clamp(0, 15).to(torch.uint8)
    return code.view(x.shape), scale.view(*x.shape[:-1], -1), zero.view(*x.shape[:-1], -1)


def quantise_by_fractions(values, to_type):
    """One group in exact arithmetic: codes, scale, zero.  ``to_type`` rounds a Fraction to the storage type."""
    x = [Fraction(v) for v in values]
    zero, scale = min(x), to_type((max(x) - min(x)) / 15)
    return [min(15, round((v - zero) / scale)) if scale else 0 for v in x], scale, zero


def _param_bytes(t):
    return np.frombuffer(t.contiguous().view(torch.uint8).numpy().tobytes(), np.uint8)


def write(pool, page, head, position, page_size, k, v):
    """One token of one head, k and v ``[d]``, into the pool (numpy uint8, modified)."""
    d = k.shape[0]
    tile = pool[page, head, position % page_size // TILE]
    t, elem = position % TILE, k.dtype.itemsize
    for i, x in enumerate((k, v)):
        code, scale, zero = quantise(x)
        byte, shift = places(d)[i]
        for b in np.unique(byte[t]):
            tile[b] = 0
        np.bitwise_or.at(tile, byte[t], (code.numpy() << shift[t]).astype(np.uint8))
        first = 16 * d + i * (d * elem // 2) + t * (d // GROUP) * 2 * elem
        tile[first : first + d // GROUP * 2 * elem] = _param_bytes(torch.stack((scale, zero), -1))


def read_tiles(tiles, d, dtype):
    """Tiles numpy ``[n, tile_bytes]`` -> keys and values ``[n * 16, d]`` in 64 bits."""
    out = []
    for i in range(2):
        byte, shift = places(d)[i]
        code = torch.from_numpy((tiles[:, byte] >> shift) & 15).double().reshape(-1, d // GROUP, GROUP)
        size = d * dtype.itemsize // 2
        first = 16 * d + i * size
        param = torch.from_numpy(tiles[:, first : first + size].copy()).view(dtype).double().reshape(-1, d // GROUP, 2)
        out.append((param[..., 1:] + code * param[..., :1]).reshape(-1, d))
    return out


def row_entries(pool, pages, length, head, d, dtype):
    """Keys and values of a row's tokens for one head, ``[length, d]`` each in 64 bits."""
    page_size = pool.shape[2] * TILE
    n = -(-length // TILE)
    tiles = np.stack([pool[pages[i * TILE // page_size], head, i % (page_size // TILE)] for i in range(n)]) if n else np.zeros((0, pool.shape[3]), np.uint8)
    k, v = read_tiles(tiles, d, dtype)
    return k[:length], v[:length]


def append(pool, table, lengths, k, v, counts):
    """k, v ``[tokens, heads, d]``: the last counts[r] tokens of every row r."""
    page_size, at = pool.shape[2] * TILE, 0
    for r, n in enumerate(counts):
        for i in range(n):
            position = lengths[r] - n + i
            if position >= 0 and 0 <= table[r][position // page_size] < pool.shape[0]:
                for h in range(k.shape[1]):
                    write(pool, table[r][position // page_size], h, position, page_size, k[at + i, h], v[at + i, h])
        at += n


def attention(q, pool, table, lengths, dtype, scale):
    """q ``[rows, tokens, heads, d]`` -> the same in 64 bits, and a bound on what fp32 arithmetic may be off by: for each query the
    largest sum of |terms| of a score and the largest entry's terms of the values (``[rows, tokens, heads]`` each)."""
    rows, tokens, hq, d = q.shape
    kv = pool.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    score_size, value_size = torch.zeros(rows, tokens, hq, dtype=torch.float64), torch.zeros(rows, tokens, hq, dtype=torch.float64)
    for r in range(rows):
        if lengths[r] == 0:
            continue
        for g in range(kv):
            k, v = row_entries(pool, table[r], lengths[r], g, d, dtype)
            k_size, v_size = _sizes(pool, table[r], lengths[r], g, d, dtype)
            for i in range(tokens):
                seen = lengths[r] - tokens + i + 1
                if seen <= 0:
                    continue
                for h in range(g * (hq // kv), (g + 1) * (hq // kv)):
                    x = q[r, i, h].double()
                    out[r, i, h] = torch.softmax(scale * (k[:seen] @ x), 0) @ v[:seen]
                    score_size[r, i, h] = abs(scale) * (k_size[:seen] @ x.abs()).max()
                    value_size[r, i, h] = v_size[:seen].max()
    return out, score_size, value_size


def _sizes(pool, pages, length, head, d, dtype):
    """|zero| + 15 scale of every entry: what the terms of a sum over entries may be as large as."""
    page_size = pool.shape[2] * TILE
    n = -(-length // TILE)
    tiles = np.stack([pool[pages[i * TILE // page_size], head, i % (page_size // TILE)] for i in range(n)])
    out = []
    for i in range(2):
        size = d * dtype.itemsize // 2
        first = 16 * d + i * size
        param = torch.from_numpy(tiles[:, first : first + size].copy()).view(dtype).double().reshape(-1, d // GROUP, 2)
        out.append((param[..., 1].abs() + 15 * param[..., 0]).repeat_interleave(GROUP, -1)[:length])
    return out


# ---- tables -------------------------------------------------------------------------------------------------------------


def fork(table, lengths, refs, parents, children):
    rows = len(table)
    pairs = [(a, b) for a, b in zip(parents, children) if a >= 0 and b >= 0]
    kids = [b for _, b in pairs]
    if any(a >= rows or b >= rows or lengths[b] != 0 for a, b in pairs) or len(set(kids)) != len(kids):
        return [list(r) for r in table], list(lengths), list(refs), -1
    new, new_len, new_refs = [list(r) for r in table], list(lengths), list(refs)
    for a, b in pairs:
        if a in kids:
            continue
        new[b], new_len[b] = list(table[a]), lengths[a]
        for p in table[a]:
            if 0 <= p < len(refs):
                new_refs[p] += 1
    return new, new_len, new_refs, 0


def resize(pool, table, lengths, refs, after):
    """Modifies the pool (numpy) where pages are copied."""
    same = [list(r) for r in table], list(lengths), list(refs)
    page_size, width = pool.shape[2] * TILE, len(table[0])
    count = lambda n: -(-n // page_size)
    if any(n < 0 or n > width * page_size for n in list(lengths) + list(after)):
        return (*same, -1)
    table, refs = [list(r) for r in table], list(refs)
    for r, (n, m) in enumerate(zip(lengths, after)):
        for i in range(count(m), count(n)):
            if not 0 <= table[r][i] < len(refs):
                return (*same, -1)
            refs[table[r][i]] -= 1
            table[r][i] = -1
    shared = []
    for r, (n, m) in enumerate(zip(lengths, after)):
        partial = m > n and n % page_size != 0
        if partial and not 0 <= table[r][count(n) - 1] < len(refs):
            return (*same, -1)
        shared.append(partial and refs[table[r][count(n) - 1]] > 1)
    need = sum(max(0, count(m) - count(n)) + s for n, m, s in zip(lengths, after, shared))
    free = [p for p, c in enumerate(refs) if c == 0]
    if need > len(free):
        return (*same, need - len(free))
    taken = iter(free)
    for r, (n, m) in enumerate(zip(lengths, after)):
        if shared[r]:
            old, new = table[r][count(n) - 1], next(taken)
            tiles = -(-(n % page_size) // TILE)
            pool[new, :, :tiles] = pool[old, :, :tiles]
            refs[old] -= 1
            refs[new] = 1
            table[r][count(n) - 1] = new
        for i in range(count(n), count(m)):
            table[r][i] = next(taken)
            refs[table[r][i]] = 1
    return table, list(after), refs, 0


def compact(pool, table, lengths, refs):
    n = sum(c > 0 for c in refs)
    holes = [p for p in range(n) if refs[p] <= 0]
    movers = [p for p in range(n, len(refs)) if refs[p] > 0]
    name, refs = dict(zip(movers, holes)), list(refs)
    for old, new in name.items():
        pool[new] = pool[old]
        refs[new], refs[old] = refs[old], 0
    refs[n:] = [0] * (len(refs) - n)
    return [[name.get(p, p) for p in row] for row in table], list(lengths), refs, n
