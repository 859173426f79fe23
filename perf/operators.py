"""Performance cases of the paged cache that holds keys and values in 4 bits: appending tokens, reading them back,
attention over it, and the upkeep of its pages (fork, resize with copy on write, compaction).

The cache.  A pool of pages, uint8 ``[pages, kv_heads, page_size / 16, tile_bytes]``; a tile is 16 consecutive tokens of
one KV head: the key codes (8 D bytes), the value codes (8 D bytes), then scale and zero point of each group of 64 channels
for the keys and for the values (``[16][D / 64][2]`` each, in the activations' type).  An entry stands for
``zero + code * scale``, code 0..15.  Codes lie in the order in which matrix instructions take them (``_places``).
A table says which pages a sequence (row) has: ``pages`` int32 ``[rows, most]`` (-1: none), ``lengths`` int32 ``[rows]``,
``refcounts`` int32 ``[pages]`` (rows that hold the page).

Sizes: heads of the two configurations in ``mega_kernel_qwen36/config.py`` and of their tensor-parallel slices, and a few
generic head layouts.  ``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

GROUP = 64  # channels that share a scale and a zero point
TILE = 16  # tokens of a tile

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ELEM = {"bf16": 2, "f16": 2, "f32": 4}

HEADS = {  # query heads, KV heads, head_dim
    "35b": (16, 2, 256),
    "35b_half": (8, 1, 256),  # one of two tensor-parallel ranks
    "27b": (24, 4, 256),
    "27b_quarter": (6, 1, 256),  # one of four tensor-parallel ranks
    "d128": (32, 8, 128),
    "d64": (8, 8, 64),  # a KV head for every query head
    "d128_one": (16, 1, 128),  # one KV head for all
}


def listed():
    return [
        # the new tokens of a small server's decode step: all latency
        {"name": "append_35b_b8_step", "op": "append", "heads": "35b", "rows": 8, "tokens": 1, "longest": 4000, "page": 64, "dtype": "bf16", "mix": 1},
        # prompts of ragged lengths that join the batch together
        {"name": "append_27b_ragged_prompts", "op": "append", "heads": "27b", "rows": 7, "tokens": 0, "longest": 6000, "page": 32, "dtype": "f16", "mix": 2},
        # one long prompt
        {"name": "append_35b_32k", "op": "append", "heads": "35b", "rows": 1, "tokens": 32768, "longest": 32768, "page": 64, "dtype": "bf16", "mix": 3},
        # one user at the start of a conversation
        {"name": "attention_35b_b1_700", "op": "attention", "heads": "35b", "rows": 1, "tokens": 1, "longest": 700, "ragged": False, "page": 64, "dtype": "bf16", "mix": 4},
        # one user with a long document
        {"name": "attention_35b_b1_32k", "op": "attention", "heads": "35b", "rows": 1, "tokens": 1, "longest": 32768, "ragged": False, "page": 64, "dtype": "bf16", "mix": 5},
        # a batch of conversations of all lengths, each checking a draft of three tokens
        {"name": "attention_27b_b12_draft", "op": "attention", "heads": "27b", "rows": 12, "tokens": 3, "longest": 9001, "ragged": True, "page": 16, "dtype": "f16", "mix": 6},
        # a full server: many long conversations at once
        {"name": "attention_35b_b48_long", "op": "attention", "heads": "35b", "rows": 48, "tokens": 1, "longest": 40000, "ragged": True, "page": 64, "dtype": "bf16", "mix": 7},
        # several answers sampled from each of a few prompts: children share the pages, the first new token copies the last one
        {"name": "branch_35b_4x3", "op": "branch", "heads": "35b", "parents": 4, "fan": 3, "longest": 1500, "page": 64, "dtype": "bf16", "mix": 8},
        {"name": "branch_27b_24x7", "op": "branch", "heads": "27b", "parents": 24, "fan": 7, "longest": 6000, "page": 64, "dtype": "bf16", "mix": 9},
        # between two steps of a busy server: rows end, start, grow by a token, take rejected tokens back
        {"name": "resize_27b_quarter_200", "op": "resize", "heads": "27b_quarter", "rows": 200, "longest": 8000, "page": 64, "dtype": "bf16", "mix": 10},
        # the pool is made dense again, so that its end can be given back
        {"name": "compact_35b_small", "op": "compact", "heads": "35b", "rows": 6, "longest": 2000, "live": 0.6, "page": 64, "dtype": "bf16", "mix": 11},
        {"name": "compact_35b_large", "op": "compact", "heads": "35b", "rows": 64, "longest": 24000, "live": 0.55, "page": 64, "dtype": "bf16", "mix": 12},
    ]


def _log_int(rng, low, high):
    """Whole numbers from low to high, evenly spread over their logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "branch", "resize", "compact"])
    case = {"op": op, "heads": rng.choice(sorted(HEADS)), "page": rng.choice([16, 32, 64, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "mix": rng.randrange(1 << 30)}
    if op == "append":
        rows = _log_int(rng, 1, 64)
        tokens = rng.choice([0, 1, 1, _log_int(rng, 2, max(2, 24000 // rows))])
        case.update(rows=rows, tokens=tokens, longest=max(tokens, _log_int(rng, 20, max(20, 48000 // rows))))
    elif op == "attention":
        rows = _log_int(rng, 1, 48)
        case.update(rows=rows, tokens=rng.choice([1, 1, 1, 2, 3, 4, 8]), longest=_log_int(rng, 3, 300000 // (rows + 5)), ragged=rng.random() < 0.7)
    elif op == "branch":
        case.update(parents=_log_int(rng, 1, 16), fan=_log_int(rng, 1, 8), longest=_log_int(rng, 10, 6000))
    elif op == "resize":
        case.update(rows=_log_int(rng, 1, 200), longest=_log_int(rng, 30, 6000))
    else:
        case.update(rows=_log_int(rng, 1, 48), longest=_log_int(rng, 40, 16000), live=rng.choice([0.3, 0.5, 0.7, 0.9]))
    return case


def _lengths(case, rows, low=1):
    """Lengths of the case's rows, the same for every seed: spread over their logarithm, the longest among them, one row
    empty where there are eight or more."""
    rng = random.Random(case["mix"])
    lengths = [_log_int(rng, min(low, case["longest"]), case["longest"]) for _ in range(rows)]
    lengths[rng.randrange(rows)] = case["longest"]
    if rows >= 8:
        lengths[(lengths.index(case["longest"]) + 1) % rows] = 0
    return lengths


def _tile_bytes(case):
    return HEADS[case["heads"]][2] * (16 + ELEM[case["dtype"]])


def _plan(case):
    """What a server knows on the host: lengths of the rows before and after the call, and what else the operator takes."""
    op = case["op"]
    if op == "append":
        after = _lengths(case, case["rows"])
        counts = [case["tokens"]] * case["rows"]
        if case["tokens"] == 0:  # whole prompts
            counts = list(after)
        after = [max(a, c) for a, c in zip(after, counts)]
        return {"lengths": after, "counts": counts}
    if op == "attention":
        low = max(1, case["longest"] // 20)
        return {"lengths": _lengths(case, case["rows"], low) if case["ragged"] else [case["longest"]] * case["rows"]}
    if op == "branch":
        parents = _lengths(case, case["parents"], max(1, case["longest"] // 10))
        return {"lengths": parents + [0] * (case["parents"] * case["fan"])}
    if op == "resize":
        rng = random.Random(case["mix"] + 1)
        lengths = _lengths(case, case["rows"], max(1, case["longest"] // 20))
        after = []
        for n in lengths:
            what = rng.random()
            if what < 0.06:
                after.append(0)  # an answer that has ended
            elif what < 0.1:
                after.append(max(0, n - rng.randrange(1, 8)))  # rejected tokens of a draft
            elif n == 0 or what < 0.13:
                after.append(_log_int(rng, 1, case["longest"]))  # a prompt that joins
            else:
                after.append(n + 1)
        return {"lengths": lengths, "after": after}
    return {"lengths": _lengths(case, case["rows"], max(1, case["longest"] // 20))}


class _Inputs:
    """Seeded tensors on the GPU.  Keys have a few channels of large mean, as trained models' keys have."""

    def __init__(self, dtype, seed):
        self.dtype, self.gen = dtype, torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *size):
        return torch.empty(size, dtype=torch.float32, device="cuda").normal_(0, 1, generator=self.gen).to(self.dtype)

    def keys(self, *size):
        x = torch.empty(size, dtype=torch.float32, device="cuda").normal_(0, 1, generator=self.gen)
        d = size[-1]
        x[..., 3 :: d // 4] += 4
        return x.to(self.dtype)

    def bytes(self, *size):
        return torch.randint(0, 256, size, dtype=torch.uint8, device="cuda", generator=self.gen)


def prepare(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    page, dtype, plan = case["page"], DTYPES[case["dtype"]], _plan(case)
    make, rng = _Inputs(dtype, seed), random.Random(seed)
    lengths, after = plan["lengths"], plan.get("after", plan["lengths"])
    rows = len(lengths)
    held = [-(-n // page) for n in lengths]
    most = max(-(-max(a, b) // page) for a, b in zip(lengths, after)) + 2
    if case["op"] == "compact":
        total = max(sum(held) + 1, int(sum(held) / case["live"]))
    else:  # room for every row's growth and a copy of its last page
        total = sum(max(h, -(-a // page)) + 2 for h, a in zip(held, after)) + 5
    ids = list(range(total))
    rng.shuffle(ids)  # a pool that has been in use: a row's pages lie anywhere
    table, refcounts, at = np.full((rows, most), -1, np.int32), np.zeros(total, np.int32), 0
    for r, n in enumerate(held):
        table[r, :n] = ids[at : at + n]
        refcounts[table[r, :n]] = 1
        at += n
    if case["op"] == "resize":  # neighbours that share a prompt's first pages, the last of them filled in part
        for r in range(0, rows - 1, 5):
            n = min(held[r], held[r + 1])
            if lengths[r] and lengths[r + 1] and n == held[r + 1]:
                refcounts[table[r + 1, :n]] -= 1
                table[r + 1, :n] = table[r, :n]
                refcounts[table[r + 1, :n]] += 1
    on = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    state = {"op": case["op"], "head_dim": d, "kv_heads": hkv, "page": page, "dtype": dtype, "lengths_host": lengths, "pages": on(table),
             "lengths": on(lengths), "refcounts": on(refcounts), "pool": make.bytes(total, hkv, page // TILE, _tile_bytes(case))}
    if case["op"] == "append":
        counts, n = plan["counts"], sum(plan["counts"])
        shape = (rows, case["tokens"], hkv, d) if case["tokens"] else (n, hkv, d)
        state.update(k=make.keys(*shape), v=make.normal(*shape), counts_host=counts, uniform=case["tokens"] > 0)
        state["cu_tokens"] = on(np.concatenate(([0], np.cumsum(counts))).astype(np.int32))
    elif case["op"] == "attention":
        state["q"] = make.normal(rows, case["tokens"], hq, d) if case["tokens"] > 1 else make.normal(rows, hq, d)
        for r, n in enumerate(lengths):  # the rows' tokens, laid into their pages row by row
            one = {"pool": state["pool"], "head_dim": d, "page": page, "dtype": dtype, "pages": state["pages"][r : r + 1], "lengths_host": [n], "counts_host": [n]}
            if n:
                _store(one, make.keys(n, hkv, d), make.normal(n, hkv, d))
    elif case["op"] == "branch":
        n, fan = case["parents"], case["fan"]
        state["parents"] = on([p for p in range(n) for _ in range(fan)])
        state["children"] = on([n + i for i in range(n * fan)])
    elif case["op"] == "resize":
        state["after"] = on(after)
    return state


# ---- the calls of a user's program ------------------------------------------------------------------------------------


def _package():
    if os.path.abspath("mega-kernel-3.6_b200") not in sys.path:  # the package lies in a folder of its own
        sys.path.insert(0, os.path.abspath("mega-kernel-3.6_b200"))
    import mega_kernel_qwen36 as mk

    return mk


def _run_own(state):
    mk = _package()
    cache = mk.Kv4Cache(state["pool"], state["head_dim"], state["dtype"])
    table = mk.PageTable(state["pages"], state["lengths"], state["refcounts"])
    if state["op"] == "append":
        if state["uniform"]:
            mk.kv4_append(cache, table, state["k"], state["v"])
            return mk.kv4_read(cache, table, state["k"].shape[1])
        mk.kv4_append(cache, table, state["k"], state["v"], cu_tokens=state["cu_tokens"])
        return mk.kv4_read(cache, table, state["k"].shape[0], cu_tokens=state["cu_tokens"])
    if state["op"] == "attention":
        return mk.kv4_attention_decode(state["q"], cache, table)
    if state["op"] == "branch":
        forked, wrong = mk.kv_pages_fork(table, state["parents"], state["children"])
        grown, missing = mk.kv_pages_resize(cache, forked, forked.lengths + 1)
        return grown.pages, grown.lengths, grown.refcounts, wrong, missing, cache.pool
    if state["op"] == "resize":
        grown, missing = mk.kv_pages_resize(cache, table, state["after"])
        return grown.pages, grown.lengths, grown.refcounts, missing, cache.pool
    dense, live = mk.kv_pages_compact(cache, table)
    return dense.pages, dense.lengths, dense.refcounts, live, cache.pool


# ---- the operators in their plain form --------------------------------------------------------------------------------


def _places(d, device):
    """Byte and shift of the code of (token, channel) in a tile's key codes and value codes, ``[16, d]`` each."""
    t = torch.arange(TILE, device=device)[:, None]
    c = torch.arange(d, device=device)[None, :]
    group = c // GROUP
    # keys: four lanes share a token, a lane has 16 channels of each group
    unit = min(16, d // 8)
    lane, i = (c % GROUP) // 16, c % 16
    inside = group * 8 + i // 2
    k_byte = ((t // 8) * (d // 8 // unit) + inside // unit) * (32 * unit) + ((t % 8) * 4 + lane) * unit + inside % unit
    # values: eight lanes share a token, a lane has 8 channels of each group
    unit = d // 16
    lane, i = (c % GROUP) // 8, c % 8
    v_byte = ((t % 2) + 2 * (t // 8)) * (32 * unit) + (lane * 4 + (t % 8) // 2) * unit + group * 4 + i // 2
    return k_byte, v_byte + 8 * d, (4 * (c % 2)).expand(TILE, d).contiguous()


def _quantise(x):
    """codes, scale and zero point of ``[..., d]``: by group of 64, in 64 bits (a code lies next to a border), the scale rounded
    to the type of x and the codes taken with the rounded scale.  A group with an infinity or a NaN stands for NaN."""
    g = x.unflatten(-1, (-1, GROUP)).double()
    low, high = g.amin(-1), g.amax(-1)
    fine = torch.isfinite(g).all(-1)
    nan = torch.full_like(low, math.nan)
    scale = torch.where(fine, (high - low) / 15, nan).to(x.dtype)
    zero = torch.where(fine, low, nan).to(x.dtype)
    step = scale.double()[..., None]
    code = torch.where(step > 0, (g - zero.double()[..., None]) / step, torch.zeros_like(g)).round().clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), scale, zero


def _token_places(state):
    """Byte offset of the tile and place in it of the last ``counts`` tokens of every row, ``[tokens]`` each."""
    pool, page = state["pool"], state["page"]
    dev = pool.device
    rows = torch.repeat_interleave(torch.arange(len(state["counts_host"]), device=dev), torch.tensor(state["counts_host"], device=dev))
    position = torch.cat([torch.arange(n - c, n, device=dev) for n, c in zip(state["lengths_host"], state["counts_host"])])
    pid = state["pages"][rows, position // page].long()
    return pid * pool.stride(0) + (position % page) // TILE * pool.stride(2), position % TILE


def _store(state, k, v):
    """Writes k and v ``[tokens, heads, d]`` as the last tokens of their rows."""
    pool, d = state["pool"], state["head_dim"]
    k_byte, v_byte, _ = _places(d, pool.device)
    base, t = _token_places(state)
    base = base[:, None] + torch.arange(k.shape[1], device=pool.device) * pool.stride(1)
    flat, params = pool.view(-1), pool.view(-1).view(k.dtype)
    for x, byte, first in ((k, k_byte, 16 * d), (v, v_byte, 16 * d + d * k.element_size() // 2)):
        code, scale, zero = _quantise(x)
        flat[base[..., None] + byte[t][:, None, 0::2]] = code[..., 0::2] | (code[..., 1::2] << 4)
        at = (base[..., None] + first) // k.element_size() + (t[:, None, None] * (d // GROUP) + torch.arange(d // GROUP, device=pool.device)) * 2
        params[at], params[at + 1] = scale, zero


def _tiles_of(tiles, d, dtype):
    """Keys and values of tiles ``[n, tile_bytes]`` as ``[n, 16, d]`` in 32 bits."""
    k_byte, v_byte, shift = _places(d, tiles.device)
    n, g = tiles.shape[0], d // GROUP
    params = tiles[:, 16 * d :].contiguous().view(dtype).view(n, 2, TILE, g, 2).float()
    out = []
    for i, byte in enumerate((k_byte, v_byte)):
        code = ((tiles[:, byte] >> shift.to(torch.uint8)) & 15).float()
        scale, zero = params[:, i, :, :, :1], params[:, i, :, :, 1:]
        out.append((code.unflatten(-1, (g, GROUP)) * scale + zero).flatten(-2))
    return out


def _load_row(state, r, length):
    """Keys and values of a row's first tokens, ``[heads, length, d]`` in 32 bits."""
    n, per = -(-length // TILE), state["page"] // TILE
    index = torch.arange(n, device=state["pool"].device)
    tiles = state["pool"][state["pages"][r].long()[index // per], :, index % per].transpose(0, 1)
    k, v = _tiles_of(tiles.reshape(n * state["kv_heads"], -1), state["head_dim"], state["dtype"])
    return [x.view(state["kv_heads"], n * TILE, -1)[:, :length] for x in (k, v)]


def _append(state):
    d, hkv = state["head_dim"], state["kv_heads"]
    _store(state, state["k"].reshape(-1, hkv, d), state["v"].reshape(-1, hkv, d))
    base, t = _token_places(state)
    order = torch.arange(len(t), device=t.device)
    found = []
    for h in range(hkv):
        tiles = torch.as_strided(state["pool"], (state["pool"].numel() // state["pool"].stride(2), state["pool"].stride(2)), (state["pool"].stride(2), 1))
        some = []
        for part in order.split(4096):
            k, v = _tiles_of(tiles[(base[part] + h * state["pool"].stride(1)) // state["pool"].stride(2)], d, state["dtype"])
            pick = torch.arange(len(part), device=t.device)
            some.append((k[pick, t[part]], v[pick, t[part]]))
        found.append([torch.cat(x) for x in zip(*some)])
    return tuple(torch.stack(x, 1).to(state["dtype"]).view(state["k"].shape) for x in zip(*found))


def _attention(state):
    q = state["q"] if state["q"].ndim == 4 else state["q"][:, None]
    rows, tokens, hq, d = q.shape
    hkv, out = state["kv_heads"], torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    ahead = torch.arange(tokens, device=q.device)
    for r, n in enumerate(state["lengths_host"]):
        if n == 0:
            continue
        k, v = _load_row(state, r, n)
        x = q[r].float().view(tokens, hkv, hq // hkv, d).permute(1, 2, 0, 3)  # [heads, group, tokens, d]
        s = torch.matmul(x, k.transpose(-1, -2)[:, None]) / math.sqrt(d)
        seen = torch.arange(n, device=q.device) <= n - tokens + ahead[:, None]
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        o = torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True).clamp_min(1e-38)
        out[r] = o.permute(2, 0, 1, 3).reshape(tokens, hq, d)
    return out.to(q.dtype).view(state["q"].shape)


def _fork(pages, lengths, refcounts, parents, children):
    new_pages, new_lengths, new_refs = pages.clone(), lengths.clone(), refcounts.clone()
    new_pages[children.long()] = pages[parents.long()]
    new_lengths[children.long()] = lengths[parents.long()]
    taken = pages[parents.long()].flatten()
    new_refs.index_add_(0, taken.clamp_min(0).long(), (taken >= 0).int())
    return new_pages, new_lengths, new_refs


def _resize(pool, page, pages, lengths, refcounts, after):
    slot = torch.arange(pages.shape[1], device=pages.device)[None, :]
    old, new = (lengths + page - 1) // page, (after + page - 1) // page
    refs = refcounts.clone()
    gone = (slot < old[:, None]) & (slot >= new[:, None])
    refs.index_add_(0, pages.clamp_min(0).flatten().long(), -gone.flatten().int())
    tail = pages.gather(1, (old - 1).clamp_min(0).long()[:, None])[:, 0].clamp_min(0).long()
    copy = (after > lengths) & (lengths % page != 0) & (refs[tail] > 1)
    need = (new - old).clamp_min(0) + copy.int()
    first = (torch.cumsum(need, 0) - need).long()
    total = need.sum()
    free = refs == 0
    free_ids = torch.sort((~free).int(), stable=True).indices.int()
    fresh = (slot >= old[:, None]) & (slot < new[:, None])
    taken = free_ids[((first + copy)[:, None] + slot - old[:, None]).clamp(0, len(free_ids) - 1)]
    out = torch.where(gone, torch.full_like(pages, -1), torch.where(fresh, taken, pages))
    copied = copy[:, None] & (slot == old[:, None] - 1)
    out = torch.where(copied, free_ids[first.clamp_max(len(free_ids) - 1)][:, None], out)
    refs.index_add_(0, tail, -copy.int())
    refs = torch.where(free & (torch.cumsum(free.int(), 0) <= total), torch.ones_like(refs), refs)
    rows = torch.nonzero(copy)[:, 0]
    tiles = (lengths[rows] % page + TILE - 1) // TILE
    which, tile = torch.nonzero(torch.arange(page // TILE, device=pages.device) < tiles[:, None], as_tuple=True)
    source, target = tail[rows[which]], free_ids[first[rows[which]]].long()
    pool[target, :, tile] = pool[source, :, tile]
    return out, after.clone(), refs, (total - free.sum()).clamp_min(0).int().view(1)


def _compact(pool, pages, lengths, refcounts):
    live = refcounts > 0
    n = live.sum()
    index = torch.arange(len(live), device=live.device)
    source = torch.nonzero(live & (index >= n))[:, 0]
    target = torch.nonzero(~live & (index < n))[:, 0]
    moved = index.int()
    moved[source] = target.int()
    pool[target] = pool[source]
    refs = refcounts.clone()
    refs[target] = refcounts[source]
    refs[source] = 0
    return torch.where(pages >= 0, moved[pages.clamp_min(0).long()], pages), lengths.clone(), refs, n.int().view(1)


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "append":
        return _append(state)
    if state["op"] == "attention":
        return _attention(state)
    pool, table = state["pool"], (state["pages"], state["lengths"], state["refcounts"])
    if state["op"] == "branch":
        forked = _fork(*table, state["parents"], state["children"])
        grown = _resize(pool, state["page"], *forked, forked[1] + 1)
        return *grown[:3], torch.zeros(1, dtype=torch.int32, device=pool.device), grown[3], pool
    if state["op"] == "resize":
        return *_resize(pool, state["page"], *table, state["after"]), pool
    return *_compact(pool, *table), pool


def work(case):
    """What a pass cannot do without.  A token of the cache has tile_bytes / 16 bytes in each head."""
    hq, hkv, d = HEADS[case["heads"]]
    plan, page = _plan(case), case["page"]
    elem, token = ELEM[case["dtype"]], hkv * _tile_bytes(case) / TILE
    lengths, rows = plan["lengths"], len(plan["lengths"])
    entries = sum(-(-n // page) for n in lengths)
    if case["op"] == "append":  # read the tokens, write them, read them again, give them back
        n = sum(plan["counts"])
        return {"bytes": n * (4 * hkv * d * elem + 2 * token) + 8 * rows, "flops": 10 * n * 2 * hkv * d}
    if case["op"] == "attention":
        tokens, n = case["tokens"], sum(lengths)
        seen = sum(max(0, m - tokens + i + 1) for m in lengths for i in range(tokens))
        return {"bytes": n * token + 2 * rows * tokens * hq * d * elem + 4 * (entries + rows), "flops": 4 * d * hq * seen}
    page_bytes = page // TILE * hkv * _tile_bytes(case)
    if case["op"] == "branch":  # each row but an empty one or one of whole pages gets its last tiles copied; tables are read and written
        most = max(-(-n // page) for n in lengths) + 2
        copied = sum((case["fan"] + 1) * -(-(n % page) // TILE) for n in lengths[: case["parents"]])
        total = sum(-(-n // page) + 2 for n in lengths) + 5
        return {"bytes": 2 * copied * TILE * token + 8 * rows * (most + 1) + 8 * total, "flops": 0}
    if case["op"] == "resize":
        most = max(-(-max(a, b) // page) for a, b in zip(lengths, plan["after"])) + 2
        total = sum(max(-(-a // page), -(-b // page)) + 2 for a, b in zip(lengths, plan["after"])) + 5
        return {"bytes": 8 * rows * most + 12 * rows + 8 * total, "flops": 0}
    total = max(entries + 1, int(entries / case["live"]))
    moved = entries * (total - entries) / total  # live pages behind the first `entries`, on average
    return {"bytes": 2 * moved * page_bytes + 8 * entries + 8 * total, "flops": 0}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def _entry_order(d):
    """For each half byte of a tile's codes, low one first: token and channel, for keys and for values."""
    keys, values = {}, {}
    for token in range(16):
        for channel in range(d):
            g, c = divmod(channel, 64)
            vector = 16 if d >= 128 else 8
            byte = 8 * g + (c % 16) // 2
            keys[2 * ((token // 8 * (d // (8 * vector)) + byte // vector) * 32 * vector + (4 * (token % 8) + c // 16) * vector + byte % vector) + c % 2] = (token, channel)
            vector = d // 16
            quarter = {(0, 0): 0, (0, 1): 1, (1, 0): 2, (1, 1): 3}[token // 8, token % 2]
            values[2 * (quarter * 32 * vector + (4 * (c // 8) + token % 8 // 2) * vector + 4 * g + (c % 8) // 2) + c % 2] = (token, channel)
    return [torch.tensor([t[0] * d + t[1] for _, t in sorted(m.items())], device="cuda") for m in (keys, values)]


def _exact_rows(state):
    """Yields each row's keys and values ``[length, heads, d]`` in 64 bits."""
    d, heads, pool = state["head_dim"], state["kv_heads"], state["pool"]
    orders = _entry_order(d)
    for r, n in enumerate(state["lengths_host"]):
        if n == 0:
            yield None, None
            continue
        some = pool[state["pages"][r, : -(-n // state["page"])].long()].permute(1, 0, 2, 3).flatten(1, 2)  # [heads, tiles, bytes]
        parts = []
        for i in range(2):
            raw = some[..., 8 * d * i : 8 * d * (i + 1)]
            halves = torch.stack((raw % 16, raw // 16), -1).flatten(-2).double()
            entries = torch.empty_like(halves)
            entries[..., orders[i]] = halves
            size = (some.shape[-1] - 16 * d) // 2
            p = some[..., 16 * d + size * i : 16 * d + size * (i + 1)].contiguous().view(state["dtype"]).double().view(heads, -1, d // 64, 2)
            x = entries.view(heads, -1, d // 64, 64)
            parts.append((p[..., 1:] + x * p[..., :1]).flatten(-2)[:, :n].transpose(0, 1))
        yield parts


def _exact_rounded(x):
    """What the cache holds for x ``[..., d]``, as the values it stands for."""
    shape, dtype = x.shape, x.dtype
    out = []
    for part in x.reshape(-1, 64).split(1 << 20):
        part = part.double()
        bottom = part.min(1, keepdim=True).values
        step = ((part.max(1, keepdim=True).values - bottom) / 15.0).to(dtype).double()
        code = torch.floor((part - bottom) / step)
        left = (part - bottom) - (code + 0.5) * step  # whether to go up; halves go to the even one
        code = code + ((left > 0) | ((left == 0) & (code % 2 == 1)))
        out.append(bottom + step * torch.where(step > 0, code.clamp(0, 15), 0.0))
    return torch.cat(out).view(shape)


def _exact_pages(state):
    """The page operators step by step on the host."""
    pages, lengths, refs = (state[n].cpu().tolist() for n in ("pages", "lengths", "refcounts"))
    pool, page = state["pool"].clone(), state["page"]
    if state["op"] == "compact":
        n, moves = sum(1 for c in refs if c > 0), {}
        holes = [p for p in range(n) if refs[p] == 0]
        for p in range(n, len(refs)):
            if refs[p] > 0:
                moves[p] = holes.pop(0)
        for a, b in moves.items():
            refs[b], refs[a] = refs[a], 0
        if moves:
            pool[list(moves.values())] = pool[list(moves)]
        return [[moves.get(p, p) for p in row] for row in pages], lengths, refs, [n], pool
    if state["op"] == "branch":
        for a, b in zip(state["parents"].tolist(), state["children"].tolist()):
            pages[b], lengths[b] = list(pages[a]), lengths[a]
            for p in pages[b]:
                if p >= 0:
                    refs[p] += 1
        after = [n + 1 for n in lengths]
    else:
        after = state["after"].tolist()
    for r, (n, m) in enumerate(zip(lengths, after)):
        for i in range(-(-m // page), -(-n // page)):
            refs[pages[r][i]] -= 1
            pages[r][i] = -1
    shared = [m > n and n % page != 0 and refs[pages[r][n // page]] > 1 for r, (n, m) in enumerate(zip(lengths, after))]
    free = iter([p for p, c in enumerate(refs) if c == 0])
    for r, (n, m) in enumerate(zip(lengths, after)):
        if shared[r]:
            i = n // page
            p = next(free)
            tiles = -(-(n % page) // 16)
            pool[p, :, :tiles] = pool[pages[r][i], :, :tiles]
            refs[pages[r][i]] -= 1
            refs[p], pages[r][i] = 1, p
        for i in range(-(-n // page), -(-m // page)):
            pages[r][i] = next(free)
            refs[pages[r][i]] = 1
    if state["op"] == "branch":
        return pages, after, refs, [0], [0], pool
    return pages, after, refs, [0], pool


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_rounded(state["k"]), _exact_rounded(state["v"])
    if case["op"] != "attention":
        return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") if isinstance(x, list) else x for x in _exact_pages(state))
    q = state["q"].double().view(len(state["lengths_host"]), -1, *state["q"].shape[-2:])
    out, each = torch.zeros_like(q), q.shape[2] // state["kv_heads"]
    for r, (keys, values) in enumerate(_exact_rows(state)):
        if keys is None:
            continue
        for i in range(q.shape[1]):
            n = keys.shape[0] - q.shape[1] + i + 1
            for h in range(state["kv_heads"]) if n > 0 else ():
                weight = torch.softmax(q[r, i, h * each : (h + 1) * each] @ keys[:n, h].T * state["head_dim"] ** -0.5, -1)
                out[r, i, h * each : (h + 1) * each] = weight @ values[:n, h]
    return out.view(state["q"].shape)
