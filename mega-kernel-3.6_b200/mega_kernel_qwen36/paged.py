"""A paged KV cache held in 4 bits: append, read, decode attention, and the upkeep of its pages.

The reference plans a ``paged_attention`` task (mpk_graph.py:352-398) and leaves it to the caller; its attention operator
takes dense caches of one length (reference.py:117-145).  Here sequences of different lengths share a pool of pages, and
keys and values take 4 bits each plus a scale and a zero point for every 64 channels: a token takes 288 bytes for a KV head
of 256 channels, keys and values together, instead of 1024 in bfloat16.

A serving step with it::

    table, missing = kv_pages_resize(cache, table, table.lengths + 1)      # room for the new tokens
    kv4_append(cache, table, k_new, v_new)                                 # [rows, 1, kv_heads, head_dim]
    out = kv4_attention_decode(q, cache, table)                            # [rows, query_heads, head_dim]

All tables live on the GPU and no call waits for the host, so steps can be captured into CUDA graphs; a captured call
follows what the tables hold at replay.

Layers that share a table have a pool each.  ``kv_pages_resize`` and ``kv_pages_compact`` copy and move the pages of the pool that they
are given, by the table as it was before: call them for every layer with that same table, each call gives the same new one, and only
the last may be in place.  A layer that gets the new table instead has no pages copied, and nothing says so.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .ops import _native

KV4_TILE = 16  # tokens of a tile
KV4_GROUP = 64  # channels that share a scale and a zero point


@dataclass(frozen=True)
class Kv4Cache:
    """Pool of pages, uint8 ``[pages, kv_heads, page_size / 16, tile_bytes]`` (``kv4_pool`` makes one).

    A tile is 16 consecutive tokens of one KV head: codes of the keys and of the values (``8 * head_dim`` bytes each, in
    the order in which tensor-core instructions take them), then scale and zero point of every group of 64 channels for keys and
    for values, in ``dtype``.  An entry stands for ``zero + code * scale``.  ``dtype`` is that of the keys and values that
    are appended, of the queries and of everything that is read: bfloat16, float16 or float32; head_dim is 64, 128 or 256."""

    pool: torch.Tensor
    head_dim: int
    dtype: torch.dtype = torch.bfloat16

    @property
    def page_size(self) -> int:
        return self.pool.shape[2] * KV4_TILE


@dataclass(frozen=True)
class PageTable:
    """Which pages the rows (sequences) hold: ``pages`` int32 ``[rows, row_pages]`` (-1 where a row has none), ``lengths`` int32
    ``[rows]``, ``refcounts`` int32 ``[pages of the pool]``: how many rows hold a page; a page with 0 is free."""

    pages: torch.Tensor
    lengths: torch.Tensor
    refcounts: torch.Tensor


def kv4_pool(pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda") -> Kv4Cache:
    """A cache with an empty pool.  page_size is a multiple of 16."""
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("dtype must be bfloat16, float16 or float32")
    if head_dim not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    if page_size <= 0 or page_size % KV4_TILE != 0:
        raise ValueError("page_size must be a multiple of 16")
    if pages <= 0 or kv_heads <= 0:
        raise ValueError("pages and kv_heads must be positive")
    tile_bytes = head_dim * (16 + dtype.itemsize)
    return Kv4Cache(torch.zeros(pages, kv_heads, page_size // KV4_TILE, tile_bytes, dtype=torch.uint8, device=device), head_dim, dtype)


def empty_page_table(rows: int, row_pages: int, cache: Kv4Cache) -> PageTable:
    """A table of rows without tokens for the cache's pool."""
    device = cache.pool.device
    return PageTable(torch.full((rows, row_pages), -1, dtype=torch.int32, device=device), torch.zeros(rows, dtype=torch.int32, device=device),
                     torch.zeros(cache.pool.shape[0], dtype=torch.int32, device=device))


def _check_dtype(cache: Kv4Cache, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != cache.dtype:
            raise ValueError(f"the cache holds {cache.dtype}, got a tensor of {t.dtype}")


def kv4_append(cache: Kv4Cache, table: PageTable, k: torch.Tensor, v: torch.Tensor, *, cu_tokens: Optional[torch.Tensor] = None) -> None:
    """Quantises keys and values into the cache, as the LAST tokens of their rows: ``table.lengths`` already count them.

    k, v ``[rows, tokens, kv_heads, head_dim]``, or with ``cu_tokens`` (int32 ``[rows + 1]``, ascending from 0) ``[tokens,
    kv_heads, head_dim]``, row r having tokens ``cu_tokens[r]`` to ``cu_tokens[r + 1] - 1``; tokens behind the last row's are
    padding.  Only the channels need to be contiguous.  Of a group of 64 channels the zero point is the least value, the scale
    ``(greatest - least) / 15`` rounded to the cache's type, and a code ``(value - zero) / scale`` rounded to the nearest (halves to
    even), at most 15; float32 takes the difference in 64 bits.  A group with an infinity or a NaN stands for NaN.  A token without a page (-1) is not written.  Pages that
    are written must not be shared: ``kv_pages_resize`` sees to that."""
    ext = _native("kv4_append", cache.pool, table.pages, table.lengths, k, v)
    _check_dtype(cache, k, v)
    ext.kv4_append(cache.pool, table.pages, table.lengths, int(cache.head_dim), k, v, cu_tokens)


def kv4_read(
    cache: Kv4Cache,
    table: PageTable,
    tokens: int,
    *,
    cu_tokens: Optional[torch.Tensor] = None,
    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The last ``tokens`` tokens of every row as dense keys and values ``[rows, tokens, kv_heads, head_dim]``; with
    ``cu_tokens`` (as in ``kv4_append``) ``[tokens, kv_heads, head_dim]``, ``tokens`` being the number for all rows.  ``out``: a
    pair of tensors to write to, without elements that share memory; what lies behind the last row's tokens is left as it was there (0 without ``out``).  Positions before
    a row's first token read as 0, positions without a page as NaN."""
    ext = _native("kv4_read", cache.pool, table.pages, table.lengths)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    k_out, v_out = (None, None) if out is None else out
    if out is not None:
        _check_dtype(cache, k_out, v_out)
    return ext.kv4_read(cache.pool, table.pages, table.lengths, int(cache.head_dim), cache.dtype, int(tokens), cu_tokens, k_out, v_out)


def kv4_attention_decode(q: torch.Tensor, cache: Kv4Cache, table: PageTable, *, scale: Optional[float] = None) -> torch.Tensor:
    """Grouped-query attention of each row's last token, q ``[rows, query_heads, head_dim]``, or of its last tokens, q ``[rows,
    tokens, query_heads, head_dim]`` (a draft being checked, a prompt's end), over the row; token i of ``tokens`` sees the positions up
    to its own, ``lengths - tokens + i``.  ``scale`` is 1 / sqrt(head_dim) by default.  A query that sees nothing (an empty row)
    gives zeros, one that meets a page outside the pool NaN.  Keys, values and queries may be of any finite size, also by token and by group of
    64 channels; of float16, weights below 2^-35 of the largest do not count at the zero points."""
    ext = _native("kv4_attention_decode", q, cache.pool, table.pages, table.lengths)
    _check_dtype(cache, q)
    if scale is None:
        scale = 1.0 / math.sqrt(cache.head_dim)
    return ext.kv4_attention_decode(q, cache.pool, table.pages, table.lengths, int(cache.head_dim), float(scale))


def _result(table: PageTable, inplace: bool, found) -> Tuple[PageTable, torch.Tensor]:
    pages, lengths, refcounts, status = found
    return (table if inplace else PageTable(pages, lengths, refcounts)), status


def kv_pages_fork(table: PageTable, parents: torch.Tensor, children: torch.Tensor, *, inplace: bool = False) -> Tuple[PageTable, torch.Tensor]:
    """Row ``children[i]`` becomes a copy of row ``parents[i]`` that shares its pages (int32 tensors; pairs with a negative index
    are skipped).  Returns the new table and an int32 status ``[1]`` on the device: 0, or -1 where an index lies beyond the rows or
    a child is not empty or comes twice; the table is then unchanged."""
    ext = _native("kv_pages_fork", table.pages, table.lengths, table.refcounts, parents, children)
    return _result(table, inplace, ext.kv_pages_fork(table.pages, table.lengths, table.refcounts, parents, children, bool(inplace)))


def kv_pages_resize(cache: Kv4Cache, table: PageTable, new_lengths: torch.Tensor, *, inplace: bool = False) -> Tuple[PageTable, torch.Tensor]:
    """Takes and frees pages so that every row has room for ``new_lengths`` (int32) tokens: 0 ends a row, fewer tokens take some
    back, more make room for an append.  A row that grows gets a copy of its last page where other rows hold that page too and it is
    filled in part.  Free pages are taken lowest number first, row after row.  Returns the new table and an int32 status ``[1]``
    on the device: 0; n > 0 where n pages are missing; -1 for a length outside the table, or for an entry outside the pool where a page
    would be freed or copied.  Where it is not 0 nothing has changed.  Where all the rows that hold a page grow, each gets a copy, and the page
    itself is free after the call."""
    ext = _native("kv_pages_resize", cache.pool, table.pages, table.lengths, table.refcounts, new_lengths)
    return _result(table, inplace, ext.kv_pages_resize(cache.pool, table.pages, table.lengths, table.refcounts, new_lengths, bool(inplace)))


def kv_pages_compact(cache: Kv4Cache, table: PageTable, *, inplace: bool = False) -> Tuple[PageTable, torch.Tensor]:
    """Moves the pages in use to the front of the pool and renames them in the table.  Returns the new table and their number,
    int32 ``[1]`` on the device: the pages from there on are free.  Every table over the pool has to be in this one."""
    ext = _native("kv_pages_compact", cache.pool, table.pages, table.lengths, table.refcounts)
    return _result(table, inplace, ext.kv_pages_compact(cache.pool, table.pages, table.lengths, table.refcounts, bool(inplace)))
