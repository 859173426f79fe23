"""Accuracy of attention over the 4-bit paged cache, by group of 64 channels and by what the softmax lets through: values of very different
sizes in one row, in one head, and behind what a query sees."""

import math

import numpy as np
import pytest
import torch

import mega_kernel_qwen36 as mk
from oracle import kv4_oracle as oracle
from test_kv4_cache import Server, check_attention

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _parameters(pool, pages, length, head, d, dtype):
    """Scales and zero points of a row's values, ``[length, d / 64]`` each in 64 bits."""
    page_size = pool.shape[2] * oracle.TILE
    tiles = np.stack([pool[pages[i * oracle.TILE // page_size], head, i % (page_size // oracle.TILE)] for i in range(-(-length // oracle.TILE))])
    first = 16 * d + d * dtype.itemsize // 2
    param = torch.from_numpy(tiles[:, first : first + d * dtype.itemsize // 2].copy()).view(dtype).double().reshape(-1, d // oracle.GROUP, 2)[:length]
    return param[..., 0], param[..., 1]


class Row:
    """Rows of one KV head whose scores are exact: the keys' first group has the entries 0 to 15 (scale 1, zero point 0) and a
    query is one channel of it, so a score is one product of a query's channel and a code.  ``copies``: so many rows hold each
    row's pages, enough of them that a warp works through several tiles in turn."""

    def __init__(self, dev, dtype, d, lengths, page_size=32, copies=1):
        self.dev, self.dtype, self.d, self.lengths, self.copies = dev, dtype, d, list(lengths), copies
        per = [-(-n // page_size) for n in lengths]
        total, width = sum(per), max(per) + 1
        self.table, at = [], 0
        for n in per:
            self.table.append(list(range(at + n - 1, at - 1, -1)) + [-1] * (width - n))
            at += n
        self.pool = np.zeros((total, 1, page_size // 16, oracle.tile_bytes(d, dtype)), np.uint8)

    def fill(self, codes, v):
        """codes: of the channel that queries look at, 0 to 14, for all tokens of all rows; v ``[tokens, d]``."""
        k = torch.zeros(len(codes), 1, self.d)
        k[:, 0, 0], k[:, 0, 1] = torch.tensor(codes, dtype=torch.float32), 15
        self.codes = codes
        oracle.append(self.pool, self.table, self.lengths, k.to(self.dtype), v[:, None].to(self.dtype), self.lengths)
        on = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)
        self.cache = mk.Kv4Cache(torch.from_numpy(self.pool).to(self.dev), self.d, self.dtype)
        each = lambda x: on(x).repeat_interleave(self.copies, 0)
        self.gpu = mk.PageTable(each(self.table), each(self.lengths), torch.full((len(self.pool),), self.copies, dtype=torch.int32, device=self.dev))

    def queries(self, step, tokens=1, heads=4):
        """Queries whose score grows by `step` (a number of few bits) with each code; the scale of the call is 1."""
        q = torch.zeros(len(self.lengths) * self.copies, tokens, heads, self.d)
        q[..., 0] = step
        return q.to(self.dtype)

    def check(self, q, out, step):
        """Limits are for each group by itself, from what the softmax leaves of its entries.  With exact scores a weight is off by the
        roundings of the factor to log 2 units (three of 2^-24 of the score's distance to the largest), of the difference, of the
        exponential (2^-22) and of its products with scale and unit (2^-24 each, 2^-22 in two halves): 2^-21 of itself and of the
        distance; zero points of bf16 meet weights of two bf16 (2^-16).  Sums: at most 2^-22 of what they hold for each tile of 16 that
        a running sum takes and for each of a few joins.  The same for the denominator.  A weight of f16 that meets a
        zero point is held down to 2^-31 of the largest, a weight times scale down to 2^-34 of the group's largest."""
        tokens, at, worst = q.shape[1], 0, 0.0
        out = out.cpu().double().view(q.shape)
        for r, n in enumerate(self.lengths):
            codes = torch.tensor(self.codes[at : at + n], dtype=torch.float64)
            at += n
            _, values = oracle.row_entries(self.pool, self.table[r], n, 0, self.d, self.dtype)
            scale, zero = _parameters(self.pool, self.table[r], n, 0, self.d, self.dtype)
            for i in range(tokens):
                seen = n - tokens + i + 1
                score = codes[:seen] * step
                weight = torch.softmax(score, 0)
                want = weight @ values[:seen]
                share = 2 * (((score.max() - score)[:, None] + 1) * 2.0**-21 + 2.0**-20 + (n / 16 + 8) * 2.0**-22)
                size = zero[:seen].abs() + 15 * scale[:seen].abs()
                limit = (weight[:, None] * size * share).sum(0) + seen * 2.0**-34 * 15 * (weight[:, None] * scale[:seen]).amax(0)
                if self.dtype is torch.bfloat16:
                    limit += 2.0**-16 * (weight[:, None] * zero[:seen].abs()).sum(0)
                if self.dtype is torch.float16:
                    limit += (torch.minimum(weight, 2.0**-31 * weight.max())[:, None] * zero[:seen].abs()).sum(0)
                limit = limit.repeat_interleave(oracle.GROUP) + want.abs() * torch.finfo(self.dtype).eps / 2 * 1.01
                limit += torch.finfo(self.dtype).smallest_normal * torch.finfo(self.dtype).eps / 2 * 1.01  # half a step of the smallest numbers
                off = (out[r * self.copies : (r + 1) * self.copies, i] - want).abs() / limit
                worst = max(worst, off.max().item())
        assert worst <= 1, f"off by {worst:.3g} of the limit"


def _sizes(dtype):
    """Factors between sizes of values that the type can hold, with ordinary values on one side."""
    return [2.0**e for e in ((8, 16, 20) if dtype is torch.float16 else (8, 12, 16, 20, 24, 60))]


def _base(dtype, factor):
    """Size of the smaller values: in f16 the larger ones have to stay below 65504."""
    return 4096.0 / factor if dtype is torch.float16 else 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,copies", [(64, 1), (128, 1), (256, 1), (64, 200), (128, 200), (256, 200)])
def test_a_token_that_no_query_heeds_may_have_values_of_any_size(cuda_device, dtype, d, copies):
    step = 4.25  # scores of 0 to 59.5: the loud tokens' weights are 2^-86 of the others'
    for factor in _sizes(dtype):
        row = Row(cuda_device, dtype, d, [16, 100, 700], copies=copies)
        gen = torch.Generator().manual_seed(7)
        v = torch.randn(816, d, generator=gen) * _base(dtype, factor)
        codes = [14] * 816
        for loud in (3, 16, 16 + 99, 116 + 350, 116 + 351, 815):  # first, middle and last tokens of a row
            codes[loud] = 0
            v[loud] *= factor
        row.fill(codes, v)
        q = row.queries(step)
        row.check(q, mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0), step)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 256])
def test_groups_of_a_head_may_have_values_of_any_size(cuda_device, dtype, d):
    for factor in _sizes(dtype):
        row = Row(cuda_device, dtype, d, [37, 300])
        gen = torch.Generator().manual_seed(8)
        v = torch.randn(337, d, generator=gen) * _base(dtype, factor)
        v[:, 64:128] *= factor
        row.fill(torch.randint(8, 15, (337,), generator=gen).tolist(), v)
        q = row.queries(0.5)
        row.check(q, mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0), 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("order", ["within a tile", "rising", "falling"])
def test_values_that_shrink_as_the_scores_grow(cuda_device, dtype, d, order):
    """Weight times value is of one size throughout, though weights and values each go over many powers of two."""
    n = 15 * 16
    step = 1.5 if dtype is torch.float16 else 5.5  # over all codes 2^-30, 2^-111
    codes = [i % 15 if order == "within a tile" else i // 16 if order == "rising" else 14 - i // 16 for i in range(n)]
    row = Row(cuda_device, dtype, d, [n], copies=1000)
    size = torch.exp(-step * torch.tensor(codes, dtype=torch.float64)) * (30000 if dtype is torch.float16 else 1e15)
    row.fill(codes, (torch.randn(n, d, generator=torch.Generator().manual_seed(9)).double().clamp(-2, 2) * size[:, None]).float())
    q = row.queries(step)
    row.check(q, mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0), step)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [1, 4])
def test_later_tokens_of_a_draft_do_not_change_earlier_queries(cuda_device, dtype, heads):
    for factor in _sizes(dtype):
        row = Row(cuda_device, dtype, 64, [70, 37, 16])
        gen = torch.Generator().manual_seed(10)
        v = torch.randn(123, 64, generator=gen) * _base(dtype, factor)
        for last in (69, 106, 122):
            v[last] *= factor
        row.fill(torch.randint(8, 15, (123,), generator=gen).tolist(), v)
        q = row.queries(0.5, tokens=4, heads=heads)
        out = mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0)
        row.check(q, out, 0.5)
        # a call that ends before the loud token
        early = mk.kv4_attention_decode(q[:, :3].contiguous().to(cuda_device), row.cache, mk.PageTable(row.gpu.pages, row.gpu.lengths - 1, row.gpu.refcounts), scale=1.0)
        assert torch.allclose(out[:, :3].double(), early.double(), rtol=2 * torch.finfo(dtype).eps, atol=_base(dtype, factor) * 2.0**-14)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_near_the_largest_numbers_and_the_smallest(cuda_device, dtype):
    gen = torch.Generator().manual_seed(11)
    for size in (torch.finfo(dtype).max / 64, 2.0**-100, torch.finfo(dtype).smallest_normal * 512):
        row = Row(cuda_device, dtype, 64, [50, 1])
        row.fill([14] * 51, (torch.randn(51, 64, generator=gen).clamp(-3, 3) / 3).double().mul(size).float())
        q = row.queries(0.5)
        row.check(q, mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0), 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("missing", [-1, 10**6])
@pytest.mark.parametrize("copies", [1, 300])
def test_a_missing_page_reaches_the_queries_that_see_it_and_no_other(cuda_device, dtype, missing, copies):
    row = Row(cuda_device, dtype, 128, [70, 64, 40, 3], page_size=32, copies=copies)
    gen = torch.Generator().manual_seed(12)
    row.fill(torch.randint(8, 15, (177,), generator=gen).tolist(), torch.randn(177, 128, generator=gen))
    q = row.queries(0.5, tokens=9)
    whole = mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0)
    pages = row.gpu.pages.clone()
    pages[:copies, 2] = missing  # positions 64 to 69: the last six queries
    pages[copies : 2 * copies, 0] = missing  # all of them
    pages[2 * copies : 3 * copies, 1] = missing  # positions 32 to 39: all but the first query, whose last position is 31
    pages[3 * copies :, 0] = missing  # the last three; the others see nothing
    assert row.table[0][2] == 0
    row.cache.pool[0].fill_(0xFF)  # NaN parameters in a page that nobody holds now, the pool's first
    out = mk.kv4_attention_decode(q.to(cuda_device), row.cache, mk.PageTable(pages, row.gpu.lengths, row.gpu.refcounts), scale=1.0).unflatten(0, (4, copies))
    whole = whole.unflatten(0, (4, copies))
    for r, good in enumerate((3, 0, 1, 6)):
        assert torch.isnan(out[r, :, good:]).all()
        assert torch.allclose(out[r, :, :good].double(), whole[r, :, :good].double(), rtol=2 * torch.finfo(dtype).eps, atol=2.0**-14)
    assert (out[3, :, :6] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq,tokens", [(128, 8, 1), (256, 3, 1), (128, 2, 5)])
def test_groups_of_a_query_may_be_of_any_size(cuda_device, dtype, d, hq, tokens):
    """One group of the keys is large where the queries are small, and another the other way round, so that both count in the scores."""
    for a in (3, 8, 12, 13) if dtype is torch.float16 else (4, 10, 15, 30, 50, 63, 90, 110):
        s = Server(cuda_device, dtype, d, 1, 32, [90, 17])
        gen = torch.Generator().manual_seed(a)
        k, v = (torch.randn(107, 1, d, generator=gen).clamp(-3, 3) for _ in range(2))
        q = torch.randn(2, tokens, hq, d, generator=gen).clamp(-3, 3)
        k[..., :64], q[..., :64] = k[..., :64] * 2.0**-a, q[..., :64] * 2.0**a
        k[..., 64:128], q[..., 64:128] = k[..., 64:128] * 2.0**a, q[..., 64:128] * 2.0**-a
        k[..., 128:] = 0
        if hq > 2:
            q[1, :, 1, 64:] = 0  # and one whose other groups are nothing
        oracle.append(s.pool, s.table, s.lengths, k.to(dtype), v.to(dtype), s.lengths)
        s.cache.pool.copy_(torch.from_numpy(s.pool))
        q = q.to(dtype)
        for scale in (0.2, -0.2):
            check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu, scale=scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("power", [-120, -100, 100, 108, 120])
def test_keys_may_be_of_any_size(cuda_device, dtype, d, power):
    """Keys as large as queries are small, and the other way round: scores of an ordinary size."""
    s = Server(cuda_device, dtype, d, 2, 32, [90, 17])
    gen = torch.Generator().manual_seed(power + 200)
    k, v = (torch.randn(107, 2, d, generator=gen).clamp(-3, 3) for _ in range(2))
    q = torch.randn(2, 2, 4, d, generator=gen).clamp(-3, 3)
    oracle.append(s.pool, s.table, s.lengths, (k * 2.0**power).to(dtype), v.to(dtype), s.lengths)
    s.cache.pool.copy_(torch.from_numpy(s.pool))
    q = (q * 2.0**-power).to(dtype)
    check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu))


# What outputs may be off by before they are rounded, relative to their root mean square, on ordinary inputs (normal values, keys with a few channels
# of mean 4, score sums of some 30 with rounding steps of 2^-24 by the dozen, divided by sqrt(d)): weights are off by some 5e-7 each, at random.
# Zero points of bf16 meet weights of 16 bits: 2^-17 / sqrt(3) of zero points 2.5 times as large as the values.
ORDINARY = {torch.float32: 2e-6, torch.float16: 3e-6, torch.bfloat16: 2.5e-5}


def misrounded(out, want, dtype):
    """Share of the outputs that are not `want` rounded to the type, and what it may be: an output is rounded elsewhere only if it lies within
    its error of the middle between two neighbours.  Twice that share, for chance."""
    nearest = want.to(dtype)
    step = torch.finfo(dtype).eps * 2.0 ** torch.floor(torch.log2(want.abs().clamp_min(torch.finfo(dtype).smallest_normal)))
    limit = 2 * (2 * ORDINARY[dtype] * want.square().mean().sqrt() / step).clamp_max(1).mean()
    return (out != nearest).double().mean().item(), limit.item()


def test_the_limits_for_ordinary_inputs_tell_halves_that_are_left_out():
    """Outputs with the error of weights or queries of 11 bits (2^-12 / sqrt(3) at random, times zero points and codes 2.5 times as large as the values)
    are beyond the limits, outputs with the error of the full kernel are not."""
    gen = torch.Generator().manual_seed(1)
    want = torch.randn(20000, generator=gen, dtype=torch.float64) * 0.05
    noise = torch.randn(20000, generator=gen, dtype=torch.float64) * 0.05
    for dtype in (torch.float16, torch.bfloat16):
        share, limit = misrounded((want + noise * ORDINARY[dtype] / 2).to(dtype), want, dtype)
        assert share <= limit
        share, limit = misrounded((want + noise * 2.5 * 2.0**-12 / math.sqrt(3)).to(dtype), want, dtype)
        assert share > limit


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq,hkv,tokens", [(64, 8, 2, 1), (128, 16, 2, 1), (256, 16, 2, 1), (256, 24, 4, 3)])
def test_ordinary_inputs_keep_all_digits(cuda_device, dtype, d, hq, hkv, tokens):
    s = Server(cuda_device, dtype, d, hkv, 64, [700, 64, 33, 1500])
    s.fill(seed=d)
    q = torch.randn(4, tokens, hq, d, generator=torch.Generator().manual_seed(13)).to(dtype)
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu).cpu()
    want = oracle.attention(q, s.pool, s.table, s.lengths, dtype, d**-0.5)[0]
    if dtype is torch.float32:
        for r in range(4):
            error = (out[r].double() - want[r]).square().mean().sqrt() / want[r].square().mean().sqrt()
            assert error <= ORDINARY[dtype], f"row {r}: {error:.3g}"
    else:
        share, limit = misrounded(out, want, dtype)
        assert share <= limit, f"{share:.4f} of the outputs, limit {limit:.4f}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, 2.0**-120])
def test_a_scale_near_zero_takes_the_mean(cuda_device, dtype, scale):
    s = Server(cuda_device, dtype, 64, 1, 16, [40, 5])
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn(45, 1, 64, generator=gen).clamp(-3, 3) for _ in range(2))
    oracle.append(s.pool, s.table, s.lengths, (k * 2.0**120).to(dtype), v.to(dtype), s.lengths)
    s.cache.pool.copy_(torch.from_numpy(s.pool))
    q = (torch.randn(2, 3, 64, generator=gen).clamp(-3, 3) * 2.0**-14).to(dtype)  # scores of 2^112 before the scale
    check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu, scale=scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("copies", [1, 300])
def test_weights_of_any_size_count_where_the_largest_meets_zeros(cuda_device, dtype, d, copies):
    """One token draws all but 2^-86 and has values of 0: the output is what the others leave.  (f16 holds weights at zero points down to 2^-31.)"""
    row = Row(cuda_device, dtype, d, [100, 300, 16], copies=copies)
    v = torch.randn(416, d, generator=torch.Generator().manual_seed(14))
    codes = [0] * 416
    for sink in (99, 100 + 140, 400):
        codes[sink], v[sink] = 14, 0
    row.fill(codes, v)
    q = row.queries(4.25)
    row.check(q, mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=1.0), 4.25)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,copies", [(64, 1), (128, 300), (256, 300)])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_scores_of_any_size(cuda_device, dtype, d, copies, order):
    """Scores so far apart that the largest draws everything, up to 2^100: tokens of the largest score share the output."""
    n = 240
    codes = {"rising": [i // 16 for i in range(n)], "falling": [14 - i // 16 for i in range(n)],
             "mixed": torch.randint(0, 15, (n,), generator=torch.Generator().manual_seed(4)).tolist()}[order]
    row = Row(cuda_device, dtype, d, [n], copies=copies)
    row.fill(codes, torch.randn(n, d, generator=torch.Generator().manual_seed(15)))
    for power in (4, 10, 14, 19, 24, 28, 33, 40, 60, 100):
        for sign in (1, -1):
            step, scale = (2.0**10, 2.0 ** (power - 10)) if power > 10 else (2.0**power, 1.0)
            q = row.queries(sign * step, tokens=2)
            row.check(q, mk.kv4_attention_decode(q.to(cuda_device), row.cache, row.gpu, scale=scale), sign * step * scale)
