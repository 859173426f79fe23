"""The 4-bit paged cache: append, read, attention and the upkeep of pages, against their definition in 64 bits
(``oracle/kv4_oracle.py``)."""

import ctypes
import itertools
import math
import random
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest
import torch

import mega_kernel_qwen36 as mk
from mega_kernel_qwen36 import cabi
from oracle import kv4_oracle as oracle

ROOT = Path(__file__).resolve().parent.parent
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---- on the CPU ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("d", [64, 128, 256])
def test_every_half_byte_of_a_tile_has_one_entry(d):
    for i, (byte, shift) in enumerate(oracle.places(d)):
        halves = sorted((2 * byte + shift // 4).ravel().tolist())
        assert halves == list(range(16 * d * i, 16 * d * (i + 1)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_oracle_quantises_as_exact_fractions_do(dtype):
    def to_type(f):  # nearest value of the type: among the neighbours of the double's rounding
        near = torch.tensor(float(f), dtype=torch.float64).to(dtype)
        around = [near, torch.nextafter(near.float(), torch.tensor(math.inf)).to(dtype), near]
        bits = near.view(torch.int16).item()
        around = [torch.tensor(b, dtype=torch.int16).view(dtype) for b in (bits - 1, bits, bits + 1) if b >= 0]
        return min((Fraction(x.item()) for x in around), key=lambda x: (abs(x - f), x.numerator % 2))

    gen = torch.Generator().manual_seed(3)
    for spread in (1.0, 1e-3, 300.0):
        x = (torch.randn(8, 64, generator=gen) * spread + spread).to(dtype)
        x[0, :16] = torch.arange(16).to(dtype) * 0.5  # many values next to borders
        code, scale, zero = oracle.quantise(x)
        for r in range(8):
            codes, s, z = oracle.quantise_by_fractions(x[r].tolist(), to_type)
            assert codes == code[r].tolist() and s == Fraction(scale[r].item()) and z == Fraction(zero[r].item())


def test_structures_match_the_c_header(tmp_path):
    import shutil
    import subprocess

    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    pairs = {"mk36_kv4_cache": cabi.Kv4Cache, "mk36_kv4_tokens": cabi.Kv4Tokens, "mk36_kv4_attention_args": cabi.Kv4AttentionArgs,
             "mk36_kv_pages_args": cabi.KvPagesArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mk36.h"', "int main(void) {"]
    for name, struct in pairs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field}));' for field, _ in struct._fields_]
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([gcc, "-std=c99", "-I", str(ROOT / "include"), str(source), "-o", str(program)], check=True)
    seen = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()
    expected = []
    for struct in pairs.values():
        expected += [ctypes.sizeof(struct)] + [getattr(struct, field).offset for field, _ in struct._fields_]
    assert [int(x) for x in seen] == expected


def _c_cache(**other):
    fields = dict(pool=16, page_table=16, lengths=16, pages=4, dtype=cabi.MK36_BF16, kv_heads=2, head_dim=128, page_size=32, rows=3, row_pages=5)
    return cabi.Kv4Cache(**{**fields, **other})


def test_c_calls_refuse_wrong_arguments():
    lib = cabi.load()

    def refused(call, status, text):
        assert call == status and text in lib.mk36_last_error()

    tokens = cabi.Kv4Tokens(k=16, v=16, tokens=1)
    for call in (lib.mk36_kv4_append, lib.mk36_kv4_read):
        refused(call(None, tokens, None), cabi.MK36_ERR_INVALID_ARG, b"cache is NULL")
        refused(call(_c_cache(), None, None), cabi.MK36_ERR_INVALID_ARG, b"tokens is NULL")
        refused(call(_c_cache(pool=None), tokens, None), cabi.MK36_ERR_INVALID_ARG, b"NULL tensor pointer")
        refused(call(_c_cache(pool=8), tokens, None), cabi.MK36_ERR_INVALID_ARG, b"16-byte aligned")
        refused(call(_c_cache(dtype=9), tokens, None), cabi.MK36_ERR_UNSUPPORTED, b"unsupported dtype 9")
        refused(call(_c_cache(rows=0), tokens, None), cabi.MK36_ERR_INVALID_ARG, b"sizes must be positive")
        refused(call(_c_cache(head_dim=96), tokens, None), cabi.MK36_ERR_UNSUPPORTED, b"head_dim must be")
        refused(call(_c_cache(page_size=24), tokens, None), cabi.MK36_ERR_INVALID_ARG, b"multiple of 16")
        refused(call(_c_cache(row_pages=1 << 27), tokens, None), cabi.MK36_ERR_UNSUPPORTED, b"tokens in a row")
        refused(call(_c_cache(pages=1 << 31), tokens, None), cabi.MK36_ERR_UNSUPPORTED, b"pages")
        refused(call(_c_cache(), cabi.Kv4Tokens(k=16, v=None, tokens=1), None), cabi.MK36_ERR_INVALID_ARG, b"NULL tensor pointer")
        refused(call(_c_cache(), cabi.Kv4Tokens(k=17, v=16, tokens=1), None), cabi.MK36_ERR_INVALID_ARG, b"aligned to their elements")
        refused(call(_c_cache(), cabi.Kv4Tokens(k=16, v=16, tokens=-1), None), cabi.MK36_ERR_INVALID_ARG, b"must not be negative")
        refused(call(_c_cache(), cabi.Kv4Tokens(k=16, v=16, tokens=1 << 31), None), cabi.MK36_ERR_UNSUPPORTED, b"too many tokens")
        assert call(_c_cache(), cabi.Kv4Tokens(tokens=0), None) == cabi.MK36_OK  # nothing to do

    def attention(cache=None, workspace=None, bytes=0, **other):
        fields = dict(q=16, out=16, query_heads=4, tokens=1, scale=1.0)
        return lib.mk36_kv4_attention_decode(cache or _c_cache(), cabi.Kv4AttentionArgs(**{**fields, **other}), workspace, bytes, None)

    refused(lib.mk36_kv4_attention_decode(_c_cache(), None, None, 0, None), cabi.MK36_ERR_INVALID_ARG, b"args is NULL")
    refused(attention(q=None), cabi.MK36_ERR_INVALID_ARG, b"NULL tensor pointer")
    refused(attention(query_heads=3), cabi.MK36_ERR_INVALID_ARG, b"divisible by kv_heads")
    refused(attention(tokens=0), cabi.MK36_ERR_INVALID_ARG, b"sizes must be positive")
    refused(attention(q=17), cabi.MK36_ERR_INVALID_ARG, b"aligned to their elements")
    refused(attention(scale=math.inf), cabi.MK36_ERR_INVALID_ARG, b"scale must be finite")
    refused(attention(cache=_c_cache(rows=1 << 20), tokens=1 << 12), cabi.MK36_ERR_UNSUPPORTED, b"query heads")

    fields = dict(page_table_in=16, lengths_in=16, refcounts_in=16, page_table_out=16, lengths_out=16, refcounts_out=16, status=16, pool=16,
                  new_lengths=16, parents=16, children=16, pages=9, rows=2, row_pages=3, count=1, kv_heads=1, page_size=16, tile_bytes=4608)
    for call, needs_pool in ((lib.mk36_kv_pages_fork, False), (lib.mk36_kv_pages_resize, True), (lib.mk36_kv_pages_compact, True)):
        def pages(**other):
            return call(cabi.KvPagesArgs(**{**fields, **other}), None, 0, None)

        refused(call(None, None, 0, None), cabi.MK36_ERR_INVALID_ARG, b"args is NULL")
        refused(pages(lengths_out=None), cabi.MK36_ERR_INVALID_ARG, b"NULL tensor pointer")
        refused(pages(rows=0), cabi.MK36_ERR_INVALID_ARG, b"sizes must be positive")
        refused(pages(pages=1 << 30), cabi.MK36_ERR_UNSUPPORTED, b"pages")
        refused(pages(rows=1 << 20, row_pages=1 << 12), cabi.MK36_ERR_UNSUPPORTED, b"table entries")
        refused(pages(), cabi.MK36_ERR_WORKSPACE, b"too small")
        if needs_pool:
            refused(pages(pool=None), cabi.MK36_ERR_INVALID_ARG, b"NULL tensor pointer")
            refused(pages(page_size=20), cabi.MK36_ERR_INVALID_ARG, b"multiple of 16")
            refused(pages(tile_bytes=100), cabi.MK36_ERR_INVALID_ARG, b"16-byte aligned")
            refused(pages(row_pages=1 << 28), cabi.MK36_ERR_UNSUPPORTED, b"tokens in a row")
    refused(lib.mk36_kv_pages_fork(cabi.KvPagesArgs(**{**fields, "children": None}), None, 0, None), cabi.MK36_ERR_INVALID_ARG, b"are missing")
    refused(lib.mk36_kv_pages_resize(cabi.KvPagesArgs(**{**fields, "new_lengths": None}), None, 0, None), cabi.MK36_ERR_INVALID_ARG, b"new_lengths is NULL")


def test_python_calls_refuse_the_cpu_and_wrong_arguments():
    cache = mk.kv4_pool(4, 2, 128, page_size=32, device="cpu")
    assert cache.pool.shape == (4, 2, 2, oracle.tile_bytes(128, torch.bfloat16)) and cache.page_size == 32
    table = mk.empty_page_table(3, 5, cache)
    assert table.pages.shape == (3, 5) and table.refcounts.shape == (4,) and (table.pages == -1).all()
    k = torch.zeros(3, 1, 2, 128, dtype=torch.bfloat16)
    ids = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: mk.kv4_append(cache, table, k, k), lambda: mk.kv4_read(cache, table, 1), lambda: mk.kv4_attention_decode(k[:, 0], cache, table),
                 lambda: mk.kv_pages_fork(table, ids, ids), lambda: mk.kv_pages_resize(cache, table, table.lengths), lambda: mk.kv_pages_compact(cache, table)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    for wrong in (dict(head_dim=96), dict(page_size=24), dict(page_size=0), dict(dtype=torch.float64), dict(pages=0)):
        with pytest.raises(ValueError):
            mk.kv4_pool(**{**dict(pages=4, kv_heads=2, head_dim=128, device="cpu"), **wrong})


# ---- on the GPU ---------------------------------------------------------------------------------------------------------


class Server:
    """A pool filled with bytes that are NaN as parameters, and rows whose pages lie anywhere in it, on both sides."""

    def __init__(self, dev, dtype, d, kv_heads, page_size, lengths, seed=0, width=2, spare=3):
        rng = random.Random(seed)
        self.dev, self.dtype, self.d, self.page_size, self.lengths = dev, dtype, d, page_size, list(lengths)
        held = [-(-n // page_size) for n in lengths]
        total = sum(held) + spare
        ids = rng.sample(range(total), total)
        self.table, self.refs = [], [0] * total
        for n in held:
            mine, ids = ids[:n], ids[n:]
            self.table.append(mine + [-1] * (max(held) + width - n))
            for p in mine:
                self.refs[p] = 1
        self.pool = np.full((total, kv_heads, page_size // 16, oracle.tile_bytes(d, dtype)), 0xFF, np.uint8)
        self.cache = mk.Kv4Cache(torch.from_numpy(self.pool.copy()).to(dev), d, dtype)
        self.upload()

    def upload(self):
        on = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)
        self.gpu = mk.PageTable(on(self.table), on(self.lengths), on(self.refs))

    def tokens(self, n, seed, spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        heads = self.pool.shape[1]
        k, v = (torch.randn(n, heads, self.d, generator=gen) * spread for _ in range(2))
        k[..., 3 :: self.d // 4] += 4 * spread
        return k.to(self.dtype), v.to(self.dtype)

    def fill(self, seed=1, spread=1.0):
        k, v = self.tokens(sum(self.lengths), seed, spread)
        oracle.append(self.pool, self.table, self.lengths, k, v, self.lengths)
        self.cache.pool.copy_(torch.from_numpy(self.pool))
        return k, v

    def same_pool(self):
        assert np.array_equal(self.cache.pool.cpu().numpy(), self.pool)


def _cu(counts, dev):
    return torch.tensor([0, *itertools.accumulate(counts)], dtype=torch.int32, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,page_size", [(64, 3, 16), (128, 2, 48), (256, 1, 64), (256, 2, 32)])
def test_append_writes_the_bytes_of_the_definition(cuda_device, dtype, d, heads, page_size):
    s = Server(cuda_device, dtype, d, heads, page_size, [1, 0, 15, 16, 17, 70, 33])
    for counts in ([1, 0, 15, 16, 17, 70, 33], [1, 0, 1, 1, 1, 1, 1], [0, 0, 3, 0, 17, 6, 20]):
        k, v = s.tokens(sum(counts), seed=sum(counts))
        oracle.append(s.pool, s.table, s.lengths, k, v, counts)
        mk.kv4_append(s.cache, s.gpu, k.to(cuda_device), v.to(cuda_device), cu_tokens=_cu(counts, cuda_device))
        s.same_pool()
    # one token for every row, also for the empty one, whose position would lie before its start
    k, v = s.tokens(7, seed=9)
    mk.kv4_append(s.cache, s.gpu, k[:, None].to(cuda_device), v[:, None].to(cuda_device))
    k, v = (torch.cat((x[:1], x[2:])) for x in (k, v))
    oracle.append(s.pool, s.table, s.lengths, k, v, [1, 0, 1, 1, 1, 1, 1])
    s.same_pool()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_at_borders_extremes_and_what_is_not_finite(cuda_device, dtype):
    s = Server(cuda_device, dtype, 64, 1, 16, [64])
    info = torch.finfo(dtype)
    g = torch.randn(64, 1, 64, generator=torch.Generator().manual_seed(5)).to(dtype)
    ramp = torch.arange(64).double()
    g[0] = 0  # one value
    g[1] = -3.5
    g[2, 0] = (ramp / 2 % 15.5).to(dtype)  # values half way between two codes
    g[3, 0] = (ramp * 0.25 - 7).to(dtype)
    g[4, 0] = (ramp / 63 * 30 - 15).to(dtype)
    g[5] = info.max
    g[6, 0, ::2], g[6, 0, 1::2] = info.max, -info.max
    g[7] *= info.tiny  # near the smallest normal number
    g[8] *= float(torch.nextafter(torch.zeros(1), torch.ones(1))) if dtype == torch.float32 else info.smallest_normal * info.eps
    g[9, 0, 7] = math.nan
    g[10, 0, 63] = math.inf
    g[11, 0, 0] = -math.inf
    g[12, 0, :32], g[12, 0, 32:] = -0.0, 0.0
    g[13] = (g[13].double() * 1e-3 + 100).to(dtype)  # a large mean
    g[14] = torch.where(torch.arange(64) == 11, torch.tensor(info.max).to(dtype) / 2, g[14])
    for i in range(15, 40):  # ranges that are multiples of 15 steps: ties by the dozen
        g[i, 0] = (torch.randint(0, 31, (64,), generator=torch.Generator().manual_seed(i)).double() / 2 * 2.0 ** (i - 26)).to(dtype)
        g[i, 0, 0], g[i, 0, 1] = 0, 15 * 2.0 ** (i - 26)
    v = g.flip(0).contiguous()
    oracle.append(s.pool, s.table, s.lengths, g, v, [64])
    mk.kv4_append(s.cache, s.gpu, g[None].to(cuda_device), v[None].to(cuda_device))
    s.same_pool()
    k_read, _ = mk.kv4_read(s.cache, s.gpu, 64)
    assert torch.isnan(k_read[0, 9:12]).all() and torch.isfinite(k_read[0, :5]).all()
    assert (k_read[0, 0] == 0).all() and (k_read[0, 1] == -3.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,page_size", [(64, 32), (128, 16), (256, 64)])
def test_read_gives_the_values_rounded_once(cuda_device, dtype, d, page_size):
    s = Server(cuda_device, dtype, d, 2, page_size, [50, 0, 7, 129])
    s.fill()
    got = mk.kv4_read(s.cache, s.gpu, 186, cu_tokens=_cu(s.lengths, cuda_device))
    for i, x in enumerate(got):
        want = torch.cat([torch.stack([oracle.row_entries(s.pool, s.table[r], n, h, d, dtype)[i] for h in range(2)], 1) for r, n in enumerate(s.lengths) if n])
        # one fp32 operation on exact operands (2^-24 of the result), then the rounding to the type
        size = want.abs()
        assert ((x.cpu().double() - want).abs() <= size * (2.0**-24 + torch.finfo(dtype).eps / 2 * (1 + 2.0**-23))).all()
    # the last two of every row; before a row's start zeros
    k, v = mk.kv4_read(s.cache, s.gpu, 8)
    assert k.shape == (4, 8, 2, d) and (k[1] == 0).all() and (v[2, 0] == 0).all()
    assert torch.equal(k[2, 1:], got[0][50:57]) and torch.equal(v[3], got[1][-8:])


@pytest.mark.gpu
def test_padding_missing_pages_and_pages_outside_the_pool(cuda_device):
    s = Server(cuda_device, torch.bfloat16, 128, 2, 16, [20, 40, 5])
    before = s.pool.copy()
    counts = [4, 30, 5]
    k, v = s.tokens(50, seed=2)  # eleven tokens of padding
    s.table[1][1], s.table[1][2] = -1, 10**6
    s.upload()
    oracle.append(s.pool, s.table, s.lengths, k, v, counts)
    mk.kv4_append(s.cache, s.gpu, k.to(cuda_device), v.to(cuda_device), cu_tokens=_cu(counts, cuda_device))
    s.same_pool()
    assert not np.array_equal(before, s.pool)
    out = tuple(torch.full((50, 2, 128), 7, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    k_read, v_read = mk.kv4_read(s.cache, s.gpu, 50, cu_tokens=_cu(counts, cuda_device), out=out)
    assert k_read is out[0] and (k_read[39:] == 7).all() and (v_read[39:] == 7).all()
    inside = torch.tensor([16 <= p < 40 for p in range(10, 40)], device=cuda_device)  # positions of row 1
    assert torch.isnan(k_read[4:34][inside]).all() and torch.isfinite(k_read[4:34][~inside]).all()
    q = torch.randn(3, 4, 128, device=cuda_device).bfloat16()
    out = mk.kv4_attention_decode(q, s.cache, s.gpu)
    assert torch.isnan(out[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_and_read_take_strided_and_unaligned_tensors(cuda_device, dtype):
    s = Server(cuda_device, dtype, 64, 3, 32, [40, 9])
    k, v = s.tokens(14, seed=4)
    oracle.append(s.pool, s.table, s.lengths, k, v, [7, 7])
    # rows of a q | k | v projection, one element off every boundary
    wide = torch.zeros(2, 7, 1 + 9 * 64, dtype=dtype, device=cuda_device)
    wide[:, :, 1 + 3 * 64 : 1 + 6 * 64] = k.view(2, 7, -1).to(cuda_device)
    wide[:, :, 1 + 6 * 64 :] = v.view(2, 7, -1).to(cuda_device)
    part = lambda i: wide[:, :, 1 + 3 * i * 64 : 1 + 3 * (i + 1) * 64].unflatten(-1, (3, 64))
    mk.kv4_append(s.cache, s.gpu, part(1), part(2))
    s.same_pool()
    plain = mk.kv4_read(s.cache, s.gpu, 7)
    wide.fill_(5)
    mk.kv4_read(s.cache, s.gpu, 7, out=(part(1), part(2)))
    assert torch.equal(part(1), plain[0]) and torch.equal(part(2), plain[1]) and (wide[:, :, : 1 + 3 * 64] == 5).all()
    # heads before tokens
    s2 = Server(cuda_device, dtype, 64, 3, 32, [40, 9])
    turned = [x.view(2, 7, 3, 64).permute(0, 2, 1, 3).contiguous().to(cuda_device).permute(0, 2, 1, 3) for x in (k, v)]
    mk.kv4_append(s2.cache, s2.gpu, *turned)
    assert torch.equal(s2.cache.pool, s.cache.pool)


def attention_tolerance(dtype, want, score_size, value_size, d, length):
    """The output's own rounding; what the scores are off by (a sum of d products in fp32 whose additions in the tensor cores cut
    off: at most 2^-22 of the sum of |terms| for each of 16 steps and as much for scales and zero points), which moves every weight by
    that share; exponentials and sums of weights (2^-20); and the weighted sum of the values, at most 2^-22 of its largest term's
    size for each tile of 16 tokens that a running sum takes, and 2^-20 for weights held in two halves."""
    share = 2 * (score_size * 32 * 2.0**-22 + 2.0**-20)
    own = torch.finfo(dtype).eps / 2
    return want.abs() * own * 1.01 + (value_size * (share + (length / 16 + 8) * 2.0**-22))[..., None]


def check_attention(s, q, out, scale=None):
    scale = 1 / math.sqrt(s.d) if scale is None else scale
    shaped = q if q.ndim == 4 else q[:, None]
    want, score_size, value_size = oracle.attention(shaped.cpu(), s.pool, s.table, s.lengths, s.dtype, scale)
    limit = attention_tolerance(s.dtype, want, score_size, value_size, s.d, max(s.lengths))
    off = (out.cpu().double().view(want.shape) - want).abs()
    assert (off <= limit).all(), f"off by {(off / limit.clamp_min(1e-300)).max().item():.2f} of the limit"
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq,hkv,page_size", [(64, 2, 2, 16), (64, 9, 3, 32), (128, 8, 1, 64), (128, 20, 2, 16), (256, 16, 2, 64), (256, 6, 1, 48), (256, 24, 1, 16)])
def test_attention_matches_the_definition(cuda_device, dtype, d, hq, hkv, page_size):
    for lengths in ([1], [0, 1, 15, 16, 17, 33, 200], [700, 3], [64, 64, 64]):
        s = Server(cuda_device, dtype, d, hkv, page_size, lengths, seed=len(lengths))
        s.fill(seed=len(lengths))
        q = torch.randn(len(lengths), hq, d, generator=torch.Generator().manual_seed(7)).to(dtype)
        want = check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu))
        assert (want[[n == 0 for n in lengths]] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [2, 3, 5, 8, 19])
def test_attention_of_several_tokens_is_causal(cuda_device, dtype, tokens):
    for d, hq, hkv in ((64, 4, 2), (128, 6, 1), (256, 8, 2)):
        s = Server(cuda_device, dtype, d, hkv, 32, [tokens, 1, 0, tokens + 14, 90, 47])
        s.fill()
        q = torch.randn(6, tokens, hq, d, generator=torch.Generator().manual_seed(tokens)).to(dtype)
        out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu)
        check_attention(s, q, out)
        assert (out[1, : tokens - 1] == 0).all() and (out[2] == 0).all()  # queries that see nothing
        # each as a call of its own, over a row that ends at its token
        one = mk.PageTable(s.gpu.pages, (s.gpu.lengths - tokens + 2).clamp_min(0), s.gpu.refcounts)
        again = mk.kv4_attention_decode(q[:, 1].contiguous().to(cuda_device), s.cache, one)
        assert torch.allclose(again.float(), out[:, 1].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [1e-30, 1e-4, 30.0, 1e4, 1e30])
def test_attention_over_values_of_any_size(cuda_device, spread):
    """Scales that f16 could not hold: weights times scales have to keep their precision."""
    s = Server(cuda_device, torch.bfloat16, 128, 1, 16, [100, 31])
    k, _ = s.tokens(131, seed=1)
    _, v = s.tokens(131, seed=2, spread=spread)
    v[50:60] *= 64  # and of different sizes in one row
    v[5:9] /= 1024
    oracle.append(s.pool, s.table, s.lengths, k, v, s.lengths)
    s.cache.pool.copy_(torch.from_numpy(s.pool))
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16()
    check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [12, 24, 26])
def test_small_weights_count_where_the_largest_meets_zeros(cuda_device, dtype, gap):
    """One key draws nearly everything and its value is 0, so that the output is made of weights near 2^-gap alone.  Weights, and weights
    times scales, are held down to 2^-31 of the largest: a term is off by at most 2^-31 of its entry's size for either, and beyond that
    as any term is."""
    d, lengths = 64, [16, 200]
    s = Server(cuda_device, dtype, d, 1, 32, lengths)
    k, v = torch.randn(2, sum(lengths), 1, d, generator=torch.Generator().manual_seed(5)).mul(torch.tensor([0.01, 1.0]).view(2, 1, 1, 1)).to(dtype)
    for sink in (3, 16 + 77):
        k[sink], v[sink] = 1, 0
    oracle.append(s.pool, s.table, s.lengths, k, v, s.lengths)
    s.cache.pool.copy_(torch.from_numpy(s.pool))
    q = torch.full((2, 8, d), gap * math.log(2) / math.sqrt(d)).to(dtype)
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu).cpu().double()
    for r, n in enumerate(lengths):
        keys, values = (torch.as_tensor(x) for x in oracle.row_entries(s.pool, s.table[r], n, 0, d, dtype))
        weight = torch.softmax(keys @ q[r].double().T / math.sqrt(d), 0)
        size = values.abs().amax(1) * 3  # of an entry: |zero| + 15 scale, the least and the range of a group
        want = weight.T @ values
        score_size = (q[r].double().abs().sum(1) * keys.abs().max() / math.sqrt(d)) * 3
        share = 2 * (score_size * 32 * 2.0**-22 + 2.0**-20)
        limit = want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + ((weight.T @ size) * (share + (n / 16 + 8) * 2.0**-22) + n * 2.0**-30 * weight.amax(0) * size.max())[:, None]
        if dtype is torch.float16:
            limit = limit + 2.0**-25  # half a step of its subnormals
        off = (out[r] - want).abs()
        assert (off <= limit).all(), f"off by {(off / limit).max().item():.2f} of the limit"


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-3, 12.0, 1e30])
def test_attention_with_queries_of_any_size(cuda_device, size):
    s = Server(cuda_device, torch.bfloat16, 64, 2, 16, [77])
    s.fill(spread=1.0)
    q = (torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(3)) * size).bfloat16()
    q[0, 0, :63] *= 1e-5  # one large channel
    scale = 0.125 if size < 100 else 0.125 / size
    check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu, scale=scale), scale)
    zero = mk.kv4_attention_decode(torch.zeros_like(q).to(cuda_device), s.cache, s.gpu)
    check_attention(s, torch.zeros_like(q), zero)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_reaches_the_queries_that_see_it_and_no_other(cuda_device, dtype):
    s = Server(cuda_device, dtype, 128, 2, 32, [50, 50, 50])
    k, v = s.tokens(150, seed=1)
    k[70, 0, 5], v[139, 1, 100] = math.nan, math.inf  # row 1 position 20 head 0; row 2 position 39 head 1
    oracle.append(s.pool, s.table, s.lengths, k, v, s.lengths)
    s.cache.pool.copy_(torch.from_numpy(s.pool))
    q = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(3)).to(dtype)
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1, :2]).all() and torch.isfinite(out[1, 2:]).all()
    assert torch.isfinite(out[2, :2]).all() and torch.isnan(out[2, 2:, 64:]).all()
    shorter = mk.PageTable(s.gpu.pages, s.gpu.lengths - 31, s.gpu.refcounts)  # 19 tokens: neither is seen
    assert torch.isfinite(mk.kv4_attention_decode(q.to(cuda_device), s.cache, shorter)).all()
    q[0, 1, 3] = math.nan
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu)
    assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, 0]).all() and torch.isfinite(out[0, 2:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq", [1, 4])
def test_a_nan_does_not_reach_earlier_queries_of_a_draft(cuda_device, dtype, hq):
    s = Server(cuda_device, dtype, 64, 1, 16, [70, 37])
    k, v = s.tokens(107, seed=1)
    k[69, 0, 5], v[70 + 35, 0, 9] = math.nan, math.inf  # the last token of row 0, the last but one of row 1
    oracle.append(s.pool, s.table, s.lengths, k, v, s.lengths)
    s.cache.pool.copy_(torch.from_numpy(s.pool))
    q = torch.randn(2, 4, hq, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu)
    assert torch.isnan(out[0, 3]).all() and torch.isnan(out[1, 2:]).all()
    early = mk.kv4_attention_decode(q[:, :2].contiguous().to(cuda_device), s.cache, mk.PageTable(s.gpu.pages, s.gpu.lengths - 2, s.gpu.refcounts))
    s.lengths = [68, 35]
    check_attention(s, q[:, :2], early)
    check_attention(s, q[:, :2], out[:, :2])


@pytest.mark.gpu
def test_attention_takes_strided_and_unaligned_queries_and_a_negative_scale(cuda_device):
    s = Server(cuda_device, torch.float16, 128, 2, 16, [45, 3, 99])
    s.fill()
    wide = torch.randn(3, 1 + 10 * 128, device=cuda_device).half()
    q = wide[:, 1 : 1 + 6 * 128].view(3, 6, 128)
    out = mk.kv4_attention_decode(q, s.cache, s.gpu, scale=-0.2)
    assert torch.equal(out, mk.kv4_attention_decode(q.contiguous(), s.cache, s.gpu, scale=-0.2))
    check_attention(s, q, out, scale=-0.2)


@pytest.mark.gpu
def test_long_ragged_batch_and_lengths_out_of_range(cuda_device):
    lengths = [2500, 0, 1, 900, 17, 1601, 333, 64, 48, 1, 2, 3, 0, 0, 5, 1000]
    s = Server(cuda_device, torch.bfloat16, 64, 2, 16, lengths, width=0)
    s.fill()
    q = torch.randn(16, 8, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu)
    check_attention(s, q, out)
    assert torch.equal(out, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu))  # the same bits every time
    wild = s.gpu.lengths.clone()
    wild[0], wild[2] = 2**31 - 1, -5  # counts as the table's 2512 tokens, and as none
    out = mk.kv4_attention_decode(q.to(cuda_device), s.cache, mk.PageTable(s.gpu.pages, wild, s.gpu.refcounts))
    assert (out[2] == 0).all() and torch.isnan(out[0]).all()  # the tail of the last page holds NaN parameters
    k, v = s.tokens(16, seed=1)
    mk.kv4_append(s.cache, mk.PageTable(s.gpu.pages, wild.clamp_max(0), s.gpu.refcounts), k[:, None].to(cuda_device), v[:, None].to(cuda_device))
    s.same_pool()  # nothing has a place


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq,hkv,tokens", [(64, 8, 1, 1), (64, 3, 3, 2), (128, 12, 2, 1), (256, 16, 2, 1), (256, 5, 1, 3)])
def test_passes_cut_into_any_number_of_pieces(cuda_device, dtype, d, hq, hkv, tokens):
    for lengths in ([2500, 0, 100, 200, 5, 400, 0, 64, 65, 900, 130, 17, 0], [1700], [300, 260]):
        s = Server(cuda_device, dtype, d, hkv, 64, lengths, seed=len(lengths))
        s.fill(seed=d)
        q = torch.randn(len(lengths), tokens, hq, d, generator=torch.Generator().manual_seed(11)).to(dtype)
        for width in (s.gpu.pages.shape[1], 2000):  # the same rows in a table with room for far more
            pages = torch.full((len(lengths), width), -1, dtype=torch.int32, device=cuda_device)
            pages[:, : s.gpu.pages.shape[1]] = s.gpu.pages
            del [torch.full((1 << k,), float("nan"), device=cuda_device) for k in range(6, 22)][:]  # what an output not written may hold
            check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, mk.PageTable(pages, s.gpu.lengths, s.gpu.refcounts)))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [129, 300])
def test_more_rows_than_threads(cuda_device, rows):
    lengths = [(r * 7) % 40 for r in range(rows)]
    s = Server(cuda_device, torch.float16, 64, 1, 16, lengths)
    s.fill()
    q = torch.randn(rows, 2, 64, generator=torch.Generator().manual_seed(3)).half()
    check_attention(s, q, mk.kv4_attention_decode(q.to(cuda_device), s.cache, s.gpu))


@pytest.mark.gpu
def test_pages_beyond_four_gigabytes(cuda_device):
    """Offsets into the pool that 32 bits do not hold."""
    cache = mk.Kv4Cache(torch.empty(250_000, 1, 4, oracle.tile_bytes(256, torch.bfloat16), dtype=torch.uint8, device=cuda_device), 256)
    assert cache.pool.numel() > 2**32
    table = mk.PageTable(torch.tensor([[249_999, 3], [7, 240_001]], dtype=torch.int32, device=cuda_device),
                         torch.tensor([100, 70], dtype=torch.int32, device=cuda_device), torch.zeros(250_000, dtype=torch.int32, device=cuda_device))
    s = Server(cuda_device, torch.bfloat16, 256, 1, 64, [100, 70])
    k, v = s.fill()
    mk.kv4_append(cache, table, k.to(cuda_device), v.to(cuda_device), cu_tokens=_cu([100, 70], cuda_device))
    q = torch.randn(2, 8, 256, generator=torch.Generator().manual_seed(3)).bfloat16()
    out = mk.kv4_attention_decode(q.to(cuda_device), cache, table)
    check_attention(s, q, out)
    assert torch.equal(mk.kv4_read(cache, table, 70)[0], mk.kv4_read(s.cache, s.gpu, 70)[0])
    table.refcounts[table.pages.flatten().long()] = 1
    dense, live = mk.kv_pages_compact(cache, table)
    assert live.item() == 4 and sorted(dense.pages.flatten().tolist()) == [0, 1, 2, 3]
    assert torch.equal(mk.kv4_attention_decode(q.to(cuda_device), cache, dense), out)


def _lists(table):
    return table.pages.tolist(), table.lengths.tolist(), table.refcounts.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("page_size,heads,d,dtype", [(16, 1, 64, torch.float16), (64, 2, 128, torch.bfloat16), (48, 1, 256, torch.float32)])
def test_forks_resizes_and_compactions_follow_the_definition(cuda_device, inplace, page_size, heads, d, dtype):
    rng = random.Random(page_size + inplace)
    rows, width, total = 40, 6, 120
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    pool = np.random.default_rng(0).integers(0, 256, (total, heads, page_size // 16, oracle.tile_bytes(d, dtype)), np.uint8)
    cache = mk.Kv4Cache(torch.from_numpy(pool.copy()).to(cuda_device), d, dtype)
    table = mk.empty_page_table(rows, width, cache)
    state = _lists(table)
    seen = set()
    for step in range(60):
        what = rng.choice(["fork", "resize", "resize", "resize", "compact"])
        old = mk.PageTable(*(x.clone() for x in (table.pages, table.lengths, table.refcounts)))
        if what == "fork":
            empty = [r for r in range(rows) if state[1][r] == 0]
            n = rng.randrange(0, min(8, len(empty)) + 1)
            parents, children = [rng.randrange(-1, rows) for _ in range(n)], rng.sample(empty, n)
            if rng.random() < 0.2 and n:
                children[0] = rng.choice([rows, rng.randrange(rows), children[-1], -1])
            *state, status = oracle.fork(*state, parents, children)
            new, got = mk.kv_pages_fork(table, on(parents), on(children), inplace=inplace)
        elif what == "resize":
            after = []
            for n in state[1]:
                x = rng.random()
                after.append(0 if x < 0.15 else max(0, n - rng.randrange(0, 2 * page_size)) if x < 0.3 else n if x < 0.4 else min(width * page_size, n + 1) if x < 0.8
                             else rng.randrange(0, width * page_size + 1))
            if rng.random() < 0.1:
                after[rng.randrange(rows)] = rng.choice([-1, width * page_size + 1])
            *state, status = oracle.resize(pool, *state, after)
            new, got = mk.kv_pages_resize(cache, table, on(after), inplace=inplace)
        else:
            *state, status = oracle.compact(pool, *state)
            new, got = mk.kv_pages_compact(cache, table, inplace=inplace)
        seen.add((what, (status > 0) - (status < 0)))
        assert (new is table) == inplace
        if not inplace:
            assert all(torch.equal(getattr(old, n), getattr(table, n)) for n in ("pages", "lengths", "refcounts"))
        table = new
        assert got.tolist() == [status], (step, what)
        assert _lists(table) == tuple(state), (step, what)
        assert np.array_equal(cache.pool.cpu().numpy(), pool), (step, what)
    assert {("resize", 0), ("resize", -1), ("fork", 0), ("compact", 1)} <= seen


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
def test_resize_changes_nothing_where_pages_are_missing(cuda_device, inplace):
    s = Server(cuda_device, torch.bfloat16, 64, 2, 16, [20, 3, 40], spare=2)
    s.fill()
    before = s.table, s.lengths, s.refs
    for after, missing in (([20, 60, 40], 1), ([33, 50, 48], 2), ([0, 80, 40], 0), ([100, 0, 0], 0)):
        # what rows give back in the call can be taken in it
        pool = s.pool.copy()
        *state, status = oracle.resize(pool, *before, after)
        table = mk.PageTable(*(x.clone() for x in (s.gpu.pages, s.gpu.lengths, s.gpu.refcounts)))
        if max(after) > 16 * len(s.table[0]):
            missing = -1
        new, got = mk.kv_pages_resize(s.cache, table, torch.tensor(after, dtype=torch.int32, device=cuda_device), inplace=inplace)
        assert got.item() == status == missing and _lists(new) == tuple(state)
        if missing:
            assert _lists(new) == before


@pytest.mark.gpu
def test_fork_refuses_children_that_are_not_empty_or_come_twice(cuda_device):
    s = Server(cuda_device, torch.bfloat16, 64, 1, 16, [20, 3, 0, 0, 0])
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    before = s.table, s.lengths, s.refs
    for parents, children, status in (([0, 0], [2, 2], -1), ([0], [1], -1), ([5], [2], -1), ([0], [5], -1), ([0, -1], [-1, 1], 0), ([], [], 0),
                                      ([0, 1, 0], [2, 3, 4], 0), ([2, 1], [3, 2], 0), ([2], [2], 0)):
        *state, want = oracle.fork(*before, parents, children)
        new, got = mk.kv_pages_fork(s.gpu, on(parents), on(children))
        assert got.item() == want == status and _lists(new) == tuple(state)
        assert status == 0 or _lists(new) == before


@pytest.mark.gpu
def test_resize_refuses_tables_that_name_pages_outside_the_pool(cuda_device):
    for slot, after in ((1, 10), (1, 25)):  # gives the page back; would copy it
        s = Server(cuda_device, torch.bfloat16, 64, 1, 16, [20, 3])
        s.table[0][slot] = 99
        s.upload()
        new, status = mk.kv_pages_resize(s.cache, s.gpu, torch.tensor([after, 3], dtype=torch.int32, device=cuda_device))
        assert status.item() == -1 and _lists(new) == (s.table, s.lengths, s.refs)


@pytest.mark.gpu
def test_many_rows_and_pages(cuda_device):
    """More rows and pages than a plan has threads, pages that are shared by many rows."""
    rows, width, total = 2500, 4, 9000
    cache = mk.kv4_pool(total, 1, 64, page_size=16, device=cuda_device)
    cache.pool.random_(0, 256)
    pool = cache.pool.cpu().numpy().copy()
    table = mk.empty_page_table(rows, width, cache)
    state, on = _lists(table), lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    rng = random.Random(1)
    after = [rng.randrange(0, 64) if r < 1000 else 0 for r in range(rows)]
    for step in range(3):
        *state, status = oracle.resize(pool, *state, after)
        table, got = mk.kv_pages_resize(cache, table, on(after))
        assert got.item() == status == 0
        if step == 0:
            parents, children = [3 if r % 2 else r % 1000 for r in range(1000, rows)], list(range(1000, rows))
            *state, status = oracle.fork(*state, parents, children)
            table, got = mk.kv_pages_fork(table, on(parents), on(children))
            assert got.item() == status == 0
        after = [max(0, min(64, n + rng.randrange(-6, 7))) for n in state[1]]
    *state, n = oracle.compact(pool, *state)
    table, got = mk.kv_pages_compact(cache, table)
    assert got.item() == n and _lists(table) == tuple(state) and np.array_equal(cache.pool.cpu().numpy(), pool)


def _serve(dev, dtype, graph=False):
    """Prompts, answers sampled from each, tokens one by one, a draft taken back, the pool made dense: logits of every step."""
    d, hq, hkv, page_size = 128, 8, 2, 32
    cache = mk.kv4_pool(60, hkv, d, page_size=page_size, dtype=dtype, device=dev)
    table = mk.empty_page_table(6, 8, cache)
    gen = torch.Generator().manual_seed(11)
    make = lambda *shape: torch.randn(*shape, generator=gen).to(dtype)
    prompts = [45, 70]
    dense = [[] for _ in range(6)]  # what every row has been given

    def check(q, out):
        for r in range(6):
            n = len(dense[r])
            if n == 0:
                assert (out[r] == 0).all()
                continue
            pool = np.zeros((-(-n // page_size), hkv, page_size // 16, cache.pool.shape[3]), np.uint8)
            k, v = (torch.stack([t[i] for t in dense[r]]) for i in range(2))
            rows = [list(range(pool.shape[0]))]
            oracle.append(pool, rows, [n], k, v, [n])
            want, a, b = oracle.attention(q[r][None], pool, rows, [n], dtype, d**-0.5)
            assert ((out[r].cpu().double() - want[0]).abs() <= attention_tolerance(dtype, want, a, b, d, n)[0]).all()

    on = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    table, missing = mk.kv_pages_resize(cache, table, on(prompts + [0] * 4))
    k, v = make(sum(prompts), hkv, d), make(sum(prompts), hkv, d)
    mk.kv4_append(cache, table, k.to(dev), v.to(dev), cu_tokens=_cu(prompts + [0] * 4, dev))
    for i in range(sum(prompts)):
        dense[0 if i < 45 else 1].append((k[i], v[i]))
    table, wrong = mk.kv_pages_fork(table, on([0, 0, 1]), on([2, 3, 5]))
    dense[2], dense[3], dense[5] = list(dense[0]), list(dense[0]), list(dense[1])
    assert missing.item() == wrong.item() == 0
    alive, growing = on([1, 1, 1, 1, 0, 1]), {0, 1, 2, 3, 5}
    k_in, v_in, q_in = (torch.empty(6, 1, h, d, dtype=dtype, device=dev) for h in (hkv, hkv, hq))
    status = torch.zeros(1, dtype=torch.int32, device=dev)

    def step():
        _, s = mk.kv_pages_resize(cache, table, table.lengths + alive, inplace=True)
        status.add_(s.abs())
        mk.kv4_append(cache, table, k_in, v_in)
        return mk.kv4_attention_decode(q_in, cache, table)

    out = None
    if graph:
        saved = [x.clone() for x in (table.pages, table.lengths, table.refcounts, cache.pool)]
        side = torch.cuda.Stream(dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for x in (k_in, v_in, q_in):
                x.zero_()
            step()
        side.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            out = step()
        for x, y in zip((table.pages, table.lengths, table.refcounts, cache.pool), saved):
            x.copy_(y)
        status.zero_()
    results = []
    for i in range(40):
        k, v, q = make(6, 1, hkv, d), make(6, 1, hkv, d), make(6, 1, hq, d)
        for x, y in ((k_in, k), (v_in, v), (q_in, q)):
            x.copy_(y)
        for r in growing:
            dense[r].append((k[r, 0], v[r, 0]))
        if graph:
            captured.replay()
        else:
            out = step()
        results.append(out.clone())
        if i % 13 == 0:
            check(q, out)
        if i == 20:  # three tokens of row 3 are taken back, row 0 ends, the pool is made dense
            lengths = table.lengths.clone()
            lengths[0], lengths[3] = 0, lengths[3] - 3
            mk.kv_pages_resize(cache, table, lengths, inplace=True)
            dense[0], dense[3] = [], dense[3][:-3]
            alive[0] = 0
            growing.discard(0)
            _, live = mk.kv_pages_compact(cache, table, inplace=True)
            assert live.item() == (table.refcounts > 0).sum().item() == (table.refcounts[: live.item()] > 0).sum().item()
    # row 4 was never alive and keeps no token, row 0 has ended: both give zeros
    check(q, out)
    assert status.item() == 0 and (out[4] == 0).all()
    return results


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_served_batch_matches_dense_attention_and_its_captured_form(cuda_device, dtype):
    eager, replayed = _serve(cuda_device, dtype), _serve(cuda_device, dtype, graph=True)
    assert all(torch.equal(a, b) for a, b in zip(eager, replayed))


@pytest.mark.gpu
def test_calls_on_two_streams_and_two_captured_graphs_do_not_meet(cuda_device):
    servers = [Server(cuda_device, torch.bfloat16, 256, 2, 64, [1500 + 100 * i, 40], seed=i) for i in range(2)]
    queries = []
    for i, s in enumerate(servers):
        k, v = s.tokens(sum(s.lengths), seed=i)
        mk.kv4_append(s.cache, s.gpu, k.to(cuda_device), v.to(cuda_device), cu_tokens=_cu(s.lengths, cuda_device))
        queries.append(torch.randn(2, 16, 256, device=cuda_device).bfloat16())
    want = [mk.kv4_attention_decode(q, s.cache, s.gpu) for q, s in zip(queries, servers)]
    graphs, outs, streams = [], [], [torch.cuda.Stream(cuda_device) for _ in range(2)]
    for q, s in zip(queries, servers):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mk.kv4_attention_decode(q, s.cache, s.gpu))
        graphs.append(g)
    torch.cuda.synchronize()
    eager = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
                eager[i].append(mk.kv4_attention_decode(queries[i], servers[i].cache, servers[i].gpu))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], want[i]) and all(torch.equal(x, want[i]) for x in eager[i])


@pytest.mark.gpu
def test_calls_without_tokens_and_in_inference_mode(cuda_device):
    s = Server(cuda_device, torch.bfloat16, 64, 2, 16, [20, 0])
    s.fill()
    none = torch.empty(2, 0, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    mk.kv4_append(s.cache, s.gpu, none, none)
    mk.kv4_append(s.cache, s.gpu, none[0], none[0], cu_tokens=_cu([0, 0], cuda_device))
    s.same_pool()
    for k, v in (mk.kv4_read(s.cache, s.gpu, 0), mk.kv4_read(s.cache, s.gpu, 0, cu_tokens=_cu([0, 0], cuda_device))):
        assert k.numel() == v.numel() == 0 and k.shape == v.shape
    nobody = torch.empty(0, dtype=torch.int32, device=cuda_device)
    same, status = mk.kv_pages_fork(s.gpu, nobody, nobody)
    assert status.item() == 0 and _lists(same) == _lists(s.gpu)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(cuda_device)
    with torch.inference_mode():
        longer, status = mk.kv_pages_resize(s.cache, s.gpu, s.gpu.lengths + 1)
        k = torch.ones(2, 1, 2, 64, dtype=torch.bfloat16, device=cuda_device)
        mk.kv4_append(s.cache, longer, k, k)
        assert status.item() == 0
        out = mk.kv4_attention_decode(q, s.cache, longer)
        assert torch.equal(mk.kv4_read(s.cache, longer, 1)[1], k)
        mk.kv_pages_compact(s.cache, longer, inplace=True)
        assert torch.equal(mk.kv4_attention_decode(q, s.cache, longer), out)
    assert (out[1] == 1).all() and not out.requires_grad


@pytest.mark.gpu
def test_calls_on_the_gpu_refuse_wrong_arguments(cuda_device):
    s = Server(cuda_device, torch.bfloat16, 128, 2, 16, [20, 3])
    k = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=cuda_device)
    long = mk.PageTable(s.gpu.pages.long(), s.gpu.lengths, s.gpu.refcounts)
    for wrong, text in (
        (lambda: mk.kv4_append(s.cache, s.gpu, k.half(), k.half()), "holds"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k, k[:, :, :1]), "kv_heads"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k[:1], k[:1]), "rows"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k[..., ::2], k[..., ::2]), "head_dim"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k, torch.cat((k, k), 1)), "match"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k.transpose(-1, -2).contiguous().transpose(-1, -2), k), "contiguous channels"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k[:, 0], k[:, 0]), "tokens"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k[:, 0], k[:, 0], cu_tokens=torch.zeros(2, dtype=torch.int32, device=cuda_device)), "rows \\+ 1"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k[:, 0], k[:, 0], cu_tokens=torch.zeros(3, device=cuda_device)), "int32"),
        (lambda: mk.kv4_append(s.cache, s.gpu, k[:, 0], k[:, 0], cu_tokens=torch.zeros(3, dtype=torch.int32)), "CUDA"),
        (lambda: mk.kv4_append(s.cache, long, k, k), "int32"),
        (lambda: mk.kv4_append(mk.Kv4Cache(s.cache.pool, 64), s.gpu, k, k), "tiles"),
        (lambda: mk.kv4_append(mk.Kv4Cache(s.cache.pool, 96), s.gpu, k, k), "head_dim"),
        (lambda: mk.kv4_append(mk.Kv4Cache(s.cache.pool[:, :1], 128), s.gpu, k, k), "contiguous"),
        (lambda: mk.kv4_read(s.cache, s.gpu, -1), "negative"),
        (lambda: mk.kv4_read(s.cache, s.gpu, 2, out=(k, k)), "shape"),
        (lambda: mk.kv4_attention_decode(q[:, :3], s.cache, s.gpu), "divisible"),
        (lambda: mk.kv4_attention_decode(q[:1], s.cache, s.gpu), "rows"),
        (lambda: mk.kv4_attention_decode(q[..., :64], s.cache, s.gpu), "head_dim"),
        (lambda: mk.kv4_attention_decode(q.float(), s.cache, s.gpu), "holds"),
        (lambda: mk.kv4_attention_decode(q, s.cache, s.gpu, scale=math.nan), "finite"),
        (lambda: mk.kv4_attention_decode(q[:, None][:, :0], s.cache, s.gpu), "token"),
        (lambda: mk.kv_pages_fork(s.gpu, s.gpu.lengths, s.gpu.lengths[:1]), "one length"),
        (lambda: mk.kv_pages_fork(long, s.gpu.lengths, s.gpu.lengths), "int32"),
        (lambda: mk.kv_pages_resize(s.cache, s.gpu, s.gpu.lengths[:1]), "each row"),
        (lambda: mk.kv_pages_resize(s.cache, mk.PageTable(s.gpu.pages, s.gpu.lengths, s.gpu.refcounts[1:]), s.gpu.lengths), "each page"),
        (lambda: mk.kv_pages_compact(s.cache, mk.PageTable(s.gpu.pages, s.gpu.lengths[:1], s.gpu.refcounts)), "each row"),
    ):
        with pytest.raises((RuntimeError, ValueError), match=text):
            wrong()
    s.same_pool()


@pytest.mark.gpu
def test_more_pages_than_a_plan_ranks_at_once(cuda_device):
    """Pages by the ten thousand: ranks carry over from one segment of 32768 to the next."""
    total, rows, width = 70_001, 300, 260
    cache = mk.Kv4Cache(torch.zeros(total, 1, 1, oracle.tile_bytes(64, torch.float16), dtype=torch.uint8, device=cuda_device), 64, torch.float16)
    cache.pool[:, 0, 0, :4] = torch.arange(total, dtype=torch.int32, device=cuda_device).view(torch.uint8).view(total, 4)  # each page knows its number
    rng = random.Random(4)
    ids, at = rng.sample(range(total), total), 0
    table, lengths, refs = [], [], [0] * total
    for r in range(rows):
        n = rng.randrange(0, width)
        lengths.append(16 * n - rng.randrange(0, 16) if n else 0)
        table.append(ids[at : at + n] + [-1] * (width - n))
        for p in ids[at : at + n]:
            refs[p] = 1
        at += n
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    gpu = mk.PageTable(on(table), on(lengths), on(refs))
    pool = cache.pool.cpu().numpy().copy()
    after = [rng.choice([0, n, min(16 * width, n + 1), rng.randrange(0, 16 * width)]) for n in lengths]
    *state, status = oracle.resize(pool, table, lengths, refs, after)
    gpu, got = mk.kv_pages_resize(cache, gpu, on(after))
    assert got.item() == status == 0 and _lists(gpu) == tuple(state)
    *state, n = oracle.compact(pool, *state)
    gpu, got = mk.kv_pages_compact(cache, gpu)
    assert got.item() == n and _lists(gpu) == tuple(state) and np.array_equal(cache.pool.cpu().numpy(), pool)
    *state, status = oracle.resize(pool, *state, [16 * width] * rows)
    gpu, got = mk.kv_pages_resize(cache, gpu, on([16 * width] * rows))
    assert got.item() == status > 0 and _lists(gpu) == tuple(state)
    # more than one segment in use, and holes in each
    for after in ([16 * 200] * rows, [16 * (240 if r % 2 else 100) for r in range(rows)], [16 * 225] * rows, [16 * (250 if r % 3 else 150) for r in range(rows)]):
        *state, status = oracle.resize(pool, *state, after)
        gpu, got = mk.kv_pages_resize(cache, gpu, on(after))
        assert got.item() == status and _lists(gpu) == tuple(state)
    assert status == 0
    *state, n = oracle.compact(pool, *state)
    gpu, got = mk.kv_pages_compact(cache, gpu)
    assert got.item() == n > 32768 and _lists(gpu) == tuple(state) and np.array_equal(cache.pool.cpu().numpy(), pool)
