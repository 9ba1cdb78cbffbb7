"""Paged caches of 8 and 4 bits, on the GPU: page numbers and values that are none, in calls of many columns and at the edge of what a row sees; items of
more tiles than a wave holds page numbers for.  Helpers and tolerances are those of tests/test_paged_quant_gpu.py."""

import math

import pytest
import torch

from paged_quant_util import QuantBatch
from sample_efficient_gpt_amd import PagedKVCache, PageTable
from test_paged_quant_gpu import BF16, DTYPES, F32, attend, both_formats, check_y, read

pytestmark = pytest.mark.gpu


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", [(6, 2, 64, BF16), (4, 2, 128, BF16), (4, 2, 32, F32), (4, 2, 64, F32), (4, 2, 128, F32)])
@pytest.mark.parametrize("page", [8, 16, 32, 64])
@pytest.mark.parametrize("prefix", [0, 45])
def test_a_bad_page_number_reaches_every_row_that_sees_it(gpu_device, H, Hkv, D, dtype, page, prefix, fmt):
    """More columns than one wave has, pages smaller than a tile of keys: the wave that reads a page is not the only one that multiplies by its keys."""
    rows, lens = [60, 200, 1], [140, 260, 90]
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=50, prefix=prefix)
    clean = attend(x)
    for b in range(2):
        for j in range(-(-lens[b] // page)):
            was = x.block_table[b, j].clone()
            x.block_table[b, j] = x.n_pages if j % 2 else -1
            y, lse = attend(x, return_lse=True)
            first, end = x.starts[b] + max(0, j * page - (lens[b] - rows[b])), x.starts[b + 1]
            assert y[first:end].isnan().all() and lse[first:end].isnan().all(), (b, j)
            others = [r for r in range(sum(rows)) if not x.starts[b] <= r < end]
            assert torch.equal(y[others], clean[others]), (b, j)
            x.block_table[b, j] = was
    for j in range(-(-prefix // page)):
        was = x.prefix_table[j].clone()
        x.prefix_table[j] = x.n_pages + 5
        assert attend(x).isnan().all(), j
        x.prefix_table[j] = was
    assert torch.equal(attend(x), clean)


@pytest.mark.parametrize("fmt,kind", [("e4m3", "nan"), ("e4m3", "-nan"), ("e4m3", "large"), ("e2m1", "large")])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(6, 2, 64, BF16), (4, 2, 128, BF16), (4, 2, 32, F32), (4, 2, 64, F32), (4, 2, 128, F32)])
@pytest.mark.parametrize("rows,lens,prefix", [([1, 1], [37, 64], 0), ([70, 1], [70, 40], 0), ([45, 3], [300, 50], 0), ([1, 50], [5, 50], 40)])
def test_a_value_that_is_none_by_its_code(gpu_device, rows, lens, prefix, H, Hkv, D, dtype, fmt, kind):
    """Pools that something else filled: the code that is NaN in 8 bits, and a scale that carries codes beyond the largest number.  Wherever the key stands
    (in a block that all rows see, or one that some do), the rows that see it have its value, and nothing else changes."""
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=51, prefix=prefix)
    clean = attend(x)
    codes, rep = x.v_pages.view(torch.uint8), H // Hkv
    for b, (n, L) in enumerate(zip(rows, lens)):
        for p in sorted({0, L // 2, L // 32 * 32, L - n, L - 2, L - 1} & set(range(L))):
            page, slot = int(x.block_table[b, p // 16]), p % 16
            was = codes[page, 1, slot].clone(), x.v_scales[page, 1, slot].clone()
            if kind == "large":  # a whole block, beyond what bf16 and fp32 hold
                codes[page, 1, slot, (D - 32) * codes.shape[3] // D:] = 0x7E if fmt == "e4m3" else 0x77
                x.v_scales[page, 1, slot, -1] = 254
                none = torch.arange(D) >= D - 32
            else:
                codes[page, 1, slot, D - 27] = 0x7F if kind == "nan" else 0xFF
                none = torch.arange(D) == D - 27
            y = attend(x)
            codes[page, 1, slot], x.v_scales[page, 1, slot] = was
            first, end = x.starts[b] + max(0, p - (L - n)), x.starts[b + 1]
            hit = torch.zeros(y.shape, dtype=torch.bool, device=gpu_device)
            hit[first:end, rep:2 * rep] = none.to(gpu_device)
            assert torch.equal(y.isnan() if kind != "large" else ~y.isfinite(), hit), (b, p)
            assert torch.equal(y[~hit], clean[~hit]), (b, p)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,lens", [([1, 1], [37, 64]), ([70, 1], [70, 40])])
def test_a_key_that_is_none_by_its_code(gpu_device, rows, lens, dtype):
    x = QuantBatch("e4m3", rows, lens, 6, 2, 64, 16, dtype, gpu_device, seed=52)
    clean = attend(x)
    for b, (n, L) in enumerate(zip(rows, lens)):
        for p in sorted({0, L // 2, L // 32 * 32, L - 1} & set(range(L))):
            at = x.k_pages.view(torch.uint8)[int(x.block_table[b, p // 16]), 1, p % 16, 5:6]
            was = at.clone()
            at.fill_(0x7F)
            y = attend(x)
            at.copy_(was)
            hit = torch.zeros(y.shape, dtype=torch.bool, device=gpu_device)
            hit[x.starts[b] + max(0, p - (L - n)):x.starts[b + 1], 3:] = True
            assert torch.equal(y.isnan(), hit) and torch.equal(y[~hit], clean[~hit]), (b, p)


def test_rows_back_from_codes_that_are_none(gpu_device):
    x = QuantBatch("e4m3", [40], [40], 2, 1, 64, 16, BF16, gpu_device, seed=53)
    codes = x.v_pages.view(torch.uint8)
    for t, (code, scale) in enumerate([(0x7F, 127), (0xFF, 127), (0x7E, 254), (0xFE, 254)]):
        at = int(x.block_table[0, t // 16]), 0, t % 16
        codes[(*at, slice(32))], x.v_scales[(*at, 0)] = code, scale
    for dtype in (BF16, F32):
        v = read(x, dtype=dtype)[1][:, 0, :32]
        assert v[:2].isnan().all() and v[2:4].isinf().all() and (v[2] > 0).all() and (v[3] < 0).all() and v[4:].isfinite().all()


@both_formats
def test_a_cache_around_pools_of_bytes(gpu_device, fmt):
    """Pools that a program made itself, as bytes where they are of 4 bits: under the prefix's table, turned into other types, attended to."""
    pages = PageTable(2, 40, 8, prefix_len=19, device=gpu_device)
    codes = [torch.empty(pages.n_pages, 2, 8, 64 if fmt == "e4m3" else 32, dtype=torch.uint8, device=gpu_device) for _ in "kv"]
    scales = [torch.empty(pages.n_pages, 2, 8, 2, dtype=torch.uint8, device=gpu_device) for _ in "kv"]
    mine = PagedKVCache(pages, 2, 64, DTYPES[fmt], *([t.view(DTYPES[fmt]) for t in codes] if fmt == "e4m3" else codes), *scales)
    plain = PagedKVCache(pages, 2, 64, DTYPES[fmt])
    g = torch.Generator().manual_seed(54)
    n = lambda *s: torch.randn(*s, generator=g).to(BF16).to(gpu_device)
    for table, rows in ((pages.prefix, 19), (pages, [30, 7])):
        table.extend(rows)
        k, v = n(table.rows, 2, 64), n(table.rows, 2, 64)
        for c in (mine, plain):
            c.of(table).append(k, v)
    q = n(pages.rows, 6, 64)
    gain = torch.ones(1, device=gpu_device)
    assert torch.equal(mine.attend(q, gain), plain.attend(q, gain))
    for dtype in (BF16, *DTYPES.values(), torch.uint8):
        a, b = mine.to(dtype), plain.to(dtype)
        assert a.dtype == b.dtype
        for table in (pages, pages.prefix):
            assert all(torch.equal(x, y) for x, y in zip(a.of(table).read()[:2], b.of(table).read()[:2]))


# Items of more than 64 tiles: a wave goes through tiles of 16 keys (more than 32 columns a kv head: 64, at heads of 128 32) and works out the places of 64 at a
# time.  How long an item is follows from the number of blocks of 32 keys, all tiles of columns and kv heads together, over 744 workgroups (heads of 128 496,
# ragged rows 480): 100 to 150 tiles in the first two, 78 and 91 in the third.  All sequences have the same pages; some rows are looked at.
@both_formats
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (32, F32), (64, F32), (128, F32)])
@pytest.mark.parametrize("kind", ["tokens", "ragged tokens", "prompt"])
def test_items_of_more_tiles_than_a_wave_holds_places_for(gpu_device, kind, D, dtype, page, fmt):
    if kind == "prompt":
        H, Hkv, B, rows, lens = 32, 4, 1, [2500 if D == 128 else 4500], [2900 if D == 128 else 5000]
    else:
        H, Hkv, B = 8, 8, 64
        rows, lens = [1] * 63 + [1 if kind == "tokens" else 2], [9600 - 3 * b for b in range(64)]
    x = QuantBatch(fmt, rows[-1:], [max(lens)], H, Hkv, D, page, dtype, gpu_device, seed=55)
    x.rows, x.lens = rows, lens
    x.starts = [sum(rows[:b]) for b in range(B + 1)]
    x.q = torch.randn(sum(rows), H, D, generator=torch.Generator().manual_seed(56)).to(dtype).to(gpu_device)
    x.block_table, x.kv_len = x.block_table.repeat(B, 1), torch.tensor(lens, dtype=torch.int32, device=gpu_device)
    x.seq_start = None if kind == "tokens" else torch.tensor(x.starts, dtype=torch.int32, device=gpu_device)
    y, lse = attend(x, return_lse=True)
    some = [(0, i) for i in (0, 1, rows[0] // 2, rows[0] - 1)] if kind == "prompt" else [(b, rows[b] - 1) for b in (0, 1, 40, 63)]
    at = [x.starts[b] + i for b, i in some]
    part = QuantBatch(fmt, [1] * 4, [1] * 4, H, Hkv, D, page, dtype, gpu_device)  # the same rows as sequences of their own
    part.lens, part.q, part.block_table = [lens[b] - rows[b] + i + 1 for b, i in some], x.q[at], x.block_table[[b for b, _ in some]]
    for name in ("g_q", "cos", "sin", "k_pages", "v_pages", "k_scales", "v_scales"):
        setattr(part, name, getattr(x, name))
    check_y(part, y[at], lse[at], part.attended())
    assert torch.equal(y, attend(x))
