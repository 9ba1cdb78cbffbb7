"""Paged caches of 8 and 4 bits with heads of 32 (float32 rows): a row is one block, and half a row of the tiles that the kernels multiply.  What is asked for,
and the tolerances, are those of tests/test_paged_quant_gpu.py, whose tests are called for this head size."""

import pytest
import torch

import test_paged_quant_gpu as base
from paged_quant_util import QuantBatch, decode, encode
from paged_util import F64
from sample_efficient_gpt_amd import MultiHeadSelfAttention, PagedKVCache, PageTable, paged_kv_append
from test_paged_quant_gpu import BF16, DTYPES, F32, append, attend, both_formats, check_pools, check_y, read

pytestmark = pytest.mark.gpu


@both_formats
@pytest.mark.parametrize("H,Hkv", [(6, 2), (4, 4)])
@pytest.mark.parametrize("rows,lens", base.RAGGED)
@pytest.mark.parametrize("page", [8, 64])
def test_append_and_read(gpu_device, rows, lens, H, Hkv, page, fmt):
    base.test_append_and_read(gpu_device, rows, lens, H, Hkv, 32, F32, page, fmt)


@both_formats
@pytest.mark.parametrize("H,Hkv", [(6, 2), (40, 1)])
@pytest.mark.parametrize("rows,lens", base.RAGGED)
@pytest.mark.parametrize("page", [8, 16, 64])
def test_attention(gpu_device, rows, lens, H, Hkv, page, fmt):
    base.test_attention(gpu_device, rows, lens, H, Hkv, 32, F32, page, fmt)


@both_formats
@pytest.mark.parametrize("H,Hkv", [(6, 2), (40, 1)])
@pytest.mark.parametrize("rows,lens,prefix", [([1], [1], 1), ([1, 1, 1], [0, 5, 70], 100), ([1] * 40, [i for i in range(40)], 515), ([3, 0, 20, 1], [3, 9, 60, 0], 64),
                                              ([150, 130], [150, 260], 333)])
@pytest.mark.parametrize("page", [8, 32])
def test_shared_prefix(gpu_device, rows, lens, prefix, H, Hkv, page, fmt):
    base.test_shared_prefix(gpu_device, rows, lens, prefix, H, Hkv, 32, F32, page, fmt)


@both_formats
@pytest.mark.parametrize("H", [16, 17, 32, 33])
@pytest.mark.parametrize("rows,lens,prefix", [([1], [2500], 0), ([1, 2, 1], [900, 77, 1300], 0), ([1], [40], 1500)])
def test_two_tiles_of_few_columns(gpu_device, rows, lens, prefix, H, fmt):
    base.test_two_tiles_of_few_columns(gpu_device, rows, lens, prefix, H, 1, 32, F32, fmt)


@both_formats
@pytest.mark.parametrize("rows,lens,page", [([1, 1, 1], [5001, 2, 3000], 16), ([1], [9000], 8), ([300, 1, 1], [2500, 1800, 40], 32), ([700], [700], 64), ([257, 100], [5000, 4500], 8)])
def test_long_caches(gpu_device, rows, lens, page, fmt):
    base.test_long_caches(gpu_device, rows, lens, page, 6, 2, 32, F32, fmt)


@both_formats
def test_bad_pages_and_lengths(gpu_device, fmt):
    x = QuantBatch(fmt, [1, 5, 1, 2, 1], [50, 40, 30, 60, 20], 6, 2, 32, 16, F32, gpu_device, seed=7)
    clean, rows = attend(x), read(x, dtype=F32)
    x.block_table[0, 1], x.block_table[1, 2], x.kv_len[2], x.kv_len[3] = x.n_pages, -1, -3, x.width * 16 + 1
    y, lse = attend(x, return_lse=True)
    assert y[:9].isnan().all() and lse[:9].isnan().all() and torch.equal(y[9:], clean[9:])
    for got, want in zip(read(x, dtype=F32), rows):
        assert torch.equal(got[0], want[0]) and got[1:9].isnan().all() and torch.equal(got[9:], want[9:])


@both_formats
def test_codes_of_all_kinds_of_values(gpu_device, fmt):
    base.test_codes_of_all_kinds_of_values(gpu_device, fmt, F32, 32)


@both_formats
def test_keys_next_to_a_border(gpu_device, fmt):
    T = 4096
    x = QuantBatch(fmt, [T], [T], 2, 2, 32, 64, F32, gpu_device)
    x.k = (x.k * (1 + torch.arange(T, device=gpu_device)[:, None, None] / T)).contiguous()
    want = x.appended_codes(eps=0.5)
    append(x, eps=0.5)
    check_pools(x, want)


@both_formats
def test_many_sequences_rows_in_none_and_strides(gpu_device, fmt):
    x = QuantBatch(fmt, [(0, 1, 1, 3, 12)[i % 5] for i in range(300)], [30 + 17 * i % 90 for i in range(300)], 4, 2, 32, 16, F32, gpu_device, seed=60, layout="apart")
    x.q = x.q.transpose(0, 1).contiguous().transpose(0, 1)
    y, lse = attend(x, gate_logits=x.gate, return_lse=True)
    check_y(x, y, lse, x.attended(gate=True))
    want = x.appended_codes(mix=True)
    append(x, v_first=x.v_first, vr_coef=x.coef)
    check_pools(x, want)
    x = QuantBatch(fmt, [1, 3, 9], [20, 40, 9], 6, 2, 32, 16, F32, gpu_device, seed=61)
    x.seq_start = torch.tensor([2, 3, 6, 8], dtype=torch.int32, device=gpu_device)
    out, k, v = torch.full_like(x.q, 7.0), *(torch.full((13, 2, 32), 7.0, device=gpu_device) for _ in "kv")
    y = attend(x)
    assert attend(x, out=out) is out and (out[[0, 1, 8, 12]] == 7).all() and (y[[0, 1, 8, 12]] == 0).all() and torch.equal(y[2:8], out[2:8])
    read(x, out=(k, v))
    assert (k[[0, 1, 8, 12]] == 7).all() and torch.equal(k[2:8], read(x, dtype=F32)[0][2:8])


@both_formats
def test_a_captured_step(gpu_device, fmt):
    x = QuantBatch(fmt, [1, 1, 1], [30, 200, 65], 6, 2, 32, 16, F32, gpu_device, seed=62, uniform=True)

    def step():
        append(x)
        return attend(x, gate_logits=x.gate), *read(x, dtype=F32)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for i in range(4):
        x.kv_len.sub_(1)
        for t in (x.q, x.k):
            t.copy_(torch.randn_like(t))
        g.replay()
        got = [t.clone() for t in y]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


@both_formats
def test_cache_and_module(gpu_device, fmt):
    """Heads of 32 through the cache: read, turned into other types and back, and under the module, against the module over an fp32 cache of the same values."""
    torch.manual_seed(63)
    d, H, Hkv = 192, 6, 2
    m = MultiHeadSelfAttention(d, H, Hkv, max_seq_len=256, qknorm=True, device=gpu_device, dtype=F32)
    with torch.no_grad():
        pages = PageTable(3, 60, 16, prefix_len=37, device=gpu_device)
        cache = PagedKVCache(pages, Hkv, 32, DTYPES[fmt])
        pages.prefix.extend(37)
        m(torch.randn(1, 37, d, device=gpu_device), kv_cache=cache.of(pages.prefix))
        for rows in ([20, 1, 33], 1, [3, 0, 2]):
            pages.extend(rows)
            x = torch.randn(1, pages.rows, d, device=gpu_device)
            y, _ = m(x, kv_cache=cache)
            plain = cache.to(F32)
            assert plain.dtype == F32 and cache.read()[0].dtype == F32 and all(torch.equal(a, b) for a, b in zip(cache.read()[:2], plain.read()[:2]))
            plain.append = lambda *a, **kw: None
            want, _ = m(x, kv_cache=plain)
            assert (y - want).norm() <= 1e-5 * want.norm()
            again = plain.to(DTYPES[fmt])
            for a, b in zip(again.read()[:2], cache.read()[:2]):
                assert torch.equal(a, b)
        other = cache.to(DTYPES["e2m1" if fmt == "e4m3" else "e4m3"])
        for got, ref in zip(other.read()[:2], cache.read()[:2]):
            to = "e2m1" if fmt == "e4m3" else "e4m3"
            assert torch.equal(got.to(F64), decode(*encode(ref.to(F64), to), to))


def test_only_float32_rows_have_heads_of_32(gpu_device):
    x = QuantBatch("e4m3", [1, 2], [20, 30], 6, 2, 32, 16, F32, gpu_device, seed=64)
    from sample_efficient_gpt_amd._lib import SegptError

    with pytest.raises(SegptError, match="head"):
        base.paged_attention(x.q.to(BF16), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales())
    with pytest.raises(SegptError, match="head"):
        paged_kv_append(x.k.to(BF16), x.v.to(BF16), x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start, **x.scales())
    with pytest.raises(SegptError, match="head"):
        read(x, dtype=BF16)
