"""PagedKVCache around pools that are handed in, no GPU: which it takes, under which tables, and what type it says it has."""

import pytest
import torch

from sample_efficient_gpt_amd import PagedKVCache, PageTable

E4M3, E2M1 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2


def _pools(n, Hkv, page, row, dtype):
    return tuple(torch.zeros(n, Hkv, page, row, dtype=torch.uint8).view(dtype) if dtype != torch.bfloat16 else torch.zeros(n, Hkv, page, row, dtype=dtype) for _ in "kv")


@pytest.mark.parametrize("dtype,row", [(E4M3, 64), (E2M1, 32), (torch.uint8, 32)])
def test_pools_with_scales(dtype, row):
    t = PageTable(2, 40, 16, prefix_len=20, device="cpu")
    k, v = _pools(t.n_pages, 2, 16, row, dtype)
    scales = tuple(torch.zeros(t.n_pages, 2, 16, 2, dtype=torch.uint8) for _ in "kv")
    kind = E4M3 if dtype == E4M3 else E2M1
    for given in (dtype, kind, torch.bfloat16):  # the pool's type counts
        c = PagedKVCache(t, 2, 64, given, k, v, *scales)
        assert c.dtype == kind and c.head_dim == 64 and c.k_pages is k and c.v_scales is scales[1]
        p = c.of(t.prefix)
        assert p.pages is t.prefix and p.dtype == kind and p.k_pages is k and p.k_scales is scales[0] and p.head_dim == 64
        assert c.to(kind) is c and c.to(dtype) is c
    c = PagedKVCache(t, 2, 64, dtype, k, v)  # scales of its own, for the pools as they are
    assert c.k_scales.shape == c.v_scales.shape == (t.n_pages, 2, 16, 2)
    c = PagedKVCache(t, 2, 64, dtype, k)
    assert c.v_pages.shape == k.shape and c.v_pages.dtype == k.dtype and c.dtype == kind


def test_bytes_without_pools_are_four_bits():
    t = PageTable(2, 40, 16, device="cpu")
    c = PagedKVCache(t, 2, 64, torch.uint8)
    assert c.dtype == E2M1 and c.k_pages.shape == (t.n_pages, 2, 16, 32) and c.k_scales.shape == (t.n_pages, 2, 16, 2)
    assert c.to(torch.uint8) is c and c.to(E4M3).to(torch.uint8).dtype == E2M1  # nothing is held yet


def test_pools_that_do_not_fit_are_refused():
    t = PageTable(2, 40, 16, device="cpu")
    k, v = _pools(t.n_pages, 2, 16, 64, E4M3)
    with pytest.raises(ValueError, match="pages"):
        PagedKVCache(t, 2, 64, E4M3, k, v[:, :1])
    with pytest.raises(ValueError, match="pages"):
        PagedKVCache(t, 2, 64, E4M3, k, v.view(torch.uint8))
    with pytest.raises(ValueError, match="pages"):
        PagedKVCache(PageTable(2, 40, 8, device="cpu"), 2, 64, E4M3, k, v)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache(t, 2, 64, E4M3, k, v, torch.zeros(t.n_pages, 2, 16, 4, dtype=torch.uint8))
    rows = _pools(t.n_pages, 2, 16, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache(t, 2, 64, torch.bfloat16, *rows, torch.zeros(t.n_pages, 2, 16, 2, dtype=torch.uint8))


def test_types_that_no_call_has_are_refused_before_anything_is_made():
    c = PagedKVCache(PageTable(2, 40, 16, device="cpu"), 2, 64)
    for dtype in (torch.float16, torch.int8, torch.float8_e5m2):
        with pytest.raises(ValueError, match="dtype"):
            c.to(dtype)
    small = PagedKVCache(PageTable(2, 40, 16, device="cpu"), 2, 32, torch.float32)
    assert small.to(E4M3).head_dim == 32
    with pytest.raises(ValueError, match="head_dim"):
        small.to(torch.bfloat16)
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCache(PageTable(2, 40, 16, device="cpu"), 2, 48, torch.float32).to(E4M3)
    for d in (16, 48, 96, 256):
        with pytest.raises(ValueError, match="head_dim"):
            PagedKVCache(PageTable(2, 40, 16, device="cpu"), 2, d, E4M3)
