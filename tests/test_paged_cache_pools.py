"""PagedKVCache around pools that are handed in, no GPU: which it takes, under which tables, and what type it says it has."""

import pytest
import torch

from sample_efficient_gpt_amd import PagedKVCache, PageTable

E4M3, E2M1 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2


def _pools(n, Hkv, page, row, dtype):
    return tuple(torch.zeros(n, Hkv, page, row, dtype=torch.uint8).view(dtype) if dtype != torch.bfloat16 else torch.zeros(n, Hkv, page, row, dtype=dtype) for _ in "kv")


def test_a_pool_of_rows_may_be_larger_than_its_table():
    """One pool under tables that hand out different parts of it, as it was taken before there were pools with scales."""
    t, small = PageTable(2, 40, 16, device="cpu"), PageTable(1, 16, 16, device="cpu")
    k, v = _pools(t.n_pages + 9, 2, 16, 64, torch.bfloat16)
    c = PagedKVCache(t, 2, 64, k_pages=k, v_pages=v)
    assert c.k_pages is k and c.v_pages is v and c.dtype == torch.bfloat16 and c.k_scales is None and c.head_dim == 64
    again = c.of(small)
    assert again.pages is small and again.k_pages is k and again.v_pages is v
    f = PagedKVCache(t, 2, 64, k_pages=k.float(), v_pages=v.float())  # the pool's type counts
    assert f.dtype == torch.float32 and f.k_scales is None and f.of(small).dtype == torch.float32


@pytest.mark.parametrize("dtype,row", [(E4M3, 64), (E2M1, 32)])
def test_so_may_one_with_scales(dtype, row):
    t = PageTable(2, 40, 16, prefix_len=20, device="cpu")
    k, v = _pools(t.n_pages + 3, 2, 16, row, dtype)
    scales = tuple(torch.zeros(t.n_pages + 3, 2, 16, 2, dtype=torch.uint8) for _ in "kv")
    c = PagedKVCache(t, 2, 64, dtype, k, v, *scales)
    assert c.of(t.prefix).k_pages is k and c.of(t.prefix).k_scales is scales[0]
    c = PagedKVCache(t, 2, 64, dtype, k, v)
    assert c.k_scales.shape == c.v_scales.shape == (t.n_pages + 3, 2, 16, 2)


def test_pools_that_do_not_fit_are_refused():
    t = PageTable(2, 40, 16, device="cpu")
    k, v = _pools(t.n_pages, 2, 16, 64, E4M3)
    with pytest.raises(ValueError, match="pages"):
        PagedKVCache(t, 2, 64, E4M3, k, v[:, :1])
    with pytest.raises(ValueError, match="page size"):
        PagedKVCache(PageTable(2, 40, 8, device="cpu"), 2, 64, E4M3, k, v)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCache(t, 2, 64, E4M3, k, v, torch.zeros(t.n_pages, 2, 16, 4, dtype=torch.uint8))
