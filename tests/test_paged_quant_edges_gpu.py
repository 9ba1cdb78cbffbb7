"""Paged caches of 8 and 4 bits, on the GPU: page numbers and values that are none, in calls of many columns and at the edge of what a row sees; items of
more tiles than a wave holds page numbers for.  Helpers and tolerances are those of tests/test_paged_quant_gpu.py."""

import math

import pytest
import torch

from paged_quant_util import QuantBatch
from test_paged_quant_gpu import BF16, F32, attend, both_formats, read

pytestmark = pytest.mark.gpu


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", [(6, 2, 64, BF16), (4, 2, 128, BF16), (4, 2, 64, F32), (4, 2, 128, F32)])
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
