"""Heads of 32 in the C ABI of paged caches of 8 and 4 bits, no GPU: asked for by a flag, for fp32 rows; every call returns from the host-side checks."""

import pytest

from paged_quant_util import FORMATS
from sample_efficient_gpt_amd import _lib
from test_paged import _params
from test_paged_quant import _quant, lib  # noqa: F401


def _small(flag, dtype=_lib.SEGPT_DTYPE_FP32):
    p = _params(dtype, 32)
    p.flags = flag
    return p


@pytest.mark.parametrize("fmt", FORMATS)
def test_heads_of_32_are_asked_for(lib, fmt):  # noqa: F811
    flag, q, t = _lib.SEGPT_FLAG_HEAD_32, _quant(fmt, 32), _lib.Tensor4
    calls = (lib.segpt_paged_append_quant, lib.segpt_paged_attn_quant, lib.segpt_paged_read)
    assert lib.segpt_paged_quant_workspace_bytes(_small(0), q) == 0
    need = lib.segpt_paged_quant_workspace_bytes(_small(flag), q)
    assert need > 0 and need % 256 == 0
    for f in calls:
        assert f(_small(0), q, None) == -5
        assert f(_small(flag, _lib.SEGPT_DTYPE_BF16), q, None) == -5
        row = 32 if fmt == "e4m3" else 16
        for pages, code in ((t(0x10000, 32 * row, 16 * row, row - 16), -6), (t(0x10000, 32 * row + 8, 16 * row, row), -6), (t(0x10008, 32 * row, 16 * row, row), -10)):
            p = _small(flag)
            p.v_pages = pages
            assert f(p, q, None) == code, pages
        for scales, code in ((t(None, 32, 16, 1), -1), (t(0x30000, 32, 16, 0), -6), (t(0x30000, -32, 16, 1), -6)):
            bad = _quant(fmt, 32)
            bad.v_scales = scales
            assert f(_small(flag), bad, None) == code, scales
    p = _small(flag)
    p.workspace_bytes = need - 1
    assert lib.segpt_paged_attn_quant(p, q, None) == -7
    over = _quant(fmt, 32)
    over.k_scales = t(0x30000, 0, 16, 1)  # pages over one another: read, but not written
    assert lib.segpt_paged_append_quant(_small(flag), over, None) == -6
    assert lib.segpt_paged_workspace_bytes(_small(flag)) == lib.segpt_paged_workspace_bytes(_small(0)) > 0  # the calls without scales do not look at it
