"""Host side of the paged caches of 8 and 4 bits, no GPU: what the C ABI and the functions refuse, the structs' layout, the tests' own definition."""

import ctypes as C
import os
import re

import pytest
import torch

from paged_quant_util import FORMATS, NUMBERS, QuantBatch, decode, encode
from sample_efficient_gpt_amd import PagedKVCache, PageTable, _lib, paged_attention, paged_kv_append, paged_kv_read
from test_paged import APPEND, ATTEND, BOTH, _params, _struct_names

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"e4m3": torch.float8_e4m3fn, "e2m1": torch.float4_e2m1fn_x2}


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _quant(fmt, D=64):
    q = _lib.PagedQuant()
    q.struct_bytes = C.sizeof(q)
    q.format = {"e4m3": _lib.SEGPT_POOL_E4M3, "e2m1": _lib.SEGPT_POOL_E2M1}[fmt]
    q.k_scales = q.v_scales = _lib.Tensor4(0x30000, 2 * 16 * D // 32, 16 * D // 32, D // 32)
    return q


def test_structs_match_the_header():
    assert _struct_names("segpt_paged_quant") == [f[0] for f in _lib.PagedQuant._fields_]
    text = open(os.path.join(ROOT, "include", "segpt_attn.h")).read()
    for name in ("SEGPT_SCALE_BLOCK", "SEGPT_POOL_E4M3", "SEGPT_POOL_E2M1"):
        assert int(re.search(r"#define\s+%s\s+(-?\d+)" % name, text)[1]) == getattr(_lib, name)


@pytest.mark.parametrize("fmt", FORMATS)
def test_bad_arguments_are_refused_before_any_launch(lib, fmt):
    calls = {"append": lib.segpt_paged_append_quant, "attn": lib.segpt_paged_attn_quant, "read": lib.segpt_paged_read}
    for name, cases in (("append", BOTH + APPEND), ("attn", BOTH + ATTEND)):
        assert calls[name](None, None, None) == -1
        for change, code in cases:
            p = _params()
            for key, value in change.items():
                setattr(p, key, value)
            # strides are bytes here: those of the cases are of rows of 64, whole 16-byte pieces where theirs are
            if code == -6 and any(k.endswith("_pages") for k in change) and fmt == "e2m1":
                continue
            assert calls[name](p, _quant(fmt), None) == code, (name, change)
    t = _lib.Tensor4
    for name, f in calls.items():
        p = _params()
        assert name == "read" or f(p, None, None) == -1
        p.D = 32
        p.dtype = _lib.SEGPT_DTYPE_FP32
        assert f(p, _quant(fmt), None) == -5
        row = 64 if fmt == "e4m3" else 32
        for change, code in [(dict(struct_bytes=8), -2), (dict(format=0), -3), (dict(format=3), -3), (dict(k_scales=t(None, 64, 32, 2)), -1), (dict(v_scales=t(0x30001, 64, 32, 2)), -10),
                             (dict(k_scales=t(0x30000, 64, 32, 1)), -6), (dict(k_scales=t(0x30000, 63, 32, 2)), -6), (dict(v_scales=t(0x30000, 64, -32, 2)), -6),
                             (dict(v_scales=t(0x30000, 64, 32, 3)), -6)]:
            q = _quant(fmt)
            for key, value in change.items():
                setattr(q, key, value)
            assert f(_params(), q, None) == code, (name, change)
        for pages, code in ((t(0x10000, 32 * row, 16 * row, row - 16), -6), (t(0x10000, 32 * row + 8, 16 * row, row), -6), (t(0x10008, 32 * row, 16 * row, row), -10)):
            p = _params()
            p.v_pages = pages
            assert f(p, _quant(fmt), None) == code, (name, pages)
    q = _quant(fmt)
    q.v_scales = t(0x30000, 0, 32, 2)  # pages over one another: read, but not written
    assert calls["append"](_params(), q, None) == -6
    p = _params()
    p.k = _lib.Rows(0x10000, 64, 64)  # rows over one another
    assert calls["read"](p, _quant(fmt), None) == -6 and calls["read"](p, None, None) == -6


@pytest.mark.parametrize("fmt", FORMATS)
def test_workspace_bytes(lib, fmt):
    need = lib.segpt_paged_quant_workspace_bytes(_params(), _quant(fmt))
    assert need > 0 and need % 256 == 0
    for change in (dict(struct_bytes=4), dict(T=0), dict(H=5), dict(dtype=9), dict(page_size=0), dict(table_width=0), dict(seq_start=None, T=7), dict(dtype=_lib.SEGPT_DTYPE_FP32, D=32)):
        p = _params()
        for key, value in change.items():
            setattr(p, key, value)
        assert lib.segpt_paged_quant_workspace_bytes(p, _quant(fmt)) == 0, change
    for change in (dict(struct_bytes=1), dict(format=7)):
        q = _quant(fmt)
        for key, value in change.items():
            setattr(q, key, value)
        assert lib.segpt_paged_quant_workspace_bytes(_params(), q) == 0
    assert lib.segpt_paged_quant_workspace_bytes(_params(), None) == 0
    p = _params()
    p.workspace_bytes = need - 1
    assert lib.segpt_paged_attn_quant(p, _quant(fmt), None) == -7
    huge = _params()
    huge.T = huge.B = 1 << 24
    huge.H = huge.Hkv = 4
    huge.q = huge.o = _lib.Rows(0x10000, 4 * 64, 64)
    huge.workspace_bytes = (1 << 63) - 1
    assert lib.segpt_paged_quant_workspace_bytes(huge, _quant(fmt)) == 0 and lib.segpt_paged_attn_quant(huge, _quant(fmt), None) == -4


def test_launches_of_more_threads_than_one_may_have(lib):
    p = _params(D=128)
    p.T, p.B, p.Hkv = 1 << 28, 1, 4
    p.k_pages = p.v_pages = _lib.Tensor4(0x10000, 4 * 16 * 128, 16 * 128, 128)
    p.k = p.v = _lib.Rows(0x10000, 4 * 128, 128)
    q = _quant("e4m3", 128)
    q.k_scales = q.v_scales = _lib.Tensor4(0x30000, 4 * 16 * 4, 16 * 4, 4)
    for call in (lib.segpt_paged_append_quant, lib.segpt_paged_read):
        assert call(p, q, None) == -4


def test_host_tensors_are_refused():
    z = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    scales = torch.zeros(3, 2, 16, 2, dtype=torch.uint8)
    for pages in (torch.zeros(3, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(3, 2, 16, 32, dtype=torch.uint8)):
        kw = dict(k_scales=scales, v_scales=scales.clone())
        with pytest.raises(AssertionError, match="device tensors"):
            paged_attention(z, pages, pages, table, lens, torch.ones(1), **kw)
        with pytest.raises(AssertionError, match="device tensors"):
            paged_kv_append(z, z, pages, pages, table, lens, **kw)
        with pytest.raises(AssertionError, match="device tensors"):
            paged_kv_read(pages, pages, table, lens, 2, **kw)
        with pytest.raises(AssertionError, match="go together"):
            paged_kv_append(z, z, pages, pages, table, lens, k_scales=scales)
        g = z.clone().requires_grad_()
        with pytest.raises(AssertionError, match="no derivative"):
            paged_kv_append(g, z, pages, pages, table, lens, **kw)
        with pytest.raises(AssertionError, match="no derivative"):
            paged_attention(g, pages, pages, table, lens, torch.ones(1), **kw)


def test_cache_shapes():
    t = PageTable(2, 40, 16, prefix_len=20, device="cpu")
    for fmt, width in (("e4m3", 64), ("e2m1", 32)):
        c = PagedKVCache(t, 2, 64, DTYPES[fmt])
        assert c.k_pages.shape == (t.n_pages, 2, 16, width) and c.k_scales.shape == c.v_scales.shape == (t.n_pages, 2, 16, 2) and c.dtype == DTYPES[fmt]
        same = c.of(t.prefix)
        assert same.k_pages is c.k_pages and same.v_scales is c.v_scales and same.head_dim == 64 and same.dtype == c.dtype
        with pytest.raises(ValueError, match="scales"):
            PagedKVCache(t, 2, 64, DTYPES[fmt], k_scales=torch.zeros(1, 2, 16, 2, dtype=torch.uint8))
    c = PagedKVCache(t, 2, 64)
    assert c.k_scales is None and c.to(torch.bfloat16) is c and c.to(torch.float8_e4m3fn).k_scales is not None  # nothing is held yet


@pytest.mark.parametrize("fmt", FORMATS)
def test_the_definition_itself(fmt):
    """The nearest number of all there are, by looking at every one of them; for 8 bits also torch's own conversion."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 64, generator=g, dtype=torch.float64) * 2.0 ** torch.randint(-20, 20, (64, 1), generator=g)
    x[0], x[1, :32], x[2, 5] = 0.0, torch.arange(32) / 8, torch.nan
    codes, scales = encode(x, fmt)
    assert scales[2, 0] == 255 and (scales[2, 1] != 255)
    x[2, 5] = 0.0
    codes, scales = encode(x, fmt)
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127).repeat_interleave(32, -1)
    top = NUMBERS[fmt][-1]
    big = x.abs().unflatten(-1, (2, 32)).amax(-1)
    assert (big <= top * s[:, ::32]).all() and ((big > top * s[:, ::32] / 2) | (scales == 17)).all()
    every = torch.cat([NUMBERS[fmt], -NUMBERS[fmt]])
    nearest = ((x / s)[..., None] - every).abs().amin(-1)
    got = decode(codes, scales, fmt)
    assert torch.equal((x - got).abs() / s, nearest)
    if fmt == "e4m3":
        assert torch.equal((x / s).float().to(torch.float8_e4m3fn).float().double() * s, got)


def test_batches():
    x = QuantBatch("e2m1", [3, 1], [20, 5], 4, 2, 64, 16, torch.bfloat16, "cpu", layout="apart")
    assert x.k_pages.shape[3] == 32 and not x.k_pages.is_contiguous()
    k, v = x.values()
    codes, scales = encode(k, "e2m1")
    # stored values are stored again as they are; a block whose largest was rounded down to 3 gets the next smaller scale, on whose grid all of it lies
    assert torch.equal(decode(codes, scales, "e2m1"), k) and (scales <= x.k_scales).all()
