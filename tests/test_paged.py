"""Host side of the paged cache, no GPU: what the C ABI refuses, the struct's layout, the table that hands out pages."""

import os
import re

import pytest
import torch

from sample_efficient_gpt_amd import PagedKVCache, PageTable, _lib, paged_attention, paged_kv_append

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _params(dtype=_lib.SEGPT_DTYPE_BF16, D=64):
    """Plausible params with addresses that are never looked at: every call below returns from the host-side checks."""
    import ctypes as C

    p = _lib.PagedParams()
    p.struct_bytes = C.sizeof(p)
    p.dtype, p.D = dtype, D
    p.T, p.B, p.H, p.Hkv = 8, 4, 6, 2
    p.n_pages, p.page_size, p.table_width = 10, 16, 5
    p.gq_numel, p.eps, p.sm_scale, p.gate_scale = D, 1e-6, 0.125, 2.0
    p.k_pages = p.v_pages = _lib.Tensor4(0x10000, 2 * 16 * D, 16 * D, D)
    p.block_table = p.kv_len = p.seq_start = p.g_q = 0x20000
    p.table_stride = 5
    p.k = p.v = _lib.Rows(0x10000, 2 * D, D)
    p.q = p.o = _lib.Rows(0x10000, 6 * D, D)
    p.workspace, p.workspace_bytes = 0x40000, 1 << 40
    return p


def _struct_names(name):
    text = open(os.path.join(ROOT, "include", "segpt_attn.h")).read()
    body = text[text.index("typedef struct %s {" % name): text.index("} %s;" % name)]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    names = []
    for decl in body.split(";"):
        first, *rest = decl.strip().split(",")
        if first:
            names.append(re.findall(r"(\w+)\s*$", first.strip())[0])
            names += [r.strip().lstrip("*") for r in rest]
    return names


def test_structs_match_the_header():
    assert _struct_names("segpt_paged_params") == [f[0] for f in _lib.PagedParams._fields_]
    assert _struct_names("segpt_rows") == [f[0] for f in _lib.Rows._fields_]
    text = open(os.path.join(ROOT, "include", "segpt_attn.h")).read()
    for name in ("SEGPT_FLAG_ZERO_REST", "SEGPT_E_PAGES"):
        assert int(re.search(r"#define\s+%s\s+(-?\d+)" % name, text)[1]) == getattr(_lib, name)


BOTH = [  # what either call refuses
    (dict(struct_bytes=8), -2), (dict(dtype=5), -3), (dict(T=0), -4), (dict(B=0), -4), (dict(Hkv=0), -4), (dict(Hkv=70000), -4),
    (dict(T=1 << 30, B=1), -4), (dict(seq_start=None, T=7), -4), (dict(D=48), -5), (dict(D=32), -5),
    (dict(n_pages=0), -14), (dict(page_size=12), -14), (dict(page_size=4), -14), (dict(page_size=1 << 17), -14), (dict(page_size=-16), -14),
    (dict(table_width=0), -14), (dict(table_width=1 << 28), -14), (dict(max_len=-1), -14),
    (dict(block_table=None), -1), (dict(kv_len=None), -1), (dict(table_stride=-1), -6), (dict(kv_len=0x20002), -10), (dict(block_table=0x20001), -10), (dict(seq_start=0x20002), -10),
    (dict(k_pages=_lib.Tensor4(None, 2048, 1024, 64)), -1), (dict(v_pages=_lib.Tensor4(0x10008, 2048, 1024, 64)), -10),
    (dict(k_pages=_lib.Tensor4(0x10000, 2048, 1024, 60)), -6), (dict(k_pages=_lib.Tensor4(0x10000, 2052, 1024, 64)), -6),
    (dict(v_pages=_lib.Tensor4(0x10000, -2048, 1024, 64)), -6), (dict(v_pages=_lib.Tensor4(0x10000, 2048, 1024, 1 << 27)), -6),
    (dict(rope_cos=0x50000, rope_len=100), -12), (dict(rope_cos=0x50000, rope_sin=0x60000, rope_len=79), -12),
    (dict(rope_cos=0x50000, rope_sin=0x60000, rope_len=80, rope_pos0=1), -12), (dict(rope_cos=0x50000, rope_sin=0x60004, rope_len=80), -12),
    (dict(rope_cos=0x50000, rope_sin=0x60000, rope_len=80, rope_pos0=-1), -12), (dict(rope_cos=0x50000, rope_sin=0x60000, rope_len=39, max_len=40), -12),
]
APPEND = [
    (dict(k=_lib.Rows(None, 128, 64)), -1), (dict(v=_lib.Rows(0x10002, 128, 64)), -10), (dict(k=_lib.Rows(0x10000, 130, 64)), -6), (dict(v=_lib.Rows(0x10000, 128, -64)), -6),
    (dict(v_first=_lib.Rows(0x10000, 128, 64)), -8), (dict(vr_coef=0x10000), -8), (dict(v_first=_lib.Rows(0x10008, 128, 64), vr_coef=0x10000), -10),
    (dict(k_pages=_lib.Tensor4(0x10000, 0, 1024, 64)), -6), (dict(v_pages=_lib.Tensor4(0x10000, 1024, 1024, 64)), -6), (dict(k_pages=_lib.Tensor4(0x10000, 2048, 64, 64)), -6),
]
ATTEND = [
    (dict(H=0), -4), (dict(H=5), -4), (dict(H=70000, Hkv=2), -4), (dict(gq_numel=3), -4), (dict(gk_numel=1), -4), (dict(g_k=0x10000), -4), (dict(g_q=None), -1),
    (dict(prefix_len=5), -8), (dict(prefix_table=0x20000), -8), (dict(prefix_table=0x20000, prefix_len=-1), -14), (dict(prefix_table=0x20001, prefix_len=5), -10),
    (dict(q=_lib.Rows(None, 384, 64)), -1), (dict(q=_lib.Rows(0x10000, 380, 64)), -6), (dict(o=_lib.Rows(0x10004, 384, 64)), -10), (dict(o=_lib.Rows(0x10000, 0, 64)), -6),
    (dict(o=_lib.Rows(0x10000, 384, 32)), -6), (dict(gate=_lib.Rows(0x10000, -6, 1)), -6), (dict(workspace=None), -7), (dict(workspace_bytes=100), -7), (dict(workspace=0x40010), -10),
    (dict(rope_cos=0x50000, rope_sin=0x60000, rope_len=84, prefix_table=0x20000, prefix_len=5), -12),
]


def test_bad_arguments_are_refused_before_any_launch(lib):
    calls = {"append": lib.segpt_paged_append, "attn": lib.segpt_paged_attn}
    for f in calls.values():
        assert f(None, None) == -1
    for name, cases in (("append", BOTH + APPEND), ("attn", BOTH + ATTEND)):
        for change, code in cases:
            p = _params()
            for key, value in change.items():
                setattr(p, key, value)
            assert calls[name](p, None) == code, (name, change)
    p = _params(_lib.SEGPT_DTYPE_FP32, 32)
    p.k = _lib.Rows(0x10000, 64, 30)  # fp32: rows of whole 16-byte pieces
    assert lib.segpt_paged_append(p, None) == -6


def test_workspace_bytes(lib):
    p = _params()
    need = lib.segpt_paged_workspace_bytes(p)
    assert need > 0 and need % 256 == 0
    p.T = 1 << 20  # prompts of a million rows whose keys are not shared out leave no partial results: scratch does not grow with them
    long = lib.segpt_paged_workspace_bytes(p)
    assert long < 1 << 30
    p.prefix_table, p.prefix_len = 0x20000, 100  # beside a prefix every row leaves some
    assert lib.segpt_paged_workspace_bytes(p) > p.T * p.H * (p.D + 2) * 4
    for change in (dict(struct_bytes=4), dict(T=0), dict(H=5), dict(dtype=9), dict(page_size=0), dict(table_width=0)):
        q = _params()
        for key, value in change.items():
            setattr(q, key, value)
        assert lib.segpt_paged_workspace_bytes(q) == 0


def test_host_tensors_are_refused():
    z = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="device tensors"):
        paged_attention(z, pages, pages, table, lens, torch.ones(1))
    with pytest.raises(AssertionError, match="device tensors"):
        paged_kv_append(z, z, pages, pages, table, lens)


def _pages_are_consistent(t):
    held = [p for pages in t._pages for p in pages] + ([] if t.prefix is None else t.prefix._pages[0])
    assert sorted(held + t._free) == list(range(t.n_pages))
    for b, (n, pages) in enumerate(zip(t.lengths, t._pages)):
        assert len(pages) == -(-n // t.page_size)
        assert t.block_table[b, : len(pages)].tolist() == pages
    assert t.kv_len.tolist() == t.lengths


def test_page_table_hands_out_and_takes_back():
    t = PageTable(3, 100, 16, n_pages=9, device="cpu")
    t.extend([17, 0, 1])
    assert t.seq_start.tolist() == [0, 17, 17, 18] and t.rows == 18
    _pages_are_consistent(t)
    t.extend(1)
    assert t.seq_start is None and t.rows == 3 and t.lengths == [18, 1, 2]
    _pages_are_consistent(t)
    with pytest.raises(RuntimeError, match="full"):
        t.extend([100 - 18, 30, 16])  # 5 + 1 + 1 pages more, five are free
    assert t.lengths == [18, 1, 2] and t.rows == 3
    _pages_are_consistent(t)
    with pytest.raises(RuntimeError, match="room for 100"):
        t.extend([83, 0, 0])
    t.release(0)
    _pages_are_consistent(t)
    t.extend([100, 1, 1])
    _pages_are_consistent(t)
    for bad in ([1, 1], [1, -1, 1]):
        with pytest.raises(ValueError):
            t.extend(bad)


def test_page_table_with_a_prefix():
    t = PageTable(2, 40, 16, prefix_len=33, device="cpu")
    assert t.n_pages == 2 * 3 + 3 and t.prefix_table.tolist() == t.prefix._pages[0] and len(t.prefix._pages[0]) == 3
    t.prefix.extend(20).extend(13)
    assert t.prefix.lengths == [33] and t.prefix.kv_len.tolist() == [33]
    t.extend(40)
    assert not t._free and len({*t._pages[0], *t._pages[1], *t.prefix._pages[0]}) == 9
    with pytest.raises(RuntimeError):
        t.prefix.extend(1)
    for bad in (dict(page_size=12), dict(page_size=4), dict(max_len=0), dict(batch=0), dict(prefix_len=-1), dict(prefix_len=100, n_pages=3)):
        with pytest.raises(ValueError):
            PageTable(**{**dict(batch=2, max_len=40, page_size=16, device="cpu"), **bad})


def test_cache_shapes():
    t = PageTable(2, 40, 16, prefix_len=20, device="cpu")
    c = PagedKVCache(t, 2, 64)
    assert c.k_pages.shape == (t.n_pages, 2, 16, 64) and c.of(t.prefix).k_pages is c.k_pages
    with pytest.raises(ValueError):
        PagedKVCache(t, 2, 64, k_pages=torch.zeros(1, 2, 16, 64), v_pages=torch.zeros(1, 2, 16, 64))
    t.extend(1)
    with pytest.raises(AssertionError, match="extended for 2 rows"):
        c.append(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64))
    with pytest.raises(AssertionError, match="holds 0 of its 20"):
        c.attend(torch.zeros(2, 2, 64), torch.ones(1))


def test_workspace_bytes_of_sizes_that_no_call_has(lib):
    """Without seq_start the rows are the same number for every sequence: fewer rows than sequences, or no multiple, is no shape."""
    for change in (dict(seq_start=None, T=1, B=2), dict(seq_start=None, T=7), dict(D=48), dict(page_size=12), dict(max_len=-1), dict(T=1 << 30, B=1),
                   dict(B=(1 << 24) + 1), dict(table_width=1 << 28), dict(prefix_table=0x20000, prefix_len=-1)):
        p = _params()
        for key, value in change.items():
            setattr(p, key, value)
        assert lib.segpt_paged_workspace_bytes(p) == 0, change
        assert lib.segpt_paged_attn(p, None) < 0, change
    p = _params()
    p.seq_start = p.k_pages.ptr = p.block_table = None  # addresses do not matter
    assert lib.segpt_paged_workspace_bytes(p) > 0


def test_launches_of_more_threads_than_one_may_have(lib):
    """2^32 and more: refused before anything is launched."""
    def change(**kw):
        p = _params()
        for key, value in kw.items():
            setattr(p, key, value)
        return p

    huge = dict(T=1 << 24, B=1 << 24, H=4, Hkv=4, workspace_bytes=(1 << 63) - 1)
    for kw in (huge, dict(huge, H=1, Hkv=1, prefix_table=0x20000, prefix_len=8), dict(huge, seq_start=None), dict(T=1 << 28, B=1, H=4, Hkv=4, prefix_table=0x20000, prefix_len=8)):
        p = change(**kw)
        p.q = p.o = _lib.Rows(0x10000, p.H * 64, 64)
        assert lib.segpt_paged_workspace_bytes(p) == 0 and lib.segpt_paged_attn(p, None) == -4, kw
    p = change(T=1 << 24, B=1 << 22, H=1, Hkv=1)
    assert lib.segpt_paged_workspace_bytes(p) > 0
    p = change(T=1 << 28, B=1, Hkv=4, D=128)
    p.k_pages = p.v_pages = _lib.Tensor4(0x10000, 4 * 16 * 128, 16 * 128, 128)
    p.k = p.v = _lib.Rows(0x10000, 4 * 128, 128)
    assert lib.segpt_paged_append(p, None) == -4


def test_page_table_keeps_the_row_ranges_that_it_handed_out():
    """A captured step holds on to ``seq_start``: it has to follow steps with one number for all sequences as well."""
    t = PageTable(3, 100, 16, device="cpu")
    t.extend(2)
    assert t.seq_start is None
    t.extend([2, 0, 1])
    held = t.seq_start
    assert held.tolist() == [0, 2, 2, 3]
    t.extend(1)
    assert t.seq_start is None and held.tolist() == [0, 1, 2, 3]
    t.extend([0, 0, 5])
    assert t.seq_start is held and held.tolist() == [0, 0, 0, 5]
    t.extend(0)
    assert held.tolist() == [0, 0, 0, 0] and t.kv_len.tolist() == [5, 3, 9] == t.lengths


def test_a_gradient_is_refused_before_anything_else():
    """Also where the call is made as a registered operator, which runs below autograd: an append would drop the gradient without a word."""
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    z, g = (torch.zeros(2, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    g.requires_grad_()
    calls = [lambda: paged_kv_append(g, z, pages, pages, table, lens), lambda: paged_kv_append(z, z, pages, pages, table, lens, v_first=g, vr_coef=torch.ones(2)),
             lambda: paged_attention(g, pages, pages, table, lens, torch.ones(1)), lambda: paged_attention(z, pages, pages, table, lens, torch.ones(1, requires_grad=True))]
    for call in calls:
        with pytest.raises(AssertionError, match="no derivative"):
            call()
        with torch.no_grad(), pytest.raises(AssertionError, match="device tensors"):
            call()


def test_module_refuses_rows_in_another_order():
    """Rows of a step with unequal numbers are packed; [B, S, d] is for S rows of every sequence."""
    from sample_efficient_gpt_amd import MultiHeadSelfAttention

    m = MultiHeadSelfAttention(128, 2, 2, max_seq_len=64, qknorm=True)
    t = PageTable(3, 64, 16, device="cpu")
    c = PagedKVCache(t, 2, 64)
    with torch.no_grad():
        t.extend([4, 1, 1])
        for shape in ((3, 2), (2, 3), (6, 1)):
            with pytest.raises(ValueError, match="1, 6, 128"):
                m(torch.zeros(*shape, 128), kv_cache=c)
        t.extend(2)
        for shape in ((2, 3), (6, 1)):
            with pytest.raises(ValueError, match="3, 2, 128"):
                m(torch.zeros(*shape, 128), kv_cache=c)
