"""Paged caches of 8 and 4 bits against their definition in float64 (tests/paged_quant_util.py), on the GPU.

Tolerances.  Codes and scales: none.  The kernel works keys and mixed values out in 64 bits, as the definition does, and the two differ in the last
bits of those; a code would differ only if a value lay within 2^-50 of a border.  Reading back: none, stored values are exact in bf16.
Attention, bf16 rows: the query in two parts is off by 2^-14 of a component, a score by 2^-14 S with S = sum |q k'|, a probability by 2^-13 S;
rounded once, where a sequence has more than 32 columns, by 2 h more (numerator and sum; h = 2^-8, half a step), else by 2^-13; y once, h |y|.  W = sum P |v|:
|dy| <= (2^-13 S + 2 h) W + h |y|, held to (2 S + 2) h W + h |y| as for pools of bf16.  That is the worst case with all roundings in one direction; as a whole a result is far nearer, 3e-3 of its
norm for roundings of y and of the probabilities, and twice that is asked for.  fp32 rows: D 2^-24 for sums of D products, as for pools of fp32."""

import math
import random

import pytest
import torch

from paged_quant_util import FORMATS, QuantBatch, decode, encode
from paged_util import EPS, F64
from sample_efficient_gpt_amd import MultiHeadSelfAttention, PagedKVCache, PageTable, paged_attention, paged_kv_append, paged_kv_read, shared_prefix_attention

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
H_BF16, H_F32 = 2.0**-8, 2.0**-24
DTYPES = {"e4m3": torch.float8_e4m3fn, "e2m1": torch.float4_e2m1fn_x2}


def append(x, eps=2.0**-20, **kw):
    kw = dict(dict(seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin), **kw)
    paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, eps=eps, **x.scales(), **kw)


def read(x, rows=None, **kw):
    kw = dict(dict(seq_start=x.seq_start), **kw)
    return paged_kv_read(x.k_pages, x.v_pages, x.block_table, x.kv_len, sum(x.rows) if rows is None else rows, **x.scales(), **kw)


def attend(x, **kw):
    kw = dict(dict(seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin, eps=EPS), **x.scales(), **kw)
    if x.prefix:
        return shared_prefix_attention(x.q, x.k_pages, x.v_pages, x.prefix_table, x.prefix, x.block_table, x.kv_len, x.g_q, **kw)
    return paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, **kw)


def pools(x):
    return [t.view(torch.uint8) for t in (x.k_pages, x.k_scales, x.v_pages, x.v_scales)]


def check_pools(x, want):
    for got, ref in zip(pools(x), want):
        assert torch.equal(got, ref), int((got != ref).sum())


def check_y(x, y, lse, ref):
    """ref: (y, lse, (2 S + 2) W + |y|) of the definition."""
    y_ref, lse_ref, bound = ref
    h = H_BF16 if x.dtype == BF16 else H_F32 * x.D
    y, none = y.to(F64), lse_ref == -math.inf
    assert torch.equal(none, lse == -math.inf) and (y[none] == 0).all()
    far = (y - y_ref).abs()
    assert (far <= h * bound + 1e-30).all(), (far - h * bound).max()
    if y_ref.numel() and y_ref.norm() > 0:
        assert far.norm() / y_ref.norm() <= (6e-3 if x.dtype == BF16 else 5e-6)
    assert (lse.to(F64) - lse_ref)[~none].abs().max() <= (0.05 if x.dtype == BF16 else 1e-4) if (~none).any() else True


HEADS = [(18, 6, 64, BF16), (16, 4, 128, BF16), (8, 8, 64, BF16), (40, 2, 64, BF16), (8, 4, 64, F32), (4, 2, 128, F32)]
RAGGED = [
    ([1], [1]), ([1], [33]), ([1, 1, 1], [64, 1, 200]),
    ([3, 1, 0, 7, 1], [3, 40, 17, 130, 129]),                # a sequence without rows
    ([33, 1, 70], [33, 500, 100]),
    ([2, 5], [1, 3]),                                        # rows before the first key
    ([1] * 70, [1 + 13 * i % 90 for i in range(70)]),        # more sequences than lanes
]
both_formats = pytest.mark.parametrize("fmt", FORMATS)


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", HEADS)
@pytest.mark.parametrize("rows,lens", RAGGED)
@pytest.mark.parametrize("page", [8, 64])
def test_append_and_read(gpu_device, rows, lens, H, Hkv, D, dtype, page, fmt):
    for i, (qk_norm, mix, rope, layout) in enumerate([(True, False, True, "phsd"), (True, True, True, "pshd"), (False, True, False, "apart"), (False, False, True, "phsd")]):
        x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=i, rope=rope, layout=layout)
        want = x.appended_codes(qk_norm=qk_norm, mix=mix, pos0=3 if rope else 0)
        append(x, qk_norm=qk_norm, v_first=x.v_first if mix else None, vr_coef=x.coef if mix else None, rope_pos0=3 if rope else 0)
        check_pools(x, want)
        k, v = read(x, dtype=dtype)
        kd, vd = x.values()
        for t, (b, p) in enumerate(x.positions()):
            for got, ref in ((k, kd), (v, vd)):
                assert torch.equal(got[t].to(F64), ref[int(x.block_table[b, p // page]), :, p % page] if p >= 0 else torch.zeros(Hkv, D, dtype=F64, device=gpu_device)), (t, b, p)


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", HEADS)
@pytest.mark.parametrize("rows,lens", RAGGED)
@pytest.mark.parametrize("page", [8, 16, 64])
def test_attention(gpu_device, rows, lens, H, Hkv, D, dtype, page, fmt):
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=1)
    y, lse = attend(x, gate_logits=x.gate, return_lse=True)
    check_y(x, y, lse, x.attended(gate=True))
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=2, rope=False, layout="apart")
    y, lse = attend(x, g_k=x.g_k, qk_norm=False, sm_scale=0.2, return_lse=True)
    check_y(x, y, lse, x.attended(g_k=x.g_k, qk_norm=False, sm_scale=0.2))


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", HEADS + [(32, 2, 128, BF16), (40, 1, 64, BF16)])
@pytest.mark.parametrize("rows,lens,prefix", [
    ([1], [1], 1), ([1, 1, 1], [0, 5, 70], 100), ([1] * 40, [i for i in range(40)], 515), ([3, 0, 20, 1], [3, 9, 60, 0], 64), ([150, 130], [150, 260], 333),
])
@pytest.mark.parametrize("page", [8, 32])
def test_shared_prefix(gpu_device, rows, lens, prefix, H, Hkv, D, dtype, page, fmt):
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, prefix=prefix, seed=3, uniform=len(set(rows)) == 1, layout="pshd")
    y, lse = attend(x, gate_logits=x.gate, return_lse=True)
    check_y(x, y, lse, x.attended(gate=True))


# 17 .. 32 columns of a kv head are two tiles of one wave each, 33 are a tile of four waves
@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", [(16, 1, 64, BF16), (17, 1, 128, BF16), (32, 1, 64, BF16), (32, 1, 128, F32), (33, 1, 64, F32)])
@pytest.mark.parametrize("rows,lens,prefix", [([1], [2500], 0), ([1, 1], [100, 1], 0), ([1, 2, 1], [900, 77, 1300], 0), ([2], [600], 0), ([1], [40], 1500), ([1, 1], [0, 9], 16)])
def test_two_tiles_of_few_columns(gpu_device, rows, lens, prefix, H, Hkv, D, dtype, fmt):
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, dtype, gpu_device, prefix=prefix, seed=41, uniform=len(set(rows)) == 1)
    y, lse = attend(x, gate_logits=x.gate, return_lse=True)
    check_y(x, y, lse, x.attended(gate=True))


# so many columns that a workgroup of the merge has more than a tile of 16 holds
@both_formats
def test_merge_of_many_small_tiles(gpu_device, fmt):
    x = QuantBatch(fmt, [2] * 1100, [2 + i % 20 for i in range(1100)], 16, 1, 64, 8, BF16, gpu_device, prefix=40, seed=42, uniform=True)
    y, lse = attend(x, return_lse=True)
    check_y(x, y, lse, x.attended())


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", [(18, 6, 64, BF16), (16, 4, 128, BF16), (8, 4, 64, F32), (4, 2, 128, F32)])
@pytest.mark.parametrize("rows,lens,page", [
    ([1, 1, 1], [5001, 2, 3000], 16), ([1], [9000], 8), ([300, 1, 1], [2500, 1800, 40], 32), ([2, 2], [4700, 9000], 8), ([700], [700], 64),
    ([257, 100], [5000, 4500], 8),  # longer than the page numbers a wave holds at a time
])
def test_long_caches(gpu_device, rows, lens, page, H, Hkv, D, dtype, fmt):
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=4, uniform=len(set(rows)) == 1)
    y, lse = attend(x, return_lse=True)
    check_y(x, y, lse, x.attended())
    again, _ = attend(x, return_lse=True)
    assert torch.equal(y, again)


@both_formats
@pytest.mark.parametrize("H,Hkv,D,dtype", [(18, 6, 64, BF16), (16, 4, 128, BF16), (8, 4, 64, F32)])
def test_only_what_a_row_sees_is_looked_at(gpu_device, H, Hkv, D, dtype, fmt):
    """Slots behind a sequence's end, other pages, and a key and a value that later rows of the same call brought hold blocks that are no number."""
    rows, lens = [40, 1, 3, 70], [40, 100, 37, 200]
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=5)
    clean = attend(x)
    used = torch.zeros(x.n_pages, 16, dtype=torch.bool)
    for b, L in enumerate(lens):
        for p in range(L):
            used[int(x.block_table[b, p // 16]), p % 16] = True
    free = (~used).to(gpu_device)[:, None, :, None]
    for s in (x.k_scales, x.v_scales):
        s[free.expand_as(s)] = 255
    first = {}
    for b, row in ((0, 20), (3, 41)):  # what this row and later ones see: a block of a value, a block of a key of kv head 0
        p = lens[b] - rows[b] + row
        x.v_scales[int(x.block_table[b, p // 16]), :, p % 16, 1] = 255
        x.k_scales[int(x.block_table[b, p // 16]), 0, p % 16, 0] = 255
        first[b] = x.starts[b] + row
    y = attend(x)
    rep = H // Hkv
    for b in range(4):
        r0, r1 = x.starts[b], x.starts[b + 1]
        cut = first.get(b, r1)
        assert torch.equal(y[r0:cut], clean[r0:cut]), b
        if cut < r1:
            assert y[cut:r1, :rep].isnan().all()                                   # the key's heads
            assert y[cut:r1, rep:, 32:64].isnan().all()                            # the value's block
            assert y[cut:r1, rep:, :32].isfinite().all() and y[cut:r1, rep:, 64:].isfinite().all()
    k, v = read(x)
    kd, vd = x.values()
    assert torch.equal(k[first[0]].isnan(), kd[int(x.block_table[0, 1]), :, 4].isnan()) and k[first[0], 0, :32].isnan().all() and v[first[0], :, 32:64].isnan().all()


@both_formats
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 128)])
def test_bad_pages_and_lengths(gpu_device, dtype, D, fmt):
    rows, lens = [1, 5, 1, 2, 1], [50, 40, 30, 60, 20]
    x = QuantBatch(fmt, rows, lens, 6, 2, D, 16, dtype, gpu_device, seed=7)
    clean, (ck, cv) = attend(x), read(x)
    x.block_table[0, 1] = x.n_pages          # just behind the pool
    x.block_table[1, 2] = -1                 # holds keys 32 .. 47
    x.kv_len[2] = -3
    x.kv_len[3] = x.width * 16 + 1
    y, lse = attend(x, return_lse=True)
    s = x.starts
    assert y[s[0]:s[1]].isnan().all() and y[s[1]:s[2]].isnan().all() and y[s[2]:s[4]].isnan().all() and lse[: s[4]].isnan().all()
    assert torch.equal(y[s[4]:], clean[s[4]:])
    for got, want in zip(read(x), (ck, cv)):  # sequence 0's row lies in another page; all rows of 1 in the one that is not there
        assert torch.equal(got[s[0]], want[s[0]]) and got[s[1]:s[4]].isnan().all() and torch.equal(got[s[4]:], want[s[4]:])
    before = [t.clone() for t in pools(x)]
    append(x)  # sequence 0's row lies in page 3, 4's row in its last page; of 3's two rows, at positions 63 and 64, the second is behind the table
    for got, was in zip(pools(x)[::2], before[::2]):
        changed = (got != was).flatten(2).any(-1).any(-1)
        assert sorted(changed.nonzero().flatten().tolist()) == sorted(int(x.block_table[b, j]) for b, j in ((0, 3), (3, 3), (4, 1)))


@both_formats
def test_rows_in_no_sequence(gpu_device, fmt):
    x = QuantBatch(fmt, [1, 3, 9], [20, 40, 9], 6, 2, 64, 16, BF16, gpu_device, seed=8)
    full = attend(x)
    x.seq_start = torch.tensor([2, 3, 6, 8], dtype=torch.int32, device=gpu_device)  # rows 0, 1 and 8 .. 12 belong to nobody
    out, k, v = torch.full_like(x.q, 7.0), torch.full((13, 2, 64), 7.0, dtype=BF16, device=gpu_device), torch.full((13, 2, 64), 7.0, dtype=BF16, device=gpu_device)
    y, lse = attend(x, return_lse=True)
    assert attend(x, out=out) is out
    rest = [0, 1, 8, 9, 10, 11, 12]
    assert (y[rest] == 0).all() and (out[rest] == 7).all() and torch.equal(y[2:8], out[2:8]) and y.isfinite().all() and not torch.equal(y, full)
    assert (lse[rest] == -math.inf).all() and lse[2:8].isfinite().all()
    got = read(x)
    back = read(x, out=(k, v))
    assert back[0] is k and back[1] is v
    for a, b in zip(got, back):
        assert (a[rest] == 0).all() and (b[rest] == 7).all() and torch.equal(a[2:8], b[2:8]) and a[2:8].abs().sum() > 0
    before = [t.clone() for t in pools(x)]
    append(x)
    assert int((pools(x)[0] != before[0]).any(-1).any(1).sum()) == 6  # six slots
    x.seq_start = torch.tensor([-5, 100, 50, 13], dtype=torch.int32, device=gpu_device)  # cut off at the rows there are; the second has none
    attend(x)
    read(x)
    append(x)
    torch.cuda.synchronize()


@both_formats
def test_max_len_limits_a_sequence(gpu_device, fmt):
    x = QuantBatch(fmt, [1, 1], [40, 41], 6, 2, 64, 16, BF16, gpu_device, seed=9)
    clean = attend(x)
    cut = dict(rope_cos=x.cos[:40], rope_sin=x.sin[:40], max_len=40)  # the tables end where the sequences do
    y = attend(x, **cut)
    assert torch.equal(y[0], clean[0]) and y[1].isnan().all()
    k, _ = read(x, max_len=40)
    assert k[0].isfinite().all() and k[1].isnan().all()
    before = pools(x)[0].clone()
    append(x, **cut)
    assert (pools(x)[0] != before).flatten(2).any(-1).any(-1).nonzero().flatten().tolist() == [int(x.block_table[0, 2])]


@both_formats
def test_pool_beyond_32_bits(gpu_device, fmt):
    Hkv, D, page = 2, 64, 64
    x = QuantBatch(fmt, [1, 4], [100, 70], 6, Hkv, D, page, BF16, gpu_device, seed=10)
    row = x.k_pages.shape[3]
    n = (5 << 30) // (Hkv * row * page)  # 5 GiB of keys
    y, rows = attend(x), read(x)
    where = torch.arange(x.n_pages, device=gpu_device) * 2 + n - 2 * x.n_pages - 1
    big = []
    for t in pools(x):
        b = torch.zeros(n, *t.shape[1:], dtype=torch.uint8, device=gpu_device)
        b[where] = t
        big.append(b.view(x.k_pages.dtype) if t.shape[3] == row else b)
    x.k_pages, x.k_scales, x.v_pages, x.v_scales = big
    x.block_table = torch.where(x.block_table >= 0, where.to(torch.int32)[x.block_table.clamp(min=0).long()], x.block_table)
    assert torch.equal(attend(x), y) and all(torch.equal(a, b) for a, b in zip(read(x), rows))
    before = pools(x)[0][where]
    append(x)
    assert int((pools(x)[0][where] != before).any(-1).any(1).sum()) == 5


@both_formats
def test_another_stream_and_a_captured_step(gpu_device, fmt):
    """Appending, attending and reading in a graph whose lengths and rows move on between replays; another stream; two graphs side by side."""
    x = QuantBatch(fmt, [1, 1, 1], [30, 200, 65], 18, 6, 64, 16, BF16, gpu_device, seed=11, uniform=True)
    z = QuantBatch(fmt, [1, 1], [30, 90], 18, 6, 64, 16, BF16, gpu_device, seed=12, uniform=True, prefix=130)

    def step(t):
        append(t, rope_pos0=t.prefix)
        return (attend(t, gate_logits=t.gate), *read(t))

    same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step(x)
        step(z)
    torch.cuda.current_stream().wait_stream(s)
    assert same(want, step(x))
    graphs = []
    for t in (x, z):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(t)
        graphs.append((g, y, t))
    for i in range(4):
        for g, y, t in graphs:
            t.kv_len.sub_(1 if i % 2 else 2)
            t.q.copy_(torch.randn_like(t.q))
            t.k.copy_(torch.randn_like(t.k))
        for g, y, t in graphs:
            g.replay()
        got = [[u.clone() for u in y] for _, y, _ in graphs]
        torch.cuda.synchronize()
        for (g, y, t), a in zip(graphs, got):
            assert same(a, step(t)), i


@both_formats
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_run_of_steps(gpu_device, fmt, dtype):
    """Ragged prompts, then single tokens, then mixed steps, through table and cache: what is held is the definition's, bit for bit, and y its attention."""
    H, Hkv, D = 6, 2, 64
    g = torch.Generator().manual_seed(13)
    pages = PageTable(3, 120, 16, device=gpu_device)
    cache = PagedKVCache(pages, Hkv, D, DTYPES[fmt])
    ang = torch.outer(torch.arange(120, dtype=F64), 10_000.0 ** (-2 * torch.arange(D // 2, dtype=F64) / D))
    cos, sin = ang.cos().float().to(gpu_device), ang.sin().float().to(gpu_device)
    gain, eps = torch.ones(1, device=gpu_device), 2.0**-20
    K, V = ([torch.zeros(0, Hkv, D, dtype=F64, device=gpu_device) for _ in range(3)] for _ in range(2))
    turn = lambda t, p: torch.cat([t[..., :32] * cos[p].to(F64)[:, None] - t[..., 32:] * sin[p].to(F64)[:, None],
                                   t[..., :32] * sin[p].to(F64)[:, None] + t[..., 32:] * cos[p].to(F64)[:, None]], -1)
    unit = lambda t: t / (t.square().mean(-1, keepdim=True) + eps).sqrt()
    for rows in ([17, 40, 5], 1, 1, [1, 30, 0], 2, [60, 1, 1]):
        pages.extend(rows)
        each = [rows] * 3 if isinstance(rows, int) else rows
        q, k, v = (torch.randn(sum(each), h, D, generator=g).to(dtype).to(gpu_device) for h in (H, Hkv, Hkv))
        cache.append(k, v, eps=eps, rope_cos=cos, rope_sin=sin)
        y = cache.attend(q, gain, eps=eps, rope_cos=cos, rope_sin=sin)
        at = 0
        for b, n in enumerate(each):
            r, first = slice(at, at + n), K[b].shape[0]
            at += n
            if n == 0:
                continue
            where = torch.arange(first, first + n, device=gpu_device)
            K[b] = torch.cat([K[b], decode(*encode(unit(turn(k[r].to(F64), where)), fmt), fmt)])
            V[b] = torch.cat([V[b], decode(*encode(v[r].to(F64), fmt), fmt)])
            Q = unit(turn(q[r].to(F64), where)) / 8.0
            hidden = torch.arange(first + n, device=gpu_device)[None] > where[:, None]
            for h in range(H):
                s = (Q[:, h] @ K[b][:, h // 3].T).masked_fill(hidden, -math.inf)
                p = torch.softmax(s, -1)
                ref, W = p @ V[b][:, h // 3], p @ V[b][:, h // 3].abs()
                S = (Q[:, h].abs() @ K[b][:, h // 3].abs().T).amax(-1, keepdim=True)
                tol = (2.0**-13 * S + 2 * H_BF16) * W + H_BF16 * ref.abs() if dtype == BF16 else H_F32 * D * ((2 * S + 2) * W + ref.abs())
                assert ((y[r, h].to(F64) - ref).abs() <= tol).all(), (rows, b, h)
        k, v, starts = cache.read()
        assert torch.equal(k.to(F64), torch.cat(K)) and torch.equal(v.to(F64), torch.cat(V)) and starts[1:].tolist() == [sum(pages.lengths[: b + 1]) for b in range(3)]
    pages.release(1)
    pages.extend([0, 3, 0])
    assert cache.read()[0].shape[0] == sum(pages.lengths) == K[0].shape[0] + K[2].shape[0] + 3


@both_formats
@pytest.mark.parametrize("at_once", [1, 40, 61, 1 << 18])
def test_another_dtype_some_sequences_at_a_time(gpu_device, fmt, at_once, monkeypatch):
    from sample_efficient_gpt_amd import paged

    monkeypatch.setattr(paged, "_ROWS_AT_ONCE", at_once)
    pages = PageTable(5, 64, 8, device=gpu_device, prefix_len=11)
    cache = PagedKVCache(pages, 2, 64)
    g = torch.Generator().manual_seed(5)
    for table, rows in ((pages.prefix, 11), (pages, [20, 0, 41, 1, 33])):
        table.extend(rows)
        cache.of(table).append(*(torch.randn(table.rows, 2, 64, generator=g).to(BF16).to(gpu_device) for _ in "kv"))
    small = cache.to(DTYPES[fmt])
    for table in (pages.prefix, pages):
        for got, ref in zip(small.of(table).read()[:2], cache.of(table).read()[:2]):
            assert torch.equal(got.to(F64), decode(*encode(ref.to(F64), fmt), fmt))


@both_formats
@pytest.mark.parametrize("prefix", [0, 70])
def test_module(gpu_device, fmt, prefix):
    """The attention module over such a cache, against the same module over a bf16 cache that holds the very values: what this one reads back."""
    torch.manual_seed(15)
    d, H, Hkv = 384, 6, 2
    m = MultiHeadSelfAttention(d, H, Hkv, max_seq_len=256, qknorm=True, value_residual=True, gating="per-head", device=gpu_device, dtype=BF16)
    with torch.no_grad():
        m.alpha1.fill_(0.8)
        m.alpha2.fill_(0.5)
        pages = PageTable(3, 60, 16, prefix_len=prefix, device=gpu_device)
        cache = PagedKVCache(pages, Hkv, d // H, DTYPES[fmt])
        if prefix:
            pages.prefix.extend(prefix)
            m(torch.randn(1, prefix, d, device=gpu_device).to(BF16), v1=torch.randn(1, Hkv, prefix, 64, device=gpu_device).to(BF16), kv_cache=cache.of(pages.prefix))
        for rows in ([20, 1, 33], 1, [3, 0, 2]):
            pages.extend(rows)
            x = torch.randn(1, pages.rows, d, device=gpu_device).to(BF16)
            v1 = torch.randn(1, Hkv, pages.rows, 64, device=gpu_device).to(BF16)
            y, _ = m(x, v1=v1, kv_cache=cache)
            plain = cache.to(BF16)
            assert plain.dtype == BF16 and plain.k_scales is None and cache.to(DTYPES[fmt]) is cache
            plain.append = lambda *a, **kw: None
            want, _ = m(x, v1=v1, kv_cache=plain)
            # y of the attention: bf16, from equal operands, its rounding and those of the probabilities on either side
            assert (y.float() - want.float()).norm() <= 1e-2 * want.float().norm()
            again = plain.to(DTYPES[fmt]) if rows != 1 else cache
            for a, b in zip(again.read()[:2], cache.read()[:2]):
                assert torch.equal(a, b)  # stored values are stored again as they are


@both_formats
def test_as_operators(gpu_device, fmt):
    """Under torch.compile the calls are nodes of the graph; results are the eager ones bit for bit, rows in no sequence keep what they held."""
    x, z = (QuantBatch(fmt, [1, 9, 3], [40, 20, 30], 6, 2, 64, 16, BF16, gpu_device, seed=16, prefix=50) for _ in range(2))
    x.seq_start = z.seq_start = torch.tensor([1, 2, 11, 12], dtype=torch.int32, device=gpu_device)

    def f(t, q, k, v, kp, vp, ks, vs, out):
        kw = dict(seq_start=t.seq_start, k_scales=ks, v_scales=vs)
        paged_kv_append(k, v, kp, vp, t.block_table, t.kv_len, rope_cos=t.cos, rope_sin=t.sin, rope_pos0=50, **kw)
        a = shared_prefix_attention(q * 1, kp, vp, t.prefix_table, 50, t.block_table, t.kv_len, t.g_q, rope_cos=t.cos, rope_sin=t.sin, **kw)
        b, lse = paged_attention(q * 1, kp, vp, t.block_table, t.kv_len, t.g_q, out=out[0], return_lse=True, **kw)
        c = paged_kv_read(kp, vp, t.block_table, t.kv_len, 13, **kw)
        paged_kv_read(kp, vp, t.block_table, t.kv_len, 13, out=(out[1], out[2]), **kw)
        return a, b * 2, lse, *c

    outs = [[torch.full_like(x.q, 7.0)] + [torch.full((13, 2, 64), 7.0, dtype=F32, device=gpu_device) for _ in range(2)] for _ in range(2)]
    with torch.no_grad():
        want = f(x, x.q, x.k, x.v, x.k_pages, x.v_pages, x.k_scales, x.v_scales, outs[0])
        got = torch.compile(lambda *a: f(z, *a), backend="aot_eager", fullgraph=True)(z.q, z.k, z.v, z.k_pages, z.v_pages, z.k_scales, z.v_scales, outs[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(*outs))
    assert all(torch.equal(a, b) for a, b in zip(pools(x), pools(z))) and (outs[0][0][[0, 12]] == 7).all() and (outs[0][1][[0, 12]] == 7).all()
    k = x.k.clone().requires_grad_()
    with pytest.raises(Exception, match="no derivative"):
        torch.compile(lambda k: f(x, x.q, k, x.v, x.k_pages, x.v_pages, x.k_scales, x.v_scales, outs[0]), backend="aot_eager", fullgraph=True)(k)


@both_formats
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_codes_of_all_kinds_of_values(gpu_device, fmt, dtype, D):
    """Zeros of either sign, ties, borders of scales, the largest and smallest numbers, and components that are not finite."""
    top = 448.0 if fmt == "e4m3" else 6.0
    blocks = [torch.zeros(32), -torch.zeros(32), torch.arange(32) * 2.0**-6, torch.linspace(-top, top, 32), torch.linspace(-top, top, 32) * (1 + 2.0**-7),
              top * 2.0 ** torch.arange(0, -32, -1), 2.0 ** torch.arange(-100, -132, -1).double(), torch.full((32,), 2.0**127), torch.full((32,), -1.9 * 2.0**127),
              torch.randn(32, generator=torch.Generator().manual_seed(1)) * 2.0**-120, torch.full((32,), 3.3e38), torch.full((32,), 1.74 * 2.0**127)]
    for bad in (math.nan, math.inf, -math.inf):
        b = torch.ones(32)
        b[17] = bad
        blocks.append(b)
    n = D // 32
    while len(blocks) % n:
        blocks.append(torch.ones(32))
    rows = torch.stack([b.float().to(dtype) for b in blocks]).view(-1, 1, D).to(gpu_device)
    T = rows.shape[0]
    x = QuantBatch(fmt, [T], [T], 1, 1, D, 16, dtype, gpu_device, rope=False)
    x.k, x.v = rows, rows.flip(0)
    want = x.appended_codes(qk_norm=False)
    append(x, qk_norm=False)
    check_pools(x, want)
    k, v = read(x, dtype=F32)
    assert torch.equal(k.isnan(), v.flip(0).isnan()) and torch.equal(k.nan_to_num(), v.flip(0).nan_to_num()) and not k.isinf().any()
    none = ~rows.view(T, n, 32).isfinite().all(-1)
    assert k.view(T, n, 32).isnan().all(-1)[none].all() and none.any()


@both_formats
def test_keys_next_to_a_border(gpu_device, fmt):
    """Prepared keys that 32 bits cannot tell from a border between two codes: 4096 rows at every length around 1 (eps 0.5 makes the scale no power of two)."""
    T, D = 4096, 128
    x = QuantBatch(fmt, [T], [T], 2, 2, D, 64, F32, gpu_device)
    x.k = (x.k * (1 + torch.arange(T, device=gpu_device)[:, None, None] / T)).contiguous()
    want = x.appended_codes(eps=0.5)
    append(x, eps=0.5)
    check_pools(x, want)


def test_read_of_pages_without_scales(gpu_device):
    from paged_util import Batch
    for dtype, D in ((BF16, 64), (BF16, 128), (F32, 32), (F32, 64), (F32, 128)):
        for rows, lens in RAGGED:
            x = Batch(rows, lens, 4, 2, D, 16, dtype, gpu_device, seed=40, layout="apart")
            k, v = paged_kv_read(x.k_pages, x.v_pages, x.block_table, x.kv_len, sum(rows), seq_start=x.seq_start)
            assert k.dtype == v.dtype == dtype
            for t, (b, p) in enumerate(x.positions()):
                for got, pool in ((k, x.k_pages), (v, x.v_pages)):
                    assert torch.equal(got[t], pool[int(x.block_table[b, p // 16]), :, p % 16] if p >= 0 else torch.zeros_like(got[t]))


@both_formats
def test_refusals(gpu_device, fmt):
    x = QuantBatch(fmt, [1, 2], [20, 30], 6, 2, 64, 16, BF16, gpu_device, seed=17)
    from sample_efficient_gpt_amd._lib import SegptError

    with pytest.raises(AssertionError, match="no derivative"):
        paged_attention(x.q.clone().requires_grad_(), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales())
    with pytest.raises(AssertionError, match="go together"):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, k_scales=x.k_scales)
    with pytest.raises(AssertionError, match="go together"):
        paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start, v_scales=x.v_scales)
    with pytest.raises(TypeError):  # codes without scales are no rows
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(TypeError):
        paged_attention(x.q.half(), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales())
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        paged_attention(x.q, x.q[:, :2, None], x.q[:, :2, None], x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales())
    with pytest.raises(TypeError, match="scales must be"):
        paged_kv_read(x.k_pages, x.v_pages, x.block_table, x.kv_len, 3, seq_start=x.seq_start, k_scales=x.k_scales.int(), v_scales=x.v_scales)
    with pytest.raises(AssertionError, match="scales must be"):
        paged_kv_read(x.k_pages, x.v_pages, x.block_table, x.kv_len, 3, seq_start=x.seq_start, k_scales=x.k_scales[:, :, :8], v_scales=x.v_scales)
    with pytest.raises(AssertionError, match="head_dim"):
        paged_attention(x.q.repeat(1, 1, 2), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales())
    with pytest.raises(AssertionError):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, k_scales=x.k_scales.cpu(), v_scales=x.v_scales)
    with pytest.raises(AssertionError):  # three rows of two sequences
        paged_kv_read(x.k_pages, x.v_pages, x.block_table, x.kv_len, 3, **x.scales())
    with pytest.raises(AssertionError):
        read(x, rows=-1)
    with pytest.raises(TypeError):
        read(x, dtype=torch.float16)
    z = torch.zeros(3, 2, 64, dtype=BF16, device=gpu_device)
    with pytest.raises(AssertionError):
        read(x, out=(z, z[:2]))
    with pytest.raises(TypeError):
        read(x, out=(z, z.float()))
    with pytest.raises(RuntimeError, match="overlap"):
        read(x, out=(z, z))
    with pytest.raises(RuntimeError, match="overlap"):
        read(x, out=(z, x.v_pages.view(torch.uint8).view(-1)[: 2 * z.numel()].view(BF16).view(z.shape)))
    with pytest.raises(RuntimeError, match="overlap"):
        paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start, k_scales=x.k_scales, v_scales=x.k_scales)
    with pytest.raises(RuntimeError, match="overlap"):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales(),
                        out=x.v_pages.view(torch.uint8).view(-1)[: 2 * x.q.numel()].view(BF16).view(x.q.shape))
    with pytest.raises(SegptError, match="stride"):
        flat = x.k_scales[:1].expand_as(x.k_scales)
        paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start, k_scales=flat, v_scales=flat.clone())
    with pytest.raises(SegptError, match="head"):  # rows of 32
        paged_kv_read(x.k_pages[..., : x.k_pages.shape[3] // 2], x.v_pages[..., : x.k_pages.shape[3] // 2], x.block_table, x.kv_len, 3, seq_start=x.seq_start,
                      k_scales=x.k_scales[..., :1], v_scales=x.v_scales[..., :1])
    empty = x.q[:0]
    assert paged_attention(empty, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start * 0, **x.scales()).shape == empty.shape
    assert read(x, rows=0, seq_start=x.seq_start * 0)[0].shape == (0, 2, 64)
    e8m0 = torch.float8_e8m0fnu
    same = paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, k_scales=x.k_scales.view(e8m0), v_scales=x.v_scales.view(e8m0))
    assert torch.equal(same, paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, **x.scales()))


@both_formats
@pytest.mark.parametrize("rows,lens,prefix", [
    ([1] * 300, [1 + 29 * i % 150 for i in range(300)], 0),                      # every sequence one token, more than a wave keeps in registers
    ([(0, 1, 1, 3, 12)[i % 5] for i in range(300)], [30 + 17 * i % 90 for i in range(300)], 0),
    ([1] * 300, [i % 40 for i in range(300)], 140),
    ([(1, 0, 14)[i % 3] for i in range(1500)], [15 + i % 20 for i in range(1500)], 33),
])
def test_many_sequences(gpu_device, rows, lens, prefix, fmt):
    for H, Hkv, D, dtype in ((6, 2, 64, BF16), (4, 2, 64, F32)):
        x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=18, prefix=prefix, uniform=len(set(rows)) == 1)
        y, lse = attend(x, return_lse=True)
        check_y(x, y, lse, x.attended())
        want = x.appended_codes(pos0=prefix)
        append(x, rope_pos0=prefix)
        check_pools(x, want)


@both_formats
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,lens", [([1, 1], [700, 90]), ([200, 1], [900, 300])])
@pytest.mark.parametrize("order", ["rising", "falling", "spike"])
def test_scores_far_apart(gpu_device, dtype, rows, lens, order, fmt):
    """Keys along the queries, so that the scores of a row run over several hundred: upwards (every tile has a new maximum), downwards (all but
    the first underflow), or with one key above all others."""
    for H, Hkv, D in ((6, 2, 64), (4, 2, 128)):
        x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=20, rope=False)
        x.q.copy_(1.0 + 0.05 * torch.randn(x.q.shape, device=gpu_device))
        x.g_q = torch.ones(1, device=gpu_device)
        for b, L in enumerate(lens):
            for p in range(L):
                size = {"rising": p / L, "falling": 1 - p / L, "spike": float(p == L // 2)}[order] * 2 - 1
                codes, scales = encode(torch.full((Hkv, D), 4.0 * size, dtype=F64, device=gpu_device), fmt)
                x.k_pages.view(torch.uint8)[int(x.block_table[b, p // 16]), :, p % 16] = codes
                x.k_scales[int(x.block_table[b, p // 16]), :, p % 16] = scales
        y, lse = attend(x, qk_norm=False, return_lse=True, sm_scale=1.0)
        y_ref, lse_ref, bound = x.attended(qk_norm=False, sm_scale=1.0)
        # scores up to 4 D: their roundings (2^-8 or D 2^-24 of that) move the sums by more than their size at bf16; y stays among the values
        assert y.isfinite().all() and lse.isfinite().all()
        h = H_BF16 if dtype == BF16 else H_F32 * D
        # Components whose value is 0 wherever a probability counts (4-bit codes often are) are sums of the others, down to 1e-56 here: what lies under
        # 2^-126 no fp32 probability holds, and 900 of them times values up to 6 are less than 900 * 6 * 2^-126 = 6.4e-35
        assert ((y.to(F64) - y_ref).abs() <= h * bound + 1e-34).all()
        assert ((lse.to(F64) - lse_ref).abs() <= h * (4.5 * D + 16)).all()


@both_formats
def test_strided_rows_gate_and_out(gpu_device, fmt):
    for H, Hkv, D, dtype in ((6, 2, 64, BF16), (4, 2, 128, BF16), (6, 2, 64, F32)):
        for rows, lens in (([1, 1, 1], [40, 9, 200]), ([60, 1, 5], [60, 100, 30])):
            x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=21)
            T = sum(rows)
            x.gate = torch.randn(T, H, 3, device=gpu_device).to(dtype)[..., 1]
            x.q = x.q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
            want, lse = attend(x, gate_logits=x.gate, return_lse=True)
            check_y(x, want, lse, x.attended(gate=True))
            wide = torch.full((H, T + 2, D + 8), 5.0, dtype=dtype, device=gpu_device)
            out = wide[:, 1:-1, :D].transpose(0, 1)
            y, lse2 = attend(x, gate_logits=x.gate, return_lse=True, out=out)
            assert y is out and torch.equal(out, want) and torch.equal(lse, lse2)
            assert (wide[:, [0, -1]] == 5).all() and (wide[..., D:] == 5).all()
            wide = torch.full((Hkv, T + 2, 2 * D + 8), 5.0, dtype=dtype, device=gpu_device)
            k, v = (wide[:, 1:-1, i * D:(i + 1) * D].transpose(0, 1) for i in range(2))  # side by side in one buffer
            read(x, out=(k, v))
            assert all(torch.equal(a, b) for a, b in zip((k, v), read(x, dtype=dtype)))
            assert (wide[:, [0, -1]] == 5).all() and (wide[..., 2 * D:] == 5).all()


@both_formats
def test_two_calls_at_once(gpu_device, fmt):
    """Calls on two streams, each with work of its own, give what they give alone."""
    xs = [QuantBatch(fmt, [1] * 8, [3000 + i for i in range(8)], 18, 6, 64, 16, BF16, gpu_device, seed=23, uniform=True),
          QuantBatch(fmt, [200, 1, 90], [900, 4000, 300], 18, 6, 64, 32, BF16, gpu_device, seed=24),
          QuantBatch(fmt, [1] * 20, [i for i in range(20)], 18, 6, 64, 32, BF16, gpu_device, seed=25, prefix=700)]
    want = [attend(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(6):
        for x, s, g in zip(xs, streams, got):
            with torch.cuda.stream(s):
                g.append(attend(x))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


@pytest.mark.parametrize("seed", range(16))
def test_batches_drawn_at_random(gpu_device, seed):
    r = random.Random(100 + seed)
    fmt = FORMATS[seed % 2]
    H, Hkv, D, dtype = r.choice(HEADS + [(24, 1, 64, BF16), (5, 5, 128, BF16), (33, 11, 64, F32)])
    page, prefix = r.choice([8, 16, 32, 64, 128]), r.choice([0, 0, 1, 31, 32, 100, 257])
    B = r.choice([1, 2, 5, 17, 65])
    rows = [r.choice([0, 1, 1, 2, 5, 11, 33, 64, 129]) for _ in range(B)] if r.random() < 0.7 else [r.choice([1, 4, 12])] * B
    if sum(rows) == 0:
        rows[0] = 1
    lens = [max(n + r.choice([0, 0, 1, 7, 64, 500]) - (r.random() < 0.2), 0) for n in rows]
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=seed, prefix=prefix, uniform=len(set(rows)) == 1, rope=r.random() < 0.7,
                   layout=r.choice(["phsd", "pshd", "apart"]))
    gate, norm = r.random() < 0.5, r.random() < 0.7
    want = x.appended_codes(qk_norm=norm, mix=True, pos0=prefix if x.cos is not None else 0)
    append(x, qk_norm=norm, v_first=x.v_first, vr_coef=x.coef, rope_pos0=prefix if x.cos is not None else 0)
    check_pools(x, want)
    y, lse = attend(x, qk_norm=norm, gate_logits=x.gate if gate else None, g_k=x.g_k, sm_scale=0.1, return_lse=True)
    check_y(x, y, lse, x.attended(qk_norm=norm, gate=gate, g_k=x.g_k, sm_scale=0.1))


@both_formats
@pytest.mark.parametrize("H,Hkv,D", [(18, 6, 64), (16, 4, 128)])
@pytest.mark.parametrize("rows,lens,prefix,most", [
    ([1] * 32, [200 + 61 * i for i in range(32)], 0, 1.1), ([1, 1], [3000, 500], 0, 1.1),                       # generated tokens
    ([1] * 32, [5 + i for i in range(32)], 1500, 1.5), ([200, 1, 1, 1], [1500, 900, 40, 1200], 0, 1.5), ([700, 300], [700, 900], 0, 1.5),
])
def test_error_of_bf16_is_that_of_its_outputs(gpu_device, rows, lens, prefix, most, H, Hkv, D, fmt):
    """Against 64 bits, in units of what rounding the exact y to bf16 costs (r, in norm).  Single tokens of up to 32 heads a kv group: query and
    probabilities are in two parts, what they leave is 2^-14 of a score and of a probability, nothing beside r.  More columns: the probabilities are rounded
    once, an independent error of the size of y's own: sqrt(2) r."""
    x = QuantBatch(fmt, rows, lens, H, Hkv, D, 16, BF16, gpu_device, seed=32, prefix=prefix, uniform=len(set(rows)) == 1)
    y_ref = x.attended()[0]
    r = (y_ref.to(BF16).to(F64) - y_ref).norm()
    assert (attend(x).to(F64) - y_ref).norm() <= most * r


@both_formats
@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("uniform", [False, True])
def test_lengths_at_the_ends_of_32_bits(gpu_device, prefix, uniform, fmt):
    """A length that is no length at all: NaN in that sequence's rows, nothing elsewhere, and nothing outside the tensors is read."""
    x = QuantBatch(fmt, [2, 2, 2, 2], [9, 40, 30, 2], 6, 2, 64, 16, BF16, gpu_device, seed=31, prefix=prefix, uniform=uniform)
    clean, (ck, _) = attend(x), read(x)
    x.kv_len[1], x.kv_len[2] = -(2**31), 2**31 - 1
    y, (k, _) = attend(x), read(x)
    assert y[2:6].isnan().all() and torch.equal(y[:2], clean[:2]) and torch.equal(y[6:], clean[6:])
    assert k[2:6].isnan().all() and torch.equal(k[:2], ck[:2]) and torch.equal(k[6:], ck[6:])
    before = pools(x)[0].clone()
    append(x, rope_pos0=prefix)
    assert int((pools(x)[0] != before).any(-1).any(1).sum()) == 4  # slots of the two sequences that have a length


@both_formats
def test_a_very_long_sequence(gpu_device, fmt):
    x = QuantBatch(fmt, [1, 2], [400_003, 5], 4, 2, 64, 64, BF16, gpu_device, seed=28)
    y, lse = attend(x, return_lse=True)
    check_y(x, y, lse, x.attended())
    z = QuantBatch(fmt, [1, 40], [3, 50], 4, 2, 64, 64, BF16, gpu_device, seed=29, prefix=200_001)
    y, lse = attend(z, return_lse=True)
    check_y(z, y, lse, z.attended())
