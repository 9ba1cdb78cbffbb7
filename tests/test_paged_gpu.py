"""The paged cache's operators against their definition in float64 (tests/paged_util.py), on the GPU.

Tolerances.  A rounding to bf16 is off by at most h = 2^-8 of the value, to fp32 by 2^-24.  Append: one rounding of a value that fp32
arithmetic knows to a few 2^-24 of the row's largest (rotation three, normaliser at most D / 8 + 8 of them).  Attention: the query is rounded
once, which moves a score by at most h * sum |qhat k'| =: h S and a probability by 2 h S (numerator and sum); a probability is rounded
once, and the sum is of the rounded ones (2 h); y once: |dy| <= h ((2 S + 2) sum P |v| + |y|), element by element.  That is the worst
case, with all roundings in one direction; as they are independent, a whole result is far nearer: three of them at h / 2 / sqrt(3) * sqrt(...)
of y's own size, 3e-3 of its norm, and twice that is asked for.  fp32: the same with 2^-24 times the roundings of a sum of D products, D."""

import math

import pytest
import torch

from paged_util import EPS, F64, Batch
from sample_efficient_gpt_amd import (KVCache, MultiHeadSelfAttention, PagedKVCache, PageTable, paged_attention, paged_kv_append,
                                      shared_prefix_attention)

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
H_BF16, H_F32 = 2.0**-8, 2.0**-24


def append(x, **kw):
    paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin, eps=EPS, **kw)


def attend(x, **kw):
    kw = dict(dict(seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin, eps=EPS), **kw)
    if x.prefix:
        return shared_prefix_attention(x.q, x.k_pages, x.v_pages, x.prefix_table, x.prefix, x.block_table, x.kv_len, x.g_q, **kw)
    return paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, **kw)


def check_pools(x, kp, vp, mix=False):
    for got, ref, one_rounding in ((x.k_pages, kp, False), (x.v_pages, vp, not mix)):
        size = ref.abs().amax(-1, keepdim=True)
        h = H_BF16 if x.dtype == BF16 else H_F32
        tol = h * ref.abs() + (x.D / 8 + 16) * H_F32 * size
        assert ((got.to(F64) - ref).abs() <= tol).all()
        if one_rounding:
            assert torch.equal(got.to(F64), ref)  # a copy


def check_y(x, y, lse, ref, norm=True):
    y_ref, lse_ref, bound = ref
    h = H_BF16 if x.dtype == BF16 else H_F32 * x.D
    y, none = y.to(F64), lse_ref == -math.inf
    assert torch.equal(none, lse == -math.inf) and (y[none] == 0).all()
    far = (y - y_ref).abs()
    assert (far <= h * bound + 1e-30).all(), (far - h * bound).max()
    if norm and y_ref.numel() and y_ref.norm() > 0:
        assert far.norm() / y_ref.norm() <= (6e-3 if x.dtype == BF16 else 5e-6)
    # bound = (2 S + 2) sum P |v| + |y|, and a score moves by h S: with |v| left out, an upper bound of S is not at hand here
    assert (lse.to(F64) - lse_ref)[~none].abs().max() <= (0.05 if x.dtype == BF16 else 1e-4) if (~none).any() else True


HEADS = [(18, 6, 64, BF16), (16, 4, 128, BF16), (8, 8, 64, BF16), (6, 2, 32, F32), (8, 4, 64, F32), (4, 2, 128, F32)]
RAGGED = [
    ([1], [1]), ([1], [33]), ([1, 1, 1], [64, 1, 200]),
    ([3, 1, 0, 7, 1], [3, 40, 17, 130, 129]),                # a sequence without rows
    ([33, 1, 70], [33, 500, 100]),
    ([2, 5], [1, 3]),                                        # rows before the first key
    ([1] * 70, [1 + 13 * i % 90 for i in range(70)]),        # more sequences than lanes
]


@pytest.mark.parametrize("H,Hkv,D,dtype", HEADS)
@pytest.mark.parametrize("rows,lens", RAGGED)
@pytest.mark.parametrize("page", [8, 16, 64])
def test_append(gpu_device, rows, lens, H, Hkv, D, dtype, page):
    for i, (qk_norm, mix, rope, layout) in enumerate([(True, False, True, "phsd"), (True, True, True, "pshd"), (False, True, False, "apart")]):
        x = Batch(rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=i, rope=rope, layout=layout)
        kp, vp = x.appended(qk_norm, mix, pos0=3 if rope else 0)
        append(x, qk_norm=qk_norm, v_first=x.v_first if mix else None, vr_coef=x.coef if mix else None, rope_pos0=3 if rope else 0)
        check_pools(x, kp, vp, mix)


@pytest.mark.parametrize("H,Hkv,D,dtype", HEADS)
@pytest.mark.parametrize("rows,lens", RAGGED)
@pytest.mark.parametrize("page", [8, 16, 64])
def test_attention(gpu_device, rows, lens, H, Hkv, D, dtype, page):
    x = Batch(rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=1)
    y, lse = attend(x, gate_logits=x.gate, return_lse=True)
    check_y(x, y, lse, x.attended(gate=True))
    x = Batch(rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=2, rope=False, layout="pshd")
    y, lse = attend(x, g_k=x.g_k, qk_norm=False, sm_scale=0.2, return_lse=True)
    check_y(x, y, lse, x.attended(g_k=x.g_k, qk_norm=False, sm_scale=0.2))


@pytest.mark.parametrize("H,Hkv,D,dtype", HEADS + [(32, 2, 128, BF16), (40, 1, 64, BF16)])
@pytest.mark.parametrize("rows,lens,prefix", [
    ([1], [1], 1), ([1, 1, 1], [0, 5, 70], 100), ([1] * 40, [i for i in range(40)], 515), ([3, 0, 20, 1], [3, 9, 60, 0], 64), ([150, 130], [150, 260], 333),
])
@pytest.mark.parametrize("page", [8, 32])
def test_shared_prefix(gpu_device, rows, lens, prefix, H, Hkv, D, dtype, page):
    x = Batch(rows, lens, H, Hkv, D, page, dtype, gpu_device, prefix=prefix, seed=3, uniform=len(set(rows)) == 1, layout="apart")
    y, lse = attend(x, gate_logits=x.gate, return_lse=True)
    check_y(x, y, lse, x.attended(gate=True))


@pytest.mark.parametrize("H,Hkv,D,dtype", [(18, 6, 64, BF16), (16, 4, 128, BF16), (8, 4, 64, F32), (4, 2, 128, F32)])
@pytest.mark.parametrize("rows,lens,page", [
    ([1, 1, 1], [5001, 2, 3000], 16), ([1], [9000], 8), ([300, 1, 1], [2500, 1800, 40], 32), ([2, 2], [4700, 9000], 8), ([700], [700], 64),
    ([257, 100], [5000, 4500], 8),  # longer than the page numbers a workgroup holds at a time
])
def test_long_caches(gpu_device, rows, lens, page, H, Hkv, D, dtype):
    x = Batch(rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=4, uniform=len(set(rows)) == 1)
    y, lse = attend(x, return_lse=True)
    check_y(x, y, lse, x.attended())
    again, _ = attend(x, return_lse=True)
    assert torch.equal(y, again)


@pytest.mark.parametrize("H,Hkv,D,dtype", [(18, 6, 64, BF16), (16, 4, 128, BF16), (6, 2, 32, F32), (8, 4, 64, F32)])
def test_only_what_a_row_sees_is_looked_at(gpu_device, H, Hkv, D, dtype):
    """Slots behind a sequence's end, other pages, and keys and values that later rows of the same call brought are not finite."""
    rows, lens = [40, 1, 3, 70], [40, 100, 37, 200]
    x = Batch(rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=5)
    clean = attend(x)
    for bad in (math.nan, math.inf, -math.inf):
        kp, vp = x.k_pages.clone(), x.v_pages.clone()
        used = torch.zeros(x.n_pages, x.page, dtype=torch.bool)
        first = {}
        for b, L in enumerate(lens):
            for p in range(L):
                used[int(x.block_table[b, p // 16]), p % 16] = True
        free = (~used).to(gpu_device)[:, None, :, None].expand_as(kp)
        x.k_pages[free] = bad
        x.v_pages[free] = bad
        for b, row in ((0, 20), (3, 41)):  # key and value that this row and later ones see
            p = lens[b] - rows[b] + row
            x.v_pages[int(x.block_table[b, p // 16]), :, p % 16, 3] = bad
            x.k_pages[int(x.block_table[b, p // 16]), 0, p % 16, 5] = bad
            first[b] = x.starts[b] + row
        y = attend(x)
        rep = H // Hkv
        for b in range(4):
            r0, r1 = x.starts[b], x.starts[b + 1]
            cut = first.get(b, r1)
            assert torch.equal(y[r0:cut], clean[r0:cut]), (bad, b)
            if cut < r1:
                assert not y[cut:r1, rep:, 3].isfinite().any()                       # the value's column
                assert y[cut:r1, rep:, 4:].isfinite().all() and y[cut:r1, rep:, :3].isfinite().all()
                if bad != bad:
                    assert y[cut:r1, :rep].isnan().all()                              # the key's heads
        x.k_pages.copy_(kp)
        x.v_pages.copy_(vp)


def test_value_that_is_infinite_is_the_answer_of_the_rows_that_see_it(gpu_device):
    for H, Hkv, D, dtype in ((6, 2, 64, BF16), (6, 2, 64, F32)):
        x = Batch([40], [40], H, Hkv, D, 16, dtype, gpu_device, seed=6)
        x.v_pages[int(x.block_table[0, 1]), :, 4, 7] = math.inf  # key 20
        y = attend(x)
        assert (y[20:, :, 7] == math.inf).all() and y[:20].isfinite().all() and y[:, :, 8:].isfinite().all()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 64)])
def test_bad_pages_and_lengths(gpu_device, dtype, D):
    rows, lens = [1, 5, 1, 2, 1], [50, 40, 30, 60, 20]
    x = Batch(rows, lens, 6, 2, D, 16, dtype, gpu_device, seed=7)
    clean = attend(x)
    x.block_table[0, 1] = x.n_pages          # just behind the pool
    x.block_table[1, 2] = -1                 # holds keys 32 .. 47
    x.kv_len[2] = -3
    x.kv_len[3] = x.width * 16 + 1
    y, lse = attend(x, return_lse=True)
    s = x.starts
    assert y[s[0]:s[1]].isnan().all() and y[s[1]:s[2]].isnan().all() and y[s[2]:s[4]].isnan().all() and lse[: s[4]].isnan().all()
    assert torch.equal(y[s[4]:], clean[s[4]:])
    before = x.k_pages.clone(), x.v_pages.clone()
    append(x)  # sequence 0's row lies in page 3, 1's rows 35 .. 39 in the page that is not there, 4's row in its last page;
    # of 3's two rows, at positions 63 and 64, the second is behind the table
    changed = (x.k_pages != before[0]).flatten(2).any(-1).any(-1), (x.v_pages != before[1]).flatten(2).any(-1).any(-1)
    for c in changed:
        assert sorted(c.nonzero().flatten().tolist()) == sorted(int(x.block_table[b, j]) for b, j in ((0, 3), (3, 3), (4, 1)))


def test_rows_behind_the_last_sequence(gpu_device):
    x = Batch([1, 3, 9], [20, 40, 9], 6, 2, 64, 16, BF16, gpu_device, seed=8)
    full = attend(x)
    x.seq_start = torch.tensor([2, 3, 6, 8], dtype=torch.int32, device=gpu_device)  # rows 0, 1 and 8 .. 12 belong to nobody
    out = torch.full_like(x.q, 7.0)
    y = attend(x)
    assert attend(x, out=out) is out
    rest = [0, 1, 8, 9, 10, 11, 12]
    assert (y[rest] == 0).all() and (out[rest] == 7).all() and torch.equal(y[2:8], out[2:8]) and y.isfinite().all() and not torch.equal(y, full)
    before = x.k_pages.clone()
    append(x)
    assert int((x.k_pages != before).any(-1).any(1).sum()) == 6  # six slots
    x.seq_start = torch.tensor([-5, 100, 50, 13], dtype=torch.int32, device=gpu_device)  # cut off at the rows there are; the second has none
    attend(x)
    append(x)
    torch.cuda.synchronize()


def test_max_len_limits_a_sequence(gpu_device):
    x = Batch([1, 1], [40, 41], 6, 2, 64, 16, BF16, gpu_device, seed=9)
    clean = attend(x)
    cut = dict(rope_cos=x.cos[:40], rope_sin=x.sin[:40], max_len=40)  # the tables end where the sequences do
    y = attend(x, **cut)
    assert torch.equal(y[0], clean[0]) and y[1].isnan().all()
    before = x.k_pages.clone()
    paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, **cut)
    assert (x.k_pages != before).flatten(2).any(-1).any(-1).nonzero().flatten().tolist() == [int(x.block_table[0, 2])]


def test_pool_beyond_32_bits(gpu_device):
    Hkv, D, page = 2, 64, 64
    n = (5 << 30) // (Hkv * D * page * 2)  # 5 GiB of keys
    x = Batch([1, 4], [100, 70], 6, Hkv, D, page, BF16, gpu_device, seed=10)
    y = attend(x)
    big_k, big_v = (torch.zeros(n, Hkv, page, D, dtype=BF16, device=gpu_device) for _ in range(2))
    where = torch.arange(x.n_pages, device=gpu_device) * 2 + n - 2 * x.n_pages - 1
    big_k[where], big_v[where] = x.k_pages, x.v_pages
    moved = torch.where(x.block_table >= 0, where.to(torch.int32)[x.block_table.clamp(min=0).long()], x.block_table)
    x.k_pages, x.v_pages, x.block_table = big_k, big_v, moved
    assert torch.equal(attend(x), y)
    kp, vp = (big_k[where].to(F64), big_v[where].to(F64))
    append(x)
    assert int((big_k[where].to(F64) != kp).any(-1).any(1).sum()) == 5


def test_another_stream_and_a_captured_step(gpu_device):
    """Appending and attending in a graph whose lengths and tables move on between replays; another stream; two graphs side by side."""
    x = Batch([1, 1, 1], [30, 200, 65], 18, 6, 64, 16, BF16, gpu_device, seed=11, uniform=True, prefix=0)
    z = Batch([1, 1], [30, 90], 18, 6, 64, 16, BF16, gpu_device, seed=12, uniform=True, prefix=130)

    def step(t):
        append(t, rope_pos0=t.prefix)
        return attend(t, gate_logits=t.gate)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step(x)
        step(z)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, step(x))
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
        got = [y.clone() for _, y, _ in graphs]
        torch.cuda.synchronize()
        for (g, y, t), a in zip(graphs, got):
            assert torch.equal(a, step(t)), i


def test_run_of_steps_against_one_pass(gpu_device):
    """Ragged prompts, then single tokens, then a mixed step, through the table and the cache: y as the definition has it on the whole history."""
    H, Hkv, D = 6, 2, 64
    for dtype in (BF16, F32):
        g = torch.Generator().manual_seed(13)
        pages = PageTable(3, 120, 16, device=gpu_device)
        cache = PagedKVCache(pages, Hkv, D, dtype)
        hist = [[], [], []]
        ang = torch.outer(torch.arange(120, dtype=F64), 10_000.0 ** (-2 * torch.arange(D // 2, dtype=F64) / D))
        cos, sin = ang.cos().float().to(gpu_device), ang.sin().float().to(gpu_device)
        gain = torch.ones(1, device=gpu_device)
        for rows in ([17, 40, 5], 1, 1, [1, 30, 0], 2, [60, 1, 1]):
            pages.extend(rows)
            each = [rows] * 3 if isinstance(rows, int) else rows
            T = sum(each)
            q, k, v = (torch.randn(T, h, D, generator=g).to(dtype).to(gpu_device) for h in (H, Hkv, Hkv))
            cache.append(k, v, rope_cos=cos, rope_sin=sin)
            y = cache.attend(q, gain, rope_cos=cos, rope_sin=sin)
            at = 0
            for b, n in enumerate(each):
                for t in range(at, at + n):
                    hist[b].append((k[t].to(F64), v[t].to(F64)))
                    K, V = (torch.stack([e[i] for e in hist[b]]) for i in (0, 1))
                    L = len(K)
                    turn = lambda x, p: torch.cat([x[..., :32] * cos[p].to(F64)[:, None] - x[..., 32:] * sin[p].to(F64)[:, None],
                                                   x[..., :32] * sin[p].to(F64)[:, None] + x[..., 32:] * cos[p].to(F64)[:, None]], -1)
                    unit = lambda x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
                    K = unit(turn(K, torch.arange(L, device=gpu_device)))
                    Q = unit(turn(q[t:t + 1].to(F64), torch.tensor([L - 1], device=gpu_device)))[0]
                    p = torch.softmax(torch.einsum("hd,lhd->hl", Q, K.repeat_interleave(3, 1)) / 8.0, -1)
                    ref = torch.einsum("hl,lhd->hd", p, V.repeat_interleave(3, 1))
                    # two roundings of the operands here (query and cached key): h S each
                    S = torch.einsum("hd,lhd->hl", Q.abs(), K.abs().repeat_interleave(3, 1)).amax(-1, keepdim=True) / 8.0
                    W = torch.einsum("hl,lhd->hd", p, V.abs().repeat_interleave(3, 1))
                    h = H_BF16 if dtype == BF16 else H_F32 * D
                    assert ((y[t].to(F64) - ref).abs() <= h * ((4 * S + 2) * W + ref.abs())).all(), (dtype, rows, b, t)
                at += n
        pages.release(1)
        pages.extend([0, 3, 0])
        assert pages.kv_len.tolist() == [len(hist[0]), 3, len(hist[2])]


@pytest.mark.parametrize("value_residual,gating,qknorm", [(False, "per-head", True), (True, "per-head", True), (True, "elementwise", False), (False, False, True)])
def test_module_with_a_paged_cache_is_the_module_with_its_cache(gpu_device, value_residual, gating, qknorm):
    """Two layers, the second handed the first one's values: prompt and steps through pages against the same through ``KVCache``."""
    torch.manual_seed(14)
    d, H, Hkv, B = 384, 6, 2, 3
    layers = [MultiHeadSelfAttention(d, H, Hkv, max_seq_len=100, qknorm=qknorm, value_residual=value_residual, gating=gating, device=gpu_device, dtype=BF16)
              for _ in range(2)]
    if value_residual:
        with torch.no_grad():
            for m in layers:
                m.alpha1.fill_(0.8)
                m.alpha2.fill_(0.5)
    pages = PageTable(B, 100, 16, device=gpu_device)
    paged = [PagedKVCache(pages, Hkv, d // H) for _ in layers]
    dense = [KVCache(), KVCache()]
    with torch.no_grad():
        for S in (45, 1, 1, 7, 1):
            x = torch.randn(B, S, d, device=gpu_device).to(BF16)
            pages.extend(S)
            outs = []
            for caches in (dense, paged):
                h, v1 = x, None
                for m, c in zip(layers, caches):
                    y, v = m(h, v1=v1, kv_cache=c)
                    v1 = v if v1 is None else v1
                    h = h + y
                outs.append((h, y, v1))
            (a, ya, va), (b, yb, vb) = outs
            assert yb.shape == ya.shape and (yb.float() - ya.float()).norm() <= 1.5e-2 * ya.float().norm(), S
            assert vb.shape == (B, Hkv, S, d // H)
            if not value_residual:
                assert torch.equal(vb, va[:, :, -S:])
            else:
                assert (vb.float() - va[:, :, -S:].float()).norm() <= 1e-2 * va.float().norm()
        assert type(paged[0]) is PagedKVCache and pages.lengths == [55] * B


def test_module_with_a_shared_prefix_and_ragged_rows(gpu_device):
    """A prompt all sequences share, filled once, then ragged rows of their own, against every sequence by itself with all of its tokens."""
    torch.manual_seed(15)
    d, H, Hkv = 384, 6, 2
    m = MultiHeadSelfAttention(d, H, Hkv, max_seq_len=256, qknorm=True, gating="per-head", device=gpu_device, dtype=BF16)
    pages = PageTable(3, 60, 16, prefix_len=70, device=gpu_device)
    cache = PagedKVCache(pages, Hkv, d // H)
    with torch.no_grad():
        common = torch.randn(1, 70, d, device=gpu_device).to(BF16)
        pages.prefix.extend(70)
        m(common, kv_cache=cache.of(pages.prefix))
        own = [torch.randn(1, n, d, device=gpu_device).to(BF16) for n in (20, 1, 33)]
        pages.extend([20, 1, 33])
        y, _ = m(torch.cat(own, 1), kv_cache=cache)
        tail = torch.randn(3, 1, d, device=gpu_device).to(BF16)
        pages.extend(1)
        y2, _ = m(tail, kv_cache=cache)
        at = 0
        for b, x in enumerate(own):
            ref = m(torch.cat([common, x, tail[b:b + 1]], 1))[0]
            n = x.shape[1]
            got = torch.cat([y[:, at:at + n], y2[b:b + 1]], 1)
            at += n
            assert (got.float() - ref[:, 70:].float()).norm() <= 1.5e-2 * ref[:, 70:].float().norm()


def test_as_operators(gpu_device):
    """Under torch.compile the calls are nodes of the graph; results are the eager ones bit for bit."""
    x = Batch([1, 9], [40, 20], 6, 2, 64, 16, BF16, gpu_device, seed=16, prefix=50)
    eager_k, eager_v = x.k_pages.clone(), x.v_pages.clone()
    paged_kv_append(x.k, x.v, eager_k, eager_v, x.block_table, x.kv_len, seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin, rope_pos0=50)
    want = shared_prefix_attention(x.q, eager_k, eager_v, x.prefix_table, 50, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin)

    def f(q, k, v, kp, vp):
        paged_kv_append(k, v, kp, vp, x.block_table, x.kv_len, seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin, rope_pos0=50)
        return shared_prefix_attention(q * 1, kp, vp, x.prefix_table, 50, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin)

    with torch.no_grad():
        got = torch.compile(f, backend="aot_eager", fullgraph=True)(x.q, x.k, x.v, x.k_pages, x.v_pages)
    assert torch.equal(got, want) and torch.equal(x.k_pages, eager_k) and torch.equal(x.v_pages, eager_v)


def test_refusals(gpu_device):
    x = Batch([1, 2], [20, 30], 6, 2, 64, 16, BF16, gpu_device, seed=17)
    from sample_efficient_gpt_amd._lib import SegptError

    with pytest.raises(AssertionError, match="no derivative"):
        paged_attention(x.q.clone().requires_grad_(), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(TypeError):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table.long(), x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(TypeError):
        paged_attention(x.q.half(), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(TypeError):
        paged_attention(x.q.float(), x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(AssertionError):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q)  # three rows of two sequences
    with pytest.raises(AssertionError):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len.cpu(), x.g_q, seq_start=x.seq_start)
    with pytest.raises(AssertionError):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, out=x.q)
    with pytest.raises(AssertionError):
        shared_prefix_attention(x.q, x.k_pages, x.v_pages, x.block_table[0, :1], 17, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(SegptError, match="rope"):
        paged_attention(x.q, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, rope_cos=x.cos[:20], rope_sin=x.sin[:20])
    with pytest.raises(SegptError, match="power of two"):
        paged_attention(x.q, x.k_pages[:, :, :12], x.v_pages[:, :, :12], x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start)
    with pytest.raises(AssertionError):
        paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start, v_first=x.v_first)
    with pytest.raises(SegptError, match="stride"):
        flat = x.k_pages[:1].expand(4, -1, -1, -1)
        paged_kv_append(x.k, x.v, flat, flat, x.block_table, x.kv_len, seq_start=x.seq_start)
    empty = x.q[:0]
    assert paged_attention(empty, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start * 0).shape == empty.shape


@pytest.mark.parametrize("rows,lens,prefix", [
    ([1] * 300, [1 + 29 * i % 150 for i in range(300)], 0),                      # every sequence one token, more than a wave keeps in registers
    ([(0, 1, 1, 3, 12)[i % 5] for i in range(300)], [30 + 17 * i % 90 for i in range(300)], 0),
    ([1] * 300, [i % 40 for i in range(300)], 140),
    ([(1, 0, 14)[i % 3] for i in range(270)], [15 + i % 40 for i in range(270)], 33),
])
@pytest.mark.parametrize("uniform", [False, True])
def test_many_sequences(gpu_device, rows, lens, prefix, uniform):
    for H, Hkv, D, dtype in ((6, 2, 64, BF16), (6, 2, 32, F32)):
        x = Batch(rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=18, prefix=prefix, uniform=uniform and len(set(rows)) == 1)
        y, lse = attend(x, return_lse=True)
        check_y(x, y, lse, x.attended())
        kp, vp = x.appended(pos0=prefix)
        append(x, rope_pos0=prefix)
        check_pools(x, kp, vp)


@pytest.mark.parametrize("H,Hkv,D,dtype", [(16, 8, 64, BF16), (16, 8, 32, F32), (16, 8, 128, BF16)])
def test_a_wave_holds_part_of_its_page_numbers(gpu_device, H, Hkv, D, dtype):
    """Tokens whose shares are longer than 64 pages, beside slots that are not finite behind every sequence's end."""
    lens = [4000 + 37 * i for i in range(64)]
    x = Batch([1] * 64, lens, H, Hkv, D, 8, dtype, gpu_device, seed=19, uniform=True)
    for b, L in enumerate(lens):
        if L % 8:
            x.k_pages[int(x.block_table[b, L // 8]), :, L % 8:] = math.nan
            x.v_pages[int(x.block_table[b, L // 8]), :, L % 8:] = math.inf
    y, lse = attend(x, return_lse=True)
    some = [0, 31, 63]
    ref = Batch([1] * 3, [lens[b] for b in some], H, Hkv, D, 8, dtype, gpu_device, seed=19)
    ref.block_table, ref.k_pages, ref.v_pages, ref.q, ref.cos, ref.sin, ref.g_q = x.block_table[some], x.k_pages, x.v_pages, x.q[some], x.cos, x.sin, x.g_q
    check_y(x, y[some], lse[some], ref.attended())
    alone = attend(ref)  # other shares, other sums
    assert (alone.double() - y[some].double()).norm() <= (6e-3 if dtype == BF16 else 1e-5) * alone.double().norm()
    assert y.isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,lens", [([1, 1], [700, 90]), ([200, 1], [900, 300])])
@pytest.mark.parametrize("order", ["rising", "falling", "spike"])
def test_scores_far_apart(gpu_device, dtype, rows, lens, order):
    """Keys along the queries, so that the scores of a row run over several hundred: upwards (every tile has a new maximum), downwards (all but
    the first underflow), or with one key above all others."""
    for H, Hkv, D in ((6, 2, 64), (4, 2, 128)):
        x = Batch(rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=20, rope=False)
        x.q.copy_(1.0 + 0.05 * torch.randn(x.q.shape, device=gpu_device))
        x.g_q = torch.ones(1, device=gpu_device)
        for b, L in enumerate(lens):
            for p in range(L):
                size = {"rising": p / L, "falling": 1 - p / L, "spike": float(p == L // 2)}[order] * 2 - 1
                x.k_pages[int(x.block_table[b, p // 16]), :, p % 16] = 4.0 * size
        y, lse = attend(x, qk_norm=False, return_lse=True, sm_scale=1.0)
        y_ref, lse_ref, bound = x.attended(qk_norm=False, sm_scale=1.0)
        # scores up to 4 D: their roundings (2^-8 or D 2^-24 of that) move the sums by more than their size at bf16; y stays among the values
        assert y.isfinite().all() and lse.isfinite().all()
        h = H_BF16 if dtype == BF16 else H_F32 * D
        assert ((y.to(F64) - y_ref).abs() <= h * bound).all()
        assert ((lse.to(F64) - lse_ref).abs() <= h * (4.5 * D + 16)).all()


def test_strided_rows_gate_and_out(gpu_device):
    for H, Hkv, D, dtype in ((6, 2, 64, BF16), (4, 2, 128, BF16), (6, 2, 32, F32)):
        for rows, lens in (([1, 1, 1], [40, 9, 200]), ([60, 1, 5], [60, 100, 30])):
            x = Batch(rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=21)
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


def test_lse_of_rows_in_no_sequence(gpu_device):
    x = Batch([1, 3, 9], [20, 40, 9], 6, 2, 64, 16, BF16, gpu_device, seed=22)
    x.seq_start = torch.tensor([2, 3, 6, 8], dtype=torch.int32, device=gpu_device)
    rest = [0, 1, 8, 9, 10, 11, 12]
    for kw in (dict(), dict(out=torch.zeros_like(x.q))):
        _, lse = attend(x, return_lse=True, **kw)
        assert (lse[rest] == -math.inf).all() and lse[2:8].isfinite().all()


def test_two_calls_at_once(gpu_device):
    """Calls on two streams, each with work of its own, give what they give alone."""
    xs = [Batch([1] * 8, [3000 + i for i in range(8)], 18, 6, 64, 16, BF16, gpu_device, seed=23, uniform=True),
          Batch([200, 1, 90], [900, 4000, 300], 18, 6, 64, 32, BF16, gpu_device, seed=24),
          Batch([1] * 20, [i for i in range(20)], 18, 6, 64, 32, BF16, gpu_device, seed=25, prefix=700)]
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


@pytest.mark.parametrize("seed", range(12))
def test_batches_drawn_at_random(gpu_device, seed):
    import random
    r = random.Random(100 + seed)
    H, Hkv, D, dtype = r.choice(HEADS + [(24, 1, 64, BF16), (5, 5, 128, BF16), (33, 11, 64, F32)])
    page, prefix = r.choice([8, 16, 32, 64, 128]), r.choice([0, 0, 1, 31, 32, 100, 257])
    B = r.choice([1, 2, 5, 17, 65])
    rows = [r.choice([0, 1, 1, 2, 5, 11, 33, 64, 129]) for _ in range(B)] if r.random() < 0.7 else [r.choice([1, 4, 12])] * B
    if sum(rows) == 0:
        rows[0] = 1
    lens = [max(n + r.choice([0, 0, 1, 7, 64, 500]) - (r.random() < 0.2), 0) for n in rows]
    x = Batch(rows, lens, H, Hkv, D, page, dtype, gpu_device, seed=seed, prefix=prefix, uniform=len(set(rows)) == 1, rope=r.random() < 0.7,
              layout=r.choice(["phsd", "pshd", "apart"]))
    gate, norm = r.random() < 0.5, r.random() < 0.7
    kp, vp = x.appended(norm, True, pos0=prefix if x.cos is not None else 0)
    append(x, qk_norm=norm, v_first=x.v_first, vr_coef=x.coef, rope_pos0=prefix if x.cos is not None else 0)
    check_pools(x, kp, vp, True)
    y, lse = attend(x, qk_norm=norm, gate_logits=x.gate if gate else None, g_k=x.g_k, sm_scale=0.1, return_lse=True)
    check_y(x, y, lse, x.attended(qk_norm=norm, gate=gate, g_k=x.g_k, sm_scale=0.1))


def test_further_refusals(gpu_device):
    x = Batch([1, 2], [20, 30], 6, 2, 64, 16, BF16, gpu_device, seed=26)
    kw = dict(seq_start=x.seq_start)
    with pytest.raises(AssertionError, match="prefix_table"):
        shared_prefix_attention(x.q, x.k_pages, x.v_pages, None, 16, x.block_table, x.kv_len, x.g_q, **kw)
    with pytest.raises(RuntimeError, match="overlap|single memory location"):
        attend(x, out=x.k_pages.flatten()[: x.q.numel()].view(x.q.shape))
    with pytest.raises(RuntimeError, match="overlap|single memory location"):
        paged_kv_append(x.k, x.v, x.k_pages, x.k_pages, x.block_table, x.kv_len, **kw)
    both = torch.stack([x.k_pages, x.v_pages], 1)  # keys and values of a page side by side are no overlap
    paged_kv_append(x.k, x.v, both[:, 0], both[:, 1], x.block_table, x.kv_len, **kw)
    paged_kv_append(x.k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, **kw)
    assert torch.equal(both[:, 0], x.k_pages) and torch.equal(both[:, 1], x.v_pages)


def test_as_an_operator_with_out(gpu_device):
    """Rows in no sequence keep what they held, also where the call is a node of a graph."""
    x = Batch([1, 9, 3], [40, 20, 30], 6, 2, 64, 16, BF16, gpu_device, seed=27)
    x.seq_start = torch.tensor([1, 2, 11, 12], dtype=torch.int32, device=gpu_device)

    def f(q, out):
        y, lse = paged_attention(q * 1, x.k_pages, x.v_pages, x.block_table, x.kv_len, x.g_q, seq_start=x.seq_start, rope_cos=x.cos, rope_sin=x.sin,
                                 out=out, return_lse=True)
        return y * 2, lse

    eager, traced = torch.full_like(x.q, 7.0), torch.full_like(x.q, 7.0)
    with torch.no_grad():
        want = f(x.q, eager)
        got = torch.compile(f, backend="aot_eager", fullgraph=True)(x.q, traced)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(traced, eager)
    assert (traced[[0, 12]] == 7).all() and not (traced[1:12] == 7).all()


def test_module_refuses_other_values(gpu_device):
    m = MultiHeadSelfAttention(384, 6, 2, max_seq_len=64, qknorm=True, value_residual=True, device=gpu_device, dtype=BF16)
    pages = PageTable(2, 64, 16, device=gpu_device)
    cache = PagedKVCache(pages, 2, 64)
    x = torch.randn(2, 5, 384, device=gpu_device).to(BF16)
    pages.extend(5)
    with torch.no_grad(), pytest.raises(ValueError, match="v1"):
        m(x, v1=torch.zeros(2, 6, 5, 64, device=gpu_device, dtype=BF16), kv_cache=cache)


def test_a_very_long_sequence(gpu_device):
    x = Batch([1, 2], [400_003, 5], 4, 2, 64, 64, BF16, gpu_device, seed=28)
    y, lse = attend(x, return_lse=True)
    check_y(x, y, lse, x.attended())
    z = Batch([1, 40], [3, 50], 4, 2, 64, 64, BF16, gpu_device, seed=29, prefix=200_001)
    y, lse = attend(z, return_lse=True)
    check_y(z, y, lse, z.attended())


@pytest.mark.parametrize("H,Hkv,D,dtype", [(6, 2, 64, BF16), (4, 2, 128, BF16), (4, 2, 64, F32)])
def test_a_long_prompt_is_the_contiguous_attention(gpu_device, H, Hkv, D, dtype):
    """10007 rows, appended and attended in pages, against the attention over contiguous keys (its own roundings: as many again)."""
    from sample_efficient_gpt_amd import qknorm_attention

    n = 10_007
    x = Batch([n], [n], H, Hkv, D, 32, dtype, gpu_device, seed=30)
    append(x)
    y = attend(x)
    with torch.no_grad():
        dense = qknorm_attention(*(t.transpose(0, 1)[None] for t in (x.q, x.k, x.v)), x.g_q, eps=EPS, rope_cos=x.cos, rope_sin=x.sin)
    dense = dense[0].transpose(0, 1).double()
    assert (y.double() - dense).norm() <= (1.2e-2 if dtype == BF16 else 1e-5) * dense.norm()


@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("uniform", [False, True])
def test_lengths_at_the_ends_of_32_bits(gpu_device, prefix, uniform):
    """A length that is no length at all: NaN in that sequence's rows, nothing elsewhere, and nothing outside the tensors is read."""
    x = Batch([2, 2, 2, 2], [9, 40, 30, 2], 6, 2, 64, 16, BF16, gpu_device, seed=31, prefix=prefix, uniform=uniform)
    clean = attend(x)
    x.kv_len[1], x.kv_len[2] = -(2**31), 2**31 - 1
    y = attend(x)
    assert y[2:6].isnan().all() and torch.equal(y[:2], clean[:2]) and torch.equal(y[6:], clean[6:])
    before = x.k_pages.clone()
    append(x, rope_pos0=prefix)
    assert int((x.k_pages != before).any(-1).any(1).sum()) == 4  # slots of the two sequences that have a length


@pytest.mark.parametrize("H,Hkv,D", [(18, 6, 64), (16, 4, 128)])
@pytest.mark.parametrize("rows,lens,prefix,most", [
    ([1] * 32, [200 + 61 * i for i in range(32)], 0, 1.1), ([1, 1], [3000, 500], 0, 1.1),                       # generated tokens
    ([1] * 32, [5 + i for i in range(32)], 1500, 1.5), ([200, 1, 1, 1], [1500, 900, 40, 1200], 0, 1.5), ([700, 300], [700, 900], 0, 1.5),
])
def test_error_of_bf16_is_that_of_its_outputs(gpu_device, rows, lens, prefix, most, H, Hkv, D):
    """Against 64 bits, in units of what rounding the exact y to bf16 costs (r, in norm).  Single tokens of up to 32 heads a kv group: query and
    probabilities are in two parts, what they leave is 2^-14 of a score and of a probability, nothing beside r.  More columns: the probabilities are rounded
    once, an independent error of the size of y's own: sqrt(2) r.  A second such rounding, of the query, would make it sqrt(3) r."""
    x = Batch(rows, lens, H, Hkv, D, 16, BF16, gpu_device, seed=32, prefix=prefix, uniform=len(set(rows)) == 1)
    y_ref = x.attended()[0]
    r = (y_ref.to(BF16).to(F64) - y_ref).norm()
    assert (attend(x).to(F64) - y_ref).norm() <= most * r


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(6, 2, 64, BF16), (4, 2, 128, BF16), (6, 2, 64, F32)])
def test_infinities_are_what_the_formula_makes_of_them(gpu_device, rows, H, Hkv, D, dtype):
    """An infinite value is the answer of the rows that see it, whichever items they are part of.  An infinite component of a key makes the score an
    infinity of the sign that the query's component gives it: NaN where that is positive, no weight where it is negative."""
    x = Batch([rows, rows], [600, 40], H, Hkv, D, 16, dtype, gpu_device, seed=33, uniform=True, rope=False)
    where = 600 - rows  # all rows of the first sequence see this key
    page, slot = int(x.block_table[0, where // 16]), where % 16
    clean = attend(x)
    v = x.v_pages[page, :, slot, 7].clone()
    for sign in (math.inf, -math.inf):
        x.v_pages[page, :, slot, 7] = sign
        y = attend(x)
        assert (y[:rows, :, 7] == sign).all() and torch.equal(y[rows:], clean[rows:])
        assert torch.equal(y[:rows, :, 8:], clean[:rows, :, 8:]) and torch.equal(y[:rows, :, :7], clean[:rows, :, :7])
    x.v_pages[page, :, slot, 7] = v
    x.q[..., 5] = torch.where(x.q[..., 5].abs() < 0.01, torch.ones_like(x.q[..., 5]), x.q[..., 5])
    x.k_pages[page, :, slot, 5] = math.inf
    y = attend(x, qk_norm=False)
    up = x.q[:rows, :, 5] > 0
    assert y[:rows][up].isnan().all() and y[:rows][~up].isfinite().all() and up.any() and (~up).any()
    x.k_pages[page, :, slot, 5] = 30.0 * 2.0**100  # finite, and as far down for the rows whose component is negative
    assert torch.equal(y[:rows][~up], attend(x, qk_norm=False)[:rows][~up])


@pytest.mark.parametrize("H,Hkv,D,dtype", [(6, 2, 64, BF16), (6, 2, 32, F32)])
@pytest.mark.parametrize("rows,lens,prefix", [
    (lambda i: 1, lambda i: 1 + 29 * i % 90, 0), (lambda i: (1, 0, 2, 14)[i % 4], lambda i: 14 + 17 * i % 60, 0), (lambda i: (1, 0, 3)[i % 3], lambda i: 3 + i % 40, 45),
    (lambda i: 3000 * (i == 255), lambda i: 3000 * (i == 255), 0),  # one prompt among sequences without rows
])
@pytest.mark.parametrize("B", [256, 257, 5000])
def test_thousands_of_sequences(gpu_device, B, rows, lens, prefix, H, Hkv, D, dtype):
    """As many as waves plan for by themselves, one more, and more than the plan's workgroup keeps in registers: some of them against the definition, the others against the same call in pieces."""
    rows, lens = [rows(i) for i in range(B)], [lens(i) for i in range(B)]
    x = Batch(rows, lens, H, Hkv, D, 16, dtype, gpu_device, seed=34, prefix=prefix, uniform=len(set(rows)) == 1)
    y, lse = attend(x, return_lse=True)
    assert torch.equal(attend(x), y)
    some = sorted(b for b in {0, 1, 2, 3, 255, 256, 257, 1022, 1023, 1024, 4095, 4096, 4097, B - 2, B - 1} if b < B)
    take = lambda bs: torch.cat([torch.arange(x.starts[b], x.starts[b + 1]) for b in bs]).to(gpu_device)

    def part(bs):
        p = Batch([rows[b] for b in bs], [lens[b] for b in bs], H, Hkv, D, 16, dtype, gpu_device, seed=34, prefix=prefix)
        p.block_table, p.kv_len, p.k_pages, p.v_pages, p.prefix_table = x.block_table[bs], x.kv_len[bs], x.k_pages, x.v_pages, x.prefix_table
        p.q, p.cos, p.sin, p.g_q = x.q[take(bs)], x.cos, x.sin, x.g_q
        return p

    few = part(some)
    if sum(lens) > 3000:
        check_y(few, y[take(some)], lse[take(some)], few.attended())
    for b0 in range(0, B, 200):
        bs = list(range(b0, min(b0 + 200, B)))
        if sum(rows[b] for b in bs):
            z = attend(part(bs))
            assert (z.to(F64) - y[take(bs)].to(F64)).norm() <= (6e-3 if dtype == BF16 else 1e-5) * z.to(F64).norm()


@pytest.mark.parametrize("ragged", [False, True])
def test_two_hundred_thousand_sequences(gpu_device, ragged):
    """Sequences of one to eight keys, in pages that many of them share: the time a call takes grows with the sequences, not with their square."""
    B, H, Hkv, D = 200_000, 4, 2, 64
    g = torch.Generator(device=gpu_device).manual_seed(35)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device)
    kp, vp, q = n(64, Hkv, 8, D).to(BF16), n(64, Hkv, 8, D).to(BF16), n(B, H, D).to(BF16)
    table = torch.randint(0, 64, (B, 1), generator=g, device=gpu_device, dtype=torch.int32)
    lens = torch.randint(1, 9, (B,), generator=g, device=gpu_device, dtype=torch.int32)
    starts = torch.arange(B + 1, device=gpu_device, dtype=torch.int32) if ragged else None
    y = paged_attention(q, kp, vp, table, lens, torch.ones(1, device=gpu_device), seq_start=starts, qk_norm=False)
    r = H // Hkv
    K, V = (p[table[:, 0].long()].float().repeat_interleave(r, 1) for p in (kp, vp))
    s = (q.float()[:, :, None] * K).sum(-1) / 8.0
    s = s.masked_fill(torch.arange(8, device=gpu_device) >= lens[:, None, None], -math.inf)
    want = (torch.softmax(s, -1)[..., None] * V).sum(2)
    assert (y.float() - want).norm() <= 3e-3 * want.norm()  # y's rounding 1.7e-3, and in fp32 sums nothing beside it
    assert ((y.float() - want).abs() <= H_BF16 * (want.abs() + 0.1)).all()


def test_row_ranges_that_overlap_beyond_32_bits(gpu_device):
    """No call is meant to have them, and their rows are undefined: but the partial results of 2^15 sequences of 2^13 rows, counted before those of the last
    sequence, come to 2^31, and nothing may be written there."""
    T, H, D, B = 1 << 13, 256, 64, (1 << 16) + 1
    q = torch.randn(T, H, D, device=gpu_device).to(BF16)
    kp, vp = torch.randn(2, 2, H, 8, D, device=gpu_device).to(BF16)
    table = torch.zeros(B, 1, dtype=torch.int32, device=gpu_device)
    lens = torch.full((B,), 8, dtype=torch.int32, device=gpu_device)
    starts = torch.zeros(B + 1, dtype=torch.int32, device=gpu_device)
    starts[1:-1:2] = T
    starts[-1] = 1
    gain = torch.ones(1, device=gpu_device)
    call = lambda s, n: shared_prefix_attention(q, kp, vp, table[0], 8, table[:n], lens[:n], gain, seq_start=s, qk_norm=False)
    one = torch.tensor([0, T], dtype=torch.int32, device=gpu_device)
    clean = call(one, 1)
    call(starts, B)
    torch.cuda.synchronize()
    assert torch.equal(call(one, 1), clean)


def test_outputs_that_overlap_inputs_are_refused(gpu_device):
    """Rows are read again after others are written.  Views of one buffer that lie side by side in every row are no overlap."""
    rows, lens, H, Hkv, D = [1, 70], [20, 90], 6, 2, 64
    x = Batch(rows, lens, H, Hkv, D, 16, BF16, gpu_device, seed=36)
    want = attend(x, gate_logits=x.gate)
    T = sum(rows)
    wide = torch.zeros(T, 2 * H * D + 64, dtype=BF16, device=gpu_device)
    q, beside = (wide[:, i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(2))
    shifted = wide[:, 3 * D:(H + 3) * D].unflatten(-1, (H, D))
    gate = wide[:, 2 * H * D:2 * H * D + H]
    q.copy_(x.q)
    gate.copy_(x.gate)
    x.q = q
    with pytest.raises(RuntimeError, match="overlap"):
        attend(x, out=shifted)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(x, gate_logits=beside[:, :, 0], out=beside)
    pools = torch.zeros(2, x.n_pages, Hkv, 16, D + 8, dtype=BF16, device=gpu_device)[..., :D]  # rows apart
    pools[0], pools[1] = x.k_pages, x.v_pages
    x.k_pages, x.v_pages = pools[0], pools[1]
    inside = pools.as_strided((T, H, D), (H * (D + 8), D + 8, 1))
    with pytest.raises(RuntimeError, match="overlap"):
        attend(x, out=inside)
    assert torch.equal(attend(x, gate_logits=gate, out=beside), want) and torch.equal(x.q, q)
    k = x.k_pages[:3].flatten(0, 1).transpose(0, 1)[:, :Hkv]  # rows of the pool itself
    starts = torch.tensor([0, 1, k.shape[0]], dtype=torch.int32, device=gpu_device)
    fresh = torch.zeros_like(k)
    for a, b, first in ((k, fresh, None), (fresh, k, None), (fresh, fresh, k)):
        with pytest.raises(RuntimeError, match="overlap"):
            paged_kv_append(a, b, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=starts, v_first=first, vr_coef=None if first is None else x.coef)


def test_a_captured_step_of_unequal_numbers_serves_equal_ones(gpu_device):
    H, Hkv, D = 6, 2, 64
    pages = PageTable(3, 100, 16, device=gpu_device)
    cache = PagedKVCache(pages, Hkv, D)
    gain = torch.ones(1, device=gpu_device)
    q, k, v = (torch.randn(6, h, D, device=gpu_device).to(BF16) for h in (H, Hkv, Hkv))

    def step(n=6):
        cache.append(k[:n], v[:n])
        return cache.attend(q[:n], gain)

    pages.extend([3, 1, 2])
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for rows in (1, [2, 0, 4], 2, [1, 0, 0], 1):
        pages.extend(rows)
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        g.replay()
        n = pages.rows
        got = y.clone()
        assert torch.equal(got[:n], step(n)) and (got[n:] == 0).all(), rows


def test_an_append_of_rows_with_a_gradient_is_refused_under_compilation(gpu_device):
    x = Batch([1, 9], [40, 20], 6, 2, 64, 16, BF16, gpu_device, seed=37)
    k = x.k.clone().requires_grad_()
    before = x.k_pages.clone()

    def f(k):
        paged_kv_append(k, x.v, x.k_pages, x.v_pages, x.block_table, x.kv_len, seq_start=x.seq_start)
        return x.k_pages * 1

    with pytest.raises(Exception, match="no derivative"):
        torch.compile(f, backend="aot_eager", fullgraph=True)(k)
    assert torch.equal(x.k_pages, before)
    with torch.no_grad():
        torch.compile(f, backend="aot_eager", fullgraph=True)(k)
    assert not torch.equal(x.k_pages, before)


@pytest.mark.parametrize("gaps", [[0, 0, 0], [1, 2, 3, 4, 5, 6, 7, 8, 9], [1 << 20, 5, 0, 1 << 19, 63, 64, 65]])
def test_an_append_behind_sequences_without_rows(gpu_device, gaps):
    """Rows of neighbouring sequences with that many in between that bring none: a row finds its own in a few loads, not in one for each of those (2^20
    of them one after the other took 100 ms)."""
    page, Hkv, D = 8, 2, 64
    has = [0]
    for n in gaps:
        has.append(has[-1] + n + 1)
    B, T = has[-1] + 1, len(has)
    rows = torch.zeros(B, dtype=torch.int32)
    rows[has] = 1
    starts = torch.cat([torch.zeros(1, dtype=torch.int32), rows.cumsum(0).int()]).to(gpu_device)
    lens = torch.randint(0, 8, (B,), dtype=torch.int32)
    lens[has] = torch.arange(1, T + 1, dtype=torch.int32) % 8 + 1
    table = torch.zeros(B, 1, dtype=torch.int32)
    table[has, 0] = torch.arange(T, dtype=torch.int32)
    k, v = (torch.randn(T, Hkv, D, device=gpu_device).to(BF16) for _ in range(2))
    kp, vp = torch.zeros(2, T, Hkv, page, D, dtype=BF16, device=gpu_device)
    want = kp.clone(), vp.clone()
    for t, b in enumerate(has):
        for w, x in zip(want, (k, v)):
            w[t, :, int(lens[b]) - 1] = x[t]
    table, lens = table.to(gpu_device), lens.to(gpu_device)
    call = lambda: paged_kv_append(k, v, kp, vp, table, lens, seq_start=starts, qk_norm=False)
    call()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    call()
    b.record()
    torch.cuda.synchronize()
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    assert a.elapsed_time(b) < 20
