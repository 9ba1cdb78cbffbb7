"""Key/value cache in pages, for sequences of unequal lengths: what fills it, what reads it, and the host side that hands out the pages.

The reference's cache (sample_efficient_gpt/transformer/attention.py:15-27) is one tensor per batch, as long as its longest sequence.
Here a sequence's rows lie in pages of a pool that all sequences share, its table says in which, and nothing is padded:

* ``paged_kv_append``          the new rows of every sequence into their pages; keys are rotated and normalised on the way (values mixed
                               with the first layer's), so that the attention reads them as they are.
* ``paged_attention``          the rows of every sequence against the pages of that sequence: one token each, whole prompts, or both
                               in one call.
* ``shared_prefix_attention``  the same for sequences that all begin with one prompt, whose pages are read once for the whole batch.
* ``PageTable``                pages of a batch of sequences, lengths and tables on the device.
* ``PagedKVCache``             the pool of one layer; ``MultiHeadSelfAttention`` takes it as ``kv_cache``.

All three calls are forward only.  Rows of a batch are packed, ``[rows, heads, head_dim]``, those of a sequence side by side.
"""

from __future__ import annotations

import math
from typing import List, Optional

import torch
from torch import Tensor

from . import _native
from .library_op import _seen_as_operator

__all__ = ["paged_kv_append", "paged_attention", "shared_prefix_attention", "PageTable", "PagedKVCache"]


@torch.library.custom_op("segpt::paged_kv_append", mutates_args=("k_pages", "v_pages"))
def _append_op(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, kv_len: Tensor, seq_start: Optional[Tensor],
               v_first: Optional[Tensor], vr_coef: Optional[Tensor], eps: float, qk_norm: bool, rope_cos: Optional[Tensor],
               rope_sin: Optional[Tensor], rope_pos0: int, max_len: Optional[int]) -> None:
    _native.load().paged_append(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, eps, qk_norm, rope_cos, rope_sin,
                                rope_pos0, max_len)


@_append_op.register_fake
def _(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, eps, qk_norm, rope_cos, rope_sin, rope_pos0, max_len):
    return None


@torch.library.custom_op("segpt::paged_attention", mutates_args=())
def _attend_op(q: Tensor, k_pages: Tensor, v_pages: Tensor, prefix_table: Optional[Tensor], prefix_len: int, block_table: Tensor, kv_len: Tensor,
               g_q: Tensor, g_k: Optional[Tensor], seq_start: Optional[Tensor], gate_logits: Optional[Tensor], gate_scale: float, eps: float,
               sm_scale: float, qk_norm: bool, rope_cos: Optional[Tensor], rope_sin: Optional[Tensor], rope_pos0: int,
               max_len: Optional[int]) -> List[Tensor]:
    return list(_native.load().paged_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits,
                                               gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len, None, True))


@_attend_op.register_fake
def _(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm,
      rope_cos, rope_sin, rope_pos0, max_len):
    return [q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)]


@torch.library.custom_op("segpt::paged_attention_out", mutates_args=("out",))
def _attend_out_op(out: Tensor, q: Tensor, k_pages: Tensor, v_pages: Tensor, prefix_table: Optional[Tensor], prefix_len: int, block_table: Tensor,
                   kv_len: Tensor, g_q: Tensor, g_k: Optional[Tensor], seq_start: Optional[Tensor], gate_logits: Optional[Tensor], gate_scale: float,
                   eps: float, sm_scale: float, qk_norm: bool, rope_cos: Optional[Tensor], rope_sin: Optional[Tensor], rope_pos0: int,
                   max_len: Optional[int]) -> Tensor:
    return _native.load().paged_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits,
                                          gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len, out, True)[1]


@_attend_out_op.register_fake
def _(out, q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm,
      rope_cos, rope_sin, rope_pos0, max_len):
    return q.new_empty(q.shape[:2], dtype=torch.float32)


def _no_gradient_asked(what, *operands):
    """The registered operators run below autograd and cannot see that a gradient is asked for."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        raise AssertionError(f"{what} has no derivative: call it under torch.no_grad() or on detached tensors")


def paged_kv_append(k, v, k_pages, v_pages, block_table, kv_len, *, seq_start=None, v_first=None, vr_coef=None, eps=1e-6, qk_norm=True,
                    rope_cos=None, rope_sin=None, rope_pos0=0, max_len=None):
    """Writes the rows k, v ``[T, Hkv, D]`` (any strides, last dim contiguous, rows 16 B aligned) into the pages of their sequences.

    k_pages, v_pages ``[pages, Hkv, page size, D]`` (any strides with a contiguous last dim; page size a power of two from 8 on), written
    in place; block_table int32 ``[B, width]``: the page that holds keys ``j * page size ..`` of sequence b is ``block_table[b, j]``;
    kv_len int32 ``[B]``: keys of a sequence INCLUDING the rows of this call; seq_start int32 ``[B + 1]``: the rows of sequence b are
    ``seq_start[b] .. seq_start[b + 1]`` (None: T / B each).  Row i of n goes to position ``p = kv_len[b] - n + i``.

    What is stored is ``rot(k) * rsqrt(mean(k^2) + eps)`` (qk_norm) with the angles of ``rope_pos0 + p`` (rope_cos / rope_sin
    ``[len, D/2]``, rope.py:36-56), and ``c1 v + c2 v_first`` (``vr_coef`` = (c1, c2), attention.py:228), each rounded once.

    max_len: no sequence holds more keys (default: what its table row can).  Lengths and tables are read on the device: a row whose position
    is negative or not below max_len, or whose page number is not in the pool, is left out.  Two rows of one call must not have one
    slot: sequences must not append into a page they share.  The rows must not lie in the pools (RuntimeError)."""
    if k.is_cuda and not _seen_as_operator(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, rope_cos, rope_sin):
        _native.load().paged_append(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, eps, qk_norm, rope_cos, rope_sin,
                                    rope_pos0, max_len)
    else:
        _no_gradient_asked("paged_kv_append", k, v, k_pages, v_pages, v_first, vr_coef)
        torch.ops.segpt.paged_kv_append(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, float(eps), bool(qk_norm),
                                        rope_cos, rope_sin, int(rope_pos0), max_len)


def _attend(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm,
            rope_cos, rope_sin, rope_pos0, max_len, out, return_lse):
    tensors = (q, k_pages, v_pages, prefix_table, block_table, kv_len, g_q, g_k, seq_start, gate_logits, rope_cos, rope_sin, out)
    if q.is_cuda and not _seen_as_operator(*tensors):
        y, lse = _native.load().paged_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits,
                                                gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len, out, return_lse)
        return (y, lse) if return_lse else y
    _no_gradient_asked("paged attention", q, k_pages, v_pages, g_q, g_k, gate_logits, out)
    args = (q, k_pages, v_pages, prefix_table, int(prefix_len), block_table, kv_len, g_q, g_k, seq_start, gate_logits, float(gate_scale), float(eps),
            float(1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale), bool(qk_norm), rope_cos, rope_sin, int(rope_pos0), max_len)
    if out is None:
        y, lse = torch.ops.segpt.paged_attention(*args)
    else:  # rows in no sequence are left as they are
        y, lse = out, torch.ops.segpt.paged_attention_out(out, *args)
    return (y, lse) if return_lse else y


def paged_attention(q, k_pages, v_pages, block_table, kv_len, g_q, g_k=None, *, seq_start=None, gate_logits=None, gate_scale=2.0, eps=1e-6,
                    sm_scale=None, qk_norm=True, rope_cos=None, rope_sin=None, rope_pos0=0, max_len=None, out=None, return_lse=False):
    """Attention of the rows q ``[T, H, D]`` (unrotated, as projected) over the pages of their sequences, filled by ``paged_kv_append``
    (pages, tables, lengths and rows as there; the same eps, qk_norm and angles).  Row i of n of a sequence sees its keys
    ``0 .. kv_len - n + i``; H is a multiple of the pages' kv heads.

    g_q, g_k scale vectors of 1 or D elements, gate_logits ``[T, H]`` with ``y = gate_scale * sigmoid(z) * o``, sm_scale by default
    ``1/sqrt(D)``: as in ``qknorm_attention``.  Returns y ``[T, H, D]`` (and the natural log-sum-exp ``[T, H]``, fp32).

    A row that sees no key gives y = 0 and lse = -inf.  Rows in no sequence (behind ``seq_start[-1]``) are zero in a y that is allocated
    here, and left as they are in ``out``, which must not overlap an input (RuntimeError); their lse is -inf.  A sequence whose length is negative or above max_len, or whose
    table has a page number that is not in the pool, gives NaN.  A key or value that is not finite takes part in the rows that see it as the formula
    has it, and shows in no other: a key with a NaN gives NaN, one with an infinity NaN or, where its score is -inf, no weight; a value
    that is not finite is what its component of y becomes."""
    return _attend(q, k_pages, v_pages, None, 0, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm,
                   rope_cos, rope_sin, rope_pos0, max_len, out, return_lse)


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k=None, *, seq_start=None, gate_logits=None,
                            gate_scale=2.0, eps=1e-6, sm_scale=None, qk_norm=True, rope_cos=None, rope_sin=None, rope_pos0=0, max_len=None, out=None,
                            return_lse=False):
    """``paged_attention`` for sequences that all begin with the same prefix_len keys, in the pages prefix_table (int32) names: every row
    sees those and then its sequence's own.  The prefix's pages are read once for all rows of the batch, not once a sequence.
    block_table and kv_len are about a sequence's own keys, which may be none; row i of n stands at ``prefix_len + kv_len - n + i`` (among
    the prefix's keys if that is below prefix_len) and sees the keys up to there; the angles of a sequence's first own position are those
    of ``rope_pos0 + prefix_len`` (append with that as ``rope_pos0``)."""
    return _attend(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale,
                   qk_norm, rope_cos, rope_sin, rope_pos0, max_len, out, return_lse)


class PageTable:
    """Which pages of a pool hold the keys of which sequence, for a batch of sequences and all layers of a model.

    ``extend(n)`` before a step makes room for its rows: n more for every sequence, or a list with a number for each.  The device
    tensors ``block_table``, ``kv_len`` and ``seq_start`` are updated in place, so that a captured step sees them: one that was captured with a
    ``seq_start`` serves any step of no more rows, one without (the same number for every sequence) those of that number.  Only an extension
    that begins a new page copies a table from the host.  ``release(b)`` ends sequence b: its pages go back, and it starts again at length 0.

    max_len: keys a sequence may hold.  n_pages: pages of the pool (default: as many as a full batch and the prefix need).
    prefix_len: a prompt all sequences begin with; ``prefix`` is the table of that one sequence, to be extended and filled once.
    """

    def __init__(self, batch, max_len, page_size=64, n_pages=None, prefix_len=0, device="cuda", *, _free=None):
        if batch < 1 or max_len < 1 or prefix_len < 0 or page_size < 8 or page_size & (page_size - 1):
            raise ValueError(f"bad page table: {batch=}, {max_len=}, {prefix_len=}, {page_size=} (a power of two from 8 on)")
        width, prefix_pages = -(-max_len // page_size), -(-prefix_len // page_size)
        self.batch, self.max_len, self.page_size, self.prefix_len = batch, max_len, page_size, prefix_len
        self.n_pages = batch * width + prefix_pages if n_pages is None else n_pages
        if self.n_pages < max(prefix_pages, 1):
            raise ValueError(f"{self.n_pages} pages do not hold a prefix of {prefix_len} keys")
        self._free = list(range(self.n_pages - 1, -1, -1)) if _free is None else _free  # the prefix's table takes from the same pool
        self.lengths = [0] * batch
        self._pages = [[] for _ in range(batch)]
        self._host = torch.zeros(batch, width, dtype=torch.int32)
        self.block_table = torch.zeros(batch, width, dtype=torch.int32, device=device)
        self.kv_len = torch.zeros(batch, dtype=torch.int32, device=device)
        self._starts = None  # handed out as seq_start by the first step of unequal numbers; kept up to date from then on
        self.seq_start, self.rows = None, 0  # of the step that was last made room for: None means rows / batch each
        self.prefix = self.prefix_table = None
        if prefix_len:
            self.prefix = PageTable(1, prefix_len, page_size, self.n_pages, device=device, _free=self._free)
            self.prefix._take([prefix_pages])
            self.prefix_table = self.prefix.block_table[0]

    def _take(self, more):
        """`more` further pages for each sequence."""
        if sum(more) > len(self._free):
            raise RuntimeError(f"the pool is full: {sum(more)} pages wanted, {len(self._free)} of {self.n_pages} free")
        if not any(more):
            return
        for b, m in enumerate(more):
            for _ in range(m):
                self._host[b, len(self._pages[b])] = self._free[-1]
                self._pages[b].append(self._free.pop())
        self.block_table.copy_(self._host)

    def extend(self, n):
        """Room for the rows of the next step; returns self.  Nothing changes if they do not fit (RuntimeError)."""
        each = [int(n)] * self.batch if not hasattr(n, "__len__") else [int(x) for x in n]
        if len(each) != self.batch or min(each) < 0:
            raise ValueError(f"extend takes a number of rows, or one for each of {self.batch} sequences")
        after = [a + x for a, x in zip(self.lengths, each)]
        if max(after) > self.max_len:
            raise RuntimeError(f"a sequence would hold {max(after)} keys, the table has room for {self.max_len}")
        self._take([max(0, -(-a // self.page_size) - len(p)) for a, p in zip(after, self._pages)])
        self.lengths, self.rows = after, sum(each)
        if len(set(each)) == 1:
            self.seq_start = None
            self.kv_len.add_(each[0])
            if self._starts is not None:
                torch.mul(self._numbers, each[0], out=self._starts)
        else:
            starts = [0]
            for x in each:
                starts.append(starts[-1] + x)
            if self._starts is None:
                self._numbers = torch.arange(self.batch + 1, dtype=torch.int32, device=self.kv_len.device)
                self._starts = torch.empty_like(self._numbers)
            self._starts.copy_(torch.tensor(starts, dtype=torch.int32))
            self.kv_len.copy_(torch.tensor(after, dtype=torch.int32))
            self.seq_start = self._starts
        return self

    def release(self, b):
        """Sequence b is over: its pages are free again, its length is 0."""
        if self._pages[b]:
            self._free.extend(reversed(self._pages[b]))
            self._pages[b] = []
        self.lengths[b] = 0
        self.kv_len[b] = 0


class PagedKVCache:
    """Pages of keys and values of one layer, ``[n_pages, Hkv, page size, D]`` each, under a ``PageTable`` that all layers share.

    A step: ``pages.extend(rows)`` once, then for every layer ``append`` and ``attend`` (``MultiHeadSelfAttention`` does both when it is given
    the cache).  ``of(table)`` is the same pool under another table, as ``cache.of(pages.prefix)`` to fill the shared prefix."""

    def __init__(self, pages, n_kv_heads, head_dim, dtype=torch.bfloat16, k_pages=None, v_pages=None):
        self.pages = pages
        shape = (pages.n_pages, n_kv_heads, pages.page_size, head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=pages.kv_len.device) if k_pages is None else k_pages
        self.v_pages = torch.empty(shape, dtype=dtype, device=pages.kv_len.device) if v_pages is None else v_pages
        if self.k_pages.shape != shape or self.v_pages.shape != shape:
            raise ValueError(f"pages must be {shape}, got {tuple(self.k_pages.shape)} and {tuple(self.v_pages.shape)}")

    def of(self, pages):
        return PagedKVCache(pages, self.k_pages.shape[1], self.k_pages.shape[3], self.k_pages.dtype, self.k_pages, self.v_pages)

    def append(self, k, v, *, v_first=None, vr_coef=None, eps=1e-6, qk_norm=True, rope_cos=None, rope_sin=None):
        """The rows ``[T, Hkv, D]`` of the step the table was last extended for."""
        t = self.pages
        assert k.shape[0] == t.rows, f"the table was extended for {t.rows} rows, got {k.shape[0]}"
        paged_kv_append(k, v, self.k_pages, self.v_pages, t.block_table, t.kv_len, seq_start=t.seq_start, v_first=v_first, vr_coef=vr_coef, eps=eps,
                        qk_norm=qk_norm, rope_cos=rope_cos, rope_sin=rope_sin, rope_pos0=t.prefix_len, max_len=t.max_len)

    def attend(self, q, g_q, g_k=None, **kw):
        """The rows ``[T, H, D]`` of that step against their sequences (and the shared prefix); keywords of ``paged_attention``."""
        t = self.pages
        assert q.shape[0] == t.rows, f"the table was extended for {t.rows} rows, got {q.shape[0]}"
        kw = dict(kw, seq_start=t.seq_start, max_len=t.max_len)
        if t.prefix is None:
            return paged_attention(q, self.k_pages, self.v_pages, t.block_table, t.kv_len, g_q, g_k, **kw)
        assert t.prefix.lengths[0] == t.prefix_len, f"the prefix holds {t.prefix.lengths[0]} of its {t.prefix_len} keys"
        return shared_prefix_attention(q, self.k_pages, self.v_pages, t.prefix_table, t.prefix_len, t.block_table, t.kv_len, g_q, g_k, **kw)
