"""Key/value cache in pages, for sequences of unequal lengths: what fills it, what reads it, and the host side that hands out the pages.

The reference's cache (sample_efficient_gpt/transformer/attention.py:15-27) is one tensor per batch, as long as its longest sequence.
Here a sequence's rows lie in pages of a pool that all sequences share, its table says in which, and nothing is padded:

* ``paged_kv_append``          the new rows of every sequence into their pages; keys are rotated and normalised on the way (values mixed
                               with the first layer's), so that the attention reads them as they are.
* ``paged_attention``          the rows of every sequence against the pages of that sequence: one token each, whole prompts, or both
                               in one call.
* ``shared_prefix_attention``  the same for sequences that all begin with one prompt, whose pages are read once for the whole batch.
* ``paged_kv_read``            stored rows back as rows.
* ``PageTable``                pages of a batch of sequences, lengths and tables on the device.
* ``PagedKVCache``             the pool of one layer; ``MultiHeadSelfAttention`` takes it as ``kv_cache``.

All calls are forward only.  Rows of a batch are packed, ``[rows, heads, head_dim]``, those of a sequence side by side.

**Pages of 8 or 4 bits.**  A pool of the rows' dtype holds a row as it is.  With ``k_scales`` and ``v_scales`` it holds codes, in blocks of 32
components with one power of two each: twice or four times as many keys in the same memory, and as many fewer bytes a generated token has to read.

* ``float8_e4m3fn`` pages ``[pages, Hkv, page size, D]``: 8 bits, 3 of them mantissa.
* ``uint8`` (or ``float4_e2m1fn_x2``) pages ``[pages, Hkv, page size, D / 2]``: 4 bits a component, 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, two
  components a byte, the first in the low half.
* scales ``uint8`` (or ``float8_e8m0fnu``) ``[pages, Hkv, page size, D / 32]``: the byte e + 127 of ``2^e``, e the smallest number from -110 on
  with which no component exceeds the largest code (448, 6).  255: the block is NaN, as one with a component that is not finite becomes.

A component is the nearest code of its exact value, ties to the even one.  What is attended to is the stored value, exactly.  Rows may be bfloat16 or
float32, head_dim 64 or 128, with float32 rows also 32.
"""

from __future__ import annotations

import math
from typing import List, Optional

import torch
from torch import Tensor

from . import _native
from .library_op import _seen_as_operator

__all__ = ["paged_kv_append", "paged_kv_read", "paged_attention", "shared_prefix_attention", "PageTable", "PagedKVCache"]


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


# ---- the same over pages of 8 or 4 bits

@torch.library.custom_op("segpt::paged_kv_append_scaled", mutates_args=("k_pages", "v_pages", "k_scales", "v_scales"))
def _append_scaled_op(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, block_table: Tensor, kv_len: Tensor,
                      seq_start: Optional[Tensor], v_first: Optional[Tensor], vr_coef: Optional[Tensor], eps: float, qk_norm: bool,
                      rope_cos: Optional[Tensor], rope_sin: Optional[Tensor], rope_pos0: int, max_len: Optional[int]) -> None:
    _native.load().paged_append_scaled(k, v, k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, v_first, vr_coef, eps, qk_norm, rope_cos,
                                       rope_sin, rope_pos0, max_len)


@_append_scaled_op.register_fake
def _(k, v, k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, v_first, vr_coef, eps, qk_norm, rope_cos, rope_sin, rope_pos0, max_len):
    return None


@torch.library.custom_op("segpt::paged_attention_scaled", mutates_args=())
def _attend_scaled_op(q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, prefix_table: Optional[Tensor], prefix_len: int,
                      block_table: Tensor, kv_len: Tensor, g_q: Tensor, g_k: Optional[Tensor], seq_start: Optional[Tensor],
                      gate_logits: Optional[Tensor], gate_scale: float, eps: float, sm_scale: float, qk_norm: bool, rope_cos: Optional[Tensor],
                      rope_sin: Optional[Tensor], rope_pos0: int, max_len: Optional[int]) -> List[Tensor]:
    return list(_native.load().paged_attention_scaled(q, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_len, g_q, g_k,
                                                      seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len,
                                                      None, True))


@_attend_scaled_op.register_fake
def _(q, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale,
      qk_norm, rope_cos, rope_sin, rope_pos0, max_len):
    return [q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)]


@torch.library.custom_op("segpt::paged_attention_scaled_out", mutates_args=("out",))
def _attend_scaled_out_op(out: Tensor, q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, prefix_table: Optional[Tensor],
                          prefix_len: int, block_table: Tensor, kv_len: Tensor, g_q: Tensor, g_k: Optional[Tensor], seq_start: Optional[Tensor],
                          gate_logits: Optional[Tensor], gate_scale: float, eps: float, sm_scale: float, qk_norm: bool, rope_cos: Optional[Tensor],
                          rope_sin: Optional[Tensor], rope_pos0: int, max_len: Optional[int]) -> Tensor:
    return _native.load().paged_attention_scaled(q, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start,
                                                 gate_logits, gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len, out, True)[1]


@_attend_scaled_out_op.register_fake
def _(out, q, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale,
      qk_norm, rope_cos, rope_sin, rope_pos0, max_len):
    return q.new_empty(q.shape[:2], dtype=torch.float32)


def _head_dim(k_pages, k_scales):
    return k_pages.shape[3] * (2 if k_scales is not None and k_pages.dtype != torch.float8_e4m3fn else 1)


@torch.library.custom_op("segpt::paged_kv_read", mutates_args=())
def _read_op(k_pages: Tensor, v_pages: Tensor, k_scales: Optional[Tensor], v_scales: Optional[Tensor], block_table: Tensor, kv_len: Tensor, rows: int,
             seq_start: Optional[Tensor], dtype: torch.dtype, max_len: Optional[int]) -> List[Tensor]:
    return list(_native.load().paged_read(k_pages, v_pages, k_scales, v_scales, block_table, kv_len, rows, seq_start, dtype, max_len, None, None))


@_read_op.register_fake
def _(k_pages, v_pages, k_scales, v_scales, block_table, kv_len, rows, seq_start, dtype, max_len):
    shape = (rows, k_pages.shape[1], _head_dim(k_pages, k_scales))
    return [k_pages.new_empty(shape, dtype=dtype), k_pages.new_empty(shape, dtype=dtype)]


@torch.library.custom_op("segpt::paged_kv_read_out", mutates_args=("k", "v"))
def _read_out_op(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Optional[Tensor], v_scales: Optional[Tensor], block_table: Tensor,
                 kv_len: Tensor, seq_start: Optional[Tensor], max_len: Optional[int]) -> None:
    _native.load().paged_read(k_pages, v_pages, k_scales, v_scales, block_table, kv_len, k.shape[0], seq_start, k.dtype, max_len, k, v)


@_read_out_op.register_fake
def _(k, v, k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, max_len):
    return None


def _no_gradient_asked(what, *operands):
    """The registered operators run below autograd and cannot see that a gradient is asked for."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        raise AssertionError(f"{what} has no derivative: call it under torch.no_grad() or on detached tensors")


def _both_scales(k_scales, v_scales):
    if k_scales is None or v_scales is None:
        raise AssertionError("k_scales and v_scales go together")


def paged_kv_append(k, v, k_pages, v_pages, block_table, kv_len, *, seq_start=None, v_first=None, vr_coef=None, eps=1e-6, qk_norm=True,
                    rope_cos=None, rope_sin=None, rope_pos0=0, max_len=None, k_scales=None, v_scales=None):
    """Writes the rows k, v ``[T, Hkv, D]`` (any strides, last dim contiguous, rows 16 B aligned) into the pages of their sequences.

    k_pages, v_pages ``[pages, Hkv, page size, D]`` (any strides with a contiguous last dim; page size a power of two from 8 on), written
    in place; block_table int32 ``[B, width]``: the page that holds keys ``j * page size ..`` of sequence b is ``block_table[b, j]``;
    kv_len int32 ``[B]``: keys of a sequence INCLUDING the rows of this call; seq_start int32 ``[B + 1]``: the rows of sequence b are
    ``seq_start[b] .. seq_start[b + 1]`` (None: T / B each).  Row i of n goes to position ``p = kv_len[b] - n + i``.

    What is stored is ``rot(k) * rsqrt(mean(k^2) + eps)`` (qk_norm) with the angles of ``rope_pos0 + p`` (rope_cos / rope_sin
    ``[len, D/2]``, rope.py:36-56), and ``c1 v + c2 v_first`` (``vr_coef`` = (c1, c2), attention.py:228), each rounded once; with k_scales and
    v_scales (see above) as codes and scales, all four tensors written in place.

    max_len: no sequence holds more keys (default: what its table row can).  Lengths and tables are read on the device: a row whose position
    is negative or not below max_len, or whose page number is not in the pool, is left out.  Two rows of one call must not have one
    slot: sequences must not append into a page they share.  The rows must not lie in the pools (RuntimeError)."""
    if k_scales is not None or v_scales is not None:
        args = (k, v, k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, v_first, vr_coef, float(eps), bool(qk_norm), rope_cos, rope_sin,
                int(rope_pos0), max_len)
        if k.is_cuda and not _seen_as_operator(k, v, k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, v_first, vr_coef, rope_cos, rope_sin):
            _native.load().paged_append_scaled(*args)
        else:
            _no_gradient_asked("paged_kv_append", k, v, k_pages, v_pages, v_first, vr_coef)
            _both_scales(k_scales, v_scales)
            torch.ops.segpt.paged_kv_append_scaled(*args)
    elif k.is_cuda and not _seen_as_operator(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, rope_cos, rope_sin):
        _native.load().paged_append(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, eps, qk_norm, rope_cos, rope_sin,
                                    rope_pos0, max_len)
    else:
        _no_gradient_asked("paged_kv_append", k, v, k_pages, v_pages, v_first, vr_coef)
        torch.ops.segpt.paged_kv_append(k, v, k_pages, v_pages, block_table, kv_len, seq_start, v_first, vr_coef, float(eps), bool(qk_norm),
                                        rope_cos, rope_sin, int(rope_pos0), max_len)


def _attend(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm,
            rope_cos, rope_sin, rope_pos0, max_len, out, return_lse, k_scales, v_scales):
    tensors = (q, k_pages, v_pages, prefix_table, block_table, kv_len, g_q, g_k, seq_start, gate_logits, rope_cos, rope_sin, out)
    if k_scales is not None or v_scales is not None:
        if q.is_cuda and not _seen_as_operator(*tensors, k_scales, v_scales):
            y, lse = _native.load().paged_attention_scaled(q, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_len, g_q, g_k,
                                                           seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len,
                                                           out, return_lse)
            return (y, lse) if return_lse else y
        _both_scales(k_scales, v_scales)
    elif q.is_cuda and not _seen_as_operator(*tensors):
        y, lse = _native.load().paged_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits,
                                                gate_scale, eps, sm_scale, qk_norm, rope_cos, rope_sin, rope_pos0, max_len, out, return_lse)
        return (y, lse) if return_lse else y
    _no_gradient_asked("paged attention", q, k_pages, v_pages, g_q, g_k, gate_logits, out)
    args = (prefix_table, int(prefix_len), block_table, kv_len, g_q, g_k, seq_start, gate_logits, float(gate_scale), float(eps),
            float(1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale), bool(qk_norm), rope_cos, rope_sin, int(rope_pos0), max_len)
    args, ops = ((q, k_pages, v_pages, *args), (torch.ops.segpt.paged_attention, torch.ops.segpt.paged_attention_out)) if k_scales is None else (
        (q, k_pages, v_pages, k_scales, v_scales, *args), (torch.ops.segpt.paged_attention_scaled, torch.ops.segpt.paged_attention_scaled_out))
    if out is None:
        y, lse = ops[0](*args)
    else:  # rows in no sequence are left as they are
        y, lse = out, ops[1](out, *args)
    return (y, lse) if return_lse else y


def paged_attention(q, k_pages, v_pages, block_table, kv_len, g_q, g_k=None, *, seq_start=None, gate_logits=None, gate_scale=2.0, eps=1e-6,
                    sm_scale=None, qk_norm=True, rope_cos=None, rope_sin=None, rope_pos0=0, max_len=None, out=None, return_lse=False, k_scales=None,
                    v_scales=None):
    """Attention of the rows q ``[T, H, D]`` (unrotated, as projected) over the pages of their sequences, filled by ``paged_kv_append``
    (pages, their scales, tables, lengths and rows as there; the same eps, qk_norm and angles).  Row i of n of a sequence sees its keys
    ``0 .. kv_len - n + i``; H is a multiple of the pages' kv heads.

    g_q, g_k scale vectors of 1 or D elements, gate_logits ``[T, H]`` with ``y = gate_scale * sigmoid(z) * o``, sm_scale by default
    ``1/sqrt(D)``: as in ``qknorm_attention``.  Returns y ``[T, H, D]`` (and the natural log-sum-exp ``[T, H]``, fp32).

    A row that sees no key gives y = 0 and lse = -inf.  Rows in no sequence (behind ``seq_start[-1]``) are zero in a y that is allocated
    here, and left as they are in ``out``, which must not overlap an input (RuntimeError); their lse is -inf.  A sequence whose length is negative or above max_len, or whose
    table has a page number that is not in the pool, gives NaN.  A key or value that is not finite takes part in the rows that see it as the formula
    has it, and shows in no other: a key with a NaN gives NaN, one with an infinity NaN or, where its score is -inf, no weight; a value
    that is not finite is what its component of y becomes."""
    return _attend(q, k_pages, v_pages, None, 0, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale, qk_norm,
                   rope_cos, rope_sin, rope_pos0, max_len, out, return_lse, k_scales, v_scales)


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k=None, *, seq_start=None, gate_logits=None,
                            gate_scale=2.0, eps=1e-6, sm_scale=None, qk_norm=True, rope_cos=None, rope_sin=None, rope_pos0=0, max_len=None, out=None,
                            return_lse=False, k_scales=None, v_scales=None):
    """``paged_attention`` for sequences that all begin with the same prefix_len keys, in the pages prefix_table (int32) names: every row
    sees those and then its sequence's own.  The prefix's pages are read once for all rows of the batch, not once a sequence.
    block_table and kv_len are about a sequence's own keys, which may be none; row i of n stands at ``prefix_len + kv_len - n + i`` (among
    the prefix's keys if that is below prefix_len) and sees the keys up to there; the angles of a sequence's first own position are those
    of ``rope_pos0 + prefix_len`` (append with that as ``rope_pos0``)."""
    return _attend(q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_len, g_q, g_k, seq_start, gate_logits, gate_scale, eps, sm_scale,
                   qk_norm, rope_cos, rope_sin, rope_pos0, max_len, out, return_lse, k_scales, v_scales)


def paged_kv_read(k_pages, v_pages, block_table, kv_len, rows, *, seq_start=None, k_scales=None, v_scales=None, dtype=None, max_len=None, out=None):
    """Stored rows back as rows: the pair (k, v) ``[rows, Hkv, D]`` that ``paged_kv_append`` would have to be given, without angles, normalisation and mix,
    for the same pages (pages, scales, tables, lengths and row ranges as there).  Row i of n of sequence b is its key ``kv_len[b] - n + i``;
    rows is the number of all rows, ``seq_start[-1]`` or a multiple of the sequences.

    dtype: of the rows; bfloat16 by default, or float32 (both exact; heads of 32 are float32) where the pages have scales, else the pages' own.  out: a pair of tensors to write to
    (any strides, last dim contiguous, rows 16 B aligned; no overlap with inputs or each other, RuntimeError), whose dtype counts.

    A row before its sequence's first key is 0.  A sequence whose length is negative or above max_len gives NaN, and so does a row whose page number is
    not in the pool.  Rows in no sequence are zero in what is allocated here, and left as they are in ``out``."""
    k, v = (None, None) if out is None else out
    if dtype is None:
        dtype = k.dtype if k is not None else torch.bfloat16 if k_scales is not None else k_pages.dtype
    if k_pages.is_cuda and not _seen_as_operator(k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, k, v):
        return _native.load().paged_read(k_pages, v_pages, k_scales, v_scales, block_table, kv_len, rows, seq_start, dtype, max_len, k, v)
    _no_gradient_asked("paged_kv_read", k_pages, v_pages, k, v)
    if out is None:
        return tuple(torch.ops.segpt.paged_kv_read(k_pages, v_pages, k_scales, v_scales, block_table, kv_len, int(rows), seq_start, dtype, max_len))
    if k.shape[0] != rows or k.dtype != dtype:
        raise AssertionError(f"out must be {rows} rows of {dtype}")
    torch.ops.segpt.paged_kv_read_out(k, v, k_pages, v_pages, k_scales, v_scales, block_table, kv_len, seq_start, max_len)
    return k, v


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


_ROWS_AT_ONCE = 1 << 18  # of a cache that is turned into one of another dtype


class PagedKVCache:
    """Pages of keys and values of one layer, ``[n_pages, Hkv, page size, D]`` each, under a ``PageTable`` that all layers share.

    dtype: bfloat16 or float32, that of the rows; or float8_e4m3fn or float4_e2m1fn_x2 (or uint8, the same), for rows of either: pages of 8 or 4 bits, with
    ``k_scales`` and ``v_scales`` beside them.  Pools that are handed in are of the table's shape; codes say themselves what they are.

    A step: ``pages.extend(rows)`` once, then for every layer ``append`` and ``attend`` (``MultiHeadSelfAttention`` does both when it is given
    the cache).  ``of(table)`` is the same pool under another table, as ``cache.of(pages.prefix)`` to fill the shared prefix.  ``read()`` is what it
    holds; ``to(dtype)`` is a cache of another dtype with the same keys and values, as of a prompt that was worked out in bfloat16 and goes on at 4 bits."""

    def __init__(self, pages, n_kv_heads, head_dim, dtype=torch.bfloat16, k_pages=None, v_pages=None, k_scales=None, v_scales=None):
        if k_pages is not None and k_pages.dtype in (torch.uint8, torch.float8_e4m3fn, torch.float4_e2m1fn_x2):
            dtype = k_pages.dtype  # pools say themselves what they are
        if dtype == torch.uint8:
            dtype = torch.float4_e2m1fn_x2  # two codes a byte, as in the functions
        scaled = dtype in (torch.float8_e4m3fn, torch.float4_e2m1fn_x2)
        if scaled and head_dim not in (32, 64, 128):
            raise ValueError(f"pages of 8 and 4 bits have a head_dim of 32, 64 or 128, got {head_dim}")
        self.pages, self.head_dim = pages, head_dim
        device, rows = pages.kv_len.device, (pages.n_pages, n_kv_heads, pages.page_size)
        shape = (*rows, head_dim // 2 if dtype == torch.float4_e2m1fn_x2 else head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device) if k_pages is None else k_pages
        self.v_pages = torch.empty(shape, dtype=self.k_pages.dtype, device=device) if v_pages is None else v_pages
        if self.k_pages.shape != shape or self.v_pages.shape != shape:
            raise ValueError(f"pages must be {shape}, got {tuple(self.k_pages.shape)} and {tuple(self.v_pages.shape)}")
        if self.k_pages.dtype != self.v_pages.dtype:
            raise ValueError(f"pages must have one dtype, got {self.k_pages.dtype} and {self.v_pages.dtype}")
        self.k_scales = self.v_scales = None
        if scaled:
            shape = (*rows, head_dim // 32)
            self.k_scales = torch.empty(shape, dtype=torch.uint8, device=device) if k_scales is None else k_scales
            self.v_scales = torch.empty(shape, dtype=torch.uint8, device=device) if v_scales is None else v_scales
            if self.k_scales.shape != shape or self.v_scales.shape != shape:
                raise ValueError(f"scales must be {shape}, got {tuple(self.k_scales.shape)} and {tuple(self.v_scales.shape)}")
        elif k_scales is not None or v_scales is not None:
            raise ValueError(f"pages of {dtype} have no scales")

    @property
    def dtype(self):
        """float4_e2m1fn_x2 also where the pages are bytes."""
        return torch.float4_e2m1fn_x2 if self.k_pages.dtype == torch.uint8 else self.k_pages.dtype

    def of(self, pages):
        return PagedKVCache(pages, self.k_pages.shape[1], self.head_dim, self.dtype, self.k_pages, self.v_pages, self.k_scales, self.v_scales)

    def append(self, k, v, *, v_first=None, vr_coef=None, eps=1e-6, qk_norm=True, rope_cos=None, rope_sin=None):
        """The rows ``[T, Hkv, D]`` of the step the table was last extended for."""
        t = self.pages
        assert k.shape[0] == t.rows, f"the table was extended for {t.rows} rows, got {k.shape[0]}"
        paged_kv_append(k, v, self.k_pages, self.v_pages, t.block_table, t.kv_len, seq_start=t.seq_start, v_first=v_first, vr_coef=vr_coef, eps=eps,
                        qk_norm=qk_norm, rope_cos=rope_cos, rope_sin=rope_sin, rope_pos0=t.prefix_len, max_len=t.max_len, k_scales=self.k_scales,
                        v_scales=self.v_scales)

    def attend(self, q, g_q, g_k=None, **kw):
        """The rows ``[T, H, D]`` of that step against their sequences (and the shared prefix); keywords of ``paged_attention``."""
        t = self.pages
        assert q.shape[0] == t.rows, f"the table was extended for {t.rows} rows, got {q.shape[0]}"
        kw = dict(kw, seq_start=t.seq_start, max_len=t.max_len, k_scales=self.k_scales, v_scales=self.v_scales)
        if t.prefix is None:
            return paged_attention(q, self.k_pages, self.v_pages, t.block_table, t.kv_len, g_q, g_k, **kw)
        assert t.prefix.lengths[0] == t.prefix_len, f"the prefix holds {t.prefix.lengths[0]} of its {t.prefix_len} keys"
        return shared_prefix_attention(q, self.k_pages, self.v_pages, t.prefix_table, t.prefix_len, t.block_table, t.kv_len, g_q, g_k, **kw)

    def read(self, dtype=None):
        """Everything the table's sequences hold, packed: ``(k, v, seq_start)``, keys as the attention multiplies them."""
        return self._read(0, len(self.pages.lengths), dtype)

    def _read(self, first, end, dtype=None):
        t = self.pages
        starts = [0]
        for n in t.lengths[first:end]:
            starts.append(starts[-1] + n)
        seq_start = torch.tensor(starts, dtype=torch.int32).to(t.kv_len.device)
        if dtype is None and self.k_scales is not None and self.head_dim == 32:
            dtype = torch.float32  # the only rows of 32 that there are
        k, v = paged_kv_read(self.k_pages, self.v_pages, t.block_table[first:end], t.kv_len[first:end], starts[-1], seq_start=seq_start, k_scales=self.k_scales,
                             v_scales=self.v_scales, dtype=dtype, max_len=t.max_len)
        return k, v, seq_start

    def to(self, dtype):
        """A cache of this dtype in pages of its own, under the same table and with the same keys and values (the shared prefix's among them).  Rows
        pass through memory of their own, some sequences at a time."""
        if dtype == torch.uint8:
            dtype = torch.float4_e2m1fn_x2
        if dtype == self.dtype:
            return self
        if dtype not in (torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float4_e2m1fn_x2):
            raise ValueError(f"no cache has the dtype {dtype}")
        if dtype == torch.bfloat16 and self.head_dim == 32:
            raise ValueError("a head_dim of 32 is one of float32 rows")
        other = PagedKVCache(self.pages, self.k_pages.shape[1], self.head_dim, dtype)
        rows = dtype if other.k_scales is None else torch.float32 if self.dtype == torch.float32 or self.head_dim == 32 else torch.bfloat16
        for t in (self.pages, self.pages.prefix):
            if t is None:
                continue
            source, b = self.of(t), 0
            while b < len(t.lengths):
                e, n = b + 1, t.lengths[b]
                while e < len(t.lengths) and n + t.lengths[e] <= _ROWS_AT_ONCE:
                    n += t.lengths[e]
                    e += 1
                if n:
                    k, v, seq_start = source._read(b, e)
                    with torch.no_grad():
                        paged_kv_append(k.to(rows), v.to(rows), other.k_pages, other.v_pages, t.block_table[b:e], t.kv_len[b:e], seq_start=seq_start,
                                        qk_norm=False, max_len=t.max_len, k_scales=other.k_scales, v_scales=other.v_scales)
                b = e
        return other
