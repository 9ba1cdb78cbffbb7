"""The operators around a paged key/value cache of 8 or 4 bits, as data: what is called, on which operands, and what it means.

A row of keys or values is stored in blocks of 32 components.  A block has one scale, the smallest power of two 2^e with
``max |x| <= 2^e top`` (held as the byte e + 127, at least 17), and each component the nearest code of ``x / 2^e``, ties to even:

* ``e4m3``  8 bits, 4 of them exponent, 3 mantissa, ``top`` 448
* ``e2m1``  4 bits, values 0, 0.5, 1, 1.5, 2, 3, 4, 6, two codes a byte, the first in the low half, ``top`` 6

* ``append``   ``paged_kv_append``: the new rows of every sequence, keys normalised and rotated on the way, into such pages.
* ``rewrite``  ``paged_kv_append``, then ``paged_kv_read`` of the rows it wrote: what the rows are from then on.
* ``read``     ``paged_kv_read``: the keys and values of whole sequences back as rows.
* ``attend``   ``paged_attention``: the rows of every sequence against its own pages.
* ``prefix``   ``shared_prefix_attention``: the same for sequences that begin with one common prompt.

``step`` says which rows a sequence brings: ``token`` one each (generation), ``mixed`` the first sequence a chunk of a long prompt
and the others one each (what a server runs), ``prompt`` all of its rows (ragged prompts side by side, no padding).
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS, _GATE_SCALE = 2.0**-20, 2.0  # the first a number of 32 bits, too: codes next to a border are the same for everybody
_BLOCK, _LEAST = 32, -110  # components of a scale, smallest exponent of one


def _case(name, op, fmt, step, B, lo, hi, heads, page, *, chunk=0, prefix=0, dtype="bf16", qk_norm=True, rope=True, gate=False, residual=False):
    H, Hkv, D = heads
    c = {"op": op, "fmt": fmt, "step": step, "B": B, "lo": lo, "hi": hi, "H": H, "Hkv": Hkv, "D": D, "page": page, "chunk": chunk, "prefix": prefix,
         "dtype": dtype, "qk_norm": qk_norm, "rope": rope, "gate": gate, "residual": residual}
    return {"name": name, **c} if name else c


def listed():
    imu, wide = (18, 6, 64), (16, 4, 128)
    return [
        # one generated token of one sequence: latency and nothing else
        _case("append_token_b1", "append", "e4m3", "token", 1, 1000, 1000, imu, 64),
        # ragged prompts entering the cache side by side: bandwidth
        _case("append_prompts_d128", "append", "e4m3", "prompt", 16, 301, 2048, wide, 32),
        # a generation step of a batch of unequal lengths, value residual on, at 4 bits; its rows come back as later steps see them
        _case("rewrite_tokens_b64", "rewrite", "e2m1", "token", 64, 17, 4000, imu, 16, residual=True),
        # sequences leaving the cache, for another one or for the host
        _case("read_seqs_b8", "read", "e4m3", "prompt", 8, 1000, 8192, imu, 64),
        _case("read_seqs_d128_b3", "read", "e2m1", "prompt", 3, 77, 3001, wide, 16),
        # one generated token against one long sequence: the latency of a chat
        _case("attend_token_b1", "attend", "e4m3", "token", 1, 4096, 4096, imu, 64),
        # a generation step of a batch of unequal lengths, gate on
        _case("attend_tokens_b32", "attend", "e4m3", "token", 32, 200, 8192, imu, 64, gate=True),
        # long contexts at 4 bits, heads of 128, small pages
        _case("attend_tokens_d128_b48", "attend", "e2m1", "token", 48, 255, 16000, wide, 16),
        # what a server runs: 512 rows of a prompt beside 31 generated tokens
        _case("attend_mixed_b32", "attend", "e4m3", "mixed", 32, 100, 8192, imu, 32, chunk=512),
        # ragged prompts of a float32 model against a cache of 4 bits
        _case("attend_prompts_fp32", "attend", "e2m1", "prompt", 3, 99, 1500, (8, 4, 64), 16, dtype="fp32"),
        # a batch of chats behind one system prompt
        _case("prefix_tokens_b32", "prefix", "e4m3", "token", 32, 1, 600, imu, 64, prefix=8192, gate=True),
        # the same with a question being read beside the answers
        _case("prefix_mixed_d128", "prefix", "e2m1", "mixed", 24, 30, 900, wide, 32, chunk=200, prefix=5001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "rewrite", "read", "attend", "attend", "attend", "prefix", "prefix"])
        fmt = "e4m3" if op == "append" else rng.choice(["e4m3", "e2m1"])
        step = "prompt" if op == "read" else rng.choice(["token", "token", "mixed", "prompt"])
        fp32 = rng.random() < 0.2
        heads = rng.choice([(4, 4, 64), (8, 4, 64), (6, 2, 32), (4, 2, 128)] if fp32 else [(18, 6, 64), (18, 6, 64), (16, 4, 128), (8, 8, 64), (16, 4, 64), (32, 2, 128)])
        hi = _log(rng, 16, 4096 if step == "prompt" else 16000)
        lo = min(hi, _log(rng, 1, hi))
        chunk = min(hi, _log(rng, 2, 700)) if step == "mixed" else 0
        prefix = _log(rng, 64, 16000) if op == "prefix" else 0
        writes = op in ("append", "rewrite")
        c = _case("", op, fmt, step, _log(rng, 1, 128), lo, hi, heads, rng.choice([8, 16, 16, 32, 64, 64, 128, 256]), chunk=chunk, prefix=prefix,
                  dtype="fp32" if fp32 else "bf16", qk_norm=rng.random() < 0.85, rope=rng.random() < 0.85, gate=op in ("attend", "prefix") and rng.random() < 0.5,
                  residual=writes and rng.random() < 0.4)
        w, most = work(c), [work(x) for x in listed()]
        if w["bytes"] <= max(x["bytes"] for x in most) and w["flops"] * (2.0 if fp32 else 1.0) <= max(x["flops"] for x in most):
            return c


def _rows(case):
    """Rows each sequence brings and the keys it holds with them: spread over lo .. hi, in no order, the same for every seed."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    lens = [lo + int(((b * 0.6180339887498949 + 0.999) % 1.0) * (hi - lo + 1)) for b in range(B)]
    if case["step"] == "prompt":
        return list(lens), lens
    if case["step"] == "mixed":
        lens[0] = hi
        return [case["chunk"]] + [1] * (B - 1), lens
    return [1] * B, lens


def _power(e):
    """2^e, float64, to the last bit."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x, fmt):
    """Codes and scales (uint8) of rows x, in float64: a value next to a border between two codes, or two scales, goes where it belongs."""
    x = x.double().unflatten(-1, (-1, _BLOCK))
    size, power = torch.frexp(x.abs().amax(-1, keepdim=True))  # size in [0.5, 1)
    e = power - 9 + (size > 0.875).int() if fmt == "e4m3" else power - 3 + (size > 0.75).int()
    e = torch.where(size == 0, _LEAST, e.clamp(min=_LEAST))
    x = x * _power(-e)
    _, power = torch.frexp(x)
    step = power.clamp(min=-5) - 4 if fmt == "e4m3" else power.clamp(min=1) - 2  # of the codes around a value
    x = (torch.round(x * _power(-step)) * _power(step)).flatten(-2)
    scales = (e.squeeze(-1) + 127).to(torch.uint8)
    if fmt == "e4m3":
        return x.float().to(torch.float8_e4m3fn).view(torch.uint8), scales
    a = x.abs()
    codes = torch.where(a <= 2, 2 * a, torch.where(a <= 4, a + 2, 7.0)).to(torch.uint8) + 8 * torch.signbit(x).to(torch.uint8)
    return codes[..., 0::2] + 16 * codes[..., 1::2], scales


def _decode(codes, scales, fmt):
    """The values, float32, that codes (uint8) and scales stand for."""
    if fmt == "e4m3":
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        x = values[torch.stack([codes & 15, codes >> 4], -1).int()].flatten(-2)
    return (x.unflatten(-1, (-1, _BLOCK)) * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


class _State:
    """What a program holds before the call."""


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    B, H, Hkv, D, page, prefix, fmt = (case[k] for k in ("B", "H", "Hkv", "D", "page", "prefix", "fmt"))
    n = lambda *s: torch.randn(*s, generator=gen, device=dev, dtype=torch.float32)
    st = _State()
    st.case = case
    st.rows, st.lens = _rows(case)
    T = sum(st.rows)
    used = [-(-L // page) for L in st.lens]
    prefix_pages = -(-prefix // page)
    width = max(used)
    total = sum(used) + prefix_pages
    pages = total + max(4, total // 16)  # a pool is never full

    # prepared keys are rows of mean square 1 (with the normalisation on), values as a projection gives them
    def pool(unit):
        codes = torch.empty(pages, Hkv, page, D if fmt == "e4m3" else D // 2, device=dev, dtype=torch.uint8)
        scales = torch.empty(pages, Hkv, page, D // _BLOCK, device=dev, dtype=torch.uint8)
        at_once = max(1, (1 << 24) // (Hkv * page * D))
        for i in range(0, pages, at_once):
            part = n(min(at_once, pages - i), Hkv, page, D)
            codes[i:i + at_once], scales[i:i + at_once] = _encode(part * torch.rsqrt(part.square().mean(-1, keepdim=True) + _EPS) if unit else part, fmt)
        return codes.view(torch.float8_e4m3fn) if fmt == "e4m3" else codes, scales

    (st.k_pages, st.k_scales), (st.v_pages, st.v_scales) = pool(case["qk_norm"]), pool(False)
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)  # pages are handed out as they become free
    table = torch.zeros(B, width, dtype=torch.int32, device=dev)
    at = prefix_pages
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    st.block_table = table
    st.prefix_table = order[:prefix_pages].clone()
    st.kv_len = torch.tensor(st.lens, dtype=torch.int32, device=dev)
    starts = [0]
    for r in st.rows:
        starts.append(starts[-1] + r)
    st.starts = starts
    st.seq_start = None if case["step"] == "token" else torch.tensor(starts, dtype=torch.int32, device=dev)

    st.gain = 1.0 + 0.02 * n(D)
    st.q = st.k = st.v = st.cos = st.sin = st.gate = st.v_first = st.coef = None
    if case["op"] == "read":
        return st
    # the rows as the module has them: slices of one projection output
    proj = n(T, (H + 2 * Hkv) * D).to(dt)
    st.q, st.k, st.v = (t.unflatten(-1, (-1, D)) for t in proj.split([H * D, Hkv * D, Hkv * D], dim=-1))
    if case["rope"]:
        length = prefix + width * page
        ang = torch.outer(torch.arange(length, device=dev, dtype=torch.float64), 10_000.0 ** (-2 * torch.arange(D // 2, device=dev, dtype=torch.float64) / D))
        st.cos, st.sin = ang.cos().float(), ang.sin().float()
    if case["gate"]:
        st.gate = n(T, H).to(dt)
    if case["residual"]:
        st.v_first = n(T, Hkv, D).to(dt)
        lam = 0.3 + 0.4 * torch.rand(1, generator=gen, device=dev)
        st.coef = torch.cat([lam, 1.0 - lam])
    return st


def _positions(st):
    """Of every row: its sequence and where it stands in it."""
    dev = st.kv_len.device
    rows = torch.tensor(st.rows, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(st.rows), device=dev), rows, output_size=sum(st.rows))
    first = st.kv_len.long() - rows - torch.tensor(st.starts[:-1], device=dev)
    return seq, first[seq] + torch.arange(sum(st.rows), device=dev)


def _rotate(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _unit(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)


def _plain_append(st):
    """In float64: the codes of a value next to a border go by its last bits."""
    case = st.case
    seq, pos = _positions(st)
    k, v = st.k.double(), st.v.double()
    if case["rope"]:
        k = _rotate(k, st.cos[pos][:, None].double(), st.sin[pos][:, None].double())
    if case["qk_norm"]:
        k = _unit(k)
    if case["residual"]:
        c = st.coef.double()
        v = c[0] * v + c[1] * st.v_first.double()
    page, slot = st.block_table[seq, pos // case["page"]].long(), pos % case["page"]
    st.k_pages.view(torch.uint8)[page, :, slot], st.k_scales[page, :, slot] = _encode(k, case["fmt"])
    st.v_pages.view(torch.uint8)[page, :, slot], st.v_scales[page, :, slot] = _encode(v, case["fmt"])


def _plain_read(st):
    case = st.case
    seq, pos = _positions(st)
    page, slot = st.block_table[seq, pos // case["page"]].long(), pos % case["page"]
    return [_decode(c.view(torch.uint8)[page, :, slot], s[page, :, slot], case["fmt"]).to(_DTYPES[case["dtype"]])
            for c, s in ((st.k_pages, st.k_scales), (st.v_pages, st.v_scales))]


def _gather(pages, scales, table, fmt):
    """The pages of some sequences side by side, [sequences, Hkv, keys, D]."""
    x = _decode(pages.view(torch.uint8)[table.long()], scales[table.long()], fmt)  # [sequences, n, Hkv, page, D]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _part(st, q, table, last):
    """Largest score, sum and products of exponentials of the rows q, [sequences, Hkv, rows, D], against the pages of their sequences;
    last: the last key each of them sees, [sequences, rows]."""
    keys, values = (_gather(p, s, table, st.case["fmt"]) for p, s in ((st.k_pages, st.k_scales), (st.v_pages, st.v_scales)))
    s = torch.matmul(q, keys.transpose(2, 3))
    s = s.masked_fill(torch.arange(s.shape[3], device=s.device) > last[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m)
    return m, e.sum(-1, keepdim=True), torch.matmul(e, values)


def _plain_attend(st):
    case = st.case
    H, Hkv, D, page, prefix = (case[k] for k in ("H", "Hkv", "D", "page", "prefix"))
    rep = H // Hkv
    _, pos = _positions(st)
    q = st.q.float()
    if case["rope"]:
        q = _rotate(q, st.cos[prefix + pos][:, None], st.sin[prefix + pos][:, None])
    if case["qk_norm"]:
        q = _unit(q)
    q = (q * st.gain / math.sqrt(D)).unflatten(1, (Hkv, rep))  # [T, Hkv, rep, D]

    def rows_of(b):  # all rows of one sequence
        rows = slice(st.starts[b], st.starts[b + 1])
        some = _part(st, q[None, rows].transpose(1, 2).flatten(2, 3), st.block_table[b:b + 1, : -(-st.lens[b] // page)], pos[None, rows].repeat_interleave(rep, 1))
        return [x[0].unflatten(1, (-1, rep)).transpose(0, 1) for x in some]

    def tokens_from(b):  # one row of each sequence from b on
        rows = slice(st.starts[b], None)
        return _part(st, q[rows], st.block_table[b:, : -(-max(st.lens[b:]) // page)], pos[rows, None].expand(-1, rep))

    if case["step"] == "token":
        parts = [tokens_from(0)]
    elif case["step"] == "mixed":
        parts = [rows_of(0)] + ([tokens_from(1)] if case["B"] > 1 else [])
    else:  # ragged prompts: one after the other
        parts = [rows_of(b) for b in range(case["B"])]
    m, l, y = (torch.cat(x) for x in zip(*parts))
    if prefix:
        end = torch.full((1, q.shape[0] * rep), prefix - 1, device=q.device)
        some = _part(st, q[None].transpose(1, 2).flatten(2, 3), st.prefix_table[None], end)
        pm, pl, py = (x[0].unflatten(1, (-1, rep)).transpose(0, 1) for x in some)
        top = torch.maximum(m, pm)
        a, c = torch.exp(m - top), torch.exp(pm - top)
        l, y = a * l + c * pl, a * y + c * py
    y = (y / l).flatten(1, 2)
    if case["gate"]:
        y = y * (_GATE_SCALE * torch.sigmoid(st.gate.float()))[..., None]
    return y.to(st.q.dtype)


def _pools(st):
    """What an append leaves, as the numbers it stands for: codes and scales (powers of two)."""
    return [st.k_pages, st.v_pages, st.k_scales.view(torch.float8_e8m0fnu), st.v_scales.view(torch.float8_e8m0fnu)]


def run(st):
    case = st.case
    if not own:
        if case["op"] in ("append", "rewrite"):
            _plain_append(st)
            return _pools(st) if case["op"] == "append" else _plain_read(st)
        return _plain_read(st) if case["op"] == "read" else _plain_attend(st)
    from sample_efficient_gpt_amd import paged_attention, paged_kv_append, paged_kv_read, shared_prefix_attention

    scales = dict(k_scales=st.k_scales, v_scales=st.v_scales)
    with torch.no_grad():
        if case["op"] in ("append", "rewrite"):
            paged_kv_append(st.k, st.v, st.k_pages, st.v_pages, st.block_table, st.kv_len, seq_start=st.seq_start, v_first=st.v_first,
                            vr_coef=st.coef, eps=_EPS, qk_norm=case["qk_norm"], rope_cos=st.cos, rope_sin=st.sin, **scales)
            if case["op"] == "append":
                return _pools(st)
        if case["op"] in ("read", "rewrite"):
            return list(paged_kv_read(st.k_pages, st.v_pages, st.block_table, st.kv_len, sum(st.rows), seq_start=st.seq_start, dtype=_DTYPES[case["dtype"]], **scales))
        kw = dict(seq_start=st.seq_start, gate_logits=st.gate, gate_scale=_GATE_SCALE, eps=_EPS, qk_norm=case["qk_norm"], rope_cos=st.cos, rope_sin=st.sin, **scales)
        if case["op"] == "attend":
            return paged_attention(st.q, st.k_pages, st.v_pages, st.block_table, st.kv_len, st.gain, **kw)
        return shared_prefix_attention(st.q, st.k_pages, st.v_pages, st.prefix_table, case["prefix"], st.block_table, st.kv_len, st.gain, **kw)


def work(case):
    rows, lens = _rows(case)
    op, H, Hkv, D, prefix = (case[k] for k in ("op", "H", "Hkv", "D", "prefix"))
    elem = 4 if case["dtype"] == "fp32" else 2
    held = D * (1.0 if case["fmt"] == "e4m3" else 0.5) + D / _BLOCK  # bytes of a stored row
    T = sum(rows)
    angles = 4.0 * D * T if case["rope"] else 0.0
    tables = 4.0 * sum(-(-L // case["page"]) for L in lens) + 4.0 * len(lens)
    if op in ("append", "rewrite", "read"):
        row = T * Hkv  # of keys, and as many of values
        writes, reads = op != "read", op != "append"
        into = row * (D * elem * (3.0 if case["residual"] else 2.0) + 2.0 * held) + angles + 8.0 * T
        back = row * 2.0 * (held + D * elem) + tables
        per = D * (10.0 + (3.0 if case["rope"] else 0.0) + (3.0 if case["residual"] else 0.0))
        return {"bytes": into * writes + back * reads, "flops": row * (per * writes + 2.0 * D * reads)}
    pairs = sum(n * (L - n) + n * (n + 1) / 2 for n, L in zip(rows, lens)) + float(T) * prefix  # (query, visible key)
    keys = sum(lens) + prefix
    gate = T * H * elem if case["gate"] else 0
    return {"bytes": 2.0 * T * H * D * elem + 2.0 * keys * Hkv * held + gate + tables + angles, "flops": 4.0 * pairs * H * D}


def exact(case, seed):
    """The definition in float64, sequence by sequence and row by row of a sequence's own list of keys; codes by search in the list of all
    numbers that there are."""
    st = prepare(case, seed)
    H, Hkv, D, page, prefix, fmt = (case[k] for k in ("H", "Hkv", "D", "page", "prefix", "fmt"))
    f64, dev = torch.float64, st.kv_len.device
    if fmt == "e4m3":
        numbers = [(m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:-1]
    else:
        numbers = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    numbers = torch.tensor(numbers, dtype=f64, device=dev)
    borders = (numbers[1:] + numbers[:-1]) / 2
    powers = torch.tensor([2.0**i for i in range(-127, 256)], dtype=f64, device=dev)  # of a scale's byte less 127

    def two_to(e):
        return powers[(e + 127).long().clamp(0, 382)]

    def stored(x):  # the values x becomes, and its scales
        blocks = x.reshape(*x.shape[:-1], -1, _BLOCK)
        big = blocks.abs().amax(-1)
        e = torch.ceil(torch.log2(big / numbers[-1]))
        e = torch.where(big == 0, float(_LEAST), e)
        e = torch.where(big <= numbers[-1] * two_to(e - 1), e - 1, e)
        e = torch.where(big > numbers[-1] * two_to(e), e + 1, e)
        scale = two_to(e.clamp(min=float(_LEAST)))
        u = (blocks / scale[..., None]).abs()
        low, high = torch.bucketize(u, borders), torch.bucketize(u, borders, right=True)
        at = torch.where((low != high) & (low % 2 == 1), high, low)  # on a border: the even one
        return (numbers[at] * blocks.sign()).reshape(x.shape), scale

    def held(codes, scales):  # the values of stored rows
        if fmt == "e4m3":
            x = codes.view(torch.float8_e4m3fn).to(f64)
        else:
            c = codes.long()
            x = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=f64, device=dev)
            x[..., 0::2], x[..., 1::2] = c % 16, c // 16
            x = numbers[(x % 8).long()] * (1 - 2 * (x >= 8).to(f64))
        return x * two_to(scales.to(f64) - 127).repeat_interleave(_BLOCK, -1)

    def turned(x, where):  # x: [rows, heads, D] at positions where
        if not case["rope"]:
            return x
        c, s = st.cos.to(f64)[where].unsqueeze(1), st.sin.to(f64)[where].unsqueeze(1)
        y = torch.empty_like(x)
        half = D // 2
        y[..., :half] = x[..., :half] * c - x[..., half:] * s
        y[..., half:] = x[..., half:] * c + x[..., :half] * s
        return y

    def scaled(x):
        return x / (x.pow(2).mean(-1, keepdim=True) + _EPS).sqrt() if case["qk_norm"] else x

    def listed_rows(pages, scales, ids, length):  # [length, Hkv, D]
        if not ids:
            return torch.zeros(0, Hkv, D, dtype=f64, device=dev)
        return torch.cat([held(pages[i], scales[i]).transpose(0, 1) for i in ids], 0)[:length]

    tables, k_codes, v_codes = st.block_table.tolist(), st.k_pages.view(torch.uint8), st.v_pages.view(torch.uint8)
    if case["op"] in ("append", "rewrite"):
        kp, vp = (st.k_pages.to(f64), st.v_pages.to(f64)) if fmt == "e4m3" else (None, None)
        ks, vs = (two_to(s.to(f64) - 127) for s in (st.k_scales, st.v_scales))
        back = [], []
        for b, (n, length) in enumerate(zip(st.rows, st.lens)):
            r0 = st.starts[b]
            k = scaled(turned(st.k[r0:r0 + n].to(f64), torch.arange(length - n, length, device=dev)))
            v = st.v[r0:r0 + n].to(f64)
            if case["residual"]:
                v = st.coef[0].to(f64) * v + st.coef[1].to(f64) * st.v_first[r0:r0 + n].to(f64)
            (kc, kk), (vc, vv) = stored(k), stored(v)
            if case["op"] == "rewrite":
                back[0].append(kc * kk.repeat_interleave(_BLOCK, -1))
                back[1].append(vc * vv.repeat_interleave(_BLOCK, -1))
                continue
            i = 0
            while i < n:  # page by page
                p = length - n + i
                m = min(n - i, page - p % page)
                at = (tables[b][p // page], slice(None), slice(p % page, p % page + m))
                for pool, new in ((kp, kc), (ks, kk), (vp, vc), (vs, vv)):
                    pool[at] = new[i:i + m].transpose(0, 1)
                i += m
        return [torch.cat(x) for x in back] if case["op"] == "rewrite" else [kp, vp, ks, vs]
    own_pages = [tables[b][: -(-length // page)] for b, length in enumerate(st.lens)]
    if case["op"] == "read":
        return [torch.cat([listed_rows(p, s, ids, length) for ids, length in zip(own_pages, st.lens)]) for p, s in ((k_codes, st.k_scales), (v_codes, st.v_scales))]
    y = torch.empty(st.q.shape, dtype=f64, device=dev)
    common = st.prefix_table.tolist()
    pk, pv = listed_rows(k_codes, st.k_scales, common, prefix), listed_rows(v_codes, st.v_scales, common, prefix)
    for b, (n, length) in enumerate(zip(st.rows, st.lens)):
        r0 = st.starts[b]
        ids = torch.tensor(own_pages[b], device=dev)
        keys, values = (torch.cat([before, held(p[ids], s[ids]).transpose(1, 2).reshape(-1, Hkv, D)[:length]])
                        for before, p, s in ((pk, k_codes, st.k_scales), (pv, v_codes, st.v_scales)))
        last = prefix + torch.arange(length - n, length, device=dev)  # the last key a row sees
        q = scaled(turned(st.q[r0:r0 + n].to(f64), last)) * st.gain.to(f64)
        hidden = torch.arange(keys.shape[0], device=dev)[None] > last[:, None]
        for h in range(H):
            g = h // (H // Hkv)
            s = (q[:, h] @ keys[:, g].T) / math.sqrt(D)
            y[r0:r0 + n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ values[:, g]
    if case["gate"]:
        y *= (_GATE_SCALE / (1.0 + torch.exp(-st.gate.to(f64)))).unsqueeze(-1)
    return y
