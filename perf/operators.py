"""The serving operators around a paged key/value cache, as data: what is called, on which operands, and what it means.

* ``append``  ``paged_kv_append``: the new rows of every sequence, keys normalised and rotated on the way (values mixed with the
  first layer's, where a model has that), into the pages its table names.
* ``attend``  ``paged_attention``: the rows of every sequence against its own pages.
* ``prefix``  ``shared_prefix_attention``: the same for sequences that begin with one common prompt, whose pages are read once for all.

``step`` says which rows a sequence brings: ``token`` one each (generation), ``mixed`` the first sequence a chunk of a long prompt
and the others one each (what a server runs), ``prompt`` all of its rows (ragged prompts side by side, no padding).
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS, _GATE_SCALE = 1e-6, 2.0


def _case(name, op, step, B, lo, hi, heads, page, *, chunk=0, prefix=0, dtype="bf16", qk_norm=True, rope=True, gate=False, residual=False):
    H, Hkv, D = heads
    c = {"op": op, "step": step, "B": B, "lo": lo, "hi": hi, "H": H, "Hkv": Hkv, "D": D, "page": page, "chunk": chunk, "prefix": prefix,
         "dtype": dtype, "qk_norm": qk_norm, "rope": rope, "gate": gate, "residual": residual}
    return {"name": name, **c} if name else c


def listed():
    imu, wide = (18, 6, 64), (16, 4, 128)
    return [
        # one generated token of one sequence: latency and nothing else
        _case("append_token_b1", "append", "token", 1, 1000, 1000, imu, 64),
        # a generation step of a batch of unequal lengths, value residual on
        _case("append_tokens_b64", "append", "token", 64, 17, 4000, imu, 16, residual=True),
        # ragged prompts entering the cache side by side: bandwidth
        _case("append_prompts_d128", "append", "prompt", 16, 301, 2048, wide, 32),
        # float32 cache of a small model
        _case("append_prompts_fp32", "append", "prompt", 3, 100, 999, (8, 4, 64), 16, dtype="fp32"),
        # one sequence, one token, a cache of some length: latency
        _case("attend_token_b1", "attend", "token", 1, 4096, 4096, imu, 64, gate=True),
        # a batch of unequal lengths: the bandwidth of the cache, and the balance
        _case("attend_tokens_b32", "attend", "token", 32, 200, 8192, imu, 64, gate=True),
        # wide heads, long caches, small pages
        _case("attend_tokens_b48_d128", "attend", "token", 48, 255, 16000, wide, 16),
        # a server's step: 512 tokens of a long prompt, and fifteen sequences generating
        _case("attend_mixed", "attend", "mixed", 16, 999, 8192, imu, 32, chunk=512, gate=True),
        # ragged prompts side by side
        _case("attend_prompts", "attend", "prompt", 6, 333, 4096, imu, 64),
        # float32: a small model's generation step
        _case("attend_tokens_fp32", "attend", "token", 8, 100, 2000, (8, 4, 64), 16, dtype="fp32"),
        # thirty-two conversations behind one system prompt
        _case("prefix_b32", "prefix", "token", 32, 1, 500, imu, 64, prefix=8192, gate=True),
        # many samples of one long document, wide heads, a prefix that ends inside a page
        _case("prefix_b128_d128", "prefix", "token", 128, 5, 300, wide, 16, prefix=16001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "append", "attend", "attend", "attend", "prefix", "prefix"])
        step = rng.choice(["token", "token", "mixed", "prompt"])
        fp32 = rng.random() < 0.2
        heads = rng.choice([(4, 4, 64), (8, 4, 64), (6, 2, 32), (4, 2, 128)] if fp32 else [(18, 6, 64), (18, 6, 64), (16, 4, 128), (8, 8, 64), (16, 4, 64), (32, 2, 128)])
        hi = _log(rng, 16, 4096 if step == "prompt" else 16000)
        lo = min(hi, _log(rng, 1, hi))
        chunk = min(hi, _log(rng, 2, 700)) if step == "mixed" else 0
        prefix = _log(rng, 64, 16000) if op == "prefix" else 0
        c = _case("", op, step, _log(rng, 1, 128), lo, hi, heads, rng.choice([8, 16, 16, 32, 64, 64, 128, 256]), chunk=chunk, prefix=prefix,
                  dtype="fp32" if fp32 else "bf16", qk_norm=rng.random() < 0.85, rope=rng.random() < 0.85, gate=op != "append" and rng.random() < 0.5,
                  residual=op == "append" and rng.random() < 0.4)
        w, most = work(c), [work(x) for x in listed()]
        scale = 8.0 if fp32 else 1.0  # the fp32 products run at a fraction of the bf16 rate
        if w["bytes"] <= max(x["bytes"] for x in most) and w["flops"] * scale <= max(x["flops"] for x in most):
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


class _State:
    """What a program holds before the call."""


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    B, H, Hkv, D, page, prefix = (case[k] for k in ("B", "H", "Hkv", "D", "page", "prefix"))
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
        x = torch.empty(pages, Hkv, page, D, device=dev, dtype=dt)
        for i in range(0, pages, 4096):
            part = n(min(4096, pages - i), Hkv, page, D)
            x[i:i + 4096] = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + _EPS) if unit else part
        return x

    st.k_pages, st.v_pages = pool(case["qk_norm"]), pool(False)
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

    # the rows as the module has them: slices of one projection output
    proj = n(T, (H + 2 * Hkv) * D).to(dt)
    st.q, st.k, st.v = (t.unflatten(-1, (-1, D)) for t in proj.split([H * D, Hkv * D, Hkv * D], dim=-1))
    st.gain = 1.0 + 0.02 * n(D)
    st.cos = st.sin = None
    if case["rope"]:
        length = prefix + width * page
        ang = torch.outer(torch.arange(length, device=dev, dtype=torch.float64), 10_000.0 ** (-2 * torch.arange(D // 2, device=dev, dtype=torch.float64) / D))
        st.cos, st.sin = ang.cos().float(), ang.sin().float()
    st.gate = n(T, H).to(dt) if case["gate"] else None
    st.v_first = st.coef = None
    if case["residual"]:
        st.v_first = n(T, Hkv, D).to(dt)
        lam = 0.3 + 0.4 * torch.rand(1, generator=gen, device=dev)
        st.coef = torch.cat([lam, 1.0 - lam])
    return st


def _positions(st):
    """Of every row: its sequence and where it stands in it."""
    dev = st.q.device
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
    case = st.case
    seq, pos = _positions(st)
    k, v = st.k.float(), st.v.float()
    if case["rope"]:
        k = _rotate(k, st.cos[pos][:, None], st.sin[pos][:, None])
    if case["qk_norm"]:
        k = _unit(k)
    if case["residual"]:
        v = st.coef[0] * v + st.coef[1] * st.v_first.float()
    page, slot = st.block_table[seq, pos // case["page"]].long(), pos % case["page"]
    st.k_pages[page, :, slot] = k.to(st.k_pages.dtype)
    st.v_pages[page, :, slot] = v.to(st.v_pages.dtype)
    return [st.k_pages, st.v_pages]


def _gather(pages, table, page):
    """The pages of some sequences side by side, [sequences, Hkv, keys, D]."""
    x = pages[table.long()].float()  # [sequences, n, Hkv, page, D]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _part(st, q, table, last):
    """Largest score, sum and products of exponentials of the rows q, [sequences, Hkv, rows, D], against the pages of their sequences;
    last: the last key each of them sees, [sequences, rows]."""
    keys, values = (_gather(p, table, st.case["page"]) for p in (st.k_pages, st.v_pages))
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
    if case["step"] == "token":
        m, l, y = _part(st, q, st.block_table, pos[:, None].expand(-1, rep))
    else:  # ragged rows: one sequence after the other
        parts = []
        for b, length in enumerate(st.lens):
            rows = slice(st.starts[b], st.starts[b + 1])
            some = _part(st, q[None, rows].transpose(1, 2).flatten(2, 3), st.block_table[b:b + 1, : -(-length // page)], pos[None, rows].repeat_interleave(rep, 1))
            parts.append([x[0].unflatten(1, (-1, rep)).transpose(0, 1) for x in some])
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


def run(st):
    case = st.case
    if not own:
        return _plain_append(st) if case["op"] == "append" else _plain_attend(st)
    from sample_efficient_gpt_amd import paged_attention, paged_kv_append, shared_prefix_attention

    with torch.no_grad():
        if case["op"] == "append":
            paged_kv_append(st.k, st.v, st.k_pages, st.v_pages, st.block_table, st.kv_len, seq_start=st.seq_start, v_first=st.v_first,
                            vr_coef=st.coef, eps=_EPS, qk_norm=case["qk_norm"], rope_cos=st.cos, rope_sin=st.sin)
            return [st.k_pages, st.v_pages]
        kw = dict(seq_start=st.seq_start, gate_logits=st.gate, gate_scale=_GATE_SCALE, eps=_EPS, qk_norm=case["qk_norm"], rope_cos=st.cos, rope_sin=st.sin)
        if case["op"] == "attend":
            return paged_attention(st.q, st.k_pages, st.v_pages, st.block_table, st.kv_len, st.gain, **kw)
        return shared_prefix_attention(st.q, st.k_pages, st.v_pages, st.prefix_table, case["prefix"], st.block_table, st.kv_len, st.gain, **kw)


def work(case):
    rows, lens = _rows(case)
    H, Hkv, D, prefix = (case[k] for k in ("H", "Hkv", "D", "prefix"))
    elem = 4 if case["dtype"] == "fp32" else 2
    T = sum(rows)
    tables = 4.0 * sum(-(-L // case["page"]) for L in lens) + 4.0 * len(lens)
    angles = 4.0 * D * T if case["rope"] else 0.0
    if case["op"] == "append":
        flops = T * Hkv * D * (4.0 + (3.0 if case["rope"] else 0.0) + (3.0 if case["residual"] else 0.0))
        return {"bytes": T * Hkv * D * elem * (5.0 if case["residual"] else 4.0) + angles + 8.0 * T, "flops": flops}
    pairs = sum(n * (L - n) + n * (n + 1) / 2 for n, L in zip(rows, lens)) + float(T) * prefix  # (query, visible key)
    keys = sum(lens) + prefix
    gate = T * H * elem if case["gate"] else 0
    return {"bytes": 2.0 * T * H * D * elem + 2.0 * keys * Hkv * D * elem + gate + tables + angles, "flops": 4.0 * pairs * H * D}


def exact(case, seed):
    """The definition in float64, sequence by sequence and row by row of a sequence's own list of keys."""
    st = prepare(case, seed)
    H, Hkv, D, page, prefix = (case[k] for k in ("H", "Hkv", "D", "page", "prefix"))
    f64 = torch.float64

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

    def stored(pages, ids, length):  # [length, Hkv, D]
        return torch.cat([pages[i].transpose(0, 1) for i in ids], 0)[:length].to(f64) if ids else torch.zeros(0, Hkv, D, dtype=f64, device=pages.device)

    tables = st.block_table.tolist()
    if case["op"] == "append":
        kp, vp = st.k_pages.to(f64), st.v_pages.to(f64)
        for b, (n, length) in enumerate(zip(st.rows, st.lens)):
            r0 = st.starts[b]
            where = torch.arange(length - n, length, device=kp.device)
            k = scaled(turned(st.k[r0:r0 + n].to(f64), where))
            v = st.v[r0:r0 + n].to(f64)
            if case["residual"]:
                v = st.coef[0].to(f64) * v + st.coef[1].to(f64) * st.v_first[r0:r0 + n].to(f64)
            i = 0
            while i < n:  # page by page
                p = length - n + i
                m = min(n - i, page - p % page)
                at = slice(p % page, p % page + m)
                kp[tables[b][p // page], :, at] = k[i:i + m].transpose(0, 1)
                vp[tables[b][p // page], :, at] = v[i:i + m].transpose(0, 1)
                i += m
        return [kp, vp]
    y = torch.empty(st.q.shape, dtype=f64, device=st.q.device)
    common = st.prefix_table.tolist()
    pk, pv = stored(st.k_pages, common, prefix), stored(st.v_pages, common, prefix)
    for b, (n, length) in enumerate(zip(st.rows, st.lens)):
        r0 = st.starts[b]
        ids = tables[b][: -(-length // page)]
        keys = torch.cat([pk, stored(st.k_pages, ids, length)])
        values = torch.cat([pv, stored(st.v_pages, ids, length)])
        last = prefix + torch.arange(length - n, length, device=y.device)  # the last key a row sees
        q = scaled(turned(st.q[r0:r0 + n].to(f64), last)) * st.gain.to(f64)
        hidden = torch.arange(keys.shape[0], device=y.device)[None] > last[:, None]
        for h in range(H):
            g = h // (H // Hkv)
            s = (q[:, h] @ keys[:, g].T) / math.sqrt(D)
            y[r0:r0 + n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ values[:, g]
    if case["gate"]:
        y *= (_GATE_SCALE / (1.0 + torch.exp(-st.gate.to(f64)))).unsqueeze(-1)
    return y
