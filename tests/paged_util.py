"""Inputs of the paged cache's operators and their definition in float64, sequence by sequence."""

import math

import torch

F64 = torch.float64
EPS = 1e-6


class Batch:
    """Ragged rows over a pool whose pages are handed out in no order.  rows / lens: per sequence, lens including the rows."""

    def __init__(self, rows, lens, H, Hkv, D, page, dtype, device, *, prefix=0, seed=0, spare=3, uniform=False, rope=True, layout="phsd", pool_values=None):
        g = torch.Generator().manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)
        self.rows, self.lens, self.H, self.Hkv, self.D, self.page, self.prefix = list(rows), list(lens), H, Hkv, D, page, prefix
        self.dtype, self.device = dtype, device
        T = sum(rows)
        used = [-(-L // page) for L in lens]
        pp = -(-prefix // page)
        self.width = max(max(used), 1)
        self.n_pages = sum(used) + pp + spare
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        table = torch.full((len(lens), self.width), -7, dtype=torch.int32)  # numbers behind a sequence's last page are never looked at
        at = pp
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        self.block_table = table.to(device)
        self.prefix_table = order[:pp].clone().to(device)
        self.spare_pages = order[at:].tolist()
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device=device)
        self.starts = [0]
        for r in rows:
            self.starts.append(self.starts[-1] + r)
        self.seq_start = None if uniform else torch.tensor(self.starts, dtype=torch.int32, device=device)
        unit = n(self.n_pages, Hkv, page, D)
        unit = unit * torch.rsqrt(unit.square().mean(-1, keepdim=True))
        self.k_pages, self.v_pages = self._pool(unit, layout), self._pool(n(self.n_pages, Hkv, page, D), layout)
        proj = n(max(T, 1), (H + 2 * Hkv) * D)[:T].to(dtype).to(device)
        self.q, self.k, self.v = (t.unflatten(-1, (-1, D)) for t in proj.split([H * D, Hkv * D, Hkv * D], dim=-1))
        self.v_first = n(T, Hkv, D).to(dtype).to(device)
        self.gate = n(T, H).to(dtype).to(device)
        self.g_q, self.g_k = (1.0 + 0.1 * n(D)).to(device), (1.0 + 0.1 * n(D)).to(device)
        self.coef = torch.tensor([0.9, -0.4], device=device)
        self.cos = self.sin = None
        if rope:
            length = prefix + self.width * page + 5
            ang = torch.outer(torch.arange(length, dtype=F64), 10_000.0 ** (-2 * torch.arange(D // 2, dtype=F64) / D))
            self.cos, self.sin = ang.cos().float().to(device), ang.sin().float().to(device)

    def _pool(self, x, layout):
        x = x.to(self.dtype).to(self.device)
        if layout == "phsd":
            return x
        if layout == "pshd":  # pages of [slot, head, D]
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.zeros(x.shape[0], x.shape[1], x.shape[2] + 1, x.shape[3] + 8, dtype=x.dtype, device=x.device)  # rows apart
        wide[:, :, :-1, :-8] = x
        return wide[:, :, :-1, :-8]

    def positions(self):
        """(sequence, position) of every row."""
        return [(b, L - n + i) for b, (n, L) in enumerate(zip(self.rows, self.lens)) for i in range(n)]

    def turned(self, x, pos):
        if self.cos is None:
            return x.to(F64)
        c, s = (t.to(F64)[pos.clamp(min=0)].unsqueeze(1) for t in (self.cos, self.sin))
        a, b = x.to(F64).chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    def appended(self, qk_norm=True, mix=False, pos0=0):
        """The two pools after the append, in float64."""
        kp, vp = self.k_pages.to(F64), self.v_pages.to(F64)
        pos = torch.tensor([p for _, p in self.positions()], device=self.device, dtype=torch.long)
        k, v = self.turned(self.k, pos + pos0), self.v.to(F64)
        if qk_norm:
            k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS)
        if mix:
            v = self.coef[0].to(F64) * v + self.coef[1].to(F64) * self.v_first.to(F64)
        for t, (b, p) in enumerate(self.positions()):
            if p < 0:
                continue
            page, slot = int(self.block_table[b, p // self.page]), p % self.page
            kp[page, :, slot], vp[page, :, slot] = k[t], v[t]
        return kp, vp

    def _list(self, pages, ids, length):
        if length == 0:
            return torch.zeros(0, self.Hkv, self.D, dtype=F64, device=self.device)
        return pages[ids[: -(-length // self.page)].long()].to(F64).transpose(1, 2).reshape(-1, self.Hkv, self.D)[:length]

    def attended(self, g_k=None, gate=False, qk_norm=True, gate_scale=2.0, sm_scale=None, pos0=0, k_pages=None, v_pages=None):
        """(y, lse, bound): float64; bound: how far roundings of qhat, probabilities and y to bf16 can move y (module docstring of the tests)."""
        H, Hkv, D = self.H, self.Hkv, self.D
        sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
        kp, vp = (self.k_pages if k_pages is None else k_pages), (self.v_pages if v_pages is None else v_pages)
        T = sum(self.rows)
        y = torch.zeros(T, H, D, dtype=F64, device=self.device)
        lse = torch.full((T, H), -math.inf, dtype=F64, device=self.device)
        bound = torch.zeros(T, H, D, dtype=F64, device=self.device)
        pk, pv = self._list(kp, self.prefix_table, self.prefix), self._list(vp, self.prefix_table, self.prefix)
        for b, (n, L) in enumerate(zip(self.rows, self.lens)):
            if n == 0:
                continue
            r = slice(self.starts[b], self.starts[b + 1])
            last = torch.arange(L - n, L, device=self.device)
            q = self.turned(self.q[r], last + self.prefix + pos0)
            if qk_norm:
                q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS)
            q = q * self.g_q.to(F64) * sm_scale * (1.0 if g_k is None else g_k.to(F64))
            keys = torch.cat([pk, self._list(kp, self.block_table[b], L)])
            vals = torch.cat([pv, self._list(vp, self.block_table[b], L)])
            sees = torch.arange(keys.shape[0], device=self.device)[None] <= self.prefix + last[:, None]
            any_key = sees.any(-1)
            for h in range(H):
                k_h, v_h = keys[:, h // (H // Hkv)], vals[:, h // (H // Hkv)]
                s = (q[:, h] @ k_h.T).masked_fill(~sees, -math.inf)
                lse[r, h] = torch.logsumexp(s, -1)
                p = torch.softmax(s, -1).masked_fill(~any_key[:, None], 0.0)
                # an unseen key takes no part, whatever is stored for it
                o = torch.stack([p[i, sees[i]] @ v_h[sees[i]] for i in range(n)]) if not v_h.isfinite().all() else p @ v_h
                y[r, h] = o
                spread = (q[:, h].abs() @ k_h.abs().T).masked_fill(~sees, 0.0).amax(-1, keepdim=True) if keys.shape[0] else torch.zeros(n, 1, dtype=F64, device=self.device)
                weight = p @ v_h.abs().nan_to_num(posinf=0.0)
                bound[r, h] = (2 * spread + 2) * weight
        if gate:
            f = (gate_scale * torch.sigmoid(self.gate.to(F64)))[..., None]
            y, bound = y * f, bound * f
        return y, lse, bound + y.abs().nan_to_num()
