"""Pools of 8 and 4 bits and their definition in float64, beside tests/paged_util.py."""

import torch

from paged_util import F64, Batch

FORMATS = ("e4m3", "e2m1")
BLOCK, LEAST, MOST = 32, -110, {"e4m3": 119, "e2m1": 125}
NUMBERS = {"e4m3": torch.tensor([m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:-1], dtype=F64),
           "e2m1": torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64)}
POWERS = torch.tensor([2.0**i for i in range(-130, 131)], dtype=F64)


def power(e):
    return POWERS.to(e.device)[(e + 130).clamp(0, 260)]


def encode(x, fmt):
    """(codes, scales): bytes that rows x (last dim a multiple of 32) are stored as."""
    numbers = NUMBERS[fmt].to(x.device)
    x = x.to(F64).unflatten(-1, (-1, BLOCK))
    big = x.abs().amax(-1)
    e = torch.full(big.shape, LEAST, dtype=torch.long, device=x.device)
    for up in (128, 64, 32, 16, 8, 4, 2, 1):  # the largest number below the answer, less one
        e = torch.where(big > numbers[-1] * power(e + up - 1), e + up, e)
    none = ~x.isfinite().all(-1) | (e > MOST[fmt])
    u = torch.where(none[..., None], 0.0, x.abs() / power(e)[..., None])
    borders = (numbers[1:] + numbers[:-1]) / 2
    low, high = torch.bucketize(u, borders), torch.bucketize(u, borders, right=True)
    codes = torch.where((low != high) & (low % 2 == 1), high, low)
    codes = (codes + (128 if fmt == "e4m3" else 8) * (x.signbit() & ~none[..., None])).flatten(-2)
    if fmt == "e2m1":
        codes = codes[..., 0::2] + 16 * codes[..., 1::2]
    return codes.to(torch.uint8), torch.where(none, 255, e + 127).to(torch.uint8)


def decode(codes, scales, fmt):
    """The values of stored rows, float64."""
    numbers, c = NUMBERS[fmt].to(codes.device), codes.view(torch.uint8).long()
    if fmt == "e2m1":
        c = torch.stack([c % 16, c // 16], -1).flatten(-2)
    half = 128 if fmt == "e4m3" else 8
    at = c % half
    x = torch.where(at < len(numbers), numbers[at.clamp(max=len(numbers) - 1)], torch.nan) * (1 - 2 * (c >= half).to(F64))
    s = scales.view(torch.uint8).long()
    return (x.unflatten(-1, (-1, BLOCK)) * torch.where(s == 255, torch.nan, power(s - 127))[..., None]).flatten(-2)


class QuantBatch(Batch):
    """A Batch whose pools are codes and scales.  layout: as there ("apart": rows and scales with room behind them, page size + 1 rows a page)."""

    def __init__(self, fmt, *a, layout="phsd", **kw):
        super().__init__(*a, layout="phsd", **kw)
        self.fmt = fmt
        (self.k_pages, self.k_scales), (self.v_pages, self.v_scales) = (self.stored(x, layout) for x in (self.k_pages, self.v_pages))

    def stored(self, x, layout):
        codes, scales = encode(x, self.fmt)
        codes, scales = self._laid_out(codes, layout, 16), self._laid_out(scales, layout, self.D // 32)
        return codes.view(torch.float8_e4m3fn) if self.fmt == "e4m3" else codes, scales

    def _laid_out(self, x, layout, room):
        if layout == "phsd":
            return x.contiguous()
        if layout == "pshd":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.full((x.shape[0], x.shape[1], x.shape[2] + 1, x.shape[3] + room), 99, dtype=x.dtype, device=x.device)
        wide[:, :, :-1, :-room] = x
        return wide[:, :, :-1, :-room]

    def scales(self):
        return dict(k_scales=self.k_scales, v_scales=self.v_scales)

    def values(self):
        return decode(self.k_pages, self.k_scales, self.fmt), decode(self.v_pages, self.v_scales, self.fmt)

    def appended_codes(self, **kw):
        """What k_pages, k_scales, v_pages, v_scales are to be after the append (bytes), and which slots it writes."""
        kc, ks, vc, vs = (t.view(torch.uint8).clone() for t in (self.k_pages, self.k_scales, self.v_pages, self.v_scales))
        k, v = self._prepared(**kw)
        (kn, kns), (vn, vns) = encode(k, self.fmt), encode(v, self.fmt)
        for t, (b, p) in enumerate(self.positions()):
            if p >= 0:
                at = (int(self.block_table[b, p // self.page]), slice(None), p % self.page)
                kc[at], ks[at], vc[at], vs[at] = kn[t], kns[t], vn[t], vns[t]
        return kc, ks, vc, vs

    def _prepared(self, qk_norm=True, mix=False, pos0=0, eps=2.0**-20):
        pos = torch.tensor([p for _, p in self.positions()], device=self.device, dtype=torch.long)
        k, v = self.turned(self.k, pos + pos0), self.v.to(F64)
        if qk_norm:
            k = k / (k.square().mean(-1, keepdim=True) + eps).sqrt()
        if mix:
            v = self.coef[0].to(F64) * v + self.coef[1].to(F64) * self.v_first.to(F64)
        return k, v

    def attended(self, **kw):
        k, v = self.values()
        return super().attended(k_pages=k, v_pages=v, **kw)
