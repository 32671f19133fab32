"""Plain float64 CPU forms of the rotation and the paged cache, and builders of caches whose
unused rows hold NaN and whose unused table entries name pages that do not exist."""

from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    """x [..., D] float64, positions broadcast over its leading dims."""
    n = inv_freq.numel()
    angle = positions.double().unsqueeze(-1) * inv_freq.double().cpu()
    c, s = angle.cos() * scale, angle.sin() * (-scale if inverse else scale)
    y = x.clone()
    if interleaved:
        a, b = x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]
        y[..., 0 : 2 * n : 2], y[..., 1 : 2 * n : 2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :n], x[..., n : 2 * n]
        y[..., :n], y[..., n : 2 * n] = a * c - b * s, b * c + a * s
    return y


def quantise(x):
    """(codes [..., D / 2], scale bytes [..., D / 32]) of x float64, nearest by distance."""
    g = x.unflatten(-1, (x.size(-1) // 32, 32))
    top = g.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(-126, 127)
    y = torch.ldexp(g.abs(), -e)
    gap = (y.unsqueeze(-1) - GRID).abs()
    near, which = gap.sort(dim=-1, stable=True)
    # (Of two codes equally near the even one.)
    tie = (near[..., 0] == near[..., 1]) & (which[..., 0] % 2 == 1)
    code = torch.where(tie, which[..., 1], which[..., 0])
    code = code + 8 * torch.signbit(g)
    scale = torch.where(top > 0, e + 127, torch.zeros_like(e)).squeeze(-1)
    bad = ~torch.isfinite(g).all(-1)
    scale = torch.where(bad, torch.full_like(scale, 255), scale).to(torch.uint8)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def values(codes, scale):
    """What codes and scale bytes stand for, float64."""
    table = torch.cat((GRID, -GRID))
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    f = torch.exp2(scale.double() - 127)
    f = torch.where(scale == 255, torch.full_like(f, math.nan), f)
    return (v.unflatten(-1, (scale.size(-1), 32)) * f.unsqueeze(-1)).flatten(-2)


def cu_of(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


class Cache:
    """A paged cache on the CPU: `lens` keys a sequence out of dense float64 keys / values."""

    def __init__(self, lens, heads, d, dv, page, dtype, bits, seed=0, rows_last=False, spare=1, room=0, empty=False):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.d, self.dv, self.page, self.dtype, self.bits = lens, heads, d, dv, page, dtype, bits
        counts = [-(-(n + room) // page) for n in lens]
        self.pages = sum(counts) + spare
        order = torch.randperm(self.pages, generator=g)
        width = max(max(counts), 1) + 2
        # Entries that no key needs name pages far outside the cache.
        self.table = torch.randint(10**6, 2**31 - 1, (len(lens), width), generator=g)
        self.table[:, 1::2] *= -1
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.table = self.table.to(torch.int32)
        self.k, self.v = [], []
        for n in lens:
            self.k.append(torch.randn(n, heads, d, generator=g, dtype=torch.float64).to(dtype))
            self.v.append(torch.randn(n, heads, dv, generator=g, dtype=torch.float64).to(dtype))
        # Rows that hold no key: NaN, or codes and scales that stand for it.
        def fresh(dim):
            shape = (self.pages, heads, page)
            if rows_last:
                shape = (self.pages, page, heads)
            if bits == 16:
                t = (torch.full((*shape, dim), math.nan, dtype=dtype),)
            else:
                t = (torch.full((*shape, dim // 2), 0x77, dtype=torch.uint8), torch.full((*shape, dim // 32), 255, dtype=torch.uint8))
            return [x.transpose(1, 2) for x in t] if rows_last else list(t)

        self.kt, self.vt = fresh(d), fresh(dv)
        if not empty:
            for b in range(len(lens)):
                self.write(b, torch.arange(lens[b]), self.k[b].double(), self.v[b].double())

    def write(self, b, pos, k, v):
        """Keys / values [n, heads, D] float64 at positions of sequence b."""
        page, row = self.table[b, pos // self.page].long(), pos % self.page
        for held, x in ((self.kt, k), (self.vt, v)):
            parts = (x.to(self.dtype),) if self.bits == 16 else quantise(x)
            for t, part in zip(held, parts):
                t[page, :, row] = part

    def held(self, b):
        """Sequence b's keys and values as the cache holds them, float64."""
        pos = torch.arange(self.lens[b])
        page, row = self.table[b, pos // self.page].long(), pos % self.page
        out = []
        for held in (self.kt, self.vt):
            parts = [t[page, :, row] for t in held]
            out.append(parts[0].double() if self.bits == 16 else values(*parts))
        return out

    def to(self, dev):
        """Keyword arguments of the operators."""
        out = {"k_cache": self.kt[0].to(dev), "v_cache": self.vt[0].to(dev), "block_table": self.table.to(dev),
               "key_lengths": torch.tensor(self.lens, dtype=torch.int32, device=dev)}
        if self.bits == 4:
            out |= {"k_scale": self.kt[1].to(dev), "v_scale": self.vt[1].to(dev)}
        return out


def attention(q, k, v, causal, scale):
    """(out, sum of |weights v|, largest |score| sum) of q [n, H, D] over k / v [m, Hk, D], the queries
    being the last n keys; float64.  Rows without keys are zero."""
    n, h, _ = q.shape
    m, group = k.size(0), h // k.size(1)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("nhd,mhd->hnm", q, k) * scale
    # What the score's error scales with: the sum of its products' magnitudes.
    mag = torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()) * abs(scale)
    if causal:
        hidden = torch.arange(m) > (torch.arange(n) + m - n).unsqueeze(1)
        s = s.masked_fill(hidden, -math.inf)
        mag = mag.masked_fill(hidden, 0.0)
    top = s.amax(-1, keepdim=True) if m else s.new_zeros(h, n, 1)
    w = torch.exp(s - top.clamp(min=-1e300))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, torch.zeros_like(w))
    out = torch.einsum("hnm,mhd->nhd", w, v)
    size = torch.einsum("hnm,mhd->nhd", w, v.abs())
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf)).squeeze(-1)
    return out, size, (mag.amax(-1) if m else mag.new_zeros(h, n)).t().unsqueeze(-1), lse
