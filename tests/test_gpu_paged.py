"""The rotation and the paged cache on the GPU against plain float64 forms on the CPU.

Tolerances.  A rounding to the result's type is off by half a step at most (``half_step``).

* Rotation: products and sine / cosine in 32 bits, each off by 2^-22 at most (sincospif's two
  units in the last place, the fused products), so ``2^-21 (|x1| + |x2|)`` and half a step.
* 4-bit codes are those of exact arithmetic: equal.
* Attention: weights rounded to 16 bits before the product with V, and in the tile kernel
  summed as rounded: two half steps of ``sum |w v|``; the result's own half step; scores off by
  ``delta`` change a weight by ``exp(+- 2 delta)``.  delta of 32-bit sums of D products: ``D 2^-24
  sum |q k|``; of the scaled MFMA, which aligns its products to the largest of a group and
  drops what lies 2^-13 below, 2^-12 of the same.  Elementwise that bound is far above what rounding
  does to a sum over many keys, so the root mean square is held too: both roundings are
  independent of the values there, sqrt(2) half steps of the result's own, and 2 delta.
"""

from __future__ import annotations

import math

import pytest
import torch

import paged_cases as P

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture()
def ops(dev, native):
    return native


def _randn(*shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64).to(dtype)


def _freq(pairs, base=1e6):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float()


# ---------------------------------------------------------------- rotation


def _check_rotated(y, x, positions, freq, interleaved, scale=1.0, inverse=False):
    ref = P.rotate(x.double(), positions, freq, interleaved, scale, inverse)
    size = P.rotate(x.double().abs(), torch.zeros_like(positions), freq, interleaved)
    n = 2 * freq.numel()
    pair = size.clone()
    if interleaved:
        pair[..., 0:n:2] += size[..., 1:n:2]
        pair[..., 1:n:2] += size[..., 0:n:2]
    else:
        pair[..., : n // 2] += size[..., n // 2 : n]
        pair[..., n // 2 : n] += size[..., : n // 2]
    tol = ref.abs() * P.half_step(x.dtype) + 2.0**-21 * scale * pair + 2.0**-25
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of its tolerance"
    assert torch.equal(y[..., n:].cpu(), x[..., n:])


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(
    "tokens,heads,heads_k,d,rd",
    [(1, 1, 1, 128, 128), (8, 16, 2, 128, 128), (37, 14, 2, 64, 64), (5, 3, 1, 128, 64), (700, 4, 4, 96, 32),
     (9, 2, 1, 20, 6), (3, 5, 2, 80, 80), (2, 1, 1, 2, 2), (11, 71, 1, 64, 48), (4, 8, 8, 256, 256), (6, 2, 2, 255, 254)],
)
def test_rotary_packed(ops, dev, dtype, interleaved, tokens, heads, heads_k, d, rd):
    q, k = _randn(tokens, heads, d, seed=1, dtype=dtype), _randn(tokens, heads_k, d, seed=2, dtype=dtype)
    pos = torch.randint(0, 2_000_000, (tokens,), generator=torch.Generator().manual_seed(3))
    freq = _freq(rd // 2)
    y, ky = ops.rotary(q.to(dev), pos.to(dev), freq.to(dev), k=k.to(dev), interleaved=interleaved)
    for out, x in ((y, q), (ky, k)):
        assert out.dtype == dtype and out.shape == x.shape
        _check_rotated(out, x, pos.unsqueeze(1), freq, interleaved)
    alone = ops.rotary(q.to(dev), pos.to(dev).int(), freq.to(dev), interleaved=interleaved)
    assert torch.equal(alone, y)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_dense_views_and_positions(ops, dev, dtype, interleaved):
    b, h, s, d = 3, 6, 50, 64
    rows = _randn(b, s, 3 * h * d, seed=4, dtype=dtype)
    x = rows[..., h * d : 2 * h * d].view(b, s, h, d).transpose(1, 2)
    xd = rows.to(dev)[..., h * d : 2 * h * d].view(b, s, h, d).transpose(1, 2)
    freq = _freq(16)
    for pos in (torch.arange(s) + 90000, torch.randint(-500, 10**6, (b, s)), torch.arange(s).unsqueeze(0)):
        y = ops.rotary(xd, pos.to(dev), freq.to(dev), interleaved=interleaved, scale=1.25)
        at = pos if pos.dim() == 1 else pos.unsqueeze(1)
        _check_rotated(y, x, at, freq, interleaved, scale=1.25)
    # Misaligned rows, a stride between dims, one head broadcast to many.
    off = torch.empty(x.numel() + 1, dtype=dtype, device=dev)[1:].view(x.shape).copy_(x)
    assert torch.equal(ops.rotary(off, pos.to(dev), freq.to(dev), interleaved=interleaved), ops.rotary(xd, pos.to(dev), freq.to(dev), interleaved=interleaved))
    wide = torch.stack((xd, xd), -1).flatten(-2)[..., ::2]
    assert torch.equal(ops.rotary(wide, pos.to(dev), freq.to(dev)), ops.rotary(xd, pos.to(dev), freq.to(dev)))
    one = xd[:, :1].expand(b, h, s, d)
    assert torch.equal(ops.rotary(one, pos.to(dev), freq.to(dev)), ops.rotary(one.contiguous(), pos.to(dev), freq.to(dev)))


def test_rotary_keeps_the_layout_and_empty_calls(ops, dev):
    freq, pos = _freq(32).to(dev), torch.arange(10, device=dev)
    x = torch.randn(2, 10, 4, 64, device=dev, dtype=BF).transpose(1, 2)
    assert ops.rotary(x, pos, freq).stride() == x.stride()
    for shape, n in (((0, 4, 64), 0), ((2, 4, 0, 64), 0), ((0, 4, 10, 64), 10)):
        y = ops.rotary(torch.empty(shape, device=dev, dtype=BF), torch.arange(n, device=dev), freq)
        assert y.shape == shape


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(ops, dev, interleaved):
    """Against the formula, and against differences (the operator is linear, so a difference
    quotient is exact but for the roundings of two results: half a step of each over the step)."""
    b, h, hk, s, d, rd = 2, 3, 2, 7, 24, 16
    freq, pos = _freq(rd // 2), torch.arange(s) + 1000
    q, k = _randn(b, h, s, d, seed=5, dtype=FP), _randn(b, hk, s, d, seed=6, dtype=FP)
    gq, gk = _randn(b, h, s, d, seed=7, dtype=FP), _randn(b, hk, s, d, seed=8, dtype=FP)
    qd, kd = q.to(dev).requires_grad_(), k.to(dev).requires_grad_()

    def call(x, y):
        return ops.rotary(x, pos.to(dev), freq.to(dev), k=y, interleaved=interleaved, scale=0.75)

    dq, dk = torch.autograd.grad(call(qd, kd), (qd, kd), (gq.to(dev), gk.to(dev)))
    _check_rotated(dq, gq, pos, freq, interleaved, scale=0.75, inverse=True)
    _check_rotated(dk, gk, pos, freq, interleaved, scale=0.75, inverse=True)
    step = 2.0
    for at in ((0, 0, 0, 0), (1, 2, 6, 15), (0, 1, 3, 9), (1, 0, 5, 23)):
        e = torch.zeros_like(q)
        e[at] = step
        with torch.no_grad():
            up, down = call((q + e).to(dev), kd)[0], call((q - e).to(dev), kd)[0]
        rows = (up.double() - down.double()).cpu() / (2 * step)
        want = float((rows * gq.double()).sum())
        # Sixteen rotated values a row, |x| below 8 here: each result off by 2^-21 * 16.
        assert abs(float(dq[at]) - want) <= 16 * 2.0**-17 * float(gq.abs().max())
    # One input alone; a broadcast gradient; nothing to differentiate.
    q1, k1 = q.to(dev).requires_grad_(), k.to(dev).requires_grad_()
    call(q1, k1)[1].sum().backward()
    assert q1.grad is None
    _check_rotated(k1.grad, torch.ones_like(k), pos, freq, interleaved, scale=0.75, inverse=True)
    y = ops.rotary(q1, pos.to(dev), freq.to(dev), interleaved=interleaved)
    y.backward(torch.ones(1, device=dev).expand(y.shape))
    _check_rotated(q1.grad, torch.ones_like(q), pos, freq, interleaved, inverse=True)
    # Twice: the gradient's own gradient is the rotation again.
    g = gq.to(dev).requires_grad_()
    (dq,) = torch.autograd.grad(ops.rotary(q1, pos.to(dev), freq.to(dev), interleaved=interleaved), q1, g, create_graph=True)
    (gg,) = torch.autograd.grad(dq, g, q.to(dev))
    _check_rotated(gg, q, pos, freq, interleaved)


# ---------------------------------------------------------------- append and read


def _append_reference(c, k, v, q, cu, freq, interleaved, scale):
    """Writes into `c` what an append does; the rotated q (float64), zeros behind the end."""
    out = None if q is None else torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(c.lens):
        lo, hi = (b, b + 1) if cu is None else (cu[b], cu[b + 1])
        pos = torch.arange(n - (hi - lo), n)
        keep = pos >= 0
        kk, at = k[lo:hi].double(), pos.unsqueeze(1)
        if freq is not None:
            kk = P.rotate(kk, at, freq, interleaved, scale)
        if out is not None:
            out[lo:hi] = P.rotate(q[lo:hi].double(), at, freq, interleaved, scale) * keep[:, None, None]
        c.write(b, pos[keep], kk[keep], v[lo:hi].double()[keep])
    return out


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize(
    "new,before,heads,heads_q,d,dv,page,rd,interleaved,rows_last",
    [
        ([1], [0], 1, 1, 64, 64, 16, 64, False, False),
        ([1, 1, 1], [5, 63, 64], 2, 16, 128, 128, 64, 128, False, False),
        ([17, 0, 40, 1], [0, 9, 30, 15], 2, 6, 128, 128, 16, 128, False, True),
        ([33, 5], [100, 0], 8, 0, 64, 64, 48, 32, True, False),
        ([8, 70, 3], [0, 0, 250], 3, 3, 96, 32, 32, 96, False, True),
        ([20, 12], [3, 4], 1, 2, 32, 64, 16, 6, False, False),
        ([9], [7], 2, 2, 256, 256, 128, 0, False, False),
        ([1, 1], [200, 7], 4, 28, 128, 96, 256, 64, True, False),
    ],
)
def test_append_and_read(ops, dev, bits, dtype, new, before, heads, heads_q, d, dv, page, rd, interleaved, rows_last):
    lens = [a + b for a, b in zip(new, before)]
    c = P.Cache(lens, heads, d, dv, page, dtype, bits, rows_last=rows_last, empty=True)
    cu, tail = (None, 0) if set(new) == {1} else (P.cu_of(new), 3)
    t = sum(new) + tail
    k, v = _randn(t, heads, d, seed=11, dtype=dtype), _randn(t, heads, dv, seed=12, dtype=dtype)
    q = _randn(t, heads_q, d, seed=13, dtype=dtype) if heads_q and rd else None
    freq = _freq(rd // 2) if rd else None
    held = c.to(dev)
    cu_d = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    got = ops.paged_append(k.to(dev), v.to(dev), **held, cu_seq=cu_d, q=None if q is None else q.to(dev),
                           inv_freq=None if freq is None else freq.to(dev), interleaved=interleaved, rotary_scale=1.5 if rd else 1.0)
    want_q = _append_reference(c, k, v, q, cu, freq, interleaved, 1.5 if rd else 1.0)
    assert (got is None) == (q is None)
    if q is not None:
        tol = want_q.abs() * P.half_step(dtype) + 2.0**-21 * 1.5 * 16
        assert bool(((got.double().cpu() - want_q).abs() <= tol).all())
        assert bool((got[sum(new):] == 0).all())
    for name, parts in (("k", c.kt), ("v", c.vt)):
        x, y = held[name + "_cache"].cpu(), parts[0]
        if bits == 4:
            # Codes and scales bit for bit, rows that no token owns as they were.
            assert torch.equal(x, y) and torch.equal(held[name + "_scale"].cpu(), parts[1])
        elif name == "v" or not rd:
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))
        else:
            assert torch.equal(x.isnan(), y.isnan())
            near = (x.double() - y.double()).abs() <= 2 * y.double().abs() * P.half_step(dtype) + 2.0**-21 * 1.5 * 16
            assert bool((near | y.isnan()).all())
    # Read back: exactly what the cache holds, zeros past the lengths.
    if not any(before):
        most = max(lens) + 5
        scales = {n: held[n] for n in held if n.endswith("scale")}
        kd, vd = ops.paged_read(held["k_cache"], held["v_cache"], held["block_table"], held["key_lengths"], most, dtype=dtype, **scales)
        if bits == 16:
            c.kt[0] = held["k_cache"].cpu()
        for b in range(len(lens)):
            for out, x in zip((kd, vd), c.held(b)):
                assert torch.equal(out[b, :, : lens[b]].double().cpu(), x.transpose(0, 1))
                assert bool((out[b, :, lens[b] :] == 0).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_append_leaves_out_what_the_cache_cannot_hold(ops, dev, bits):
    """Pages that do not exist, keys before the first and past what the table names, tokens past
    the offsets' end: every other row keeps its bytes, and q rows without a place are zero."""
    c = P.Cache([40, 40, 3, 500], 2, 64, 64, 16, BF, bits, empty=True, spare=4)
    c.table[0, 1] = -1
    c.table[1, 2] = c.pages
    new = [40, 40, 5, 30]
    cu = P.cu_of(new)
    width = 4
    held = c.to(dev)
    held["block_table"] = held["block_table"][:, :width].contiguous()
    t = sum(new) + 2
    k, v, q = (_randn(t, 2, 64, seed=s, dtype=BF) for s in (1, 2, 3))
    freq = _freq(32)
    got = ops.paged_append(k.to(dev), v.to(dev), **held, cu_seq=torch.tensor(cu, dtype=torch.int32, device=dev),
                           q=q.to(dev), inv_freq=freq.to(dev))
    for b, n in enumerate(c.lens):
        pos = torch.arange(n - new[b], n)
        held_by = [(p >= 0 and p < width * 16) for p in pos.tolist()]
        ok = [h and 0 <= int(c.table[b, p // 16]) < c.pages for h, p in zip(held_by, pos.tolist())]
        rows = torch.arange(cu[b], cu[b + 1])
        assert bool((got[rows[~torch.tensor(held_by)].to(dev)] == 0).all())
        sel = torch.tensor(ok)
        if bool(sel.any()):
            c.write(b, pos[sel], P.rotate(k[rows[sel]].double(), pos[sel].unsqueeze(1), freq), v[rows[sel]].double())
    for name, parts in (("k", c.kt), ("v", c.vt)):
        x, y = held[name + "_cache"].cpu(), parts[0]
        if bits == 4:
            assert torch.equal(x, y) and torch.equal(held[name + "_scale"].cpu(), parts[1])
        else:
            assert torch.equal(x.isnan(), y.isnan())
    # A reader takes page 0 for a page that does not exist, and stays in bounds.
    scales = {n: held[n] for n in held if n.endswith("scale")}
    kd, _ = ops.paged_read(held["k_cache"], held["v_cache"], held["block_table"], held["key_lengths"], 600, dtype=BF, **scales)
    assert bool((kd[3, :, 64:] == 0).all())
    out = ops.sdpa_paged(q.to(dev), **held, cu_seq_q=torch.tensor(cu, dtype=torch.int32, device=dev), max_q=40, max_k=600)
    assert out.shape == q.shape and bool((out[sum(new):] == 0).all())


@pytest.mark.parametrize("dtype,interleaved", [(BF, False), (HF, True), (FP, True)])
def test_large_inputs_as_their_parts(ops, dev, dtype, interleaved):
    """64 MB of inputs and more are read past the caches: bit for bit what their parts give."""
    tokens, heads, d, rd = 5000, 56 if dtype is FP else 64, 128, 96
    x = torch.randn(tokens, heads, d, device=dev).to(dtype)
    freq, pos = _freq(rd // 2).to(dev), torch.arange(tokens, device=dev) * 3
    assert x.numel() * x.element_size() >= 2**26
    whole = ops.rotary(x, pos, freq, interleaved=interleaved)
    part = torch.cat([ops.rotary(a, b, freq, interleaved=interleaved) for a, b in zip(x.split(1250), pos.split(1250))])
    assert torch.equal(whole, part)
    _check_rotated(whole[:40], x[:40].cpu(), pos[:40].cpu().unsqueeze(1), freq.cpu(), interleaved)
    if dtype is FP:
        return
    k, v, q = x[:, :16], x[:, 16:32], x[:, 32:]
    cache = [ops.paged_cache(tokens // 50, 16, 64, d, dtype=dtype, device=dev) for _ in range(2)]
    table = torch.arange(tokens // 50, dtype=torch.int32, device=dev).unsqueeze(0)

    def call(held, lo, hi):
        cu = torch.tensor([0, hi - lo], dtype=torch.int32, device=dev)
        return ops.paged_append(k[lo:hi], v[lo:hi], **held, block_table=table, key_lengths=cu[1:], cu_seq=cu, q=q[lo:hi],
                                inv_freq=freq, interleaved=interleaved)

    one = call(cache[0], 0, tokens)
    # (The second part's tokens are keys 2500 .. of the sequence.)
    first = call(cache[1], 0, 2500)
    cu = torch.tensor([0, 2500], dtype=torch.int32, device=dev)
    second = ops.paged_append(k[2500:], v[2500:], **cache[1], block_table=table, cu_seq=cu, q=q[2500:], inv_freq=freq,
                              key_lengths=torch.tensor([tokens], dtype=torch.int32, device=dev), interleaved=interleaved)
    assert torch.equal(one, torch.cat((first, second)))
    for n in ("k_cache", "v_cache"):
        assert torch.equal(cache[0][n], cache[1][n])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("interleaved,rd,scale", [(False, 128, 1.0), (True, 128, -0.7), (False, 64, 1.0), (True, 40, 1.0), (False, 24, 1.3)])
def test_append4_codes_of_many_values(ops, dev, dtype, interleaved, rd, scale):
    """Three million rotated values, thousands of them within what 32 bits are off of a border
    between two codes: bit for bit the codes of exact arithmetic."""
    d, page, heads = 128, 64, 8
    new, before = [2000, 1000, 7], [5000, 0, 100]
    if rd < 64:
        new, before = [90, 40, 7], [3000, 0, 100]
    c = P.Cache([a + b for a, b in zip(new, before)], heads, d, d, page, dtype, 4, empty=True)
    held, cu, t = c.to(dev), P.cu_of(new), sum(new)
    k, v = _randn(t, heads, d, seed=31, dtype=dtype), _randn(t, heads, d, seed=32, dtype=dtype)
    k[:40] *= 2.0**-60 if dtype is BF else 2.0**-20
    k[40:60, :, ::7] = 0
    freq = _freq(rd // 2)
    ops.paged_append(k.to(dev), v.to(dev), **held, cu_seq=torch.tensor(cu, dtype=torch.int32, device=dev),
                     inv_freq=freq.to(dev), interleaved=interleaved, rotary_scale=scale)
    _append_reference(c, k, v, None, cu, freq, interleaved, scale)
    for name, parts in (("k", c.kt), ("v", c.vt)):
        assert torch.equal(held[name + "_scale"].cpu(), parts[1])
        assert torch.equal(held[name + "_cache"].cpu(), parts[0])


def test_append4_next_to_borders(ops, dev):
    """Rotated values within 2^-24 of a border between two codes: codes of exact arithmetic."""
    d = 32
    # One pair a row turned by an angle so small that its first dim moves off a border by a few
    # 10^-8, either way; 6 sets the row's scale to 1.
    n = 512
    x = torch.zeros(n, 1, d, dtype=torch.float64)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    at = torch.arange(n)
    x[:, 0, 0] = borders[at % 7] * (1 - 2 * (at // 7 % 2))
    x[:, 0, d // 2] = 1 - 2 * (at // 14 % 2)
    x[:, 0, 1] = 6.0
    x = x.to(BF)
    freq = torch.zeros(d // 2)
    freq[0] = 1e-9
    held = ops.paged_cache(n // 16, 1, 16, d, dtype=BF, bits=4, device=dev)
    table = torch.arange(n // 16, dtype=torch.int32, device=dev).unsqueeze(0)
    ops.paged_append(x.to(dev), x.to(dev), held["k_cache"], held["v_cache"], table,
                     torch.tensor([n], dtype=torch.int32, device=dev), cu_seq=torch.tensor([0, n], dtype=torch.int32, device=dev),
                     inv_freq=freq.to(dev), k_scale=held["k_scale"], v_scale=held["v_scale"])
    codes, scale = P.quantise(P.rotate(x.double(), at.unsqueeze(1), freq))
    assert torch.equal(held["k_cache"].transpose(1, 2).reshape(n, 1, d // 2).cpu(), codes)
    assert torch.equal(held["k_scale"].transpose(1, 2).reshape(n, 1, 1).cpu(), scale)


def test_append4_of_special_values(ops, dev):
    """Zeros, values on a border between two codes, the smallest and largest, infinities and NaN."""
    d = 32
    rows = [torch.zeros(d), torch.full((d,), -0.0)]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75])
    row = torch.cat((borders, -borders, torch.zeros(d - 20)))
    rows += [row, row * 2.0**-100, row * 2.0**100, torch.linspace(-8, 8, d)]
    tiny = torch.full((d,), 2.0**-133)
    rows += [tiny, torch.full((d,), 3.3e38), torch.cat((torch.tensor([math.inf]), torch.ones(d - 1))),
             torch.cat((torch.tensor([math.nan]), torch.ones(d - 1))), torch.cat((torch.tensor([-math.inf, 0.0]), torch.ones(d - 2)))]
    x = torch.stack(rows).to(BF).unsqueeze(1)
    n = x.size(0)
    held = ops.paged_cache(1, 1, 16, d, dtype=BF, bits=4, device=dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    ops.paged_append(x.to(dev), x.to(dev), held["k_cache"], held["v_cache"], table, lens, k_scale=held["k_scale"],
                     v_scale=held["v_scale"], cu_seq=torch.tensor([0, n], dtype=torch.int32, device=dev))
    kd, vd = ops.paged_read(held["k_cache"], held["v_cache"], table, lens, n, k_scale=held["k_scale"], v_scale=held["v_scale"])
    codes, scale = P.quantise(x.double())
    fine = torch.isfinite(x).all(-1)
    for name, out in (("k", kd), ("v", vd)):
        assert torch.equal(held[name + "_scale"][0, 0, :n].cpu(), scale[:, 0])
        assert torch.equal(held[name + "_cache"][0, 0, :n].cpu()[fine[:, 0]], codes[:, 0][fine[:, 0]])
        assert bool(out[0, 0].cpu()[~fine[:, 0]].isnan().all())
        want = P.values(codes, scale)[:, 0].to(BF)
        assert torch.equal(out[0, 0].cpu()[fine[:, 0]], want[fine[:, 0]])


# ---------------------------------------------------------------- attention


def _check_attention(out, lse, c, q, cu, causal, scale, four, dtype):
    tokens = 0
    for b, n in enumerate(c.lens):
        lo, hi = (b, b + 1) if cu is None else (cu[b], cu[b + 1])
        tokens = hi
        if hi == lo:
            continue
        k, v = c.held(b)
        ref, size, mag, want_lse = P.attention(q[lo:hi].double(), k, v, causal, scale)
        delta = mag * (2.0**-12 if four else c.d * 2.0**-24)
        step = P.half_step(dtype)
        tol = size * (2 * step + 2 * delta) + ref.abs() * step + 2.0**-24
        err = (out[lo:hi].double().cpu() - ref).abs()
        assert bool((err <= tol).all()), f"sequence {b}: {float((err / tol).max()):.3g} of its tolerance"
        rms = lambda x: float(x.square().mean().sqrt())  # noqa: E731
        if n > 0 and rms(ref) > 0:
            # (Few keys: the weights' rounding is not averaged, so the elementwise bound holds alone.)
            if n >= 16:
                bound = math.sqrt(2) * step * max(1.0, rms(size) / (math.sqrt(n) * rms(ref))) + 2 * float(delta.max()) + 1e-6
                assert rms(err) / rms(ref) <= bound, (b, rms(err) / rms(ref), bound)
        if lse is not None:
            got = lse[:, lo:hi].double().cpu()
            assert torch.equal(got.isinf(), want_lse.isinf())
            fin = ~want_lse.isinf()
            off = (got - want_lse).abs()[fin]
            # (The tile kernel sums rounded weights.)
            assert off.numel() == 0 or float(off.max()) <= 2 * step + 2 * float(delta.max()) + 1e-5
    assert bool((out[tokens:] == 0).all())


def _attend(ops, dev, new, before, heads, group, d, dv, page, dtype, bits, causal=True, scale=None, rows_last=False,
            tail=0, seed=0, max_k=None):
    lens = [a + b for a, b in zip(new, before)]
    c = P.Cache(lens, heads, d, dv, page, dtype, bits, rows_last=rows_last, seed=seed)
    cu = None if set(new) == {1} and tail == 0 else P.cu_of(new)
    t = sum(new) + tail
    q = _randn(t, heads * group, d, seed=21 + seed, dtype=dtype)
    held = c.to(dev)
    cu_d = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    scales = (held.pop("k_scale", None), held.pop("v_scale", None))
    out, lse = torch.ops.ktt._sdpa_paged(q.to(dev), *held.values(), cu_d, max(new) if cu else None, max_k or max(lens),
                                         causal, scale, True, *scales)
    _check_attention(out, lse, c, q, cu, causal, 1 / math.sqrt(d) if scale is None else scale, bits == 4 and max(new) * group <= 32, dtype)
    return out


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize(
    "keys,heads,group,d,page",
    [([1], 1, 1, 64, 16), ([16, 17, 31, 32, 33], 2, 8, 128, 16), ([777], 2, 7, 64, 16), ([0, 5, 0], 1, 4, 128, 64),
     ([1000, 3, 129, 128], 3, 5, 96, 48), ([2500, 40], 1, 16, 256, 128), ([90, 300], 2, 32, 64, 32),
     ([600], 1, 17, 128, 256), ([4097], 1, 1, 32, 64), ([130, 61], 2, 3, 192, 16), ([300, 0, 5], 1, 48, 64, 32)],
)
def test_single_tokens(ops, dev, bits, dtype, keys, heads, group, d, page):
    _attend(ops, dev, [1] * len(keys), [n - 1 for n in keys], heads, group, d, d, page, dtype, bits)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize(
    "new,before,heads,group,d,dv,page",
    [
        ([4, 4, 4], [600, 0, 31], 2, 7, 64, 64, 32),  # drafts
        ([2, 0, 3], [20, 5, 0], 2, 2, 128, 128, 16),
        ([5, 9], [1200, 4], 1, 3, 128, 64, 48),
        ([33], [0], 1, 1, 64, 64, 16),  # one row over a decode workgroup
        ([70, 1, 0, 200], [0, 300, 10, 90], 2, 4, 128, 128, 16),
        ([150, 64], [2000, 0], 1, 8, 64, 32, 64),
        ([40, 100], [7, 1000], 2, 2, 96, 96, 32),
        ([65], [130], 1, 4, 256, 256, 48),
        ([50], [60], 2, 2, 32, 192, 16),
        ([300, 20], [5, 0], 8, 2, 128, 128, 128),
    ],
)
def test_several_tokens(ops, dev, bits, dtype, causal, new, before, heads, group, d, dv, page):
    _attend(ops, dev, new, before, heads, group, d, dv, page, dtype, bits, causal=causal, rows_last=len(new) == 2, tail=len(new) - 1)


@pytest.mark.parametrize("bits", [16, 4])
def test_row_tiles_that_fill_the_chip(ops, dev, bits):
    """Enough 128-row workgroups for the wide tile kernel, ragged lengths."""
    new, before = [700, 600, 512, 333, 700, 650, 90, 1], [300, 0, 64, 500, 10, 77, 0, 45]
    _attend(ops, dev, new, before, 8, 2, 64, 64, 16, BF, bits)
    name = _kernel(new, 8, 2, 64)
    assert name in ("tile64", "tile128")


def _kernel(new, heads, group, d):
    from kohakutt_amd import capi

    a = capi.PagedAttnArgs()
    c = a.cache
    c.k = c.v = c.block_table = c.key_lengths = c.cu_seqlens = 0x1000
    c.dtype, c.bits, c.pages, c.page_size, c.heads_kv, c.head_dim, c.head_dim_v = capi.KMI_BF16, 16, 8, 64, heads, d, d
    c.table_width, c.table_stride, c.batch, c.tokens = 64, 64, len(new), sum(new)
    a.q = a.out = 0x1000
    a.heads_q, a.max_q, a.max_k = heads * group, max(new), 4096
    a.scale = 1.0
    return capi.paged_attn_kernel(a)


@pytest.mark.parametrize("new,kernel", [([1] * 4, "decode16"), ([4], "decode32"), ([40], "tile64"), ([300] * 4, "tile128"), ([2000] * 32, "tile128")])
def test_kernels_by_rows(native, new, kernel):
    assert _kernel(new, 2, 8, 128) == kernel


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(ops, dev, bits, scale):
    _attend(ops, dev, [1, 1], [200, 50], 2, 4, 64, 64, 16, BF, bits, scale=scale)
    _attend(ops, dev, [40, 3], [100, 50], 2, 4, 64, 64, 16, BF, bits, scale=scale)


@pytest.mark.parametrize("bits", [16, 4])
def test_calls_repeat_bit_for_bit_and_sequences_are_independent(ops, dev, bits):
    for new, before in (([1, 1, 1], [900, 41, 300]), ([60, 3, 20], [100, 41, 700])):
        one = _attend(ops, dev, new, before, 2, 4, 128, 128, 32, BF, bits)
        two = _attend(ops, dev, new, before, 2, 4, 128, 128, 32, BF, bits)
        assert torch.equal(one, two)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,before", [([5, 3], [-2, -3]), ([40, 6, 3], [-20, -6, -2]), ([200, 90], [-150, -1])])
@pytest.mark.parametrize("causal", [True, False])
def test_more_queries_than_keys(ops, dev, bits, new, before, causal):
    """The first queries of a sequence see no key (all of them where it holds none)."""
    _attend(ops, dev, new, before, 2, 4, 64, 64, 16, BF, bits, causal=causal, tail=2)


@pytest.mark.parametrize("count", [63, 64, 65, 130])
def test_many_sequences(ops, dev, count):
    """Past the sequences that a workgroup sorts by their lengths, single tokens and tiles."""
    new = [1 + (7 * b) % 41 for b in range(count)]
    before = [(13 * b) % 90 for b in range(count)]
    _attend(ops, dev, new, before, 2, 4, 64, 64, 16, BF, 16)
    _attend(ops, dev, [1] * count, before, 2, 4, 64, 64, 16, BF, 16)
    _attend(ops, dev, [min(n, 3) for n in new], before, 2, 4, 64, 64, 16, BF, 4)


@pytest.mark.parametrize("bits", [16, 4])
def test_workspaces_full_of_nan(ops, dev, bits):
    """What a workspace held before is never read: partial rows of empty splits, the rows past a
    sequence's length in the copy of a 4-bit cache."""
    for new, before, at in (([1, 1], [5000, 3], {}), ([90, 40], [4000, 0], {}), ([200, 3], [10, 50], {"max_k": 9000})):
        c = P.Cache([a + b for a, b in zip(new, before)], 2, 64, 64, 16, BF, bits)
        held = c.to(dev)
        q = _randn(sum(new), 8, 64, seed=2, dtype=BF).to(dev)
        cu = torch.tensor(P.cu_of(new), dtype=torch.int32, device=dev)
        args = {"cu_seq_q": cu, "max_q": max(new), "max_k": max(c.lens), **at}
        torch.cuda.empty_cache()
        spoilt = [torch.full((2**n,), math.nan, device=dev) for n in range(8, 25)]
        torch.cuda.synchronize()
        del spoilt
        out = ops.sdpa_paged(q, **held, **args)
        _check_attention(out, None, c, q.cpu(), P.cu_of(new), True, 0.125, bits == 4 and max(new) * 4 <= 32, BF)


@pytest.mark.parametrize("bits", [16, 4])
def test_sequences_that_share_pages(ops, dev, bits):
    """A common prefix held once: each sequence reads it as its own, bit for bit."""
    c = P.Cache([96, 96, 96], 2, 64, 64, 16, BF, bits)
    held = c.to(dev)
    pages = held["block_table"]
    for rows in (1, 3, 30):
        q = _randn(3 * rows, 8, 64, seed=rows, dtype=BF).to(dev)
        cu = torch.arange(0, 3 * rows + 1, rows, dtype=torch.int32, device=dev)
        args = {"cu_seq_q": cu, "max_q": rows, "max_k": 96}
        shared = pages.clone()
        shared[1:, :5] = pages[0, :5]
        copied = {**held}
        for n in held:
            if n.endswith(("cache", "scale")):
                x = held[n].clone()
                for b in (1, 2):
                    x[pages[b, :5].long()] = held[n][pages[0, :5].long()]
                copied[n] = x
        one = ops.sdpa_paged(q, **{**held, "block_table": shared}, **args)
        two = ops.sdpa_paged(q, **copied, **args)
        assert torch.equal(one, two)


@pytest.mark.parametrize("new,before", [([1, 1, 1], [900, 41, 300]), ([60, 3, 2], [100, 41, 700]), ([130, 8], [4, 900])])
def test_many_rows_behind_the_last_sequence(ops, dev, new, before):
    """More of them than one workgroup zeroes (64 KB of output each), whole calls and split ones."""
    _attend(ops, dev, new, before, 2, 4, 128, 128, 32, BF, 16, tail=700)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows,kernel", [(1, "decode16"), (5, "decode32"), (40, "tile64")])
@pytest.mark.parametrize("keys,at", [(48, 3), (700, 650), (9000, 100), (33, 32)])
def test_a_nan_key_is_not_lost(ops, dev, bits, rows, kernel, keys, at):
    """One key that is NaN: every query that sees it is NaN, in calls split over their keys too
    (where the part that holds it has no maximum or sum), those before it are as ever."""
    heads, group, d = 2, 4, 64
    c = P.Cache([keys], heads, d, d, 16, BF, bits)
    held = c.to(dev)
    page, row = int(held["block_table"][0, at // 16]), at % 16
    if bits == 16:
        held["k_cache"][page, :, row] = math.nan
    else:
        held["k_scale"][page, :, row] = 255
    q = _randn(rows, heads * group, d, seed=1, dtype=BF).to(dev)
    cu = torch.tensor([0, rows], dtype=torch.int32, device=dev)
    assert _kernel([rows], heads, group, d) == kernel
    for causal in (True, False):
        out = ops.sdpa_paged(q, **held, cu_seq_q=cu, max_q=rows, max_k=keys, is_causal=causal)
        sees = torch.arange(rows) + keys - rows >= at if causal else torch.ones(rows, dtype=torch.bool)
        assert torch.equal(out.isnan().all(-1).all(-1).cpu(), sees)
        assert torch.equal(out.isnan().any(-1).any(-1).cpu(), sees)


@pytest.mark.parametrize("bits", [16, 4])
def test_pages_past_32_bits(ops, dev, bits):
    """Pages a gigabyte apart (offsets past 2^32 bytes): every operator bit for bit as over a dense cache."""
    heads, group, d, page = 2, 4, 64, 32
    new, before = [1, 40, 3], [60, 30, 0]
    lens = [a + b for a, b in zip(new, before)]
    c = P.Cache(lens, heads, d, d, page, BF, bits)
    held = c.to(dev)
    pages = held["k_cache"].size(0)
    assert pages >= 6
    far = dict(held)
    step = 2**29 if bits == 16 else 2**30 - 16
    span = heads * page * held["k_cache"].size(3)
    store = torch.empty(step * (pages - 1) + 2 * span, dtype=held["k_cache"].dtype, device=dev)
    for n, first in (("k_cache", 0), ("v_cache", span)):
        x = held[n]
        far[n] = torch.as_strided(store, x.shape, (step, page * x.size(3), x.size(3), 1), first)
        far[n].copy_(x)
    cu = torch.tensor(P.cu_of(new), dtype=torch.int32, device=dev)
    t = sum(new)
    k, v, q = (_randn(t, n, d, seed=s, dtype=BF).to(dev) for n, s in ((heads, 1), (heads, 2), (heads * group, 3)))
    freq = _freq(d // 2).to(dev)
    qr = [ops.paged_append(k, v, **h, cu_seq=cu, q=q, inv_freq=freq) for h in (held, far)]
    assert torch.equal(qr[0], qr[1])
    for n in held:
        assert torch.equal(held[n].contiguous().view(torch.uint8), far[n].contiguous().view(torch.uint8)), n
    for args in ({"cu_seq_q": cu, "max_q": max(new)}, {"cu_seq_q": cu, "max_q": 1}, {}):
        qq = qr[0] if args else qr[0][: len(new)]
        one, two = (ops.sdpa_paged(qq, **h, **args, max_k=max(lens)) for h in (held, far))
        if args.get("max_q") == 1:
            one, two = one[cu[:-1].long()], two[cu[:-1].long()]
        assert torch.equal(one, two)
    scales = {n: held[n] for n in held if n.endswith("scale")}
    one, two = (ops.paged_read(h["k_cache"], h["v_cache"], h["block_table"], h["key_lengths"], max(lens), **scales)
                for h in (held, far))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.parametrize("bits", [16, 4])
def test_default_bounds_and_a_wide_table(ops, dev, bits):
    """max_k from the table's width (far more than any length), strided q and table."""
    c = P.Cache([70, 300], 2, 64, 64, 16, BF, bits)
    held = c.to(dev)
    wide = torch.full((2, 4000), -5, dtype=torch.int32, device=dev)
    wide[:, : held["block_table"].size(1)] = held["block_table"]
    held["block_table"] = wide[:, :3000]
    q = _randn(2, 8, 64, seed=1, dtype=BF)
    big = torch.zeros(2, 24, 64, dtype=BF, device=dev)
    big[:, 8:16] = q.to(dev)
    out = ops.sdpa_paged(big[:, 8:16], **held)
    _check_attention(out, None, c, q, None, True, 0.125, bits == 4, BF)
    # Keys past max_k are not read: the first 64 of each sequence.
    cut = ops.sdpa_paged(q.to(dev), **held, max_k=64, is_causal=False)
    c.lens = [64, 64]
    _check_attention(cut, None, c, q, None, False, 0.125, bits == 4, BF)


@pytest.mark.parametrize("bits", [16, 4])
def test_no_keys_at_all(ops, dev, bits):
    """max_k of zero, a table of no pages, lengths of zero: zeros, and log-sum-exps of minus infinity."""
    c = P.Cache([40, 7], 2, 64, 64, 16, BF, bits)
    held = c.to(dev)
    q = torch.randn(80, 8, 64, dtype=BF, device=dev)
    cu = torch.tensor([0, 40, 80], dtype=torch.int32, device=dev)
    none = {**held, "block_table": held["block_table"][:, :0]}
    zero = {**held, "key_lengths": torch.zeros_like(held["key_lengths"])}
    for kw in ({**held, "max_k": 0}, none, zero):
        for qq, at in ((q[:2], {}), (q, {"cu_seq_q": cu, "max_q": 40})):
            out = ops.sdpa_paged(qq, **kw, **at)
            assert bool((out == 0).all())
    k, v = (torch.zeros(2, 2, 64, dtype=BF, device=dev) for _ in "kv")
    before = {n: t.clone() for n, t in held.items()}
    ops.paged_append(k, v, **none)
    ops.paged_append(k, v, **zero)
    assert all(torch.equal(before[n].view(torch.uint8), held[n].view(torch.uint8)) for n in held)
    kd, vd = ops.paged_read(none["k_cache"], none["v_cache"], none["block_table"], none["key_lengths"], 20,
                            k_scale=held.get("k_scale"), v_scale=held.get("v_scale"))
    assert bool((kd == 0).all()) and bool((vd == 0).all())


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("bits", [16, 4])
def test_serving_run_and_graph(ops, dev, bits):
    """Prompts, then tokens one by one through append and attention, eager and as one captured
    graph replayed with growing lengths; every step against float64 over what the cache holds."""
    heads, group, d, page, steps = 2, 4, 64, 16, 4
    new = [37, 5, 20]
    c = P.Cache(new, heads, d, d, page, BF, bits, empty=True, room=2 * steps + 2)
    freq = _freq(d // 2)
    freq_d = freq.to(dev)
    held = c.to(dev)
    scales = {n: held[n] for n in held if n.endswith("scale")}
    base = (held["k_cache"], held["v_cache"], held["block_table"], held["key_lengths"])

    def step(k, v, q, cu, max_q, max_k):
        qr = ops.paged_append(k, v, *base, cu_seq=cu, q=q, inv_freq=freq_d, **scales)
        return qr, ops.sdpa_paged(qr, *base, cu_seq_q=cu, max_q=max_q, max_k=max_k, **scales)

    def check(k, v, qr, out, cu):
        _append_reference(c, k, v, None, cu, freq, False, 1.0)
        if bits == 16:
            near = (held["k_cache"].double().cpu() - c.kt[0].double()).abs() <= 2.0**-7 * c.kt[0].double().abs() + 2.0**-17
            assert bool((near | c.kt[0].isnan()).all())
            c.kt[0] = held["k_cache"].cpu()
        else:
            assert torch.equal(held["k_cache"].cpu(), c.kt[0])
        rows = max(new) if cu else 1
        _check_attention(out, None, c, qr.cpu(), cu, True, d**-0.5, bits == 4 and rows * group <= 32, BF)

    cu = P.cu_of(new)
    t = sum(new)
    k, v, q = (_randn(t, n, d, seed=s, dtype=BF) for n, s in ((heads, 1), (heads, 2), (heads * group, 3)))
    qr, out = step(k.to(dev), v.to(dev), q.to(dev), torch.tensor(cu, dtype=torch.int32, device=dev), max(new), max(new))
    check(k, v, qr, out, cu)

    kd, vd, qd = (torch.zeros(3, n, d, dtype=BF, device=dev) for n in (heads, heads, heads * group))
    most = max(new) + 2 * steps + 2
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    for i in range(2 * steps):
        k, v, q = (_randn(3, n, d, seed=100 + 3 * i + j, dtype=BF) for j, n in enumerate((heads, heads, heads * group)))
        kd.copy_(k), vd.copy_(v), qd.copy_(q)
        held["key_lengths"].add_(1)
        c.lens = [n + 1 for n in c.lens]
        if i < steps:
            qr, out = step(kd, vd, qd, None, None, most)
        else:
            if i == steps:
                torch.cuda.synchronize()
                with torch.cuda.graph(graph, stream=stream):
                    gqr, gout = step(kd, vd, qd, None, None, most)
            graph.replay()
            qr, out = gqr, gout
        torch.cuda.synchronize()
        check(k, v, qr, out, None)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,rows", [(256, 1), (256, 5), (192, 1), (96, 3), (256, 40), (128, 150)])
def test_captured_attention(ops, dev, bits, d, rows):
    """Every kind of kernel in a graph (those with more than 64 KB of LDS among them), replayed while
    lengths and queries change."""
    lens = [700, 300, rows]
    c = P.Cache(lens, 2, d, d, 32, BF, bits)
    held = c.to(dev)
    q = torch.zeros(3 * rows, 8, d, dtype=BF, device=dev)
    cu = torch.arange(0, 3 * rows + 1, rows, dtype=torch.int32, device=dev)
    args = {**held, "cu_seq_q": cu, "max_q": rows, "max_k": 700}
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.sdpa_paged(q, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sdpa_paged(q, **args)
    for seed in range(3):
        q.copy_(_randn(3 * rows, 8, d, seed=seed, dtype=BF))
        held["key_lengths"].copy_(torch.tensor([700 - 100 * seed, 300 - seed, rows], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.sdpa_paged(q, **args))
        c.lens = held["key_lengths"].tolist()
        _check_attention(out, None, c, q.cpu(), list(range(0, 3 * rows + 1, rows)), True, d**-0.5, bits == 4 and rows * 4 <= 32, BF)


def test_two_streams_at_once(ops, dev):
    """Calls in flight on two streams keep their own workspaces."""
    c = [P.Cache([3000, 2000], 1, 64, 64, 16, BF, 16, seed=s) for s in (0, 1)]
    q = [_randn(2, 8, 64, seed=s, dtype=BF) for s in (5, 6)]
    held, qd = [x.to(dev) for x in c], [x.to(dev) for x in q]
    want = [ops.sdpa_paged(qd[i], **held[i], max_k=3000) for i in (0, 1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.sdpa_paged(qd[i], **held[i], max_k=3000))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
        _check_attention(want[i], None, c[i], q[i], None, True, 0.125, False, BF)


def test_training_step_through_rotary_and_attention(ops, dev):
    """rotary before varlen attention, gradients to the projections' rows (float64 autograd)."""
    import torch.nn.functional as F

    s, h, hk, d = 40, 4, 2, 64
    freq, pos = _freq(d // 2), torch.arange(s)
    q, k, v = (_randn(s, n, d, seed=i, dtype=BF) for i, n in ((1, h), (2, hk), (3, hk)))
    g = _randn(s, h, d, seed=4, dtype=BF)
    leaves = [x.to(dev).requires_grad_() for x in (q, k, v)]
    qr, kr = ops.rotary(leaves[0], pos.to(dev), freq.to(dev), k=leaves[1])
    out = ops.sdpa_varlen(qr, kr, leaves[2], [0, s], is_causal=True)
    grads = torch.autograd.grad(out, leaves, g.to(dev))
    ref = [x.double().requires_grad_() for x in (q, k, v)]
    # (Autograd through plain torch: the rotation without in-place writes.)
    ang = pos.double().unsqueeze(-1) * freq.double()
    c, sn = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    rot = lambda x: torch.cat((x[..., :32] * c - x[..., 32:] * sn, x[..., 32:] * c + x[..., :32] * sn), -1)  # noqa: E731
    qq, kk = rot(ref[0]).transpose(0, 1), rot(ref[1]).transpose(0, 1).repeat_interleave(2, 0)
    vv = ref[2].transpose(0, 1).repeat_interleave(2, 0)
    o = F.scaled_dot_product_attention(qq.unsqueeze(0), kk.unsqueeze(0), vv.unsqueeze(0), is_causal=True)[0].transpose(0, 1)
    want = torch.autograd.grad(o, ref, g.double())
    for a, b in zip(grads, want):
        rel = float((a.double().cpu() - b).norm() / b.norm())
        # Roundings on the way, one half step (2^-8) each at most: q and k rotated, P, dP's row
        # sums, dS, the gradient, its rotation: independent, so their root sum of squares.
        assert rel <= math.sqrt(8) * 2.0**-8, rel


# ---------------------------------------------------------------- refusals


def _rotary_call(dev, **kw):
    args = {
        "x": torch.zeros(2, 4, 5, 64, dtype=BF, device=dev),
        "positions": torch.arange(5, device=dev),
        "inv_freq": torch.ones(32, device=dev),
        "k": torch.zeros(2, 1, 5, 64, dtype=BF, device=dev),
    }
    return {**args, **kw}


@pytest.mark.parametrize(
    "make,msg",
    [
        (lambda dev: {"x": torch.zeros(2, 4, 5, 64, dtype=torch.float64, device=dev)}, "bf16, fp16 or fp32"),
        (lambda dev: {"x": torch.zeros(5, 64, dtype=BF, device=dev)}, "must be"),
        (lambda dev: {"k": torch.zeros(2, 1, 6, 64, dtype=BF, device=dev)}, "k must match"),
        (lambda dev: {"k": torch.zeros(2, 1, 5, 64, dtype=HF, device=dev)}, "k must match"),
        (lambda dev: {"k": torch.zeros(2, 1, 5, 32, dtype=BF, device=dev)}, "k must match"),
        (lambda dev: {"positions": torch.arange(4, device=dev)}, "positions must be"),
        (lambda dev: {"positions": torch.zeros(3, 5, dtype=torch.int64, device=dev)}, "positions must be"),
        (lambda dev: {"positions": torch.zeros(5, device=dev)}, "int32 or int64"),
        (lambda dev: {"positions": torch.arange(5)}, "int32 or int64 on the tensors' device"),
        (lambda dev: {"inv_freq": torch.ones(33, device=dev)}, "at most 32"),
        (lambda dev: {"inv_freq": torch.ones(0, device=dev)}, "at most 32"),
        (lambda dev: {"inv_freq": torch.ones(32)}, "on the tensors' device"),
        (lambda dev: {"inv_freq": torch.ones(32, dtype=torch.float64, device=dev)}, "fp32"),
        (lambda dev: {"inv_freq": torch.ones(32, device=dev, requires_grad=True)}, "no gradient"),
        (lambda dev: {"inv_freq": torch.ones(32, device=dev, requires_grad=True),
                      "x": torch.zeros(2, 4, 5, 64, dtype=BF, device=dev, requires_grad=True)}, "no gradient"),
    ],
)
def test_rotary_refuses(ops, dev, make, msg):
    with pytest.raises((ValueError, RuntimeError), match=msg):
        ops.rotary(**_rotary_call(dev, **make(dev)))


def _cache_calls(dev, bits=16):
    """Arguments of an append and of an attention call that are accepted."""
    cache = {n: t for n, t in P.Cache([40, 7], 2, 64, 64, 16, BF, bits).to(dev).items()}
    k = torch.zeros(2, 2, 64, dtype=BF, device=dev)
    return cache, {"k": k, "v": k.clone(), **cache}, {"q": torch.zeros(2, 8, 64, dtype=BF, device=dev), **cache}


_BAD_CACHES = [
    (lambda c: {"v_cache": c["v_cache"][1:]}, "must be \\[pages"),
    (lambda c: {"k_cache": c["k_cache"][0]}, "must be \\[pages"),
    (lambda c: {"k_cache": c["k_cache"][:, :, :8], "v_cache": c["v_cache"][:, :, :8]}, "multiple of 16"),
    (lambda c: {"k_cache": c["k_cache"].float()}, "bf16 or fp16"),
    (lambda c: {"k_cache": c["k_cache"].half(), "v_cache": c["v_cache"].half()}, "not"),
    (lambda c: {"block_table": c["block_table"].long()}, "block_table must be int32"),
    (lambda c: {"block_table": c["block_table"][0]}, "block_table must be int32"),
    (lambda c: {"block_table": c["block_table"].cpu()}, "on one device"),
    (lambda c: {"block_table": c["block_table"].t().contiguous().t()}, "rows must be contiguous"),
    (lambda c: {"key_lengths": c["key_lengths"].long()}, "key_lengths must be int32"),
    (lambda c: {"key_lengths": c["key_lengths"][:1]}, "key_lengths must be int32"),
    (lambda c: {"k_cache": c["k_cache"].transpose(2, 3).contiguous().transpose(2, 3)}, "contiguous"),
    (lambda c: {"k_scale": c["k_cache"].to(torch.uint8)}, "four uint8 tensors"),
]


@pytest.mark.parametrize("make,msg", _BAD_CACHES)
def test_bad_caches_are_refused(ops, dev, make, msg):
    cache, append, attend = _cache_calls(dev)
    bad = make(cache)
    with pytest.raises((ValueError, RuntimeError), match=msg):
        ops.paged_append(**{**append, **bad})
    with pytest.raises((ValueError, RuntimeError), match=msg):
        ops.sdpa_paged(**{**attend, **bad})


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize(
    "make,msg",
    [
        (lambda a, dev: {"k": a["k"][:1]}, "must be \\[T, heads, D\\]"),
        (lambda a, dev: {"k": a["k"][:, :, :32], "v": a["v"]}, "the cache holds"),
        (lambda a, dev: {"k": a["k"][:, :1], "v": a["v"][:, :1]}, "the cache holds"),
        (lambda a, dev: {"k": a["k"].half()}, "one type"),
        (lambda a, dev: {"k": a["k"].repeat(2, 1, 1), "v": a["v"].repeat(2, 1, 1)}, "one token per sequence"),
        (lambda a, dev: {"cu_seq": torch.tensor([0, 2], dtype=torch.int32, device=dev)}, "offsets must be"),
        (lambda a, dev: {"cu_seq": torch.tensor([0, 1, 2], device=dev)}, "offsets must be"),
        (lambda a, dev: {"cu_seq": torch.tensor([0, 1, 2], dtype=torch.int32)}, "offsets must be"),
        (lambda a, dev: {"q": torch.zeros(2, 8, 64, dtype=BF, device=dev)}, "needs inv_freq"),
        (lambda a, dev: {"q": torch.zeros(3, 8, 64, dtype=BF, device=dev), "inv_freq": torch.ones(32, device=dev)}, "q must be"),
        (lambda a, dev: {"inv_freq": torch.ones(40, device=dev)}, "at most 32"),
        (lambda a, dev: {"inv_freq": torch.ones(32, device=dev, requires_grad=True)}, "no_grad"),
        (lambda a, dev: {"k": a["k"].clone().requires_grad_()}, "no_grad"),
    ],
)
def test_append_refuses(ops, dev, bits, make, msg):
    _, append, _ = _cache_calls(dev, bits)
    with pytest.raises((ValueError, RuntimeError), match=msg):
        ops.paged_append(**{**append, **make(append, dev)})


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize(
    "make,msg",
    [
        (lambda a, dev: {"q": a["q"].float()}, "bf16 or fp16"),
        (lambda a, dev: {"q": a["q"][0]}, "q must be"),
        (lambda a, dev: {"q": a["q"][:, :7]}, "must divide"),
        (lambda a, dev: {"q": a["q"][:, :, :32].contiguous()}, "the cache holds"),
        (lambda a, dev: {"q": a["q"].repeat(2, 1, 1)}, "one token per sequence"),
        (lambda a, dev: {"max_q": -1}, "not be negative"),
        (lambda a, dev: {"max_k": -1}, "not be negative"),
        (lambda a, dev: {"q": a["q"].clone().requires_grad_()}, "no_grad"),
        (lambda a, dev: {"cu_seq_q": torch.tensor([0, 2], dtype=torch.int32, device=dev)}, "offsets must be"),
    ],
)
def test_attention_refuses(ops, dev, bits, make, msg):
    _, _, attend = _cache_calls(dev, bits)
    with pytest.raises((ValueError, RuntimeError), match=msg):
        ops.sdpa_paged(**{**attend, **make(attend, dev)})


def test_four_bit_gaps_are_refused(ops, dev):
    cache, append, attend = _cache_calls(dev, 4)
    for bad, msg in (
        ({"v_scale": None}, "four uint8 tensors"),
        ({"k_scale": cache["k_scale"].to(torch.int8)}, "four uint8 tensors"),
        ({"k_scale": cache["k_scale"][..., :1]}, "scales must be"),
        ({"k_scale": cache["k_scale"].cpu()}, "scales must be"),
        ({"k_cache": cache["k_cache"][..., :24], "v_cache": cache["v_cache"][..., :24]}, "scales must be"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=msg):
            ops.paged_append(**{**append, **bad})
        with pytest.raises((ValueError, RuntimeError), match=msg):
            ops.sdpa_paged(**{**attend, **bad})
    with pytest.raises((ValueError, RuntimeError), match="max_k"):
        ops.paged_read(**cache, max_k=-1)
    with pytest.raises((ValueError, RuntimeError), match="bf16 or fp16"):
        ops.paged_read(**cache, max_k=4, dtype=torch.float32)
