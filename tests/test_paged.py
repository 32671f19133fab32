"""The rotation and the paged cache on the CPU: refusals before any launch (C ABI and torch
ops on meta tensors), struct layouts, frequency scaling, and the plain forms the GPU tests
compare with."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

import kohakutt_amd
import paged_cases as P
from kohakutt_amd import capi

HEADER = Path(__file__).resolve().parent.parent / "include" / "kohakutt_amd.h"


@pytest.mark.parametrize("struct,cls", [("kmi_rotary_args", "RotaryArgs"), ("kmi_paged_cache", "PagedCache"),
                                        ("kmi_paged_append_args", "PagedAppendArgs"),
                                        ("kmi_paged_attn_args", "PagedAttnArgs")])
def test_struct_layout_matches_header_field_order(struct, cls):
    text = HEADER.read_text()
    start = text.index("{", text.index("typedef struct " + struct)) + 1
    body = re.sub(r"/\*.*?\*/", "", text[start : text.index("} " + struct + ";")], flags=re.S)
    names = []
    for decl in body.split(";"):
        for part in decl.split(","):
            idents = re.findall(r"[A-Za-z_]\w*", re.sub(r"\[.*?\]", "", part))
            if idents:
                names.append(idents[-1])
    assert names == [f[0] for f in getattr(capi, cls)._fields_]


# ---------------------------------------------------------------- C ABI


def _set(obj, kw):
    for name, value in kw.items():
        at = obj
        *path, last = name.split("__")
        for p in path:
            at = getattr(at, p)
        if isinstance(value, (list, tuple)):
            getattr(at, last)[:] = value
        else:
            setattr(at, last, value)
    return obj


def _cache(c, bits=16):
    c.k = c.v = c.block_table = c.key_lengths = 0x1000
    c.k_scale = c.v_scale = 0x1000 if bits == 4 else 0
    c.dtype, c.bits, c.pages, c.page_size, c.heads_kv, c.head_dim, c.head_dim_v = capi.KMI_BF16, bits, 4, 16, 2, 64, 64
    c.k_stride[:] = c.v_stride[:] = [2 * 16 * 64, 16 * 64, 64]
    c.table_stride = c.table_width = 8
    c.batch = c.tokens = 3


def _rotary(**kw):
    a = capi.RotaryArgs()
    a.x[0] = a.y[0] = a.positions = a.inv_freq = 0x1000
    a.heads[0], a.dtype, a.position_bits = 4, capi.KMI_BF16, 64
    a.batch, a.seq, a.head_dim, a.rotary_dim, a.scale = 1, 5, 64, 64, 1.0
    return _set(a, kw)


def _append(bits=16, **kw):
    a = capi.PagedAppendArgs()
    _cache(a.cache, bits)
    a.k = a.v = 0x1000
    a.k_stride[:] = a.v_stride[:] = [128, 64]
    return _set(a, kw)


def _attn(bits=16, **kw):
    a = capi.PagedAttnArgs()
    _cache(a.cache, bits)
    a.q = a.out = 0x1000
    a.q_stride[:] = a.o_stride[:] = [256, 64]
    a.heads_q, a.max_q, a.max_k, a.causal, a.scale = 4, 1, 128, 1, 0.125
    return _set(a, kw)


CACHE_REFUSALS = [
    (dict(cache__dtype=capi.KMI_F32), "BF16 or F16"),
    (dict(cache__bits=8), "16 or 4"),
    (dict(cache__head_dim=84), "multiples of 8"),
    (dict(cache__head_dim_v=264), "multiples of 8"),
    (dict(cache__pages=0), "pages must be positive"),
    (dict(cache__page_size=24), "multiple of 16"),
    (dict(cache__page_size=0), "multiple of 16"),
    (dict(cache__heads_kv=0), "heads_kv"),
    (dict(cache__k=0), "null k"),
    (dict(cache__block_table=0), "null k"),
    (dict(cache__v=0x1008), "16-byte aligned"),
    (dict(cache__k_stride=[1024, 64, 4]), "multiples of 8"),
    (dict(cache__v_stride=[-1024, 64, 64]), "negative"),
    (dict(cache__k_stride=[1024, 64, 1 << 25]), "row strides"),
    (dict(cache__batch=-1), "batch"),
    (dict(cache__table_width=1 << 27), "2^30"),
    (dict(cache__tokens=-1), "tokens"),
    (dict(cache__tokens=4), "one token per sequence"),
]


@pytest.mark.parametrize("kw,msg", CACHE_REFUSALS)
def test_c_abi_refuses_bad_caches(kw, msg):
    lib = capi.lib()
    for make, call in ((_append, lambda a: lib.kmi_paged_append(ctypes.byref(a), None)),
                       (_attn, lambda a: lib.kmi_paged_attn(ctypes.byref(a), None, 0, None))):
        assert call(make(**kw)) == capi.KMI_EINVAL
        assert msg in lib.kmi_last_error().decode()


@pytest.mark.parametrize(
    "make,call,kw,msg",
    [
        (_rotary, "kmi_rotary", dict(dtype=9), "dtype"),
        (_rotary, "kmi_rotary", dict(head_dim=257), "head_dim"),
        (_rotary, "kmi_rotary", dict(rotary_dim=66), "rotary_dim"),
        (_rotary, "kmi_rotary", dict(rotary_dim=7), "rotary_dim"),
        (_rotary, "kmi_rotary", dict(rotary_dim=0), "rotary_dim"),
        (_rotary, "kmi_rotary", dict(position_bits=16), "position_bits"),
        (_rotary, "kmi_rotary", dict(inv_freq=0), "null"),
        (_rotary, "kmi_rotary", dict(seq=-1), "sizes"),
        (_rotary, "kmi_rotary", dict(batch=1 << 14, seq=1 << 14), "tokens"),
        (_append, "kmi_paged_append", dict(k=0), "null k"),
        (_append, "kmi_paged_append", dict(k=0x1004), "16-byte aligned"),
        (_append, "kmi_paged_append", dict(v_stride=[128, 60]), "multiples of 8"),
        (_append, "kmi_paged_append", dict(rotary_dim=64), "inv_freq"),
        (_append, "kmi_paged_append", dict(rotary_dim=66, inv_freq=0x1000), "rotary_dim"),
        (_append, "kmi_paged_append", dict(q=0x1000, q_out=0x1000, heads_q=2), "needs rotary_dim"),
        (_append, "kmi_paged_append", dict(q=0x1000, heads_q=2, rotary_dim=64, inv_freq=0x1000), "q_out"),
        (_attn, "kmi_paged_attn", dict(q=0), "null q"),
        (_attn, "kmi_paged_attn", dict(heads_q=5), "divide"),
        (_attn, "kmi_paged_attn", dict(q_stride=[256, 60]), "q strides"),
        (_attn, "kmi_paged_attn", dict(o_stride=[256, 62]), "out strides"),
        (_attn, "kmi_paged_attn", dict(max_q=4), "max_q"),
        (_attn, "kmi_paged_attn", dict(max_k=-1), "max_k"),
        (_attn, "kmi_paged_attn", dict(out=0x1004), "8-byte aligned"),
    ],
)
def test_c_abi_refuses_bad_calls(make, call, kw, msg):
    lib = capi.lib()
    a = make(**kw)
    extra = (None, 0, None) if call == "kmi_paged_attn" else (None,)
    assert getattr(lib, call)(ctypes.byref(a), *extra) == capi.KMI_EINVAL
    assert msg in lib.kmi_last_error().decode()


def test_c_abi_refuses_null_and_four_bit_gaps():
    lib = capi.lib()
    assert lib.kmi_rotary(None, None) == capi.KMI_EINVAL
    assert lib.kmi_paged_append(None, None) == capi.KMI_EINVAL
    assert lib.kmi_paged_read(None, None, None, 0, None) == capi.KMI_EINVAL
    assert lib.kmi_paged_attn(None, None, 0, None) == capi.KMI_EINVAL
    assert lib.kmi_paged_attn_workspace_bytes(None, None) == capi.KMI_EINVAL
    for kw in (dict(cache__head_dim=40), dict(cache__k_scale=0), dict(cache__k_stride=[1024, 64, 24]),
               dict(cache__k_scale_stride=[-1, 0, 0])):
        a = _attn(bits=4, **kw)
        assert lib.kmi_paged_attn(ctypes.byref(a), None, 0, None) == capi.KMI_EINVAL
    a = _attn()
    for args in ((None, 0x1000, 64), (0x1000, 0x1008, 64), (0x1000, 0x1000, -1), (0x1000, 0x1000, 1 << 40)):
        assert lib.kmi_paged_read(ctypes.byref(a.cache), *args, None) == capi.KMI_EINVAL


def test_workspace_is_asked_for_and_its_absence_refused():
    # Few sequences over many keys are split; a 4-bit cache under row tiles is widened.
    a = _attn(cache__table_width=1 << 12, max_k=1 << 16)
    n = capi.paged_attn_workspace_bytes(a)
    assert n > 0
    for ws, size in ((None, 0), (0x1000, n - 1), (0x1008, n)):
        assert capi.lib().kmi_paged_attn(ctypes.byref(a), ws, size, None) == capi.KMI_EWORKSPACE
    a = _attn(bits=4, cache__cu_seqlens=0x1000, cache__tokens=300, max_q=100)
    assert capi.paged_attn_workspace_bytes(a) >= 3 * 2 * 128 * 128 * 2
    # Nothing to do: no launch, no workspace.
    assert capi.lib().kmi_paged_attn(ctypes.byref(_attn(cache__batch=0, cache__tokens=0, max_q=0)), None, 0, None) == capi.KMI_OK
    assert capi.lib().kmi_paged_append(ctypes.byref(_append(cache__batch=0, cache__tokens=0)), None) == capi.KMI_OK
    assert capi.lib().kmi_rotary(ctypes.byref(_rotary(seq=0)), None) == capi.KMI_OK


# ---------------------------------------------------------------- torch


def test_cpu_tensors_have_no_kernel():
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="CPU"):
        kohakutt_amd.rotary(x, torch.arange(3), torch.ones(32))
    held = kohakutt_amd.paged_cache(2, 2, 16, 64, device="cpu")
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="CPU"):
        kohakutt_amd.sdpa_paged(x, **held, block_table=table, key_lengths=lens)


def test_paged_cache_tensors_and_refusals():
    c = kohakutt_amd.paged_cache(3, 2, 32, 64, head_dim_v=96, dtype=torch.float16, device="cpu")
    assert c["k_cache"].shape == (3, 2, 32, 64) and c["v_cache"].shape == (3, 2, 32, 96) and "k_scale" not in c
    c = kohakutt_amd.paged_cache(3, 2, 32, 64, bits=4, device="cpu")
    assert c["k_cache"].shape == (3, 2, 32, 32) and c["v_scale"].shape == (3, 2, 32, 2)
    assert all(t.dtype == torch.uint8 for t in c.values())
    for kw, msg in ((dict(bits=8), "bits"), (dict(page_size=20), "page size"), (dict(head_dim=12), "head dims"),
                    (dict(head_dim=40, bits=4), "head dims"), (dict(head_dim=512), "head dims")):
        with pytest.raises(ValueError, match=msg):
            kohakutt_amd.paged_cache(**{**dict(pages=1, heads=1, page_size=16, head_dim=64, device="cpu"), **kw})


# ---------------------------------------------------------------- frequencies


def test_rotary_frequencies():
    plain, scale = kohakutt_amd.rotary_frequencies(64, base=1e4)
    want = 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert plain.dtype == torch.float32 and scale == 1.0
    assert torch.equal(plain, want.float())
    linear, _ = kohakutt_amd.rotary_frequencies(64, 1e4, {"type": "linear", "factor": 4})
    assert torch.equal(linear, (want / 4).float())
    ntk, _ = kohakutt_amd.rotary_frequencies(64, 1e4, {"type": "ntk", "factor": 4})
    # The fastest pair as it was, the slowest stretched by the factor.
    assert float(ntk[0]) == 1.0 and float(ntk[-1]) == pytest.approx(float(want[-1]) / 4, rel=1e-6)
    n = 4096
    turns = want * n / (2 * math.pi)
    bands, _ = kohakutt_amd.rotary_frequencies(64, 1e4, {"type": "bands", "factor": 8, "original": n})
    for f, w, t in zip(bands.double(), want, turns):
        keep = min(max((float(t) - 1) / 3, 0.0), 1.0)
        assert float(f) == pytest.approx(float(w) * (keep + (1 - keep) / 8), rel=1e-6)
    yarn, scale = kohakutt_amd.rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 8, "original": n})
    assert scale == pytest.approx(0.1 * math.log(8) + 1)
    ratio = yarn.double() / want
    # Pairs that turn more than 32 times are kept, those under one turn stretched, none rises.
    assert bool((ratio[turns > 40] > 0.99999).all())
    assert torch.allclose(ratio[turns < 0.8], torch.full_like(ratio[turns < 0.8], 1 / 8), rtol=1e-5)
    assert bool((ratio.diff() <= 1e-7).all())
    assert kohakutt_amd.rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 8, "original": n, "scale": 1.5})[1] == 1.5


@pytest.mark.parametrize(
    "dim,scaling,msg",
    [
        (7, None, "even"),
        (0, None, "even"),
        (64, {"type": "cubic", "factor": 2}, "one of"),
        (64, {"factor": 2}, "one of"),
        (64, {"type": "linear"}, "takes"),
        (64, {"type": "linear", "factor": 2, "low": 1}, "takes"),
        (64, {"type": "linear", "factor": 0.5}, "at least 1"),
        (64, {"type": "linear", "factor": math.nan}, "at least 1"),
        (2, {"type": "ntk", "factor": 2}, "more than one pair"),
        (64, {"type": "bands", "factor": 2, "original": 4096, "low": 4, "high": 4}, "above"),
        (64, {"type": "yarn", "factor": 2, "original": 4096, "slow": 4, "fast": 4}, "above"),
    ],
)
def test_rotary_frequencies_refuses(dim, scaling, msg):
    with pytest.raises(ValueError, match=msg):
        kohakutt_amd.rotary_frequencies(dim, scaling=scaling)


# ---------------------------------------------------------------- the plain forms themselves


def test_plain_codes_are_the_nearest():
    x = torch.randn(50, 64, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    codes, scale = P.quantise(x)
    got = P.values(codes, scale)
    unit = torch.exp2(scale.double() - 127).repeat_interleave(32, -1)
    for value in P.GRID.tolist():
        for sign in (1, -1):
            assert bool(((got - x).abs() <= (sign * value * unit - x).abs()).all())


def test_plain_attention_is_torchs():
    q, k, v = (torch.randn(n, h, 32, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    out, size, _, lse = P.attention(q, k, v, True, 0.2)
    for h in range(4):
        s = q[:, h] @ k[:, h // 2].t() * 0.2
        s = s.masked_fill(torch.arange(9) > torch.arange(4, 9).unsqueeze(1), -math.inf)
        assert torch.allclose(out[:, h], s.softmax(-1) @ v[:, h // 2])
        assert torch.allclose(lse[h], s.logsumexp(-1))
    assert bool((size >= out.abs() - 1e-12).all())
    none, _, _, _ = P.attention(q, k[:3], v[:3], True, 0.2)
    assert bool((none[:2] == 0).all())


def test_traced_calls_know_their_shapes():
    """Fake CUDA tensors trace through the ops without a launch (no GPU is there)."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 10, 4, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        k = torch.empty(2, 10, 2, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        pos, freq = torch.empty(10, dtype=torch.int64, device="cuda"), torch.empty(16, device="cuda")
        y, ky = kohakutt_amd.rotary(x, pos, freq, k=k)
        assert y.stride() == x.stride() and ky.shape == k.shape
        assert kohakutt_amd.rotary(x, pos, freq).shape == x.shape
        z = kohakutt_amd.rotary(x.detach().requires_grad_(), pos, freq)
        assert z.requires_grad and z.shape == x.shape
        for bits in (16, 4):
            held = kohakutt_amd.paged_cache(5, 2, 16, 64, head_dim_v=96, bits=bits)
            table, lens = torch.empty(3, 2, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
            q, kk, v = (torch.empty(3, n, d, dtype=torch.bfloat16, device="cuda") for n, d in ((4, 64), (2, 64), (2, 96)))
            assert kohakutt_amd.paged_append(kk, v, **held, block_table=table, key_lengths=lens) is None
            got = kohakutt_amd.paged_append(kk, v, **held, block_table=table, key_lengths=lens, q=q, inv_freq=freq)
            assert got.shape == q.shape
            rk, rv = kohakutt_amd.paged_read(**held, block_table=table, key_lengths=lens, max_k=20)
            assert rk.shape == (3, 2, 20, 64) and rv.shape == (3, 2, 20, 96) and rk.dtype == torch.bfloat16
            out = kohakutt_amd.sdpa_paged(q, **held, block_table=table, key_lengths=lens)
            assert out.shape == (3, 4, 96) and out.dtype == torch.bfloat16
