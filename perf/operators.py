"""Workloads of the paged-cache operators, for timing and for comparing two builds.

The operators of a serving (and, for the rotation, a training) attention layer:

* ``kohakutt_amd.rotary`` -- the position rotation of queries and keys, and its gradient;
* ``kohakutt_amd.paged_append`` -- new keys and values into the pages of a cache, rotated
  on the way, in 16 bits or in 4 (32 values under one power-of-two scale);
* ``kohakutt_amd.paged_read`` -- a cache's keys and values as dense tensors;
* ``kohakutt_amd.sdpa_paged`` -- attention over such a cache, single tokens and chunks.

* ``listed()`` -- the fixed cases; ``draw(rng)`` -- one more case of the same ranges.
* ``prepare(case, seed)`` -- what a program holds before the call, on the GPU.
* ``run(state)`` -- one call: the operators' plain torch form, or (``own``) the kernels.
* ``exact(case, seed)`` -- the same outputs in float64, written apart from the plain form.
* ``work(case)`` -- bytes and FLOPs the call cannot do without.
"""

import importlib
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, **kw):
    case = {
        "name": name,
        "op": op,  # rotary | append | read | attention
        "dtype": "bf16",
        "bits": 16,  # of the cache's values
        "seqs": 1,  # sequences (rotary in training: batch entries)
        "new": 1,  # new tokens of the longest sequence
        "keys": 1,  # keys of the longest sequence, the new ones among them
        "ragged": False,  # the other sequences are shorter
        "heads_q": 1,
        "heads_kv": 1,
        "dim": 128,
        "page": 64,
        "rotary_dim": 0,  # rotated dims of a head (0: the whole head)
        "interleaved": False,
        "far": 0,  # first position of the rotation
        "train": False,
    }
    case.update(kw)
    return case


def listed():
    return [
        # One decoding step of eight sequences deep in a long context: the rotation of
        # their queries and keys, launch latency alone.
        _case("rotary_decode_8_16_2x128", "rotary", seqs=8, heads_q=16, heads_kv=2, far=100000),
        # A training batch whose heads rotate their first half in interleaved pairs.
        _case("rotary_train_4x4096_16_8x128", "rotary", seqs=4, new=4096, heads_q=16, heads_kv=8, rotary_dim=64,
              interleaved=True, train=True),
        # One decoding step of 64 sequences: a token each into the pages, queries rotated too.
        _case("append_decode_64_16_2x128", "append", seqs=64, keys=1000, ragged=True, heads_q=16, heads_kv=2),
        # Prompts of eight sequences, some behind a shared prefix, into small pages.
        _case("append_prompt_8x2048_16_8x128", "append", dtype="f16", seqs=8, new=2048, keys=2560, ragged=True,
              heads_q=16, heads_kv=8, page=16),
        # Prompts into a 4-bit cache, and the cache read back (for a layer without a kernel
        # for it, or to move a sequence elsewhere).
        _case("append4_read_4x2048_8x128", "append", bits=4, seqs=4, new=2048, keys=2048, ragged=True, heads_q=0,
              heads_kv=8),
        # Keys and values of 16 ragged sequences out of their pages.
        _case("read_16x1001_2x64", "read", seqs=16, keys=1001, ragged=True, heads_kv=2, dim=64, page=32),
        # A token of one short sequence (14 query heads over 2): latency.
        _case("paged_decode_1x777_14_2x64", "attention", keys=777, heads_q=14, heads_kv=2, dim=64, page=16),
        # Decoding with a full batch of long sequences: the cache's bytes.
        _case("paged_decode_64x8192_16_2x128", "attention", seqs=64, keys=8192, heads_q=16, heads_kv=2),
        # A chunk of each of four long prompts over what their pages already hold.
        _case("paged_chunk_4x1024_8192_32_8x128", "attention", dtype="f16", seqs=4, new=1024, keys=8192, ragged=True,
              heads_q=32, heads_kv=8, page=128),
        # Four drafted tokens of three sequences checked at once, over a 4-bit cache.
        _case("paged4_draft_3x4_5001_14_2x64", "attention", bits=4, seqs=3, new=4, keys=5001, ragged=True, heads_q=14,
              heads_kv=2, dim=64, page=32),
        # The full batch of long sequences over a 4-bit cache.
        _case("paged4_decode_64x8192_16_2x128", "attention", bits=4, seqs=64, keys=8192, heads_q=16, heads_kv=2),
        # A ragged chunk of two prompts over a 4-bit cache with small pages.
        _case("paged4_chunk_2x777_4500_16_8x128", "attention", bits=4, seqs=2, new=777, keys=4500, ragged=True,
              heads_q=16, heads_kv=8, page=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "read", "attention", "attention", "attention"])
    heads_kv = rng.choice([1, 2, 4, 8])
    case = {
        "op": op,
        "dtype": rng.choice(["bf16", "bf16", "f16"]),
        "bits": 16,
        "seqs": _log_int(rng, 1, 64),
        "new": 1,
        "keys": 1,
        "ragged": rng.random() < 0.7,
        "heads_q": heads_kv * rng.choice([1, 2, 4, 7, 8]),
        "heads_kv": heads_kv,
        "dim": rng.choice([32, 64, 64, 96, 128, 128, 128, 256]),
        "page": rng.choice([16, 32, 48, 64, 128, 256]),
        "rotary_dim": 0,
        "interleaved": False,
        "far": 0,
        "train": False,
    }
    if op == "rotary":
        case["dtype"] = rng.choice(["bf16", "f16", "f32"])
        case["new"] = _log_int(rng, 1, 4096)
        case["far"] = rng.choice([0, _log_int(rng, 1, 1000000)])
        case["rotary_dim"] = rng.choice([0, case["dim"] // 2])
        case["interleaved"] = rng.random() < 0.5
        case["train"] = rng.random() < 0.5
        width = case["new"] * case["dim"] * (case["heads_q"] + case["heads_kv"])
        case["seqs"] = max(1, min(case["seqs"], 50_000_000 // (4 * width)))
        case["page"], case["ragged"] = 16, False
        return case
    case["bits"] = rng.choice([16, 4])
    if op == "append":
        case["new"] = rng.choice([1, _log_int(rng, 2, 2048)])
        case["keys"] = case["new"] + rng.choice([0, _log_int(rng, 1, 1000)])
        case["rotary_dim"] = rng.choice([0, 0, case["dim"] // 2])
        case["interleaved"] = rng.random() < 0.3
        case["heads_q"] = rng.choice([0, case["heads_q"]]) if case["bits"] == 16 else 0
        width = case["keys"] * case["dim"] * case["heads_kv"]
        case["seqs"] = max(1, min(case["seqs"], 17_000_000 // width))
    elif op == "read":
        case["keys"] = _log_int(rng, 1, 8192)
        case["heads_q"] = 0
        width = case["keys"] * case["dim"] * case["heads_kv"]
        case["seqs"] = max(1, min(case["seqs"], 17_000_000 // width))
    else:
        case["keys"] = _log_int(rng, 1, 16384)
        case["new"] = min(case["keys"], rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 1500)]))
        width = case["keys"] * case["dim"] * case["heads_kv"]
        case["seqs"] = max(1, min(case["seqs"], 120_000_000 // width))
        scores = case["new"] * case["keys"] * case["heads_q"]
        case["seqs"] = max(1, min(case["seqs"], 500_000_000 // scores))
    return case


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """(new tokens, keys) of each sequence; the first is the longest."""
    rng = random.Random(17)
    new, keys = [case["new"]], [case["keys"]]
    for _ in range(case["seqs"] - 1):
        n = rng.randint(max(1, case["new"] // 4), case["new"]) if case["ragged"] else case["new"]
        before = case["keys"] - case["new"]
        if case["ragged"]:
            before = rng.randint(before // 4, before)
        new.append(n)
        keys.append(n + before)
    return new, keys


def _quantise_plain(x):
    """x [..., D] as codes (uint8, two to a byte, the even dim in the low bits) and scale
    bytes of 32 dims: 2^(floor(log2 max|x|) - 2), biased by 127; e2m1 values, ties to the
    even code, saturating at 6."""
    g = x.double().unflatten(-1, (x.size(-1) // 32, 32))
    top = g.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(top)[1] - 3).clamp(-127, 127)
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127))
    y = torch.ldexp(g.abs(), -exponent)
    # Codes 0 .. 7 stand for 0, 0.5, 1, 1.5, 2, 3, 4, 6; a border belongs to the even code.
    code = (y > 0.25).to(torch.uint8)
    for border, even_above in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (y >= border) if even_above else (y > border)
    code = torch.where(torch.signbit(g), code + 8, code).flatten(-2)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return packed, (exponent.squeeze(-1) + 127).to(torch.uint8)


def _values_plain(packed, scale):
    """What codes and scale bytes stand for, float32."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=packed.device)
    table = torch.cat((table, -table))
    v = torch.stack((table[(packed & 15).long()], table[(packed >> 4).long()]), -1).flatten(-2)
    v = torch.ldexp(v.unflatten(-1, (scale.size(-1), 32)), (scale.int() - 127).unsqueeze(-1))
    return v.flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = _DTYPES[case["dtype"]], "cuda"
    hq, hk, d = case["heads_q"], case["heads_kv"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dt)

    state = {"case": case}
    rd = case["rotary_dim"] or d
    # Frequencies of a head's rotated pairs, base 10^6, as a long-context model has them.
    state["inv_freq"] = (1.0 / 1e6 ** (torch.arange(0, rd, 2, dtype=torch.float64) / rd)).float().to(dev)
    if case["op"] == "rotary":
        b, s = case["seqs"], case["new"]
        if case["train"]:
            # Heads as views of the projections' [B, S, H D] rows.
            for name, h in (("q", hq), ("k", hk)):
                state[name] = normal(b, s, h * d).view(b, s, h, d).transpose(1, 2).requires_grad_()
                state["g" + name] = normal(b, h, s, d)
            state["positions"] = torch.arange(s, device=dev) + case["far"]
        else:
            state["q"], state["k"] = normal(b * s, hq, d), normal(b * s, hk, d)
            start = torch.randint(0, max(1, case["far"]), (b, 1), generator=gen, device=dev) + case["far"]
            state["positions"] = (start + torch.arange(s, device=dev)).flatten()
        return state

    new, keys = _lengths(case)
    page = case["page"]
    counts = [-(-n // page) for n in keys]
    pages = sum(counts)
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    starts = [sum(counts[:i]) for i in range(len(counts))]
    at = torch.arange(max(counts), device=dev).unsqueeze(0)
    count = torch.tensor(counts, device=dev).unsqueeze(1)
    index = (torch.tensor(starts, device=dev).unsqueeze(1) + at).clamp(max=pages - 1)
    state["table"] = torch.where(at < count, order[index], torch.full_like(order[index], -1))
    state["lengths"] = torch.tensor(keys, dtype=torch.int32, device=dev)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    state["cu"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
    state["single"] = case["new"] == 1
    cache = {}
    for name in ("k", "v"):
        shape = (pages, hk, page)
        if case["op"] == "append" and case["bits"] == 4:
            cache[name] = torch.zeros(*shape, d // 2, dtype=torch.uint8, device=dev)
            cache[name + "_scale"] = torch.zeros(*shape, d // 32, dtype=torch.uint8, device=dev)
        elif case["op"] == "append":
            cache[name] = torch.zeros(*shape, d, dtype=dt, device=dev)
        else:
            x = normal(*shape, d)
            if name == "k":  # a few dims of a head's keys are larger than the others
                x[..., :: max(1, d // 4)] *= 3
            if case["bits"] == 4:
                parts = [_quantise_plain(c) for c in x.split(max(1, 8_000_000 // (hk * page * d)))]
                cache[name] = torch.cat([p for p, _ in parts])
                cache[name + "_scale"] = torch.cat([e for _, e in parts])
            else:
                cache[name] = x
    state["cache"] = cache
    tokens = offsets[-1]
    if case["op"] == "append":
        state["k"], state["v"] = normal(tokens, hk, d), normal(tokens, hk, d)
    if hq and case["op"] != "read":
        state["q"] = normal(tokens, hq, d)
    state["tokens"] = tokens
    state["max_k"] = max(keys)
    return state


# ---------------------------------------------------------------- the framework's calls


def _package():
    if "kohakutt_amd" not in sys.modules:  # the package of the tree that the process runs in
        sys.path.insert(0, os.path.abspath("kohaku-tt_amd"))
        importlib.import_module("kohakutt_amd")
    return sys.modules["kohakutt_amd"]


def _run_own(state):
    ops, case = _package(), state["case"]
    if case["op"] == "rotary":
        q, k = ops.rotary(state["q"], state["positions"], state["inv_freq"], k=state["k"],
                          interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": q, "k": k}
        gq, gk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["gq"], state["gk"]))
        return {"q": q, "k": k, "gq": gq, "gk": gk}
    cache, cu = state["cache"], None if state["single"] else state["cu"]
    held = (cache["k"], cache["v"], state["table"], state["lengths"])
    scales = {"k_scale": cache.get("k_scale"), "v_scale": cache.get("v_scale")}
    if case["op"] == "append":
        q = ops.paged_append(state["k"], state["v"], *held, cu_seq=cu, q=state.get("q"), inv_freq=state["inv_freq"],
                             interleaved=case["interleaved"], **scales)
        if case["bits"] == 16:
            return {"k": cache["k"], "v": cache["v"]} if q is None else {"q": q, "k": cache["k"], "v": cache["v"]}
    if case["op"] != "attention":
        k, v = ops.paged_read(*held, max_k=state["max_k"], dtype=_DTYPES[case["dtype"]], **scales)
        return {"k": k, "v": v}
    return ops.sdpa_paged(state["q"], *held, cu_seq_q=cu, max_q=case["new"], max_k=state["max_k"], is_causal=True,
                          **scales)


# ---------------------------------------------------------------- the plain forms


def _rotated(x, positions, inv_freq, interleaved, back=False):
    """x [..., D] rotated by positions (broadcast over x's leading dims) in x's type."""
    angle = positions.double().unsqueeze(-1) * inv_freq.double()
    c, s = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    if back:
        s = -s
    rd = 2 * inv_freq.numel()
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., : rd // 2], x[..., rd // 2 : rd])
    y1, y2 = a * c - b * s, b * c + a * s
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((y, x[..., rd:]), -1)


def _token_places(state):
    """Each new token's sequence and position."""
    cu, lengths = state["cu"].long(), state["lengths"].long()
    seq = torch.repeat_interleave(torch.arange(lengths.numel(), device=cu.device), cu[1:] - cu[:-1],
                                  output_size=state["tokens"])
    return seq, lengths[seq] - cu[seq + 1] + torch.arange(state["tokens"], device=cu.device)


def _gathered(state, name, dtype):
    """The cache's `name` as [B, Hkv, max_k, D], zeros past each length."""
    cache, page = state["cache"], state["case"]["page"]
    pos = torch.arange(state["max_k"], device="cuda")
    where = state["table"][:, pos // page].long().clamp(min=0)
    x = cache[name][where, :, pos % page]
    if state["case"]["bits"] == 4:
        x = _values_plain(x, cache[name + "_scale"][where, :, pos % page])
    keep = pos < state["lengths"].unsqueeze(1)
    return torch.where(keep[:, :, None, None], x.to(dtype), torch.zeros((), dtype=dtype, device="cuda")).transpose(1, 2)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "rotary":
        pos = state["positions"] if case["train"] else state["positions"].unsqueeze(1)
        out = {}
        for name in ("q", "k"):
            x = state[name].detach()
            out[name] = _rotated(x.float(), pos, state["inv_freq"], case["interleaved"]).to(x.dtype)
            if case["train"]:
                g = state["g" + name].float()
                out["g" + name] = _rotated(g, pos, state["inv_freq"], case["interleaved"], back=True).to(x.dtype)
        return out
    cache, dt = state["cache"], _DTYPES[case["dtype"]]
    if case["op"] == "append":
        seq, pos = _token_places(state)
        page, slot = state["table"][seq, pos // case["page"]].long(), pos % case["page"]
        out = {}
        if case["bits"] == 4:  # (64 bits: values next to a border between two codes)
            k = _rotated(state["k"].double(), pos.unsqueeze(1), state["inv_freq"], case["interleaved"])
            for name, x in (("k", k), ("v", state["v"])):
                cache[name][page, :, slot], cache[name + "_scale"][page, :, slot] = _quantise_plain(x)
            return {name: _gathered(state, name, dt) for name in ("k", "v")}
        k = _rotated(state["k"].float(), pos.unsqueeze(1), state["inv_freq"], case["interleaved"])
        cache["k"][page, :, slot] = k.to(dt)
        cache["v"][page, :, slot] = state["v"]
        if "q" in state:
            q = _rotated(state["q"].float(), pos.unsqueeze(1), state["inv_freq"], case["interleaved"])
            out["q"] = q.to(dt)
        out["k"], out["v"] = cache["k"], cache["v"]
        return out
    if case["op"] == "read":
        return {name: _gathered(state, name, dt) for name in ("k", "v")}
    # Attention: the queries padded to [B, Hkv, Lq G, D], every key of the batch in float32.
    b, hk, d = case["seqs"], case["heads_kv"], case["dim"]
    group, most = case["heads_q"] // hk, case["new"]
    seq, pos = _token_places(state)
    row = torch.arange(state["tokens"], device="cuda") - state["cu"].long()[seq]
    q = torch.zeros(b, most, hk, group, d, device="cuda")
    q[seq, row] = state["q"].float().unflatten(1, (hk, group))
    last = torch.full((b, most), -1, device="cuda")
    last[seq, row] = pos  # the last key each query sees
    k, v = _gathered(state, "k", torch.float32), _gathered(state, "v", torch.float32)
    s = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(b, hk, most * group, d), k.transpose(-1, -2).contiguous())
    hidden = torch.arange(state["max_k"], device="cuda") > last.unsqueeze(-1)
    s = s.view(b, hk, most, group, -1).mul_(1.0 / math.sqrt(d))
    s.masked_fill_(hidden[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hk, most * group, -1), v).view(b, hk, most, group, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3, 4)
    return o[seq, row].flatten(1, 2).to(dt)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- 64 bits


def _exact_turned(x, positions, inv_freq, interleaved, back=False):
    """x [T, H, D] float64, pairs as complex numbers times e^(i position frequency)."""
    n = inv_freq.numel()
    angle = torch.outer(positions.double(), inv_freq.double())
    turn = torch.polar(torch.ones_like(angle), -angle if back else angle).unsqueeze(1)
    y = x.clone()
    if interleaved:
        y[..., : 2 * n] = torch.view_as_real(torch.view_as_complex(x[..., : 2 * n].reshape(*x.shape[:2], n, 2).contiguous()) * turn).reshape(*x.shape[:2], 2 * n)
    else:
        z = torch.complex(x[..., :n], x[..., n : 2 * n]) * turn
        y[..., :n], y[..., n : 2 * n] = z.real, z.imag
    return y


def _exact_fp4(x):
    """The values that x's nearest codes stand for, float64 (by distance, not by borders)."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    g = x.reshape(-1, 32)
    top = g.abs().amax(1, keepdim=True)
    unit = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top)) - 2), torch.ones_like(top))
    y = (g.abs() / unit).clamp(max=6.0)
    above = torch.searchsorted(grid, y.contiguous()).clamp(max=7)
    below = (above - 1).clamp(min=0)
    up, down = grid[above] - y, y - grid[below]
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (grid[pick] * torch.sign(g) * unit).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    f = state["inv_freq"]
    if case["op"] == "rotary":
        out = {}
        for name in ("q", "k"):
            for key, back in ((name, False), ("g" + name, True)):
                if key not in state:
                    continue
                x = state[key].detach()
                if case["train"]:
                    b, h, s, d = x.shape
                    rows = x.transpose(1, 2).reshape(b * s, h, d).double()
                    y = _exact_turned(rows, state["positions"].repeat(b), f, case["interleaved"], back)
                    out[key] = y.view(b, s, h, d).transpose(1, 2)
                else:
                    out[key] = _exact_turned(x.double(), state["positions"], f, case["interleaved"], back)
        return out
    new, keys = _lengths(case)
    cache, page, cu = state["cache"], case["page"], state["cu"].tolist()
    table = state["table"].cpu()

    def held(name, i):
        """Sequence i's [keys, Hkv, D] in float64."""
        ids = table[i, : -(-keys[i] // page)].long().cuda()

        def rows(x):
            return x[ids].transpose(1, 2).flatten(0, 1)[: keys[i]]

        x = rows(cache[name])
        if case["bits"] == 16:
            return x.double()
        sign = 1.0 - 2.0 * torch.stack(((x >> 3) & 1, x >> 7), -1).flatten(-2).double()
        low = torch.stack((x & 7, (x >> 4) & 7), -1).flatten(-2)
        # e2m1: exponent bits 0 hold 0 and 0.5, else (2 + mantissa) 2^(exponent - 2).
        mag = torch.where(low < 2, low.double() / 2, (2 + (low & 1)).double() * torch.exp2((low >> 1).double() - 2))
        return sign * mag * torch.exp2(rows(cache[name + "_scale"]).double() - 127).repeat_interleave(32, -1)

    if case["op"] == "append":
        pos = torch.cat([torch.arange(n - m, n, device="cuda") for m, n in zip(new, keys)])
        k, v = _exact_turned(state["k"].double(), pos, f, case["interleaved"]), state["v"].double()
        if case["bits"] == 4:
            k, v = _exact_fp4(k), _exact_fp4(v)
            out = {n: torch.zeros(case["seqs"], case["heads_kv"], state["max_k"], case["dim"], dtype=torch.float64, device="cuda") for n in "kv"}
            for i in range(case["seqs"]):
                for name, x in (("k", k), ("v", v)):
                    out[name][i, :, keys[i] - new[i] : keys[i]] = x[cu[i] : cu[i + 1]].transpose(0, 1)
            return out
        out = {"k": torch.zeros_like(cache["k"], dtype=torch.float64), "v": torch.zeros_like(cache["v"], dtype=torch.float64)}
        for i in range(case["seqs"]):
            p = torch.arange(keys[i] - new[i], keys[i])
            ids = table[i, p // page].long().cuda()
            for name, x in (("k", k), ("v", v)):
                out[name][ids, :, (p % page).cuda()] = x[cu[i] : cu[i + 1]]
        if "q" in state:
            out["q"] = _exact_turned(state["q"].double(), pos, f, case["interleaved"])
        return out
    if case["op"] == "read":
        out = {}
        for name in ("k", "v"):
            out[name] = torch.zeros(case["seqs"], case["heads_kv"], state["max_k"], case["dim"], dtype=torch.float64, device="cuda")
            for i in range(case["seqs"]):
                out[name][i, :, : keys[i]] = held(name, i).transpose(0, 1)
        return out
    group = case["heads_q"] // case["heads_kv"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        k, v = held("k", i), held("v", i)
        sees = torch.arange(keys[i], device="cuda") <= torch.arange(keys[i] - new[i], keys[i], device="cuda").unsqueeze(1)
        for h in range(case["heads_q"]):
            s = state["q"][cu[i] : cu[i + 1], h].double() @ k[:, h // group].t() / math.sqrt(case["dim"])
            p = torch.softmax(torch.where(sees, s, torch.full_like(s, -math.inf)), -1)
            out[cu[i] : cu[i + 1], h] = p @ v[:, h // group]
    return out


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    hq, hk, d = case["heads_q"], case["heads_kv"], case["dim"]
    if case["op"] == "rotary":
        values = case["seqs"] * case["new"] * (hq + hk) * d
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * values * es, "flops": passes * 3 * values}
    new, keys = _lengths(case)
    # Bytes of a key (or value) row in the cache.
    row = d * es if case["bits"] == 16 else d // 2 + d // 32
    if case["op"] == "append":
        values = sum(new) * d
        total = 2 * sum(new) * hk * (d * es + row) + 2 * values * hq * es
        if case["bits"] == 4:
            total += 2 * sum(keys) * hk * row + 2 * case["seqs"] * max(keys) * hk * d * es
        return {"bytes": total, "flops": 3 * values * (hq + hk)}
    if case["op"] == "read":
        return {"bytes": 2 * sum(keys) * hk * row + 2 * case["seqs"] * max(keys) * hk * d * es, "flops": 0}
    # Query r of n new ones over m keys sees m - n + r + 1 of them.
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, keys))
    return {"bytes": 2 * sum(keys) * hk * row + 2 * sum(new) * hq * d * es, "flops": 4 * pairs * hq * d}
