"""Positions and the paged cache: the rotation of queries and keys, appending to a cache
whose rows lie in pages, reading it back, and attention over it.

* ``rotary(x, positions, inv_freq, k=...)`` -- rotary positions, differentiable
  (``ktt::_rotary``); ``rotary_frequencies`` makes ``inv_freq``, scaled for long contexts.
* ``paged_cache(...)`` -- the tensors of a cache, 16-bit or 4-bit.
* ``paged_append(k, v, k_cache, v_cache, ...)`` -- new keys and values into the pages, the
  rotation applied on the way (``ktt::_paged_append``).
* ``sdpa_paged(q, k_cache, v_cache, ...)`` -- attention over the pages
  (``ktt::_sdpa_paged``): the paged counterpart of ``sdpa`` and ``sdpa_varlen``.
* ``paged_read(k_cache, v_cache, ...)`` -- a cache as dense ``[B, H, S, D]`` tensors, as
  ``sdpa(key_lengths=)`` takes them (``ktt::_paged_read``).

A cache is ``k_cache`` / ``v_cache`` ``[pages, heads, page size, D]`` (any strides with
contiguous rows, so ``[pages, page size, heads, D].transpose(1, 2)`` too; the page size is a
multiple of 16).  Key p of sequence b is row ``p % page_size`` of page
``block_table[b, p // page_size]`` (int32 ``[B, n]``); ``key_lengths`` (int32 ``[B]``) counts
each sequence's keys, the new tokens of the call being the last of them.  Packed tokens
``[T, heads, D]`` belong to sequences by ``cu_seq`` (int32 ``[B + 1]``); without it there is
one token per sequence, T = B.  All three stay on the GPU and are read by the kernels alone, so
a captured graph follows what they hold at its replay.  What is out of range there never
reaches memory it should not: lengths are clamped to what ``block_table`` (and ``max_k``) can
hold, an append leaves out tokens whose page does not exist, a reader takes page 0 for it.

A 4-bit cache holds two e2m1 codes to a byte (``uint8 [pages, heads, page size, D / 2]``, the
even dim in the low bits) and one power-of-two scale byte for 32 dims of a row (``k_scale`` /
``v_scale``, ``uint8 [pages, heads, page size, D / 32]``): 4.25 bits a value.  The scale is
``2^(floor(log2 max|x|) - 2)``; values round to the nearest code, ties to the even one, and
saturate at 6 times the scale.  A group that holds a NaN or an infinity reads back as NaN.
"""

from __future__ import annotations

import math

import torch

# (The overloads themselves: a call through the packet resolves them each time.)
_ROTARY = torch.ops.ktt._rotary.default
_APPEND = torch.ops.ktt._paged_append.default
_READ = torch.ops.ktt._paged_read.default
_SDPA = torch.ops.ktt._sdpa_paged.default

__all__ = ["rotary", "rotary_frequencies", "paged_cache", "paged_append", "paged_read", "sdpa_paged"]


# ---------------------------------------------------------------- rotation


def rotary_frequencies(dim, base=10000.0, scaling=None, device=None):
    """``(inv_freq, scale)`` of ``rotary`` for `dim` rotated dims: fp32 ``[dim / 2]`` with
    ``base^(-2 i / dim)``, and the factor on the rotated values (1 unless said below).

    `scaling` stretches the frequencies for contexts longer than the trained one:

    * ``{"type": "linear", "factor": f}`` -- every frequency over f.
    * ``{"type": "ntk", "factor": f}`` -- the base times ``f^(dim / (dim - 2))``: the slowest
      pair stretched by f, the fastest not at all.
    * ``{"type": "bands", "factor": f, "original": n, "low": 1.0, "high": 4.0}`` -- pairs that
      turn fewer than `low` times in the n trained positions over f, those that turn more than
      `high` times as they are, a straight blend in the number of turns between.
    * ``{"type": "yarn", "factor": f, "original": n, "slow": 1.0, "fast": 32.0}`` -- the blend
      linear in the pair's index between the pairs that turn `fast` and `slow` times (rounded
      outward), and a scale of ``0.1 ln f + 1`` (``"scale"`` overrides it)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"kohakutt_amd.rotary_frequencies: dim must be even and positive, got {dim}")
    pair = torch.arange(0, dim, 2, dtype=torch.float64)
    plain = dict(scaling) if scaling else {"type": "none"}
    kind = plain.pop("type", None)
    known = {
        "none": (set(), set()),
        "linear": ({"factor"}, set()),
        "ntk": ({"factor"}, set()),
        "bands": ({"factor", "original"}, {"low", "high"}),
        "yarn": ({"factor", "original"}, {"slow", "fast", "scale"}),
    }
    if kind not in known:
        raise ValueError(
            f"kohakutt_amd.rotary_frequencies: scaling type must be one of {', '.join(known)}, got {kind!r}"
        )
    needed, optional = known[kind]
    if needed - set(plain) or set(plain) - needed - optional:
        raise ValueError(
            f"kohakutt_amd.rotary_frequencies: {kind} scaling takes {sorted(needed | optional)} "
            f"(needed: {sorted(needed)}), got {sorted(plain)}"
        )
    factor, scale = float(plain.get("factor", 1.0)), 1.0
    if not factor >= 1.0:
        raise ValueError(f"kohakutt_amd.rotary_frequencies: factor must be at least 1, got {factor}")
    if kind == "ntk":
        if dim == 2:
            raise ValueError("kohakutt_amd.rotary_frequencies: ntk scaling needs more than one pair")
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-pair / dim)
    if kind == "linear":
        freq = freq / factor
    elif kind == "bands":
        low, high = float(plain.get("low", 1.0)), float(plain.get("high", 4.0))
        if not high > low:
            raise ValueError(f"kohakutt_amd.rotary_frequencies: high must be above low, got {high} and {low}")
        turns = freq * plain["original"] / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
    elif kind == "yarn":
        slow, fast = float(plain.get("slow", 1.0)), float(plain.get("fast", 32.0))
        if not fast > slow:
            raise ValueError(f"kohakutt_amd.rotary_frequencies: fast must be above slow, got {fast} and {slow}")

        def pair_of(turns):  # the (fractional) pair that turns so often in the trained positions
            return dim * math.log(plain["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / factor * ramp
        scale = float(plain.get("scale", 0.1 * math.log(factor) + 1.0))
    return freq.to(torch.float32).to(device), scale


def rotary(x, positions, inv_freq, k=None, interleaved=False, scale=1.0):
    """Rotary positions: the first ``2 * len(inv_freq)`` dims of every head of `x` turned in
    pairs by ``position * inv_freq``, the others as they are.

    `x` is ``[B, H, S, D]`` (views of projections are read in place) or packed ``[T, H, D]``,
    bf16, fp16 or fp32, D up to 256; `positions` int32 or int64 ``[S]`` or ``[B, S]`` (``[T]``
    for packed tensors) on the GPU; `inv_freq` fp32.  Pair i is dims ``(i, i + len(inv_freq))``,
    or ``(2 i, 2 i + 1)`` with `interleaved`; rotated values are multiplied by `scale`.
    Angles are formed in 64 bits, so positions of millions keep theirs.

    Returns the rotated tensor, in x's memory layout; with `k` (another tensor of the same
    tokens, any number of heads) both, from one launch.  Differentiable in x and k (the
    gradient is the rotation back)."""
    y, ky = _ROTARY(x, k, positions, inv_freq, interleaved, scale)
    return y if k is None else (y, ky)


# ---------------------------------------------------------------- the cache


def paged_cache(pages, heads, page_size, head_dim, head_dim_v=None, dtype=torch.bfloat16, bits=16, device="cuda"):
    """The tensors of an empty cache, as keyword arguments of the functions below:
    ``{"k_cache": ..., "v_cache": ...}``, with ``k_scale`` and ``v_scale`` for ``bits=4``."""
    if bits not in (16, 4):
        raise ValueError(f"kohakutt_amd.paged_cache: bits must be 16 or 4, got {bits}")
    if page_size < 16 or page_size % 16:
        raise ValueError(f"kohakutt_amd.paged_cache: the page size must be a multiple of 16, got {page_size}")
    out = {}
    for name, d in (("k", head_dim), ("v", head_dim if head_dim_v is None else head_dim_v)):
        step = 8 if bits == 16 else 32
        if d < step or d > 256 or d % step:
            raise ValueError(
                f"kohakutt_amd.paged_cache: head dims of a {bits}-bit cache must be multiples of {step} up to 256, got {d}"
            )
        if bits == 16:
            out[name + "_cache"] = torch.zeros(pages, heads, page_size, d, dtype=dtype, device=device)
        else:
            out[name + "_cache"] = torch.zeros(pages, heads, page_size, d // 2, dtype=torch.uint8, device=device)
            out[name + "_scale"] = torch.zeros(pages, heads, page_size, d // 32, dtype=torch.uint8, device=device)
    return out


def paged_append(k, v, k_cache, v_cache, block_table, key_lengths, cu_seq=None, q=None, inv_freq=None,
                 interleaved=False, rotary_scale=1.0, k_scale=None, v_scale=None):
    """Writes the new keys `k` ``[T, Hkv, D]`` and values `v` ``[T, Hkv, Dv]`` into the cache:
    token r of sequence b becomes key ``key_lengths[b] - Lq_b + r``.

    With `inv_freq` keys are rotated at that position on the way (as ``rotary`` does, with
    `interleaved` and `rotary_scale`), and so is `q` ``[T, H, D]``, if given, in the same
    launch.  A 4-bit cache (`k_scale`, `v_scale`) is quantised on the way.  Tokens behind the
    last sequence write nothing; their rows of the rotated q are zero.  Returns the rotated q, or
    None without q.  Takes no gradients."""
    return _APPEND(k, v, k_cache, v_cache, block_table, key_lengths, cu_seq, q, inv_freq,
                   interleaved, rotary_scale, k_scale, v_scale)


def paged_read(k_cache, v_cache, block_table, key_lengths, max_k, dtype=None, k_scale=None, v_scale=None):
    """The cache's keys and values as dense ``[B, Hkv, max_k, D]`` and ``[B, Hkv, max_k, Dv]``
    tensors, zeros past each sequence's length (`dtype`: of a 4-bit cache's values, bf16 unless
    given)."""
    if dtype is None:
        dtype = torch.bfloat16 if k_scale is not None else k_cache.dtype
    return _READ(k_cache, v_cache, block_table, key_lengths, max_k, dtype, k_scale, v_scale)


def sdpa_paged(q, k_cache, v_cache, block_table, key_lengths, cu_seq_q=None, max_q=None, max_k=None, is_causal=True,
               scale=None, k_scale=None, v_scale=None):
    """Scaled dot-product attention of packed queries `q` ``[T, H, D]`` (bf16 or fp16) over a
    paged cache; returns ``[T, H, Dv]``.  Heads of the cache must divide q's (GQA).

    With `is_causal`, query r of a sequence sees its first ``key_lengths[b] - Lq_b + r + 1``
    keys (the new tokens are the cache's last keys), else all ``key_lengths[b]``; a query that
    sees none gets zeros, as do rows behind the last sequence.

    `max_q` (1 without `cu_seq_q`, else T unless given) must cover every sequence's queries:
    rows past it hold unspecified values.  `max_k` bounds the keys: those past it are not read
    (by default every key that `block_table` can name, which sizes a launch for that many and, over
    a 4-bit cache with more than 32 query rows per cache head, a 16-bit copy of them, so give the
    batch's longest length where it is known).  No gradient."""
    return _SDPA(q, k_cache, v_cache, block_table, key_lengths, cu_seq_q, max_q, max_k, is_causal,
                 scale, False, k_scale, v_scale)[0]


# ---------------------------------------------------------------- tracing


def _rotary_shapes(x, second, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    return torch.empty_like(x), None if second is None else torch.empty_like(second)


def _append_shapes(k, v, k_cache, v_cache, block_table, key_lengths, cu_seq=None, q=None, inv_freq=None,
                   interleaved=False, rotary_scale=1.0, k_scale=None, v_scale=None):
    return None if q is None else q.new_empty(q.shape)


def _read_shapes(k_cache, v_cache, block_table, key_lengths, max_k, dtype, k_scale=None, v_scale=None):
    wide = 1 if k_scale is None else 2
    return tuple(
        t.new_empty((block_table.size(0), t.size(1), max_k, wide * t.size(3)), dtype=dtype) for t in (k_cache, v_cache)
    )


def _sdpa_shapes(q, k_cache, v_cache, block_table, key_lengths, cu_seq_q=None, max_q=None, max_k=None, is_causal=True,
                 scale=None, stats=False, k_scale=None, v_scale=None):
    wide = 1 if v_scale is None else 2
    out = q.new_empty((q.size(0), q.size(1), wide * v_cache.size(3)))
    return out, q.new_empty((q.size(1), q.size(0)), dtype=torch.float32) if stats else None


def install() -> None:
    """Registers the shapes of the ops' results, for tracing (``torch.compile``)."""
    torch.library.register_fake("ktt::_rotary", _rotary_shapes)
    torch.library.register_fake("ktt::_paged_append", _append_shapes)
    torch.library.register_fake("ktt::_paged_read", _read_shapes)
    torch.library.register_fake("ktt::_sdpa_paged", _sdpa_shapes)
