"""64-bit restatements of the serving-step extensions: the paged plan, the normed and rotated
queries and keys with their gradients, 4-bit groups, and attention over what they stand for.

The reference has none of these; the attention arithmetic is that of
python/triton_llm/reference/paged_attention.py:14-40 with a causal mask aligned to the end of the
context, the rotation that of python/triton_llm/reference/norm_rope.py:12-40. Test infrastructure
only.
"""
from __future__ import annotations

import math

import numpy as np

GROUP = 32


def paged_plan(table, seq_lens, n_new, free, *, block_size, max_tokens):
    """(slots, positions, cu, new_lens, taken, table), a sequence at a time."""
    table = np.array(table, dtype=np.int64)
    slots, positions = np.full(max_tokens, -1, np.int64), np.zeros(max_tokens, np.int64)
    cu, new_lens, taken, asked = [0], [], 0, 0
    for b, (length, n) in enumerate(zip(seq_lens, n_new)):
        length, n = max(0, int(length)), max(0, int(n))
        have, want = -(-length // block_size), -(-(length + n) // block_size)
        fits = want <= table.shape[1]
        need = want - have if fits else 0
        start, end = asked, asked + need
        asked = end
        row = cu[-1]
        cu.append(row + n)
        ok = fits and (need == 0 or end <= len(free)) and row + n <= max_tokens
        if ok:
            table[b, have:want] = free[start:end]
            taken += need
        for t in range(n):
            if row + t < max_tokens:
                pos = length + t
                positions[row + t] = pos
                if ok:
                    slots[row + t] = table[b, pos // block_size] * block_size + pos % block_size
        new_lens.append(length + n if ok else length)
    return slots, positions, np.array(cu), np.array(new_lens), taken, table


def axis_of_pair(sections, interleaved):
    half = sum(sections)
    axes = np.zeros(half, np.int64)
    if interleaved:
        for a in range(1, len(sections)):
            for i in range(sections[a]):
                if a + i * len(sections) < half:
                    axes[a + i * len(sections)] = a
        return axes
    return np.repeat(np.arange(len(sections)), sections)


def _turn(cos, sin, positions, sections, interleaved):
    axes = axis_of_pair(sections, interleaved)
    i = np.arange(len(axes))
    row = np.asarray(positions)[axes].T  # [T, D / 2]
    return (np.float64(cos)[row, i] + 1j * np.float64(sin)[row, i])[:, None]


def norm_rope(x, w, cos, sin, positions, sections, interleaved=False, eps=1e-6):
    x, half = np.float64(x), x.shape[-1] // 2
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.float64(w)
    z = (y[..., :half] + 1j * y[..., half:]) * _turn(cos, sin, positions, sections, interleaved)
    return np.concatenate([z.real, z.imag], -1)


def norm_rope_grad(dz, x, w, cos, sin, positions, sections, interleaved=False, eps=1e-6):
    """(dx, dw, size of the terms of dx, size of the terms of dw): the last two for error bounds."""
    x, dz, w, half = np.float64(x), np.float64(dz), np.float64(w), x.shape[-1] // 2
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    t = _turn(cos, sin, positions, sections, interleaved)
    dy = (dz[..., :half] + 1j * dz[..., half:]) * t.conj()
    size = (np.abs(dz[..., :half]) + np.abs(dz[..., half:]))
    size = np.concatenate([size, size], -1)
    dy = np.concatenate([dy.real, dy.imag], -1)
    g = dy * w
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdims=True))
    gs = size * np.abs(w)
    dx_size = r * (gs + np.abs(x) * r * r * (gs * np.abs(x)).mean(-1, keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx, (dy * x * r).sum(axes), dx_size, (size * np.abs(x) * r).sum(axes)


def quantise(x):
    """(codes, scales, zeros) of x [..., D] (fp32 values): each step in fp32, as defined."""
    g = np.float32(x).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        s = ((hi - lo) * np.float32(1 / 15)).astype(np.float16)
        z = lo.astype(np.float16)
        # a rounded-up scale must not put the largest code past fp16's range
        past = (hi < 65520) & (15 * np.float32(s) + np.float32(z) >= 65520)
        s = np.where(past, np.nextafter(s, np.float16(0)), s)
        # nor is a group with a value that fp16 has no room for a group of numbers
        s = np.where((lo > -65520) & (hi < 65520), s, np.float16(np.nan))
        sf, zf = np.float32(s), np.float32(z)
        inv = np.where(sf > 0, np.float32(1) / sf, np.float32(0))
        codes = np.clip(np.rint((g - zf) * inv), 0, 15)
    return codes, s.astype(np.float64), z.astype(np.float64)


def dequantise(codes, s, z):
    """(the values, the sizes of their two terms added up), [..., D] in 64 bits."""
    shape = (*codes.shape[:-2], codes.shape[-2] * GROUP)
    with np.errstate(invalid="ignore"):
        return (codes * s + z).reshape(shape), (codes * s + np.abs(z)).reshape(shape)


def attention(q, k, v, k_size, v_size, *, scale, causal, n_new):
    """Newest n_new tokens of one sequence: q [n, Hq, D], k, v [len, Hkv, D] (the values) and the
    sizes of their terms. Returns (o, A, E): A the weighted sum of v_size, E the largest error bound
    of a score: 2^-12 of its terms (keys rounded to 11 bits) and 2^-21 of the sizes (fp32 sums)."""
    n, hq, d = q.shape
    length, hkv = k.shape[:2]
    g = hq // hkv
    o, a, e = np.empty((n, hq, d)), np.empty((n, hq, d)), np.empty((n, hq, 1))
    for h in range(hq):
        kk, vv, ks, vs = (x[:, h // g] for x in (k, v, k_size, v_size))
        for s in range(n):
            m = length - n_new + s + 1 if causal else length
            m = min(max(m, 0), length)
            if m == 0:
                o[s, h], a[s, h], e[s, h] = math.nan, 0, 0
                continue
            qq = np.float64(q[s, h])
            x = kk[:m] @ qq * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            o[s, h], a[s, h] = p @ vv[:m], p @ vs[:m]
            e[s, h] = scale * ((np.abs(kk[:m]) @ np.abs(qq)).max() * 2.0 ** -12
                               + (ks[:m] @ np.abs(qq)).max() * 2.0 ** -21)
    return o, a, e
