"""Paged 8-bit KV cache: block tables, release, writer and attention, restated in
plain numpy loops and 64 bits.  The reference has no counterpart (it keeps one
contiguous cache a sequence), so parity is unpinned there; the e4m3 codec is
``oracle.codecs``' (pinned), and ``tests/test_oracle_paged.py`` checks each
function by a property that it does not use itself.
"""
from __future__ import annotations

import math

import numpy as np

from . import codecs as C

BLOCK = 64


def step(lengths, new, table, tokens, page, free=None, count=0):
    """-> dict of the outputs; `table` is updated in place."""
    r, width = table.shape
    starts = np.zeros(r + 1, np.int32)
    lengths_out = np.array(lengths, np.int32)
    seq = np.zeros(r, np.int32)
    positions, slots = np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
    end, taken, left = 0, 0, count
    for i in range(r):
        held, n = max(int(lengths[i]), 0), max(int(new[i]), 0)
        begin, end = end, end + n
        starts[i + 1] = min(end, tokens)
        lengths_out[i] = held
        if end > tokens or held + n > width * page:
            continue
        need = -(-(held + n) // page) - -(-held // page)
        taken += need
        if free is not None and need and taken > count:
            continue
        if free is not None:
            for j in range(need):
                table[i, -(-held // page) + j] = free[count - 1 - (taken - need) - j]
            left -= need
        lengths_out[i] = seq[i] = held + n
        for t in range(n):
            p = held + t
            positions[begin + t] = p
            if 0 <= table[i, p // page] < 2 ** 31 // page:
                slots[begin + t] = table[i, p // page] * page + p % page
    return dict(starts=starts, lengths=lengths_out, seq_lens=seq, positions=positions, slots=slots,
                free_count=np.array([left], np.int32))


def trim(lengths, keep, table, page, free, count):
    """-> (lengths, count); `free` is updated in place."""
    out = np.zeros_like(lengths)
    for i in reversed(range(len(lengths))):
        held = min(max(int(lengths[i]), 0), table.shape[1] * page)
        out[i] = min(max(int(keep[i]), 0), held)
        for col in reversed(range(-(-int(out[i]) // page), -(-held // page))):
            if count < len(free):
                free[count] = table[i, col]
            count += 1
    return out, min(count, len(free))


def key_byte(token, dim, d):
    return (((token // 16) * (d // 64) + dim // 64) * 64 + (dim % 64) // 16 * 16 + token % 16) * 16 + dim % 16


def value_byte(token, dim):
    return ((dim // 16) * 64 + (token % 16) // 4 * 16 + dim % 16) * 16 + (token // 16) * 4 + token % 4


def block_maps(d):
    """Byte of (token, dim) in a block: keys, values, each [64, d]."""
    t, c = np.arange(BLOCK)[:, None], np.arange(d)[None, :]
    return key_byte(t, c, d), value_byte(t, c)


def scale_exp(amax: float) -> int:
    """The least e >= -126 with amax <= 448 2^e."""
    if amax <= 0:
        return -126
    e = math.ceil(math.log2(amax / 448.0))
    while amax > 448.0 * 2.0 ** e:
        e += 1
    while amax <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return max(e, -126)


def largest_code(e: int) -> float:
    """The largest e4m3 value that is below 2^128 times 2^e."""
    return min(448.0, 1.875 * 2.0 ** (127 - e))


def write(k, v, codes, scales, table, starts, seq):
    """k, v [T, Hkv, D] float64 -> codes [P, NB, Hkv, 2, 64 D] and scales [P, NB, Hkv, 2] updated in place."""
    nb, hkv, d = codes.shape[1], codes.shape[2], codes.shape[4] // BLOCK
    maps = block_maps(d)
    for i in range(len(seq)):
        n = int(starts[i + 1]) - int(starts[i])
        held = int(seq[i]) - n
        if n <= 0 or held < 0:
            continue
        for b in range(held // BLOCK, -(-(held + n) // BLOCK)):
            page, sub = int(table[i, b // nb]), b % nb
            if not 0 <= page < codes.shape[0]:
                continue
            lo, hi = max(held - BLOCK * b, 0), min(held + n - BLOCK * b, BLOCK)
            row = int(starts[i]) + BLOCK * b - held
            for h in range(hkv):
                for part, x in enumerate((k, v)):
                    new = x[row + lo:row + hi, h]
                    finite = np.abs(new[np.isfinite(new)])
                    e = scale_exp(float(finite.max()) if finite.size else 0.0)
                    at, unit = maps[part], codes[page, sub, h, part]
                    if lo:
                        was = int(scales[page, sub, h, part]) - 127
                        if e > was:
                            old = C.e4m3_decode(unit[at[:lo]]).astype(np.float64) * 2.0 ** (was - e)
                            unit[at[:lo]] = C.e4m3_encode(old.astype(np.float32))
                        e = max(e, was)
                    else:
                        unit[at[hi:]] = 0
                    top = largest_code(e)
                    y = np.where(np.isnan(new), new, np.clip(new * 2.0 ** -e, -top, top))
                    unit[at[lo:hi]] = C.e4m3_encode(y.astype(np.float32))
                    scales[page, sub, h, part] = e + 127


def gather(codes, scales, table_row, length):
    """The keys and values of one request, [Hkv, length, D] float64 each (scale byte 255: not a number).
    2^128 and more, which bf16 and fp32 do not have, are infinite keys and values that are not numbers."""
    nb, hkv, d = codes.shape[1], codes.shape[2], codes.shape[4] // BLOCK
    maps = block_maps(d)
    out = [np.full((hkv, -(-length // BLOCK) * BLOCK, d), np.nan) for _ in range(2)]
    for b in range(-(-length // BLOCK)):
        page = int(table_row[b // nb])
        if not 0 <= page < codes.shape[0]:
            continue
        for part in (0, 1):
            e = scales[page, b % nb, :, part].astype(np.int64) - 127
            s = np.where(e == 128, np.nan, np.exp2(e.astype(np.float64)))
            x = C.e4m3_decode(codes[page, b % nb, :, part]).astype(np.float64)[:, maps[part]]
            x = x * s[:, None, None]
            past = np.abs(x) >= 2.0 ** 128
            out[part][:, BLOCK * b:BLOCK * (b + 1)] = np.where(past, np.nan if part else np.copysign(np.inf, x), x)
    return out[0][:, :length], out[1][:, :length]


def attention(q, codes, scales, table, starts, seq, scale, sink=None, window=0):
    """q [T, Hq, D] float64 -> (o, tolerance) [T, Hq, D].

    tolerance bounds a kernel that takes the scores and statistics in fp32, the
    probabilities of the value product in bf16 and rounds the result to bf16
    (u = 2^-24; a rounding to bf16 is off by at most 2^-8 relative):
      score  |ds| <= (D + 2) u scale sum|q k| + 4 u |s|   (products and sums, two scalings, the exponent's argument)
      p      off by a factor within 2 max|ds| + 2^-22 + 2^-8 (both maximum and score; exp; the rounding)
      sums   L u a term over the L keys
      range  an exponential below 2^-126, fp32's smallest normal number, may be taken as zero: at most
             2^-126 |v| a key, with l >= 1 (the key of the maximum)
      a denominator that sums the rounded probabilities: o' - o = sum p d (v - o) / l' with |d| <= 2^-8,
             so 2^-8 |o| beside the 2^-8 A of the numerator
    so |do| <= A (2^-8 + 2 (2 max|ds| + 2^-22 + L u)) + 2^-8 |o| with A = sum p |v| / l (the second
    summand twice: numerator and denominator) and L 2^-126 max|v| and 2^-8 |o|, and the last rounding's 2^-8 of what it rounds."""
    t, hq, d = q.shape
    hkv = codes.shape[2]
    nb = codes.shape[1]
    o, tol = np.zeros((t, hq, d)), np.zeros((t, hq, d))
    u = 2.0 ** -24
    for i in range(len(seq)):
        s0, s1 = int(starts[i]), int(starts[i + 1])
        length = int(seq[i])
        if s1 <= s0 or length <= 0:
            continue
        k, v = gather(codes, scales, table[i], length)
        here = np.repeat([0 <= int(p) < codes.shape[0] for p in table[i]], nb * BLOCK)[:length]
        for j in range(s0, s1):
            pos = length - (s1 - s0) + j - s0
            lo = max(0, pos + 1 - window) if window else 0
            see = np.arange(lo, max(pos + 1, lo))
            see = see[here[see]]
            if not see.size:
                continue
            for h in range(hq):
                kk, vv = k[h // (hq // hkv), see], v[h // (hq // hkv), see]
                s = kk @ q[j, h] * scale
                m = s.max() if not np.isnan(s).any() else np.nan
                low = m == -np.inf  # every score: weights of 0, which leave the sink, or 0 / 0
                p = np.zeros_like(s) if low else np.exp(s - m) if np.isfinite(m) else np.full_like(s, np.nan)
                den = p.sum() + (math.exp(sink[h] - (0.0 if low else m)) if sink is not None else 0.0)
                den = den if den else np.nan
                o[j, h] = p @ vv / den
                ds = float(np.max((d + 2) * u * abs(scale) * (np.abs(kk) @ np.abs(q[j, h])) + 4 * u * np.abs(s)))
                a = p @ np.abs(vv) / den
                tol[j, h] = a * (2.0 ** -8 + 2 * (2 * ds + 2.0 ** -22 + see.size * u))
                tol[j, h] += 2.0 ** -8 * np.abs(o[j, h])
                tol[j, h] += see.size * 2.0 ** -126 * np.abs(vv).max(0)
                tol[j, h] += 2.0 ** -8 * (np.abs(o[j, h]) + tol[j, h])
    return o, tol
