"""Plain 64-bit restatement of the attention core (include/cpq.h: cpq_rope_*, cpq_kv_*,
cpq_paged_attn) in numpy, for tests: loops over requests, pages and heads, no tricks.

The cache is codes as numbers (float64 [pages, heads, block, D]) and float32 scales
[pages, heads]; rotary scaling follows ggml_rope_ext (YaRN paper's ramp over pairs)."""
from __future__ import annotations

import math

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}
MIN_SCALE = 2.0 ** -100


def rope_frequencies(n_dims, base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0,
                     beta_slow=1.0, n_ctx_orig=0, freq_factors=None):
    """Radians per position of each pair, and the magnitude."""
    w, m = [], attn_factor
    if ext_factor:
        pair = lambda beta: n_dims * math.log(n_ctx_orig / (beta * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(0.0, math.floor(pair(beta_fast))), min(n_dims - 1.0, math.ceil(pair(beta_slow)))
        m *= 1.0 + 0.1 * math.log(1.0 / freq_scale)
    for i in range(n_dims // 2):
        f = base ** (-2.0 * i / n_dims)
        if freq_factors is not None:
            f /= freq_factors[i]
        mix = ext_factor * (1.0 - min(1.0, max(0.0, (i - low) / max(0.001, high - low)))) if ext_factor else 0.0
        w.append(f * freq_scale * (1.0 - mix) + f * mix)
    return np.array(w), m


def rope(x, pos, n_dims, half, **params):
    """x [T, heads, D] float64 rotated to pos [T]."""
    w, m = rope_frequencies(n_dims, **params)
    turns = np.array([[(int(p) * float(f)) % (2 * math.pi) for f in w] for p in pos])
    c, s = (m * np.cos(turns))[:, None, :], (m * np.sin(turns))[:, None, :]
    y = x.copy()
    h = n_dims // 2
    a, b = (slice(0, h), slice(h, n_dims)) if half else (slice(0, n_dims, 2), slice(1, n_dims, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def kv_slots(ctx, new, table, free, taken, block, n_rows):
    """The outputs of cpq_kv_slots as a dict; table is changed in place."""
    n, width = table.shape
    start, at = [], 0
    pos, slot = np.zeros(n_rows, np.int32), np.full(n_rows, -1, np.int64)
    kv_len = np.zeros(n, np.int32)
    given, asked = 0, 0
    for r in range(n):
        c, a = int(ctx[r]), int(new[r])
        start.append(min(at, n_rows))
        good = c >= 0 and a >= 0 and -(-(c + a) // block) <= width
        need = -(-(c + a) // block) - -(-c // block) if good else 0
        first, asked = asked, asked + need
        rows = max(a, 0)
        if good and (need == 0 or asked <= len(free) - taken) and at + rows <= n_rows:
            held = -(-c // block)
            for j in range(need):
                table[r, held + j] = free[taken + first + j]
            if need:
                given = max(given, asked)
            kv_len[r] = c + a
            for i in range(rows):
                p = c + i
                pos[at + i] = p
                if table[r, p // block] >= 0:
                    slot[at + i] = int(table[r, p // block]) * block + p % block
        at += rows
    start.append(min(at, n_rows))
    return {"seq_start": np.array(start, np.int32), "kv_len": kv_len, "pos": pos, "slot": slot, "taken": taken + given}


def code_values(fmt):
    """Every number a code stands for, ascending, and whether its pattern is even."""
    if fmt == "int8":
        v = np.arange(-127, 128, dtype=np.float64)
        return v, v % 2 == 0
    mags = [j / 8 * 2.0 ** -6 for j in range(8)] + [(1 + j / 8) * 2.0 ** e for e in range(-6, 9) for j in range(8)]
    mags = np.array(mags[:-1])
    even = np.arange(len(mags)) % 2 == 0
    return np.concatenate([-mags[:0:-1], mags]), np.concatenate([even[:0:-1], even])


def nearest_code(y, fmt):
    """The code value nearest to y (float64), ties to the even pattern; NaN to 0."""
    v, even = code_values(fmt)
    y = np.nan_to_num(np.asarray(y, np.float64), nan=0.0, posinf=v[-1], neginf=v[0])
    border = (v[1:] + v[:-1]) / 2
    i = np.searchsorted(border, y, side="left")
    tie = (i < len(border)) & (border[np.minimum(i, len(border) - 1)] == y) & ~even[i]
    return v[i + tie]


def kv_append(codes, scale, x, slot, fmt):
    """Writes rows x [T, heads, D] into codes/scale in place (one of K, V)."""
    pages, heads, block, _ = codes.shape
    t = 0
    while t < len(slot):
        s = int(slot[t])
        if s < 0 or s >= pages * block:
            t += 1
            continue
        page, off = divmod(s, block)
        n = 1
        while t + n < len(slot) and off + n < block and slot[t + n] == s + n:
            n += 1
        for h in range(heads):
            part = np.asarray(x[t:t + n, h], np.float64)
            mag = np.abs(part)
            top = mag[np.isfinite(mag)].max(initial=0.0)
            new = np.float32(top / TOP[fmt])
            if new < MIN_SCALE:
                new = np.float32(0)
            if off:
                old = scale[page, h]
                new = max(new, old)
                if new != old:
                    codes[page, h, :off] = nearest_code(codes[page, h, :off] * np.float64(old) / np.float64(new), fmt)
            with np.errstate(all="ignore"):
                codes[page, h, off:off + n] = nearest_code(part / np.float64(new), fmt) if new > 0 else 0.0
            scale[page, h] = new
        t += n


def attention(q, k, v, scale, causal):
    """One sequence, one query head: q [n, D] against k, v [m, D]; (out, lse, sum of |terms| of the largest score)."""
    n, m = len(q), len(k)
    out, lse, size = np.zeros((n, v.shape[1])), np.full(n, -np.inf), 0.0
    for i in range(n):
        seen = min(max(m - n + i + 1, 0), m) if causal else m
        if seen == 0:
            continue
        z = scale * (k[:seen] @ q[i])
        size = max(size, float((abs(scale) * (np.abs(k[:seen]) @ np.abs(q[i]))).max()))
        top = z.max()
        p = np.exp(z - top)
        lse[i] = top + math.log(p.sum())
        out[i] = p @ v[:seen] / p.sum()
    return out, lse, size


def paged_attn(q, k_vals, v_vals, table, seq_start, kv_len, scale, causal):
    """q [T, heads, D] over a cache of values [pages, kv heads, block, D]; returns (out, lse, size) with NaN in
    rows that belong to no sequence."""
    t, hq, d = q.shape
    pages, hkv, block, _ = k_vals.shape
    group = hq // hkv
    out, lse, size = np.full(q.shape, np.nan), np.full((t, hq), np.nan), 0.0
    for s in range(len(kv_len)):
        a, b = int(seq_start[s]), int(seq_start[s + 1])
        kv = max(int(kv_len[s]), 0)
        m = min(kv, table.shape[1] * block)  # keys behind the table's blocks are not seen
        ids = [int(table[s, j // block]) for j in range(m)]
        places = [j % block for j in range(m)]
        there = np.array([0 <= i < pages for i in ids], bool)
        for h in range(hkv):
            for g in range(group):
                qs = q[a:b, h * group + g]
                for i in range(b - a):
                    seen = min(max(kv - (b - a) + i + 1, 0), m) if causal else m
                    idx = [j for j in range(seen) if there[j]]
                    ks = np.array([k_vals[ids[j], h, places[j]] for j in idx]).reshape(len(idx), d)
                    vs = np.array([v_vals[ids[j], h, places[j]] for j in idx]).reshape(len(idx), d)
                    o, l, z = attention(qs[i:i + 1], ks, vs, scale, False)
                    out[a + i, h * group + g], lse[a + i, h * group + g], size = o[0], l[0], max(size, z)
    return out, lse, size
