"""Rotation on several axes with the paged append, paged attention and draft verification in 64 bits, from their formulas, on the host."""
import math

import numpy as np
import torch

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}         # torch.finfo(t).eps


def half_step(y, dtype):
    """The most that rounding y to dtype moves it: half of eps relative to the value, half of the smallest step below the normal numbers."""
    return y.abs() * (EPS[dtype] / 2) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def axes_rope(qkv, pos, inv_freq, axis, heads, kv_heads, dim, adjacent, mscale):
    """-> q, k, v (T, heads, dim) float64 and how far 32-bit arithmetic and one rounding may leave q and k from them."""
    t, half = qkv.shape[0], len(inv_freq)
    x = qkv.double().view(t, heads + 2 * kv_heads, dim)
    angle = torch.zeros(t, half, dtype=torch.float64)
    for i in range(half):
        if 0 <= int(axis[i]) < pos.shape[0]:
            angle[:, i] = pos[int(axis[i])].double() * float(inv_freq[i])
    c, s = angle.cos()[:, None] * mscale, angle.sin()[:, None] * mscale
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if adjacent else (slice(0, half), slice(half, 2 * half))
    y, off = x.clone(), torch.zeros_like(x)
    n = heads + kv_heads
    a, b = x[:, :n, first], x[:, :n, second]
    y[:, :n, first], y[:, :n, second] = a * c - b * s, b * c + a * s
    # a reduced angle of at most pi rounded to 32 bits (1e-7), its sine and cosine to two units (2.4e-7), times mscale, two products and a sum (2^-24 each)
    slack = (a.abs() + b.abs()) * mscale * (1e-7 + 2.4e-7 + 4 * 2.0 ** -24)
    off[:, :n, first], off[:, :n, second] = slack, slack
    off = off + half_step(y.abs() + off, qkv.dtype)
    off[:, :n, 2 * half:] = 0.0
    off[:, n:] = 0.0
    return y[:, :heads], y[:, heads:n], y[:, n:], off[:, :heads], off[:, heads:n]


def rows_of(cache, table, b, n):
    """Rows 0 .. n - 1 of sequence b (n, kv_heads, dim) float64; zeros behind a page number outside the pool."""
    pages, size = cache.shape[:2]
    out = torch.zeros(n, *cache.shape[2:], dtype=torch.float64)
    for i in range(0, n, size):
        page = int(table[b, i // size]) if i // size < table.shape[1] else -1
        m = min(size, n - i)
        if 0 <= page < pages:
            out[i:i + m] = cache[page, :m].double()
    return out


def attention(q, k_cache, v_cache, table, lens, starts, scale, window):
    """q (T, heads, dim) on the host -> (out float64, how far the kernels may be off; rows of no sequence: NaN)."""
    t, heads, dim = q.shape
    hk, dtype = k_cache.shape[2], q.dtype
    out = torch.full((t, heads, dim), math.nan, dtype=torch.float64)
    off = torch.zeros_like(out)
    room = table.shape[1] * k_cache.shape[1]
    for b in range(len(lens)):
        lo, hi, n = int(starts[b]), int(starts[b + 1]), int(lens[b])
        if lo == hi:
            continue
        have = max(0, min(n, room))
        k, v = rows_of(k_cache, table, b, have), rows_of(v_cache, table, b, have)
        at = torch.arange(n - (hi - lo), n)
        j = torch.arange(have)
        seen = j[None] <= at[:, None]
        if window:
            seen &= j[None] > at[:, None] - window
        for h in range(heads):
            kk, vv = k[:, h // (heads // hk)], v[:, h // (heads // hk)]
            x = q[lo:hi, h].double()
            s = torch.where(seen, x @ torch.nan_to_num(kk.T, 0, 0, 0) * scale, -math.inf)
            top = s.amax(1, keepdim=True) if have else torch.zeros(hi - lo, 1)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            vz = torch.nan_to_num(vv, 0, 0, 0)
            o, spread = p @ vz, p @ vz.abs()
            # Each score's 32-bit sum of dim products and the exponent's own arithmetic move it by up to `lean`, so quotients by twice that; sums over the
            # keys and the join of their parts add a unit for each key at the most; probabilities are rounded to the type once, the result once.
            size = torch.where(seen, x.abs() @ torch.nan_to_num(kk.T, 0, 0, 0).abs() * scale, 0.0).amax(1, keepdim=True) if have else torch.zeros(hi - lo, 1)
            lean = size * (dim + 8) * 2.0 ** -24 + 2.0 ** -21
            err = spread * (EPS[dtype] / 2 + 2 * lean + 2 * (have + 64) * 2.0 ** -24)
            out[lo:hi, h], off[lo:hi, h] = o, err + half_step(o.abs() + err, dtype)
    return out, off


def verify(target, draft, drafted, accept, sample, count):
    """numpy in 64 bits, one sequence at a time."""
    target = np.asarray(target, dtype=np.float64)
    draft = None if draft is None else np.asarray(draft, dtype=np.float64)
    b, k1, vocab = target.shape
    k = k1 - 1
    accepted, tokens = np.zeros(b, np.int32), np.full((b, k + 1), -1, np.int32)
    for i in range(b):
        n = k if count is None else min(max(int(count[i]), 0), k)
        taken = 0
        while taken < n:
            x = int(drafted[i, taken])
            if not 0 <= x < vocab or not float(accept[i, taken]) * (1.0 if draft is None else draft[i, taken, x]) < target[i, taken, x]:
                break
            tokens[i, taken] = x
            taken += 1
        row = target[i, taken].copy()
        rest = row.copy()
        if taken < n:
            if draft is not None:
                rest -= draft[i, taken]
            elif 0 <= int(drafted[i, taken]) < vocab:
                rest[int(drafted[i, taken])] -= 1.0
        clean = lambda w: np.where((w > 0) & np.isfinite(w), w, 0.0)  # noqa: E731
        rest = clean(rest)
        if not rest.sum() > 0:
            rest = clean(row)
        accepted[i] = taken
        if rest.sum() > 0:
            total = np.cumsum(rest)
            past = np.nonzero((total > float(sample[i]) * total[-1]) & (rest > 0))[0]
            tokens[i, taken] = past[0] if len(past) else np.nonzero(rest)[0][-1]
    return accepted, tokens
