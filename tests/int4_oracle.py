"""Rows of a 4-bit cache, and what is done to logits, in 64 bits, from their formulas, on the host."""
import math

import numpy as np
import torch

GROUP = 32
BITS = {torch.float16: (11, -14), torch.bfloat16: (8, -126)}         # of a value, and the exponent of the smallest normal one
TOP = {torch.float16: 65504.0, torch.bfloat16: (2 - 2.0 ** -7) * 2.0 ** 127}
PLACE = [4 * (i // 2) + 16 * (i % 2) for i in range(8)]              # bit of each column in 32


def to_type(x, dtype, how=np.rint):
    """float64 numpy -> the numbers of dtype (as float64): to the nearest (ties to even), or `how`."""
    x = np.asarray(x, dtype=np.float64)
    bits, least = BITS[dtype]
    fine = np.isfinite(x)
    exponent = np.maximum(np.frexp(np.where(fine, x, 0.0))[1] - 1, least)
    unit = np.exp2(exponent.astype(np.float64) - (bits - 1))
    with np.errstate(over="ignore"):
        y = how(np.where(fine, x, 0.0) / unit) * unit
    y = np.where(np.abs(y) > TOP[dtype], np.copysign(np.inf, y), y)
    return np.where(fine, y, x)


def bits_of(x, dtype):
    """Numbers of dtype in float64 -> their 16 bits."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).view(torch.int16).numpy().view(np.uint16)


def encode(x, dtype):
    """Rows (..., dim) of numbers of dtype -> bytes (..., 5 dim / 8), uint8 torch."""
    v = x.double().numpy()
    v = v.reshape(*v.shape[:-1], -1, GROUP)
    with np.errstate(invalid="ignore"):
        low, high = v.min(-1, keepdims=True), v.max(-1, keepdims=True)
        good = np.isfinite(v).all(-1, keepdims=True)
        step = to_type(np.where(good, (high - low) / 15, 0.0), dtype, np.floor)
        some = step >= 2.0 ** -126
        code = np.where(good & some, np.minimum(np.rint((v - low) / np.where(some, step, 1.0)), 15.0), 0.0).astype(np.uint32)
    code = code.reshape(*v.shape[:-2], -1, 8)
    words = sum(code[..., i] << PLACE[i] for i in range(8)).astype("<u4")
    pair = np.concatenate([bits_of(step, dtype), bits_of(np.where(good, low, 0.0), dtype)], -1)
    pair = np.where(good, pair, 0x7fff).astype("<u2")
    lead = words.shape[:-1]
    return torch.from_numpy(np.concatenate([np.ascontiguousarray(words).view(np.uint8).reshape(*lead, -1),
                                            np.ascontiguousarray(pair.reshape(*lead, -1)).view(np.uint8).reshape(*lead, -1)], -1))


def pairs(rows, dtype):
    """Steps and lowest values (..., groups) float64 of rows of bytes."""
    n = rows.shape[-1] // 5 * 4
    meta = rows[..., n:].contiguous().view(dtype).double().numpy()
    return meta[..., 0::2], meta[..., 1::2]


def decode(rows, dtype):
    """Bytes (..., 5 dim / 8) -> the numbers of dtype that they stand for (..., dim), torch."""
    n = rows.shape[-1] // 5 * 4
    words = np.ascontiguousarray(rows[..., :n].contiguous().numpy()).view("<u4")
    code = np.stack([words >> s & 15 for s in PLACE], -1).reshape(*words.shape[:-1], -1, GROUP)
    step, low = pairs(rows, dtype)
    with np.errstate(invalid="ignore"):
        y = to_type(low[..., None] + step[..., None] * code, dtype)
    return torch.from_numpy(y.reshape(*words.shape[:-1], -1)).to(dtype)


def off_by(rows, dtype):
    """How far a row's values may be from what was written: half a step, and 15 times what rounding the step down may take off it (a step of the type below
    the step itself) at the upper end, with the rounding of what is read."""
    step, low = pairs(rows, dtype)
    eps = 2.0 ** (1 - BITS[dtype][0])
    least = 2.0 ** (BITS[dtype][1] - BITS[dtype][0] + 1)
    whole = step / 2 + 15 * (step * eps + least)
    return torch.from_numpy(np.repeat((whole + (np.abs(low) + 15 * step) * eps / 2 + least)[..., None], GROUP, -1).reshape(*step.shape[:-1], -1))


def adjust(logits, out_dtype, tokens=None, token_seq=None, token_lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None, bias_starts=None,
           bias_words=None, bias=None, temperature=None, mask=None, mask_row=None):
    """numpy float64 -> (out, how far 32-bit arithmetic and one rounding may be off).  Logits on the host; every other argument as a list or tensor."""
    z = logits.double().numpy().copy()
    r, v = z.shape
    unit = 2.0 ** -24
    off = np.zeros_like(z)
    with np.errstate(all="ignore"):
        for i in range(r):
            if tokens is not None:
                s = i if token_seq is None else int(token_seq[i])
                n = min(max(int(token_lens[i]), 0), tokens.shape[1]) if 0 <= s < tokens.shape[0] else 0
                words = tokens[s, :n].numpy() if n else np.zeros(0, np.int32)
                behind = words[max(0, 0 if prompt_lens is None else int(prompt_lens[i])):]
                words, behind = (w[(w >= 0) & (w < v)] for w in (words, behind))
                seen, count = np.unique(words), np.bincount(behind, minlength=v)
                rep, freq, pres = (d if x is None else float(x[i]) for x, d in ((repetition, 1.0), (frequency, 0.0), (presence, 0.0)))
                z[i, seen] = np.where(z[i, seen] > 0, z[i, seen] / rep, z[i, seen] * rep)
                off[i, seen] += unit * np.abs(z[i, seen])
                some = count > 0
                less = freq * count[some] + pres
                # a product, two differences
                off[i, some] += unit * (3 * (np.abs(freq * count[some]) + abs(pres)) + 2 * np.abs(z[i, some]))
                z[i, some] -= less
            if bias_starts is not None:
                for b in range(max(int(bias_starts[i]), 0), min(int(bias_starts[i + 1]), len(bias))):
                    w = int(bias_words[b])
                    if 0 <= w < v:
                        z[i, w] += float(bias[b])
                        off[i, w] += unit * np.abs(z[i, w]) * 2
            heat = 0.0 if temperature is None else float(temperature[i])
            if heat >= 2.0 ** -126:
                z[i] /= heat
                off[i] = off[i] / heat + 2.5 * unit * np.abs(z[i])   # the reciprocal's rounding and the product's
            m = -1 if mask is None else i if mask_row is None else int(mask_row[i])
            if mask is not None and 0 <= m < mask.shape[0]:
                word = np.arange(v)
                z[i, (mask[m].numpy().view(np.uint32)[word >> 5] >> (word & 31) & 1) == 0] = -math.inf
        eps = {torch.float32: 2.0 ** -23}.get(out_dtype) or 2.0 ** (1 - BITS[out_dtype][0])
        least = 2.0 ** -149 if out_dtype == torch.float32 else 2.0 ** (BITS[out_dtype][1] - BITS[out_dtype][0])
        top = TOP.get(out_dtype, (2 - 2.0 ** -23) * 2.0 ** 127)
        z = np.where(np.abs(z) > top * (1 + eps / 4), np.copysign(math.inf, z), z)   # beyond what the type holds, half a step of its largest number included
        return z, off * 1.01 + (np.abs(z) + off) * eps / 2 + least
