"""Plain 64-bit forms of the key/value cache's operators (numpy): rotary
embedding, the Q4_0 / Q8_0 block rule (its 32-bit steps), and attention."""
import math

import numpy as np

YARN = dict(base=150000.0, factor=32.0, original_len=4096, beta_fast=32.0, beta_slow=1.0)


def rope_freqs(dim, base, factor=1.0, original_len=0, beta_fast=0.0, beta_slow=0.0):
    h = dim // 2
    i = np.arange(h)
    f = float(base) ** (-i / h)
    if factor <= 1:
        return f, 1.0
    lo, hi = (h * math.log(original_len / (b * 2 * math.pi)) / math.log(base) for b in (beta_fast, beta_slow))
    ramp = np.clip((i - lo) / (hi - lo), 0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1


def rotate(x, pos, rope):
    """x [rows][heads][dim] fp32 at positions pos [rows]: rounded once to fp32."""
    dim = x.shape[-1]
    f, m = rope_freqs(dim, **rope)
    a = np.asarray(pos, np.float64)[:, None, None] * f
    c, s = np.cos(a) * m, np.sin(a) * m
    u, v = x[..., :dim // 2].astype(np.float64), x[..., dim // 2:].astype(np.float64)
    with np.errstate(all="ignore"):
        return np.concatenate([u * c - v * s, v * c + u * s], -1).astype(np.float32)


def quantize(x, bits):
    """(codes, fp16 scales) of the blocks of 32 of x (fp32): GGML's rule, |d| capped."""
    b = np.ascontiguousarray(x, np.float32).reshape(-1, 32)
    f = np.float32
    with np.errstate(all="ignore"):
        if bits == 4:
            top = b[np.arange(len(b)), np.abs(b).argmax(1)]
            d = np.clip(top / f(-8), f(-8188), f(8188))
        else:
            d = np.minimum(np.abs(b).max(1) / f(127), f(515.5))
        r = np.where(d != 0, f(1) / np.where(d != 0, d, f(1)), f(0)).astype(f)
        t = b * r[:, None]
        if bits == 4:
            q = np.floor(t + f(8.5))
            q = np.where(np.isnan(q), 8, np.clip(q, 0, 15)) - 8
        else:
            q = np.trunc(t.astype(np.float64) + np.copysign(0.5, t))
            q = np.where(np.isnan(q), 0, np.clip(q, -127, 127))
    shape = x.shape[:-1] + (x.shape[-1] // 32,)
    return q.astype(np.int32).reshape(shape + (32,)), d.astype(np.float16).reshape(shape)


def stored(k, v, bits):
    """What a store of (rotated) k and v [rows][heads][dim] reads back as."""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    out = []
    for x, mark in ((k, np.nan), (v, 0.0)):
        q, d = quantize(np.where(bad[..., None], np.float32(0), x), bits)
        y = (q * d.astype(np.float32)[..., None]).reshape(x.shape).astype(np.float32)
        out.append(np.where(bad[..., None], np.float32(mark), y))
    return out


def attend(q, k, v, first, scale, window=0, sinks=None):
    """q [rows][heads][dim] at positions first, first + 1, .. over k, v
    [positions][kv_heads][dim] in 64 bits.  Returns (out, tol): tol bounds a
    computation whose products keep 2^-22, whose sums round to fp32.

    A score q . k over dim = D: q is off by at most 2^-22 of itself in each
    element, the smallest of the four partial products (2^-11 times 2^-11) is
    left out, and 3 D products are added, each sum off by half a step:
    (2 * 2^-22 + 3 D 2^-24) * sum |q_d k_d| * scale, and the exponential's
    argument (times log2 e, minus the maximum, two roundings) 2 * 2^-24 of its
    size, which is at most 2 sum |q_d k_d| scale.  The weights are off by that
    exponent's error (numerator and denominator: twice), by 2^-22 in their
    split and by the exponential's own 2^-22 twice; the sum over positions of
    weights times values adds rounding of 3 adds a position in groups of 32:
    at most 3 n 2^-24 of sum p |v| (and n 2^-24 in the denominator)."""
    rows, heads, dim = q.shape
    g = heads // k.shape[1]
    n = k.shape[0]
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, tol = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    for i in range(rows):
        pos = first + i
        lo = max(0, pos - window + 1) if window else 0
        hi = min(n, pos + 1)
        if hi <= lo:
            continue
        for h in range(heads):
            kk, vv = k[lo:hi, h // g], v[lo:hi, h // g]
            with np.errstate(all="ignore"):
                s = kk @ q[i, h] * scale
                size = float(np.nan_to_num((np.abs(kk) @ np.abs(q[i, h])).max()) * scale)
                top = s.max()
                if sinks is not None:
                    top = max(top, sinks[h])
                p = np.exp(s - top)
                den = p.sum() + (math.exp(sinks[h] - top) if sinks is not None else 0.0)
                out[i, h] = p @ vv / den
                mass = p @ np.abs(vv) / den
            c = 2 * size * (2 * 2.0 ** -22 + 3 * dim * 2.0 ** -24 + 4 * 2.0 ** -24) + 6 * 2.0 ** -22 + 4 * (hi - lo) * 2.0 ** -24
            tol[i, h] = c * mass + 2.0 ** -24 * np.abs(out[i, h])
    return out, tol
