"""Plain implementations of the serving operators in 64 bits, on the CPU, from
their formulas alone, and the bounds that a computation in the kernels' number
formats keeps."""
import math

import numpy as np
import torch

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx_encode(x):
    """Blocks of 32 along the last axis of fp32 values: (codes packed two to a
    byte, scale bytes).  Nearest of the eight magnitudes, ties to the even
    code; the smallest power of two with the largest magnitude at 6 or below."""
    x = np.asarray(x, np.float32).astype(np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    byte = np.empty(top.shape, np.int64)
    for i in np.ndindex(top.shape):
        t = top[i]
        if not np.isfinite(b[i]).all():
            byte[i] = 255
            continue
        e = -126
        if t > 0:
            e = max(-126, math.frexp(t)[1] - 5)
            while t > math.ldexp(6.0, e):
                e += 1
        byte[i] = e + 127
    with np.errstate(all="ignore"):
        y = b / np.exp2((byte - 127).astype(np.float64))[..., None]
        dist = np.abs(np.abs(y)[..., None] - MAGNITUDES)
        code = np.argmin(dist + 1e-9 * (np.arange(8) % 2), -1)   # of two equally near the even code
    code = np.where(np.signbit(y), code + 8, code).reshape(x.shape)
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), byte.astype(np.uint8)


def mx_values(codes, scales):
    """float64 values of packed codes and scale bytes (255: NaN)."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)
    val = MAGNITUDES[c & 7] * np.where(c >= 8, -1.0, 1.0)
    s = np.exp2(scales.astype(np.float64) - 127)
    s[scales == 255] = np.nan
    return val * np.repeat(s, 32, -1)


def rotate(x, positions, cos, sin):
    """x [rows, heads, dim] float64 -> fp32 values, positions outside the table unrotated."""
    half = x.shape[-1] // 2
    out = x.copy()
    for r, p in enumerate(positions):
        if 0 <= p < cos.shape[0]:
            c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
            out[r, :, :half] = x[r, :, :half] * c - x[r, :, half:] * s
            out[r, :, half:] = x[r, :, :half] * s + x[r, :, half:] * c
    return out.astype(np.float32)


def attention(q, k, v, q_offsets, kv_lens, table, page, q_heads, window, sinks, scale, num_pages):
    """q [rows, q_heads, dim], k and v [pages, kv_heads, page, dim] in float64
    -> (out, bound on sum_j w_j |v_j|, bound on the scores' products
    scale sum |q k|, keys seen), by row.  Rows that no sequence names are NaN."""
    rows, _, dim = q.shape
    group = q_heads // k.shape[1]
    out = np.full((rows, q_heads, dim), np.nan)
    mag, prod = np.zeros_like(out), np.zeros((rows, q_heads))
    seen = np.zeros(rows, np.int64)
    for b in range(len(kv_lens)):
        n = q_offsets[b + 1] - q_offsets[b]
        for i in range(n):
            r, p = q_offsets[b] + i, kv_lens[b] - n + i
            keys = [j for j in range(p + 1) if (j > p - window or j < sinks) and 0 <= table[b][j // page] < num_pages]
            seen[r] = len(keys)
            out[r] = 0.0
            if not keys:
                continue
            at = np.array([table[b][j // page] for j in keys]), np.array([j % page for j in keys])
            for h in range(q_heads):
                kk, vv = k[at[0], h // group, at[1]], v[at[0], h // group, at[1]]
                s = scale * (kk @ q[r, h])
                prod[r, h] = scale * (np.abs(kk) @ np.abs(q[r, h])).max()
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h] = w @ vv
                mag[r, h] = w @ np.abs(vv)
    return out, mag, prod, seen


def attention_bound(out, mag, prod, seen, dim, out_dtype, weight_bits):
    """How far an output may be from the exact one.  Unit steps u = 2^-24.
    Scores: exact products (three bf16 terms or fp32), at most 3 dim + 3 sums,
    the scaling and the base's change: (3 dim + 8) u prod each, taken twice (a
    key's own and the maximum's); exp2 within 2^-22.  Weights: rounded to
    weight_bits.  Sums over the keys: n u for the products and for the weights'
    total, and for the joins of parts at most 70 more steps each.  The result
    is rounded once to its type."""
    u = 2.0 ** -24
    weight = 2 * (3 * dim + 8) * u * prod + 2.0 ** -22 + 2.0 ** -weight_bits
    rel = 2 * weight[..., None] + 2 * (seen[:, None, None] + 70) * u
    eps = torch.finfo(out_dtype).eps / 2
    return mag * rel * (1 + eps) + eps * np.abs(out) + 1e-30


def logits(x, row, hist, plen, rep, freq, pres, bias, allowed):
    """One row of fp32 logits, every step rounded to fp32.  bias: {id: value}."""
    f = np.float32
    out = x.astype(np.float32).copy()
    seen, count = {}, {}
    for i, t in enumerate(hist):
        if 0 <= t < x.size:
            seen[t] = True
            if i >= plen:
                count[t] = count.get(t, 0) + 1
    with np.errstate(all="ignore"):
        for t in seen:
            out[t] = f(out[t] / f(rep)) if out[t] > 0 else f(out[t] * f(rep))
        for t, c in count.items():
            out[t] = f(f(out[t] - f(f(freq) * f(c))) - f(pres))
        for t, b in bias.items():
            if 0 <= t < x.size:
                out[t] = f(out[t] + f(b))
    if allowed is not None:
        out[~allowed] = -np.inf
    return out
