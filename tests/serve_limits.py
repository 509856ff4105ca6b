"""How near the outputs of attention come to the exact ones, as a root mean
square, and what they come to when softmax weights or queries keep fewer bits:
limits that hold the kernels to the bits they state, where a bound of summed
worst cases would let a term of a number go unnoticed.

The distance is taken from the exact outputs rounded to the output's type, so
that the type's own rounding, the largest part of a bf16 output's error, is
left out of it.

fp32 outputs.  With 24-bit weights, queries and sums the distance is a few 2^-24
(1.2e-7 to 5e-7).  Weights or queries of 16 bits are off by up to 2^-17, uniformly:
2^-17 / sqrt(3) = 4.4e-6 at the lower end of a binade, rms over many keys 5e-6 to
8e-6.  The limit stands between: 1.2e-6.

bf16 outputs.  An error far below the output's step (h = 2^-7 to 2^-8 of it) moves
an output by a whole step, with probability |error| / h: a distance of
sqrt(E|error| h).  Weights of 16 bits: sqrt(2.6e-6 * 5.6e-3) = 1.2e-4; terms cut off
instead of rounded, twice the error and of one sign, 2e-4.  Weights of 8 bits are
off by 2^-9 / sqrt(3) = 1.1e-3 and more, as much as half a step: with the step's
rounding 2.2e-3 to 2.8e-3, and with 7 bits 3.5e-3 and more.  Limits between: 7e-4
for 16 bits, 3.1e-3 for 8."""
import math

import numpy as np
import torch

LIMIT = {24: 1.2e-6, 16: 7e-4, 8: 3.1e-3}


def distance(got, want, dtype):
    """got, want: float64 arrays (want exact)."""
    near = torch.from_numpy(np.ascontiguousarray(want)).to(dtype).double().numpy()
    return math.sqrt(((got - near) ** 2).mean() / (want ** 2).mean())


def keep(x, bits):
    """x rounded to that many significant bits."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(np.ldexp(m, bits)), e - bits)


def attention(q, k, v, q_offsets, kv_lens, table, page, q_heads, window, sinks, scale, query_bits, weight_bits):
    """Attention of rows that all see a key, queries and weights (relative to the
    row's largest) held to so many bits, the weights' sum to all, else in 64."""
    out = np.empty(q.shape)
    q = keep(q, query_bits)
    for b in range(len(kv_lens)):
        n, have = q_offsets[b + 1] - q_offsets[b], kv_lens[b]
        j = np.arange(have)
        at = np.asarray(table[b])[j // page], j % page
        for i in range(n):
            p = have - n + i
            seen = (j <= p) & ((j > p - window) | (j < sinks))
            for h in range(q_heads):
                g = h // (q_heads // k.shape[1])
                s = scale * (k[at[0], g, at[1]][seen] @ q[q_offsets[b] + i, h])
                w = np.exp(s - s.max())
                out[q_offsets[b] + i, h] = keep(w, weight_bits) @ v[at[0], g, at[1]][seen] / w.sum()
    return out
