"""Plain implementations in 64 bits, on the CPU and from their formulas alone,
of a decode step's operators around the cache, with the bounds that the kernels'
number formats keep."""
import numpy as np

EPS32 = 2.0 ** -24   # half a step of fp32, relative
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def rope(x, positions, freq, dim, layout, amplitude=1.0, inverse=False):
    """x [rows, heads * dim] float64 -> (turned values, bound of an fp32 result).

    The sines carry the rounding of an angle of at most pi / 4 (2.5 half steps of
    it: to fp32, times pi / 2), of their last steps (2) and of the amplitude (2):
    6 half steps; the two products and the sum add 2.  The 64-bit angle is off by
    some 2^-51 of itself on either side."""
    rows = x.shape[0]
    half = len(freq)
    out = x.reshape(rows, -1, dim).copy()
    bound = np.zeros_like(out)
    a = out.copy()
    i0, i1 = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2),
                                                                              slice(1, 2 * half, 2))
    live = positions >= 0
    angle = positions.astype(np.float64)[:, None] * freq
    c, s = np.cos(angle)[:, None] * amplitude, np.sin(angle)[:, None] * amplitude * (-1 if inverse else 1)
    y0, y1 = a[..., i0] * c - a[..., i1] * s, a[..., i0] * s + a[..., i1] * c
    off = (np.abs(a[..., i0]) + np.abs(a[..., i1])) * abs(amplitude) * (8 * EPS32 + np.abs(angle)[:, None] * 2.0 ** -50)
    out[live, :, i0], out[live, :, i1] = y0[live], y1[live]
    bound[live, :, i0], bound[live, :, i1] = off[live], off[live]
    return out.reshape(rows, -1), bound.reshape(rows, -1)


def q4_values(codes, scales, zeros):
    """float64 weight [out, in] of packed codes, float64 scales and zeros (None: 8)."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).astype(np.float64)
    group = c.shape[1] // scales.shape[1]
    z = np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64)
    return (c - np.repeat(z, group, 1)) * np.repeat(scales, group, 1)


def linear_q4(x, codes, scales, zeros, bias):
    """float64 x [rows, in] -> (y, bound of an fp32 result).

    Within a group the products x (1 + c / 16) and x are exact and their sums take
    a step (2^-23: a sum may cut) for each of the group's inputs, of at most the
    sum of magnitudes; then three roundings, and one for each group and each of up
    to 16 waves (three terms each) that are joined, and the bias."""
    w = q4_values(codes, scales, zeros)
    group, groups = w.shape[1] // scales.shape[1], scales.shape[1]
    ax = np.abs(x).reshape(x.shape[0], groups, group).sum(-1)             # [rows, groups]
    z = np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64)
    per = 16 * np.abs(scales) * (2 + 1 + z / 16)
    y = x @ w.T
    bound = (3 * group + 8) * 2 * EPS32 * (ax @ per.T) + (groups + 64) * EPS32 * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias
        bound = bound + 2 * EPS32 * (np.abs(y) + np.abs(bias))
    return y, bound


def quantise_q4(w, group, with_zeros, scales_bf16):
    """fp32 w -> (codes [out, in] unpacked, scales fp32, zeros or None), each step
    rounded to fp32 as the interface says."""
    f = np.float32
    g = w.astype(f).reshape(w.shape[0], -1, group)
    lo, hi = np.minimum(g.min(-1), 0).astype(f), np.maximum(g.max(-1), 0).astype(f)
    s = (hi / f(15) - lo / f(15)).astype(f) if with_zeros else (np.maximum(hi, -lo) / f(7)).astype(f)
    if scales_bf16:
        b = s.view(np.uint32).astype(np.uint64)
        s = (((b + 0x7FFF + ((b >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(f)
    s = np.where(s == 0, f(1), s)
    z = np.clip(np.rint((-lo / s).astype(f)), 0, 15) if with_zeros else np.full(s.shape, 8.0, f)
    c = np.clip(np.rint((g / s[..., None]).astype(f)) + z[..., None], 0, 15)
    return c.astype(np.uint8).reshape(w.shape), s, z.astype(np.uint8) if with_zeros else None


def logprobs(x, tokens, top):
    """float64 logits [rows, vocab], tokens [rows, n] -> dict of values and bounds.

    Under the row's probabilities p and distances d = max - x: the exponent of a
    term carries 2 half steps of d and the exponential 2 more, a sum of up to 2^17
    terms in a tree of at most 100 steps on the way 100; the logarithm 4 of
    itself; a result the roundings of x - max and of itself."""
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        m = x.max(1)
        base = np.where(np.isfinite(m), m, 0.0)[:, None]
        d = base - x
        e = np.exp(-d)
        S = e.sum(1)
        dd = np.where(e > 0, d, 0.0)
        W = (e * dd).sum(1)
        empty = np.isneginf(x).all(1)
        mean = W / S
        logS = np.where(empty, 0.0, np.log(S))
        entropy = np.where(empty, 0.0, logS + mean)
        t_lse = EPS32 * (2 * mean + 104 + 4 * np.abs(logS))
        t_ent = t_lse + EPS32 * ((e * dd * (2 * dd + 104)).sum(1) / S + mean * (2 * mean + 104) + 2 * entropy)
        order = np.where(np.isnan(x), -np.inf, x)
        ids = np.argsort(-order, axis=1, kind="stable")[:, :top]
        bad = np.isnan(x).any(1) | np.isposinf(x).any(1)

        def of(at):
            v = np.take_along_axis(x, at, 1) - base - logS[:, None]
            v[bad] = np.nan
            tol = t_lse[:, None] + 2 * EPS32 * (np.abs(np.take_along_axis(d, at, 1)) + np.abs(v))
            return v, tol

        lp, lp_tol = of(np.clip(tokens, 0, vocab - 1))
        outside = (tokens < 0) | (tokens >= vocab)
        lp, lp_tol = np.where(outside, 0.0, lp), np.where(outside, 0.0, lp_tol)
        top_lp, top_tol = of(ids)
        entropy = np.where(bad, np.nan, entropy)
    return {"logprobs": lp, "logprobs_tol": lp_tol, "entropy": entropy, "entropy_tol": np.where(empty, 0.0, t_ent),
            "top_ids": ids, "top_logprobs": top_lp, "top_logprobs_tol": top_tol}


def assert_within(got, want, bound, what=""):
    got, want, bound = (np.asarray(a, np.float64) for a in (got, want, bound))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(all="ignore"):
        ok = same | (np.isfinite(want) & (np.abs(got - want) <= bound))
    if not ok.all():
        i = tuple(np.argwhere(~ok)[0])
        raise AssertionError(f"{what}: {np.count_nonzero(~ok)} of {ok.size} off, first at {i}: {got[i]!r} for "
                             f"{want[i]!r}, bound {bound[i]!r}")
