"""Plain forms in 64 bits of the operators between a decoder layer's projections, and the error bounds their tests use."""
import math

import numpy as np

import oracle

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # a rounding to the type, relative to the value
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}     # half a step of the type's smallest values
CODE = {"f16": 1, "bf16": 2, "f32": 3}


def narrow(x, t):
    """float array -> the bits (or floats) a buffer of type t holds, and their values in 64 bits."""
    x = np.ascontiguousarray(x, np.float32)
    if t == "f32":
        return x, x.astype(np.float64)
    if t == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float64)
    b = oracle.bf16_bits(x)
    return b, widen(b, t)


def widen(bits, t):
    if t == "bf16":
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return bits.astype(np.float64)


def buffer_type(t):
    return {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}[t]


# ------------------------------------------------------------------------------------------------ adapters
def adapters(X, slot, base, A, B, scale):
    """Y and a bound on a 32-bit evaluation's error: every sum of n terms is off by at most (n + 2) half steps of 2^-24 of the sum
    of its terms' magnitudes -- doubled, as the matrix unit's own order and truncation are not specified -- and a
    rounding of the result."""
    Y = base.copy()
    bound = np.abs(base) * 2.0 ** -22
    for m, s in enumerate(slot):
        if 0 <= s < len(A) and A[s] is not None and len(A[s]):
            a, b = A[s], B[s]
            h = a @ X[m]
            mag = np.abs(a) @ np.abs(X[m])
            Y[m] = base[m] + scale[s] * (b @ h)
            bound[m] += abs(scale[s]) * (np.abs(b) @ mag) * (X.shape[1] + a.shape[0] + 16) * 2.0 ** -23 + np.abs(base[m]) * a.shape[0] * 2.0 ** -22
    return Y, bound + 2.0 ** -140


# ------------------------------------------------------------------------------------------------ heads
def rotate_norm(x, pos, gain, eps, freq, interleaved, t):
    """x [T][heads][D] -> values and a bound: the norm's sum of D squares, its root and products, then two products and a sum with
    sines good to 2^-21, in 32 bits; one rounding to t."""
    T, H, D = x.shape
    y = x.copy()
    if gain is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * gain
    n = len(freq)
    mag = np.abs(y)
    if n:
        a_i, b_i = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
        ang = pos.astype(np.float64)[:, None] * np.asarray(freq)[None, :]
        c, s = np.cos(ang)[:, None, :], np.sin(ang)[:, None, :]
        a, b = y[..., a_i].copy(), y[..., b_i].copy()
        y[..., a_i], y[..., b_i] = a * c - b * s, b * c + a * s
        m = np.abs(a) + np.abs(b)
        mag[..., a_i] = mag[..., b_i] = m
    return y, np.abs(y) * HALF_STEP[t] + mag * (D + 24) * 2.0 ** -24 * 1.01 + mag * 2.0 ** -21 + TINY[t]


# ------------------------------------------------------------------------------------------------ attention
def attention(q, k, v, q_start, kv_start, kv_len, scale, t):
    """q [Tq][Hq][D], k and v [rows][Hkv][D] in 64 bits -> {row: (out [Hq][D], bound)} for the rows of the sequences.

    The bound, A = sum p |v| / sum p being an output's mean magnitude: p is rounded to t, p (1 + d), in the numerator and in the
    denominator, which moves o by sum p d (v - o) / sum p: half a step of sum p |v - o| / sum p;
    a score's 32-bit sum of D products and its scaling are off by (D + 8) 2^-23 of scale * sum |q||k|, which moves p by as
    much relatively, in the numerator and in the denominator; the exponential and the sums over n keys in 32 bits add (n + 64) 2^-23;
    fp16 loses p below 2^-32 of the largest, 2^-31 of sum |v| at most; the result is rounded once."""
    out = {}
    group = q.shape[1] // k.shape[1]
    for b in range(len(q_start) - 1):
        n, m, k0 = q_start[b + 1] - q_start[b], kv_len[b], kv_start[b]
        for i in range(n):
            seen = min(m, max(0, m - n + i + 1))
            o, e = np.zeros(q.shape[1:]), np.full(q.shape[1:], TINY[t])
            if seen:
                for h in range(q.shape[1]):
                    Q, K, V = q[q_start[b] + i, h], k[k0:k0 + seen, h // group], v[k0:k0 + seen, h // group]
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = (K @ Q) * scale
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        o[h] = p @ V
                        A, spread = p @ np.abs(V), p @ np.abs(V - o[h])
                        some = np.isfinite(s)
                        ds = scale * (np.abs(K[some]) @ np.abs(Q)).max(initial=0.0) * (q.shape[2] + 8) * 2.0 ** -23
                        e[h] = spread * HALF_STEP[t] * 1.01 + A * (2 * ds + (seen + 64) * 2.0 ** -23) + 2.0 ** -31 * np.abs(V).sum(0) * (t == "f16") + np.abs(o[h]) * HALF_STEP[t] + TINY[t]
            out[q_start[b] + i] = (o, e)
    return out


def frequencies(rotated, base=10000.0):
    return [base ** (-2.0 * j / rotated) for j in range(rotated // 2)]


def softmax_scale(dim):
    return 1.0 / math.sqrt(dim)
