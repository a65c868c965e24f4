"""Inputs and a bound that read single softmax weights out of the windowed prefill (harness code, not product
code).

tests/bounded_ref.py holds the windowed prefill to the allowance of the plain one, whose scores are f16 and whose
exponentials are f16x2; the windowed kernel has f32 scores and exponentials and rounds once, each numerator
to f16 for the PV product. Here

- q and k are multiples of 1/4 up to 2, so a score q.k is a multiple of 1/16 up to 512: every partial sum is exact
  in f32 whatever its order, and the score error is zero;
- key i has a value in dim i % 128 only, so output dim d of a row that sees at most 128 consecutive keys (and no
  sinks) is one weight times one value: p_i v_i.

Then for the weight p_i = 2^x_i / l (x in log2 units below the running maximum, which lies at most 8 under
the true one, so some numerator is at least 1 and l >= 1; A = sum_i p_i |v_i|, V = sum_i |v_i| in the dim)

    |out - exact| <= (2^-11 + 2^-15 + N 2^-22) A + 2^-25 V     (+ 2^-8 |exact| for a bf16 output)

2^-11: half a step of the numerator's f16; 2^-25: the same below f16's normal range. 2^-15: scale * log2(e) in
f32 and the product's rounding, (2^-23 + 2^-24) ln 2 |x| <= 2^-17 for |x| <= 64 (a smaller weight is below 2^-25 as it
is), in the weight and in the sum; ex2.approx 2^-22; the f32 row sum's order, at most 32 additions per key tile
and thread 2^-19; rescaling, reciprocal and product 2^-21; the log-sum-exp join of split runs, 2^-24 |lse| + 2^-22
<= 2^-18. N: the tensor core's additions of 16 keys each, every one of which may truncate the sum so far.
"""
from __future__ import annotations

import numpy as np

SCALE = np.float32(1.0 / np.sqrt(128.0))


def quarters(rng, shape):
    return (rng.integers(-8, 9, shape) / 4.0).astype(np.float32)


def one_dim_values(rng, n_keys, n_head_kv):
    """v [n_keys][n_head_kv][128]: key i has a value of 1 to 2 in dim i % 128."""
    v = np.zeros((n_keys, n_head_kv, 128), np.float32)
    v[np.arange(n_keys), :, np.arange(n_keys) % 128] = 1.0 + rng.integers(0, 1024, (n_keys, n_head_kv)) / 1024.0
    return v


def reference(q, k, v, seen, scale):
    """Exact outputs and bounds of one sequence: q [T][Hq][128], k / v [S][Hkv][128], seen [T][S]."""
    T, Hq, _ = q.shape
    G = Hq // k.shape[1]
    out, tol = np.zeros((T, Hq, 128)), np.zeros((T, Hq, 128))
    cols = np.flatnonzero(seen.any(0))
    s = seen[:, cols]
    some = s.any(1)
    steps = (s.sum(1, keepdims=True) + 2 * 128) / 16.0 + 1.0
    for h in range(Hq):
        kk, vv = k[cols, h // G].astype(np.float64), np.abs(v[cols, h // G].astype(np.float64))
        x = np.where(s, q[:, h].astype(np.float64) @ kk.T * float(scale), -np.inf)
        m = np.where(some, x.max(1, initial=-np.inf), 0.0)[:, None]
        e = np.exp(x - m)
        p = e / np.where(some, e.sum(1), 1.0)[:, None]
        a = p @ vv  # the values are positive
        out[:, h] = a
        tol[:, h] = (2.0 ** -11 + 2.0 ** -15 + steps * 2.0 ** -22) * a + 2.0 ** -25 * (s @ vv)
    return out, tol


def restated(q, k, v, seen, scale, f16_scores):
    """The kernel's arithmetic for rows of one pass (f32 scores, numerators rounded to f16, f32 sums), or the
    same with the scores below the maximum rounded to f16 first (a loss that the bound has to see)."""
    T, Hq, _ = q.shape
    G = Hq // k.shape[1]
    c = np.float32(np.float32(scale) * np.float32(1.4426950408889634))
    out = np.zeros((T, Hq, 128))
    for h in range(Hq):
        s = q[:, h] @ k[:, h // G].T  # exact in f32
        s = np.where(seen, s, np.float32(-np.inf))
        mu = (s.max(1, keepdims=True) * c).astype(np.float32)
        x = (s.astype(np.float64) * c - mu).astype(np.float32)  # one fused multiply-add
        if f16_scores:
            x = x.astype(np.float16).astype(np.float32)
        e = np.exp2(x).astype(np.float32)
        out[:, h] = (e.astype(np.float16).astype(np.float32) @ v[:, h // G]) / e.sum(1, keepdims=True, dtype=np.float32)
    return out
