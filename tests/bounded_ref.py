"""f64 restatements of the bounded-cache operators, the error bounds their kernels are held to, and
the inputs the tests share (harness code, not product code).

Bounds. The split kernel computes a score as an f32 sum of 128 exact f16 products (at most
128 * 2^-24 of sum_d |q_d k_d|, each way), takes ex2.approx of a score in log2 units (relative 2^-22,
plus the rounding of a product of magnitude <= 64: 64 * 2^-24), rounds the probability to f16
for the V product (half a step: 2^-11, or 2^-25 absolute below f16's normal range, and no probability
exceeds 1 against a softmax sum of at least 1), and sums in f32. With E the score error in natural
units, A = sum_i p_i |v_i| and V = sum_i |v_i| over the visible keys:

    |out - exact| <= (2^-11 + 2 E + 2^-16) A + 2^-25 V     (+ 2^-8 |exact| for a bf16 output)
    |lse - exact| <= E + 2^-16 + 2^-22 |exact|
    |w - exact|   <= (2 E + 2^-16) w                         per softmax weight w

2^-16 covers ex2.approx, the scores' rounding in log2 units, the f32 sums (at most 2^15 keys, whose
pairwise and split partial sums stay far below 2^-17) and the log-sum-exp merges. The q8_0 decode
computes exact integer dots scaled in f32, so E there is 16 * 2^-24 of the same magnitude, and
rounds P * d_v to f16: the same relative bound, and 2^-25 * 127 absolute per key.

The prefill multiplies on the tensor cores (a product sum may truncate: 2^-23 in E), rounds the scores
less the running maximum (log2 units, at most 8 above zero, as far below as the key lies under the
row's maximum) to f16 - ln 2 * 2^-11 * |x| of the probability - and takes ex2.approx.f16x2 of them
(relative 2^-9.9); the row sum adds the same rounded probabilities, so with d_i the sum of these

    |out - exact| <= sum_i p_i d_i (|v_i| + |out|) + 2^-25 sum_i (|v_i| + |out|)

The windowed prefill takes its exponentials of f32 scores and in f32, which these bounds cover.
"""
from __future__ import annotations

import numpy as np
import torch

from tests.helpers import random_cache, random_q, scattered_block_tables

SCALE = 1.0 / np.sqrt(128.0)


def f16(a):
    """f16 values of a bit array, on the GPU."""
    return torch.from_numpy(a.view(np.int16)).cuda().view(torch.float16)


def vals(a):
    return np.asarray(a).view(np.float16).astype(np.float64)


def window_mask(positions, n_keys, window, n_sink):
    """[T][S] visibility for queries at `positions` over keys 0..n_keys-1."""
    at = np.asarray(positions, np.int64)[:, None]
    key = np.arange(n_keys, dtype=np.int64)[None]
    return (key <= at) & ((key > at - window) | (key < n_sink))


def quantise_q8(x, product=False):
    """(integers, f16 scales) of rows [..., 128] as ggml's quantize_row_q8_0; product: the block scale as
    amax * (1 / 127) in f32 (the query of the bounded-cache decode)."""
    x = np.asarray(x, np.float32)
    blk = x.reshape(*x.shape[:-1], 4, 32)
    amax = np.abs(blk).max(-1, keepdims=True)
    d = (amax * (np.float32(1) / np.float32(127)) if product else amax / np.float32(127)).astype(np.float32)
    inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, np.float32(1)), np.float32(0)).astype(np.float32)
    q = np.rint(blk * inv).astype(np.int8)
    return q.reshape(x.shape), d[..., 0].astype(np.float16)


def dequant(q, d):
    return q.astype(np.float64) * np.repeat(d.astype(np.float64), 32, axis=-1)


def attend(q, k, v, seen, q8=False, prefill=False):
    """Exact attention of one sequence: q [T][Hq][128], k / v [S][Hkv][128] f64, seen [T][S]. Returns
    out, lse, weights [S] (summed over rows and heads) and the bounds of each (see above)."""
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    out, t_out = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    lse, t_lse = np.full((T, Hq), -np.inf), np.zeros((T, Hq))
    w, t_w = np.zeros(k.shape[0]), np.zeros(k.shape[0])
    rows, cols = np.flatnonzero(seen.any(1)), np.flatnonzero(seen.any(0))
    if not rows.size:
        return out, lse, w, t_out, t_lse, t_w
    s = seen[np.ix_(rows, cols)]
    for h in range(Hq):
        kk, vv, qq = k[cols, h // G], v[cols, h // G], q[rows, h]
        x = np.where(s, qq @ kk.T * SCALE, -np.inf)
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        l = m + np.log(e.sum(1, keepdims=True))
        p = np.exp(x - l)
        o = p @ vv
        mag = np.where(s, np.abs(qq) @ np.abs(kk).T, 0.0).max(1, keepdims=True)
        E = SCALE * (16 if q8 else 128) * 2.0 ** (-23 if prefill else -24) * mag
        n, absv = s.sum(1, keepdims=True), np.abs(vv)
        if prefill:
            X = np.where(s, (m - x) / np.log(2.0), 0.0) + 8.0
            d = np.log(2.0) * 2.0 ** -11 * X + 2.0 ** -9.9 + 2 * E + 2.0 ** -16
            t = (p * d) @ absv + (p * d).sum(1, keepdims=True) * np.abs(o) + 2.0 ** -25 * (s @ absv + n * np.abs(o))
        else:
            t = (2.0 ** -11 + 2 * E + 2.0 ** -16) * (p @ absv) + 2.0 ** -25 * (127.0 * n if q8 else s @ absv)
        out[rows, h], t_out[rows, h], lse[rows, h] = o, t, l[:, 0]
        t_lse[rows, h] = (E + 2.0 ** -16 + 2.0 ** -22 * np.abs(l))[:, 0]
        w[cols] += p.sum(0)
        t_w[cols] += ((2 * E + 2.0 ** -16) * p).sum(0)
    return out, lse, w, t_out, t_lse, t_w


def close(got, want, tol, bf16=False, what="out"):
    got = np.asarray(got, np.float64)
    lim = tol + (2.0 ** -8 * np.abs(want) if bf16 else 0.0) + 1e-30
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin]), f"{what}: infinities differ"
    d = np.abs(got[fin] - want[fin])
    worst = (d / lim[fin]).max() if d.size else 0.0
    assert not np.isnan(got).any() and worst <= 1.0, f"{what}: {worst} of its bound (max error {d.max()})"


class Batch:
    """Sequences of the given lengths with scattered pages, as f16 tensors or q8_0 planes, and the
    values the scores use (host, f64)."""

    def __init__(self, lens, Hq, Hkv, seed=0, q8=False, q_dtype=torch.float16, sharp=2.0, n_q=None):
        rng = np.random.default_rng(seed)
        self.lens, self.Hq, self.Hkv, self.q8 = list(lens), Hq, Hkv, q8
        bt, n_pages = scattered_block_tables(rng, self.lens)
        self.kb, self.vb = random_cache(rng, n_pages, Hkv)
        self.bt_host = bt
        q = random_q(rng, len(self.lens) if n_q is None else n_q, Hq) * np.float32(sharp)
        self.q = torch.from_numpy(q).cuda().to(q_dtype)
        qv = self.q.float().cpu().numpy()
        if q8:
            import localstack_b200 as L

            planes = [quantise_q8(vals(x)) for x in (self.kb, self.vb)]
            self.k_host, self.v_host = (dequant(*p) for p in planes)
            self.cache = tuple(L.Q8Cache.from_planes(torch.from_numpy(a).cuda(), torch.from_numpy(d).cuda())
                               for a, d in planes)
            self.q_host = dequant(*quantise_q8(qv, product=True))
        else:
            self.k_host, self.v_host = vals(self.kb), vals(self.vb)
            self.cache = (f16(self.kb), f16(self.vb))
            self.q_host = qv.astype(np.float16).astype(np.float64)
        self.bt = torch.from_numpy(bt).cuda()
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def cells(self, b, n=None):
        p = np.arange(self.lens[b] if n is None else n)
        return self.bt_host[b, p // 32].astype(np.int64) * 32 + p % 32

    def decode_ref(self, b, window=1 << 30, n_sink=0):
        n = self.lens[b]
        c = self.cells(b)
        return attend(self.q_host[b:b + 1], self.k_host[c], self.v_host[c],
                      window_mask([n - 1], n, window, n_sink) if n else np.zeros((1, 0), bool), self.q8)

    def poison(self, visible):
        """Puts NaN and infinities into every cell but those of visible[b] (positions) of each sequence."""
        keep = np.zeros(self.k_host.shape[0], bool)
        for b, pos in enumerate(visible):
            keep[self.cells(b)[np.asarray(pos, np.int64)]] = True
        bad = torch.from_numpy(~keep).cuda()
        for i, c in enumerate(self.cache):
            t = c.d if self.q8 else c
            t[bad] = float("nan") if i == 0 else float("inf")
