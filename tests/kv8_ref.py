"""Plain numpy form of the 8-bit K/V cache (codes as defined, attention in 64 bits) and the error bounds its tests use."""
import numpy as np

BLOCK = 16
EPS = 2.0 ** -24          # half a step of f32, relative


def quantise(x):
    """rows [n <= 16, D] of one block -> (codes, scale): the exact product (f32 x f32 fits f64) rounded once."""
    amax = np.float32(np.abs(x).max()) if x.size else np.float32(0)
    if np.isnan(x).any() or np.isinf(x).any():
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    if amax < np.float32(2.0 ** -100):
        return np.zeros(x.shape, np.int8), np.float32(0)
    inv, scale = np.float32(127) / amax, amax / np.float32(127)
    return np.rint(x.astype(np.float64) * np.float64(inv)).astype(np.int8), np.float32(scale)


class RefCache:
    def __init__(self, n_ctx, Hkv, D):
        n = -(-n_ctx // BLOCK) * BLOCK
        self.Hkv, self.D = Hkv, D
        self.codes = np.zeros((2, n, Hkv, D), np.int8)
        self.scale = np.zeros((2, n // BLOCK, Hkv), np.float32)
        self.open = (-1, 0, None)             # block appended to last, its rows, unrounded [2, rows, Hkv, D]

    def values(self, lo=0, hi=None):
        hi = self.codes.shape[1] if hi is None else hi
        return self.codes[:, lo:hi].astype(np.float32) * np.repeat(self.scale, BLOCK, 1)[:, lo:hi, :, None]

    def append(self, k, v, pos):
        x, end = np.stack([k, v]), pos + len(k)
        keep = None
        for b in range(pos // BLOCK, (end - 1) // BLOCK + 1):
            r0, r1 = max(pos - b * BLOCK, 0), min(end - b * BLOCK, BLOCK)
            rows = np.zeros((2, r1, self.Hkv, self.D), np.float32)
            if r0:
                rows[:, :r0] = self.values(b * BLOCK, b * BLOCK + r0)
                if self.open[0] == b:
                    held = min(r0, self.open[1])
                    rows[:, :held] = self.open[2][:, :held]
            rows[:, r0:r1] = x[:, b * BLOCK + r0 - pos:b * BLOCK + r1 - pos]
            self.put(b, rows)
            keep = (b, r1, rows)
        self.open = keep

    def put(self, b, rows):
        self.codes[:, b * BLOCK:(b + 1) * BLOCK] = 0
        for j in range(2):
            for h in range(self.Hkv):
                c, s = quantise(rows[j, :, h])
                self.codes[j, b * BLOCK:b * BLOCK + len(c), h], self.scale[j, b, h] = c, s

    def evict(self, dst, T, keep, sink, recent, mass):
        kept = np.empty((self.Hkv, keep), np.int32)
        for h in range(self.Hkv):
            mid = np.arange(sink, T - recent)
            m = mass[h, sink:T - recent].astype(np.float64)
            m = np.where(np.isnan(m), -np.inf, m)
            nan = np.isnan(mass[h, sink:T - recent])
            heavy = mid[np.lexsort((mid, nan, -m))][:keep - sink - recent]
            kept[h] = np.sort(np.concatenate([np.arange(sink), heavy, np.arange(T - recent, T)]))
        val = self.values()
        for b in range(-(-keep // BLOCK)):
            at = kept[:, b * BLOCK:(b + 1) * BLOCK]
            rows = np.stack([val[:, at[h], h] for h in range(self.Hkv)], 2)
            dst.put(b, rows)
            for h in range(self.Hkv):
                p = at[h]
                if len(p) == BLOCK and p[0] % BLOCK == 0 and p[-1] == p[0] + BLOCK - 1:
                    dst.codes[:, b * BLOCK:(b + 1) * BLOCK, h] = self.codes[:, p[0]:p[0] + BLOCK, h]
                    dst.scale[:, b, h] = self.scale[:, p[0] // BLOCK, h]
            dst.open = (b, at.shape[1], rows)
        return kept, np.take_along_axis(mass, kept.astype(np.int64), 1)


def attention(val, q, n_past, mass=None):
    """q [M, H, D] over values [2, T, Hkv, D], row i sees t <= n_past + i -> (out, mass, tolerance of out, tolerance of mass), all in 64 bits.

    Tolerances (worst case, to first order in EPS, for any order of f32 sums of at most 64 terms before the next level):
      score   a product rounds each factor once and sums D terms: |ds| <= (D + 16) EPS max|q| sum_i |k_i| / sqrt(D) =: e; this also covers
              a query held as a fixed-point number of 23 bits relative to max|q| (its error is max|q| 2 EPS per entry)
      weight  p = exp(s - m) / l: relative error <= 2 e (its own score and the sum's), plus 8 EPS for exp and the quotient, plus the sum's
              own rounding, (T / 16 + 64) EPS at most when sixteen positions or more are added per step
      out     sum p v: the weights' error times sum p |v|, plus (T / 16 + 96) EPS of the same for its own sum and the weights' rounding to a
              fixed-point number of 22 bits relative to the largest p * scale of their tile (64 positions: at most 64 * 2 EPS * max|v|)
      mass    the weights' error summed, plus EPS per addition"""
    M, H, D = q.shape
    k, v = val[0].astype(np.float64), val[1].astype(np.float64)
    T, G = n_past + M, H // val.shape[2]
    k, v = k[:T], v[:T]
    out, tol = np.empty((M, H, D)), np.empty((M, H, D))
    msum, mtol = np.zeros((val.shape[2], T)), np.zeros((val.shape[2], T))
    adds = np.zeros((val.shape[2], T))
    for h in range(H):
        j = h // G
        s = q[:, h].astype(np.float64) @ k[:, j].T / np.sqrt(D)
        seen = np.arange(T)[None] <= n_past + np.arange(M)[:, None]
        s = np.where(seen, s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ np.where(seen.any(0)[:, None], v[:, j], 0)
        e = np.where(seen, (D + 16) * EPS * np.abs(q[:, h]).max(1)[:, None] * np.abs(k[:, j]).sum(1)[None] / np.sqrt(D), 0).max(1)
        w = 2 * e + (8 + T / 16 + 64) * EPS
        pv, vmax = p @ np.abs(v[:, j]), np.abs(v[:, j]).max()
        tol[:, h] = pv * (w + (T / 16 + 96) * EPS)[:, None] + 128 * EPS * vmax * p.max(1)[:, None] + 1e-30
        msum[j] += p.sum(0)
        mtol[j] += (p * w[:, None]).sum(0)
        adds[j] += seen.sum(0)
    if mass is None:
        return out, None, tol, None
    total = mass[:, :T].astype(np.float64) + msum
    return out, total, tol, mtol + EPS * (adds + 4) * (np.abs(mass[:, :T]) + msum) + 1e-30
