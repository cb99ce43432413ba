"""CPU oracle of the 8-bit paged cache, the attention over it and the 4-bit products - TEST INFRASTRUCTURE ONLY.

float64 numpy from the formats' definitions: a block of 16 tokens x 128 dims of one K/V head holds codes u = m + 128 and
an exponent E, value m * 2^(E - 133); E = 255 reads as NaN. A 4-bit weight is (u - 8) * s."""

import numpy as np

BLOCK = 16


def exponent_field(x):
    """Largest float32 exponent field of x."""
    return int((np.asarray(x, np.float32).view(np.uint32) >> 23 & 255).max())


def encode(x, E):
    if E == 255:
        return np.full(np.shape(x), 128, np.uint8)
    m = np.clip(np.rint(np.ldexp(np.asarray(x, np.float64), 133 - E)), -128, 127)
    return (m + 128).astype(np.uint8)


def decode(u, E):
    if E == 255:
        return np.full(np.shape(u), np.nan)
    return np.ldexp(u.astype(np.float64) - 128, int(E) - 133)


class Cache:
    """One layer: codes (pages, hkv, page, 128) and exponents (pages, hkv, page / 16) of keys or values."""

    def __init__(self, codes, exps):
        self.codes, self.exps, self.page = codes, exps, codes.shape[2]

    def place(self, table, pos):
        return int(table[pos // self.page]), pos % self.page

    def append(self, table, length, x):
        """x (n, hkv, 128) float32 at positions length - n .. length - 1."""
        n, hkv = x.shape[:2]
        first = length - n
        for blk in range(first // BLOCK, (length + BLOCK - 1) // BLOCK):
            lo, hi = max(first, blk * BLOCK), min(length, (blk + 1) * BLOCK)
            if lo >= hi:
                continue
            pg, at = self.place(table, blk * BLOCK)
            older = lo - blk * BLOCK
            for h in range(hkv):
                E = exponent_field(x[lo - first:hi - first, h])
                if older:
                    old = int(self.exps[pg, h, at // BLOCK])
                    E = max(E, old)
                    c = self.codes[pg, h, at:at + older]
                    m = np.rint(np.ldexp(c.astype(np.float64) - 128, old - E))
                    self.codes[pg, h, at:at + older] = (m + 128).astype(np.uint8)
                self.codes[pg, h, at + older:at + hi - blk * BLOCK] = encode(x[lo - first:hi - first, h], E)
                self.exps[pg, h, at // BLOCK] = E

    def read(self, table, length, missing=()):
        """(length, hkv, 128) float64."""
        hkv = self.codes.shape[1]
        out = np.zeros((length, hkv, 128))
        for blk in range((length + BLOCK - 1) // BLOCK):
            pg, at = self.place(table, blk * BLOCK)
            hi = min(length, (blk + 1) * BLOCK) - blk * BLOCK
            if not 0 <= pg < len(self.codes):
                continue
            for h in range(hkv):
                out[blk * BLOCK:blk * BLOCK + hi, h] = decode(self.codes[pg, h, at:at + hi], self.exps[pg, h, at // BLOCK])
        return out


def attention(q, k, v, limit, present=None):
    """q (n, heads, 128), k / v (len, hkv, 128), limit (n) last visible position -> (o (n, heads, 128), bound): bound is
    the error that half-step fp16 weights and fp32 scores leave before the output's own rounding:
    2 * 2^-11 * sum w|v| (each weight and the sum of weights off by 2^-11), the scores' fp32 sums of 128 products (128
    half steps of 2^-24 of sum |q k|, doubled for the tensor core's truncation) carried through the exponential into
    weights and sum, and weights below fp16's normal range: the split kernel keeps weights times 2^4 and, in a block whose
    V exponent is d <= 8 below the largest, times 2^-d, so they are off by 2^-25 2^(d - 4) there (the largest weight being
    >= 1) and |v| <= 2^(E - d - 126) for the largest exponent E: together at most 2^-29 2^(E - 126) <= 2^-28 max |v| a key.
    The prompt kernel keeps them times 2^7 (off by 2^-32 of the largest) and takes blocks whose values are below 2^-29 of the
    largest as zeros, which is no more."""
    n, heads, _ = q.shape
    grp = heads // k.shape[1]
    o, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(heads):
        kh, vh = k[:, h // grp], v[:, h // grp]
        for r in range(n):
            keep = np.arange(len(k)) <= limit[r]
            if present is not None:
                keep &= present
            if not keep.any():
                continue
            s = kh[keep] @ q[r, h] / np.sqrt(128)
            w = np.exp(s - s.max())
            w /= w.sum()
            es = (np.abs(kh[keep]) @ np.abs(q[r, h])).max() / np.sqrt(128) * 128 * 2.0 ** -23
            va = np.abs(vh[keep])
            o[r, h] = w @ vh[keep]
            bound[r, h] = (2 ** -10 + 4 * es) * (w @ va) + 2.0 ** -28 * keep.sum() * va.max() + 1e-30
    return o, bound


def quantize_w4(B, group):
    """B (K, N) float32 -> (codes uint8 (K, N), scales float32 holding bf16 (K / group, N))."""
    from .bfp16_oracle import bf16_round
    K, N = B.shape
    g = np.asarray(B, np.float32).reshape(K // group, group, N)
    ext = np.take_along_axis(g, np.abs(g).argmax(1)[:, None], 1)[:, 0]
    s = bf16_round((ext * np.float32(-0.125)).astype(np.float32))
    with np.errstate(divide="ignore", invalid="ignore"):
        m = np.rint((g / s[:, None]).astype(np.float32))
    m = np.where(s[:, None] == 0, 0, np.clip(m, -8, 7))
    return (m + 8).astype(np.uint8).reshape(K, N), s


def linear_w4(x, codes, scales):
    """float64 product and the bound of its fp32 sum: K half steps of 2^-24 of sum |x w|, doubled for the tensor core's
    truncation."""
    K = codes.shape[0]
    w = (codes.astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), K // len(scales), 0)
    x = np.asarray(x, np.float64)
    return x @ w, K * 2.0 ** -23 * (np.abs(x) @ np.abs(w)) + 1e-30
