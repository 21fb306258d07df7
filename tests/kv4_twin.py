"""The 4-bit cache on the host: its quantiser, its page layout and attention over it, in 64 bits."""

import numpy as np


def groups(hd):
    return max(1, hd // 64), min(64, hd)


def quantise(x):
    """(codes, scales, offsets) of f32 rows [..., hd]; scales and offsets f16 [..., groups]."""
    n, g = groups(x.shape[-1])
    x = x.astype(np.float64).reshape(*x.shape[:-1], n, g)
    with np.errstate(all="ignore"):
        low, high = x.min(-1), x.max(-1)
        scale = np.minimum((high - low) / 15, 65504.0).astype(np.float32).astype(np.float16)
        offset = np.clip(low, -65504.0, 65504.0).astype(np.float32).astype(np.float16)
        wide = scale.astype(np.float64)[..., None]
        codes = np.where(wide > 0, np.clip(np.rint((x - offset.astype(np.float64)[..., None]) / wide), 0, 15), 0)
        bad = ~np.isfinite(x).all(-1)
    scale[bad] = offset[bad] = np.nan
    codes[bad] = 0
    return codes.astype(np.uint8).reshape(*codes.shape[:-2], n * g), scale, offset


def values(codes, scale, offset):
    n, g = groups(codes.shape[-1])
    c = codes.astype(np.float64).reshape(*codes.shape[:-1], n, g)
    return (c * scale.astype(np.float64)[..., None] + offset.astype(np.float64)[..., None]).reshape(codes.shape)


class Pool:
    """One layer's pages as bytes, and single rows of it by (page, slot)."""

    def __init__(self, pages, page, kv, hd, fill=0):
        self.page, self.kv, self.hd = page, kv, hd
        self.n = groups(hd)[0]
        self.bytes = np.full((pages, page * kv * (hd + 8 * self.n)), fill, np.uint8)

    def _at(self, which, head, slot):
        head_bytes = self.page * (self.hd + 8 * self.n)
        base = head * head_bytes + which * (head_bytes // 2)
        return base + slot * (self.hd // 2), base + self.page * (self.hd // 2) + slot * self.n * 4

    def put(self, page, slot, which, codes, scale, offset):
        """codes [kv, hd], scale and offset [kv, groups] of one token (which: 0 K, 1 V)."""
        for h in range(self.kv):
            c, p = self._at(which, h, slot)
            self.bytes[page, c:c + self.hd // 2] = codes[h, 0::2] | (codes[h, 1::2] << 4)
            self.bytes[page, p:p + 4 * self.n] = np.stack([scale[h], offset[h]], -1).reshape(-1).view(np.uint8)

    def get(self, page, slot, which):
        """f64 [kv, hd]."""
        out = []
        for h in range(self.kv):
            c, p = self._at(which, h, slot)
            raw = self.bytes[page, c:c + self.hd // 2]
            par = self.bytes[page, p:p + 4 * self.n].copy().view(np.float16).reshape(self.n, 2)
            out.append(values(np.stack([raw & 15, raw >> 4], -1).reshape(-1), par[:, 0], par[:, 1]))
        return np.stack(out)


def magnitudes(codes, scale, offset):
    """scale * code + |offset|: the sizes of the two terms that a value is made of."""
    return values(codes, scale, np.abs(offset))


def attention(q, k, v, scale, queries, k_mag, v_mag, weight=0.0):
    """(out, bound) of q [queries, heads, hd] over k, v [n, kv, hd]: in f64, and how far an evaluation
    in f32 may be that keeps scale * code and offset apart (k_mag, v_mag: their sizes, added).

    A score is a sum of hd products and hd/64 offsets; every partial sum is at most
    Q = scale * sum |q| k_mag and each of at most 16 cutting accumulations and 8 roundings is off by at
    most 2^-22 of it (q's high and remainder parts by 2^-21): 2^-17 Q in all.  A weight exp(score - top)
    is then off by a factor of exp(2 * 2^-17 Q) (its own score and the top), and by 2^-20 for exp2,
    products, sums and quotient; `weight` is the further relative rounding of the weights.  Both act on
    terms of size p v_mag, in the numerator as in the sum that divides it."""
    n, kv, hd = k.shape
    heads = q.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for j in range(queries):
        m = n - queries + j + 1
        if m <= 0:
            continue
        for h in range(heads):
            at = (slice(0, m), h * kv // heads)
            with np.errstate(invalid="ignore"):
                s = k[at] @ q[j, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[j, h] = p @ v[at]
                d = 2.0 ** -17 * (k_mag[at] @ np.abs(q[j, h])).max() * scale
                bound[j, h] = (2 * np.expm1(2 * d) + 2.0 ** -20 + weight) * (p @ v_mag[at])
    return out, bound
