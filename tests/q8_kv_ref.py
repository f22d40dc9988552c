"""The int8 K/V cache in numpy, from its definition (include/thaDNN/thaDNN_q8_kv.hpp): the layout, what a store
leaves in it token block by token block, and attention over what it holds in 64 bits."""
import numpy as np

TINY = np.float32(2.0 ** -126)


def rounded(x, scale):
    """round(x / scale), half away from zero, of fp32 x and one fp32 scale; 0 where the scale is 0 or NaN."""
    if not scale > 0:
        return np.zeros(x.shape, np.int8)
    with np.errstate(over="ignore", under="ignore"):
        y = (x.astype(np.float32) / np.float32(scale)).astype(np.float64)
    return (np.sign(y) * np.floor(np.abs(y) + 0.5)).astype(np.int8)


class Cache:
    """Codes as [B, L, H, slots, lanes] for keys and values alike, scales as [B, L, H, slots / block]."""

    def __init__(self, B, L, H, hs, S, block, rng):
        self.B, self.L, self.H, self.hs, self.S, self.block = B, L, H, hs, S, block
        unit = max(64, block)
        self.slots, self.lanes = -(-S // unit) * unit, -(-hs // 16) * 16
        # what an earlier user of the memory left there
        self.codes = {w: rng.integers(-128, 128, (B, L, H, self.slots, self.lanes)).astype(np.int8) for w in "kv"}
        self.scales = {w: rng.uniform(0, 3, (B, L, H, self.slots // block)).astype(np.float32) for w in "kv"}
        for w in "kv":
            self.scales[w][rng.random(self.scales[w].shape) < 0.2] = np.nan

    def sizes(self):
        return self.B, self.L, self.H, self.hs, self.S, self.block

    def memory(self, w):
        """The codes as the device holds them."""
        c = self.codes[w]
        if w == "v":
            c = c.reshape(*c.shape[:3], self.slots // 16, 16, self.lanes).swapaxes(-1, -2)
        return np.ascontiguousarray(c)

    def of_memory(self, w, flat):
        c = flat.reshape(self.codes[w].shape)
        if w == "v":
            c = flat.reshape(*self.codes[w].shape[:3], self.slots // 16, self.lanes, 16).swapaxes(-1, -2)
            c = c.reshape(self.codes[w].shape)
        return c

    def span(self, pos, n):
        return max(pos, 0), min(pos + n, self.S)

    def store(self, layer, pos, n, k, v):
        """k, v [B, n_tokens, H, hs]; pos, n lists."""
        for w, x in (("k", k), ("v", v)):
            for b in range(len(pos)):
                first, last = self.span(pos[b], min(max(n[b], 0), x.shape[1]))
                if first >= last:
                    continue
                for at in range(first // self.block * self.block, last, self.block):
                    lo, hi = max(at, first), min(at + self.block, last)
                    for h in range(self.H):
                        self._block(w, b, layer, h, at, lo, hi, x[b, lo - pos[b]:hi - pos[b], h])

    def _block(self, w, b, layer, h, at, lo, hi, x):
        j = at // self.block
        codes, scales = self.codes[w][b, layer, h], self.scales[w][b, layer, h]
        top = np.abs(x).max()
        scale = np.float32(top) / np.float32(127) if np.isfinite(x).all() else np.float32(np.nan)
        if scale < TINY:
            scale = np.float32(0)
        if lo > at:
            was = scales[j]
            if np.isnan(was):
                scale = was
            elif scale <= was:
                scale = was
            else:
                old = codes[at:lo, :self.hs].astype(np.float32) * was
                codes[at:lo, :self.hs] = rounded(old, scale)
        codes[lo:hi, :self.hs] = rounded(x, scale)
        scales[j] = scale

    def values(self, w, layer, dtype=np.float32):
        """[B, H, slots, hs] that the codes stand for."""
        scale = np.repeat(self.scales[w][:, layer], self.block, axis=-1)[..., None].astype(dtype)
        return self.codes[w][:, layer, :, :, :self.hs].astype(dtype) * scale

    def attend(self, layer, pos, n, n_tokens, q, mul, some=None):
        """q [B, n_tokens, H * mul, hs] -> (out in 64 bits, bound of an fp32-accurate result's error), rows that are
        not computed (or not among `some`) NaN.

        The bound, with u = 2^-24 and T keys in sight: a score is off by at most E = u (hs sum |q||k| + 2 max|q|
        sum |k|) / sqrt(hs) (a sum of hs rounded products, or a query held in 24 bits of its largest component) and
        by 8u of its own size (scaling, the subtracted maximum); a softmax weight by 2 (E + 8u max|x|) of itself, by
        32u from its exponential and products, and by u of the largest weight where it is held in 24 bits; sums of T terms by T u each. Every
        such part is multiplied by a value of at most max|v|."""
        u = 2.0 ** -24
        k, v = self.values("k", layer, np.float64), self.values("v", layer, np.float64)
        out = np.full((len(pos), n_tokens, self.H * mul, self.hs), np.nan)
        bound = np.zeros(out.shape)
        for b in range(len(pos)):
            for i in range(min(max(n[b], 0), n_tokens)):
                p = pos[b] + i
                if some is not None and i not in some:
                    continue
                if p < 0 or p >= self.S:
                    out[b, i] = 0
                    continue
                for h in range(self.H * mul):
                    kk, vv, qq = k[b, h // mul, :p + 1], v[b, h // mul, :p + 1], q[b, i, h].astype(np.float64)
                    x = kk @ qq / np.sqrt(self.hs)
                    e = np.exp(x - x.max())
                    out[b, i, h] = e @ vv / e.sum()
                    err = u * (self.hs * (np.abs(kk) @ np.abs(qq)) + 2 * np.abs(qq).max() * np.abs(kk).sum(1)).max() / np.sqrt(self.hs)
                    bound[b, i, h] = np.abs(vv).max() * (2 * (err + 8 * u * np.abs(x).max()) + (4 * (p + 1) + 64) * u)
        return out, bound
