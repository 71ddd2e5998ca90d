"""MXFP4 in numpy, and caches in it with their plain 64-bit mathematics, for
the tests of the operators in four bits."""
import numpy as np

from tests.paged_case import Case, dev

GROUP = 32
CODES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
CODES = np.concatenate([CODES, -CODES])


def spread(scales, cols):
    """Scale bytes [..., groups] as the power of two of each of cols columns (NaN for 255)."""
    p = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return np.repeat(p, GROUP, -1)[..., :cols]


def unpack(codes):
    c = np.empty(codes.shape[:-1] + (2 * codes.shape[-1],), np.uint8)
    c[..., 0::2], c[..., 1::2] = codes & 15, codes >> 4
    return c


def values(codes, scales):
    """What codes [..., cols / 2] and scales [..., groups] stand for, in 64 bits."""
    c = unpack(codes)
    return CODES[c] * spread(scales, c.shape[-1])


def groups(x, fill=0.0):
    """[..., groups, 32] of [..., cols], the last group filled up."""
    cols = x.shape[-1]
    n = -(-cols // GROUP)
    y = np.full(x.shape[:-1] + (n * GROUP,), fill, x.dtype)
    y[..., :cols] = x
    return y.reshape(x.shape[:-1] + (n, GROUP))


def encode(x):
    """Codes and scales of rows x [..., cols] of exactly given values: the smallest power of two that the group's largest
    magnitude exceeds at most 7 times, then the nearest code, the even one of two."""
    cols = x.shape[-1]
    g = groups(np.asarray(x, np.float64))
    with np.errstate(invalid="ignore"):
        top = np.abs(g).max(-1)
        m, e = np.frexp(top)  # top = m 2^e, 7 = 0.875 * 2^3
        e = np.where(m <= 0.875, e - 3, e - 2)
        odd, tiny = ~np.isfinite(top), top < 2.0 ** -100
        a = np.abs(np.ldexp(g, -np.where(odd | tiny, 0, e)[..., None]))
        # distance to each code; of two nearest the one with an even last bit
        d = np.abs(np.minimum(a, 6.0)[..., None] - CODES[:8])
        d = np.where(np.isnan(d), 0, d)
        best = d.min(-1, keepdims=True)
        even = np.arange(8) % 2 == 0
        c = np.where((d == best) & even, np.arange(8), np.where(d == best, 16 + np.arange(8), 99)).min(-1) % 16
    c = (c + 8 * np.signbit(g)).astype(np.uint8)
    c[odd | tiny] = 0
    s = np.where(odd, 255, np.where(tiny, 0, e + 127)).astype(np.uint8)
    c = c.reshape(x.shape[:-1] + (-1,))[..., :cols]
    return (c[..., 0::2] | c[..., 1::2] << 4).astype(np.uint8), s


def half_step(a, step):
    """How far rounding can move a value of magnitude a (up to 7 steps) to a multiple of its step."""
    return step * np.where(a <= 2 * step, 0.25, np.where(a <= 4 * step, 0.5, 1.0))


class MxCase(Case):
    """Case over a cache in MXFP4. Slots that hold no token are NaN by their scales."""

    def __init__(self, hkv, hd, page, seqs, seed=0, spare=2, fill=True):
        super().__init__("e4m3", hkv, hd, page, seqs, seed, spare, fill=False)
        self.dtype = "mxfp4"
        shape = (self.pages, hkv, page)
        self.k, self.v = (np.full(shape + (hd // 2,), 0x77, np.uint8) for _ in "kv")
        self.ks, self.vs = (np.full(shape + (-(-hd // GROUP),), 255, np.uint8) for _ in "kv")
        if fill:
            for s, (n, _) in enumerate(seqs):
                for p in range(n):
                    self.put(s, p)

    def put(self, s, p):
        at = self.slot(s, p)
        for pool, scales in ((self.k, self.ks), (self.v, self.vs)):
            pool[at] = self.rng.integers(0, 256, (self.hkv, self.hd // 2))
            scales[at] = self.rng.integers(121, 128, (self.hkv, scales.shape[-1]))

    def row(self, which, s, p):
        page = self.table[s, p // self.page]
        if not 0 <= page < self.pages:
            return None
        pool, scales = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        return values(pool[page, :, p % self.page], scales[page, :, p % self.page])

    def cache(self, hip):
        return hip.PagedKV(dev(self.k), dev(self.v), dev(self.ks), dev(self.vs))

    def attention(self, q, hq, causal=True, limit=None):
        """Output and its error bound, as Case.attention's, but for the scores: q (scaled, 2^-24 of each) is held to
        2^-24 of the largest magnitude in each 32 columns, and ten matrix instructions a score (five terms, 256 columns)
        sum their products to 2^-23 of the sum of their magnitudes each: off by e = 24 * 2^-24 sum_d top_d |k_d|, top_d
        that largest magnitude."""
        out = np.zeros((self.tokens, hq, self.hd))
        tol = np.zeros_like(out)
        for s, (length, n) in enumerate(self.seqs):
            if not n or not length:
                continue
            (k, ok), (v, _) = self.rows("k", s), self.rows("v", s)
            for i in range(n):
                t, pos = self.cu[s] + i, length - n + i
                T = min(pos + 1 if causal else length, length if limit is None else limit)
                see = np.flatnonzero(ok[:max(T, 0)])
                if not len(see):
                    continue
                for h in range(hq):
                    kk, vv = k[see, h * self.hkv // hq], v[see, h * self.hkv // hq]
                    x = q[t, h].astype(np.float64) / np.sqrt(self.hd)
                    sc = (x * kk).sum(1)
                    top = np.repeat(np.abs(groups(x)).max(-1), GROUP)[:self.hd]
                    with np.errstate(invalid="ignore", over="ignore"):
                        p = np.exp(sc - sc.max())
                        p /= p.sum()
                        e = 24 * 2.0 ** -24 * (top * np.abs(kk)).sum(1).max()
                        e += (sc.max() - sc.min()) * 2.0 ** -23 + 2.0 ** -20 + len(see) * 2.0 ** -24
                        out[t, h] = p @ vv
                        tol[t, h] = 2 * e * (p @ np.abs(vv)) + 2.0 ** -124 * np.abs(vv).sum(0)
        return out, tol
