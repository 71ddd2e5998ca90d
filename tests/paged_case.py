"""Caches in pages, ragged batches and their plain 64-bit mathematics, for the
tests of the paged operators."""
import numpy as np
import torch


def bits_e4m3():
    """The value of each e4m3 code (sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7f and 0xff are NaN)."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = (-x if c & 128 else x) if c & 127 != 127 else np.nan
    return v


E4M3 = bits_e4m3()
UNUSED = {"bf16": 0x7fc0, "e4m3": 0x7f}  # NaN: what no token may see


class Case:
    """Sequences of (cached length, new tokens) over shuffled pages. Slots that hold no token are NaN."""

    def __init__(self, dtype, hkv, hd, page, seqs, seed=0, spare=2, fill=True):
        self.rng = np.random.default_rng(seed)
        self.dtype, self.hkv, self.hd, self.page, self.seqs = dtype, hkv, hd, page, seqs
        need = [-(-n // page) for n, _ in seqs]
        self.pages = max(1, sum(need) + spare)
        self.max_pages = max(1, max(need, default=0))
        order = self.rng.permutation(self.pages)
        self.table = np.full((len(seqs), self.max_pages), self.pages + 7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).astype(np.int32)
        self.lens = np.array([n for n, _ in seqs], np.int32)
        self.tokens = int(self.cu[-1])
        shape = (self.pages, hkv, page, hd)
        self.k, self.v = (np.full(shape, UNUSED[dtype], np.uint16 if dtype == "bf16" else np.uint8) for _ in "kv")
        self.ks, self.vs = (np.full(shape[:3], np.nan, np.float32) for _ in "kv")
        if fill:
            for s, (n, _) in enumerate(seqs):
                for p in range(n):
                    self.put(s, p)

    def slot(self, s, p):
        return self.table[s, p // self.page], slice(None), p % self.page

    def put(self, s, p):
        at, shape = self.slot(s, p), (self.hkv, self.hd)
        for pool, scales in ((self.k, self.ks), (self.v, self.vs)):
            if self.dtype == "bf16":
                x = self.rng.standard_normal(shape).astype(np.float32)
                pool[at] = (x.view(np.uint32) >> 16).astype(np.uint16)
            else:
                c = self.rng.integers(0, 254, shape)
                pool[at] = np.where(c % 128 == 127, 0, c)
                scales[at] = np.exp(self.rng.standard_normal(self.hkv)).astype(np.float32) / 100

    def row(self, which, s, p):
        """[hkv, hd] in 64 bits, or None where position p of sequence s is on no page."""
        page = self.table[s, p // self.page]
        if not 0 <= page < self.pages:
            return None
        pool, scales = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        x = pool[page, :, p % self.page]
        if self.dtype == "bf16":
            return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        return E4M3[x] * scales[page, :, p % self.page].astype(np.float64)[:, None]

    def rows(self, which, s):
        """[length, hkv, hd] and which of them are on a page."""
        r = [self.row(which, s, p) for p in range(self.lens[s])]
        ok = np.array([x is not None for x in r], bool)
        zero = np.zeros((self.hkv, self.hd))
        return np.array([zero if x is None else x for x in r]).reshape(-1, self.hkv, self.hd), ok

    def cache(self, hip):
        if self.dtype == "bf16":
            return hip.PagedKV(dev(self.k.view(np.int16)), dev(self.v.view(np.int16)))
        return hip.PagedKV(dev(self.k), dev(self.v), dev(self.ks), dev(self.vs))

    def batch(self, hip, extra=0, **bounds):
        return hip.PagedBatch(dev(self.cu), dev(self.lens), dev(self.table), self.tokens + extra, **bounds)

    def attention(self, q, hq, causal=True, limit=None):
        """Output and its error bound [tokens, hq, hd] for q f32 [tokens, hq, hd].

        The bound follows the arithmetic. A score is a sum of hd products of q (scaled and split, 2^-24 each and
        less) with exact cache values in f32, then one scale factor: off by e = (hd + 8) 2^-24 sum_d |q_d k_d|. A
        weight exp(s - m) is off by a factor of 1 +- (e + |s - m| 2^-23 + 2^-21): its argument's rounding, and the
        exponential's own few units. Weighted sums over T keys add T 2^-24, rescaling and joining parts, dividing
        and the weight sum 2^-20: the output is off by at most twice the largest of these (numerator and
        denominator) times sum_j p_j |v_j|. A weight below f32's normal range, 2^-126 of the largest, is held to
        fewer bits or none, and so is a term of its split, 2^-8 and 2^-16 of it: that adds at most 2^-126 for each
        of three terms of each key, 2^-124 sum_j |v_j|."""
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
                    prod = q[t, h].astype(np.float64) * kk / np.sqrt(self.hd)
                    sc = prod.sum(1)
                    with np.errstate(invalid="ignore", over="ignore"):
                        p = np.exp(sc - sc.max())
                        p /= p.sum()
                        e = (self.hd + 8) * 2.0 ** -24 * np.abs(prod).sum(1).max()
                        e += (sc.max() - sc.min()) * 2.0 ** -23 + 2.0 ** -20 + len(see) * 2.0 ** -24
                        out[t, h] = p @ vv
                        tol[t, h] = 2 * e * (p @ np.abs(vv)) + 2.0 ** -124 * np.abs(vv).sum(0)
        return out, tol


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()
