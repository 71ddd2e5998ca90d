"""Inputs whose results rest on single parts of the four-bit kernels' operands:
x's and q's last 6-bit term, a weight's last bf16 term, a group's scale byte.
Bounds count roundings of U = 2^-24 and are derived where they stand; what a
lost part would do to the same results is computed beside them.

Two facts of the arithmetic are used throughout. A matrix instruction adds four
groups of 32 products to a sum, one after another (test_one_instruction): with
one product p in a group, the sum so far loses what lies below a unit in p's
last place, 2 U of p, and the result is rounded, U. And where one product of a
sum is nonzero, nothing but that product's own terms is rounded: x (24 bits) is
the sum of five terms, of which the last four add up to at most 2^-4 of x; times
a code (0.5 to 6) they need 23 bits, so adding them up, smallest first, is exact
and the first term's addition alone is not: off by 3 U (1 + 1 / 16) < 3.25 U."""
import numpy as np

from tests.mx_case import GROUP, MxCase, groups

U = 2.0 ** -24


def cut(x, terms):
    """x [..., cols] as the sum of its first terms: multiples of 2^(e - 5 t - 3), e the exponent of the largest of 32."""
    g = groups(np.asarray(x, np.float64))
    top = np.abs(g).max(-1, keepdims=True)
    e = np.floor(np.log2(np.where(top > 0, top, 1)))
    rest = g.copy()
    for t in range(terms):
        step = 2.0 ** (e - 5 * t - 3)
        rest -= np.round(rest / step) * step
    return (g - rest).reshape(x.shape[:-1] + (-1,))[..., :x.shape[-1]]


# The choices of the Linear's kernel that one value a row is sent through.
KERNELS = [("gemv", 1, 4100, 4096), ("gemv", 3, 50, 264), ("gemv split", 2, 300, 9000), ("gemv5", 5, 3000, 2048),
           ("gemv5", 16, 100, 520), ("gemv5 split", 4, 300, 6000), ("gemv5 made", 13, 5000, 2048), ("gemv5 made", 9, 90, 5160),
           ("gemv5 made split", 16, 1000, 9000), ("gemm128x256", 1000, 4200, 1032), ("gemm128x128", 600, 6000, 520),
           ("gemm64x128", 500, 4000, 1160), ("gemm64x64", 64, 16300, 600), ("gemm32x64", 128, 4001, 2056),
           ("gemm32x32", 64, 4000, 1096)]
ONE_VALUE = 3.25 * U  # of |x w|


def one_value_rows(rng, M, K):
    """x of one value a row, of 24 bits whose last five, the fifth term's, stand for 9 to 23 units: four terms leave 9 at
    least, 2^-20.8 of the value. And where."""
    at = rng.integers(0, K, M)
    x = np.zeros((M, K), np.float32)
    bits = rng.integers(1 << 18, 1 << 19, M) * 32 + 2 * rng.integers(4, 12, M) + 1
    x[np.arange(M), at] = np.ldexp(bits, rng.integers(-40, -10, M)) * rng.choice([-1, 1], M)
    return x, at


# [query heads, KV heads, head columns, new tokens]: both row tiles of the kernel for few rows, the kernel for many, and
# (a second sequence of one token beside many rows) the one launch of both
HEADS = [(2, 1, 64, 1), (16, 8, 128, 1), (4, 1, 80, 1), (3, 1, 256, 1), (14, 2, 64, 1), (20, 1, 80, 1), (8, 1, 256, 1),
         (32, 4, 128, 1), (2, 1, 64, 40), (16, 8, 128, 40), (8, 1, 256, 10), (6, 2, 96, 20), (14, 2, 64, 30), (3, 3, 16, 50)]


class Parts(MxCase):
    """Keys of one nonzero column, each row's q one nonzero column there, and values that give every output column the
    weight of one key: so a score is one product, and an output one weight over the sum of weights.

    The bounds, relative to an output (every row sees all T keys): the scale's and q's rounding 2 U, the score's product
    3.25 U, all of |s| in log2; what weights are relative to, up to 8 past the largest score, is taken from a score once
    (in the matrix instruction, 3 U, or after it, U) and from another such reference up to three times (a rescaling, the
    join of waves, that of key ranges), U each, and U where it is set: 7 U of max |s| + 8. ln 2 times these is the error of one weight, and 20 U more its
    exponentials' last places (1 unit, 2 U, each), the products with them and with V, the division."""

    @staticmethod
    def weight_error(largest):
        return np.log(2) * (5.25 * largest + 7 * (largest + 8)) * U + 20 * U

    def __init__(self, hkv, hd, T, n, seed, page, k_scale):
        super().__init__(hkv, hd, page, [(T, n), (33, 1)], seed)
        self.column = int(self.rng.integers(0, hd))
        self.owner = self.rng.permutation(max(T, hd))[:hd] % T
        for s, (length, _) in enumerate(self.seqs):
            for p in range(length):
                at = self.slot(s, p)
                self.k[at], self.ks[at], self.v[at], self.vs[at] = 0, k_scale, 0, 127
        nibble = self.rng.integers(1, 8, (2, hd)) | 8 * self.rng.integers(0, 2, (2, hd))
        for s, (length, _) in enumerate(self.seqs):
            for d in range(hd):
                self.v[self.slot(s, self.owner[d] % length)][:, d // 2] |= np.uint8(nibble[s, d] << 4 * (d % 2))

    def set_key(self, s, p, code):
        self.k[self.slot(s, p)][:, self.column // 2] = code << 4 * (self.column % 2)

    def scaled(self, q, dtype=np.float32):
        """q as the kernels hold it: times log2(e) / sqrt(hd), rounded twice."""
        return (q * np.float32(np.log2(np.e) / np.sqrt(self.hd))).astype(dtype)


def last_term_of_q(hkv, hd, hq, T, n, seed, page=16):
    """One key of a sequence has a score of 48 (log2), the others 0: outputs of theirs are 2^-48 of values, and rest on
    q's bits below 2^-19, which its fifth term holds. Returns case, q, bound, and the outputs' change without that term."""
    c = Parts(hkv, hd, T, n, seed, page, 127 + 3)
    for s, (length, _) in enumerate(c.seqs):
        c.set_key(s, length // 2, 7)  # 6 * 2^3
    q = np.zeros((c.tokens, hq, hd), np.float32)
    aim = np.ldexp(np.float64((1 << 23) + 15), -23) * np.sqrt(hd) / np.log2(np.e)
    q[..., c.column] = aim * (1 + c.rng.integers(-1, 2, (c.tokens, hq)) * 2.0 ** -23)
    held = c.scaled(q[..., c.column:c.column + 1])
    lost = held.astype(np.float64) - cut(held, 4)
    # (the denominator: one weight of 2^48 and the others', which round to nothing beside it)
    return c, q, Parts.weight_error(48.0), np.expm1(np.log(2) * 48 * np.abs(lost)).max((1, 2))


def last_term_of_weights(hkv, hd, hq, T, n, seed, page=16):
    """Scores within 3 (log2), weights of all 24 bits: returns case, q, bound and the most that outputs lose with weights
    cut to two bf16 terms. Beside its own weight an output rests on the sum of all, to the same relative error and one
    rounding of each addition of a lane (a quarter of the keys) and of some joins."""
    c = Parts(hkv, hd, T, n, seed, page, 127 - 1)
    code = c.rng.integers(0, 16, (2, max(T, 33)))
    for s, (length, _) in enumerate(c.seqs):
        for p in range(length):
            c.set_key(s, p, int(code[s, p]))
    q = np.zeros((c.tokens, hq, hd), np.float32)
    q[..., c.column] = c.rng.uniform(0.5, 1, (c.tokens, hq)) * np.sqrt(hd) / np.log2(np.e)
    value = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])[code[0, :T] & 7] * np.where(code[0, :T] & 8, -0.5, 0.5)
    s2 = c.scaled(q[:n, :, c.column], np.float64)[..., None] * value
    w = np.exp2(s2 - s2.max(-1, keepdims=True) - 8).astype(np.float32)
    first = (w.view(np.uint32) & 0xffff0000).view(np.float32)
    second = ((w - first).view(np.uint32) & 0xffff0000).view(np.float32)
    lost = ((w - first - second) / w)[..., c.owner].max((1, 2))
    return c, q, 2 * Parts.weight_error(3.0) + (T / 4 + 12) * U, lost
