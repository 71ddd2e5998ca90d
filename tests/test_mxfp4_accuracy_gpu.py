"""The four-bit kernels hold f32's bits where a result rests on them: the last
of x's and q's five 6-bit terms, the last of a weight's three bf16 terms, and
the scale byte of each, in every kernel that the Linear and attention choose."""
import numpy as np
import pytest

from tests.mx_accuracy import HEADS, KERNELS, ONE_VALUE, U, last_term_of_q, last_term_of_weights, one_value_rows
from tests.mx_case import values
from tests.test_mxfp4_linear_gpu import call, inputs, weight
from tests.test_paged_attention_gpu import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,M,N,K", KERNELS)
def test_one_value_a_row(gpu, name, M, N, K):
    assert gpu.kernel_choice("linear_mxfp4", M, N, K) == name
    rng = np.random.default_rng(K)
    codes, scales = weight(rng, N, K)
    W = values(codes, scales)
    for _ in range(max(1, 24 // M)):
        x, at = one_value_rows(rng, M, K)
        want = x[np.arange(M), at].astype(np.float64)[:, None] * W[:, at].T
        off = np.abs(call(gpu, x, codes, scales) - want) / np.maximum(np.abs(want), 1e-300)
        assert (off <= ONE_VALUE).all(), f"off by {off.max() / U} U"


@pytest.mark.parametrize("name,M,N,K", KERNELS)
def test_whole_rows(gpu, name, M, N, K):
    """The error's norm. Five terms leave 1.8 U of the norm for these x (residues up to U of a group's largest value, evenly
    spread). A wave adds up 45 instructions at most, 180 groups of 32 products, to a sum that grows as a random walk does;
    of an addition off by up to 2 U, evenly spread, 1.15 U each, they leave 1.15 sqrt(180 / 2) U = 11 U. Twice that, for
    roundings that lean one way: 23 U. Four terms leave 55 U."""
    rng, x, codes, scales = inputs(K, M, N, K)
    want = x.astype(np.float64) @ values(codes, scales).T
    off = np.linalg.norm(call(gpu, x, codes, scales) - want) / np.linalg.norm(want)
    assert off <= 23 * U, f"off by {off / U} U of the norm"


@pytest.mark.parametrize("hq,hkv,hd,n", HEADS)
@pytest.mark.parametrize("T,page", [(70, 16), (400, 16), (400, 1 << 15)])
@pytest.mark.parametrize("part", [last_term_of_q, last_term_of_weights])
def test_attention(gpu, hq, hkv, hd, n, T, page, part):
    # (400 keys are four key ranges by pages of 16 and, since a range may then be longer, one by pages of 2^15)
    c, q, tol, _ = part(hkv, hd, hq, T, n, hd + T, page)
    want, _ = c.attention(q, hq, causal=False)
    off = np.abs(attend(gpu, c, q, hq, causal=False, max_new=n) - want) / np.abs(want)
    assert (off <= tol).all(), f"off by {off.max() / U} U, the bound is {tol / U}"
