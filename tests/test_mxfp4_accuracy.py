"""The bounds of the four-bit kernels' accuracy tests are narrow enough: a part
of an operand that is lost, here in the oracle, passes none of them."""
import numpy as np
import pytest

from tests.mx_accuracy import (HEADS, KERNELS, ONE_VALUE, U, cut, last_term_of_q, last_term_of_weights, one_value_rows)


def test_five_terms_are_x_and_four_are_not():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 96)) * np.exp2(rng.integers(-3, 3, (50, 96)))).astype(np.float32)
    top = np.abs(x.reshape(50, 3, 32)).max(-1).repeat(32, -1)
    assert (np.abs(cut(x, 5) - x) <= U * top).all()
    assert (np.abs(cut(x, 4) - x) > 4 * U * top).any(1).all()


@pytest.mark.parametrize("name,M,N,K", KERNELS)
def test_the_linears_bound_shows_a_lost_term(name, M, N, K):
    rng = np.random.default_rng(K)
    lost = np.concatenate([(cut(x, 4) - x)[np.arange(M), at] / x[np.arange(M), at]
                           for x, at in (one_value_rows(rng, M, K) for _ in range(max(1, 24 // M)))])
    assert (np.abs(lost) > 2 * ONE_VALUE).all()


@pytest.mark.parametrize("hq,hkv,hd,n", HEADS)
@pytest.mark.parametrize("T", [70, 400])
@pytest.mark.parametrize("part", [last_term_of_q, last_term_of_weights])
def test_attentions_bounds_show_a_lost_term(hq, hkv, hd, n, T, part):
    c, q, tol, lost = part(hkv, hd, hq, T, n, seed=hd + T)
    want, _ = c.attention(q, hq, causal=False)
    assert np.isfinite(want).all() and (want[:n] != 0).all()
    # what is lost would take some output past its bound in next to every token of the first sequence
    assert (lost[:n] > tol).mean() >= 0.9 and lost[:n].max() > 1.2 * tol
