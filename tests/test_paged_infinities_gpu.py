"""gorch_hip_paged_attention with infinite values at keys of next to no weight:
a row that sees one gets it, however the call splits its keys into ranges."""
import numpy as np
import pytest

from tests.paged_case import Case
from tests.test_paged_attention_gpu import attend, check

pytestmark = pytest.mark.gpu

# column: values of keys 5 and 6
ODD = {2: (0x7f80, None), 3: (None, 0xff80), 4: (0x7f80, 0xff80), 5: (0xffc1, None)}


@pytest.mark.parametrize("seqs,hd,name", [
    # one range; ranges of few rows, of many, of both; heads that fill a tile in part
    ([(60, 1)], 64, "few4"), ([(900, 1)], 64, "few4 split"), ([(900, 3)], 128, "few4 split"),
    ([(900, 10)], 64, "few16 split"), ([(900, 50)], 64, "many split"), ([(900, 50)], 112, "many split"),
    ([(900, 50)], 256, "many split"), ([(900, 1), (900, 60)], 64, "few4+many split")])
def test_infinite_values_of_low_scores(gpu, seqs, hd, name):
    c = Case("bf16", 1, hd, 16, seqs, seed=hd)
    # every row asks for one late key, whose score is some 20 |q|^2 / sqrt(hd) = 20 sqrt(hd), 160 or more; the others'
    # are a few units, so their weights beside it are below 2^-200, less than f32 holds
    q = np.repeat(c.rng.standard_normal((1, 1, hd)).astype(np.float32), c.tokens, 0)
    q *= np.float32(np.sqrt(hd) / np.sqrt((q[0].astype(np.float64) ** 2).sum()))
    for s, (length, n) in enumerate(seqs):
        late = length - n - 1
        c.k[c.slot(s, late)] = ((20 * q[0]).view(np.uint32) >> 16).astype(np.uint16)
        for col, codes in ODD.items():
            for p, code in zip((5, 6), codes):
                if code is not None:
                    c.v[c.slot(s, p)][:, col] = code
    bounds = dict(max_new=max(n for _, n in seqs), max_kv=max(n for n, _ in seqs))
    assert gpu.kernel_choice("paged_attention", c.tokens, len(seqs), 1, 1, hd, *bounds.values()) == name
    with np.errstate(invalid="ignore"):
        want, tol = c.attention(q, 1)
    assert (want[..., 2] == np.inf).all() and (want[..., 3] == -np.inf).all() and np.isnan(want[..., 4:6]).all()
    got = attend(gpu, c, q, 1, **bounds)
    np.testing.assert_array_equal(got[..., 2:6], want[..., 2:6].astype(np.float32))
    fine = np.isfinite(want)
    check(got[fine], want[fine], tol[fine])
