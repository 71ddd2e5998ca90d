"""gorch_hip_process_logits against its definition in 64 bits: each rule alone
and all together, ragged histories and bias lists, ids out of range and listed
twice, vocabularies of odd sizes, masks that allow nothing, infinite and NaN
logits, in place."""
import numpy as np
import pytest
import torch

from tests.paged_case import dev, host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def definition(x, r):
    """The rules in 64 bits and the f32 result's bound: a quotient or product, a product and two differences, a sum:
    at most five roundings (U each) of no more than the sum of the magnitudes."""
    rows, n = x.shape
    out, tol = x.astype(np.float64), np.zeros((rows, n))
    for i in range(rows):
        said = np.zeros(n, np.int64)
        seen = np.zeros(n, bool)
        if "history" in r:
            h = r["history"][i]
            if "history_lens" in r:
                h = h[:max(0, r["history_lens"][i])]
            p = max(0, r["prompt_lens"][i]) if "prompt_lens" in r else 0
            ok = (h >= 0) & (h < n)
            seen[h[ok]] = True
            np.add.at(said, h[p:][ok[p:]], 1)
        y = out[i]
        if "repetition" in r:
            rep = np.float64(r["repetition"][i])
            y[seen] = np.where(y[seen] > 0, y[seen] / rep, y[seen] * rep)
        mag = np.abs(y)
        for name, amount in (("frequency", said), ("presence", said > 0)):
            if name in r:
                y -= amount * np.float64(r[name][i])
                mag += amount * np.abs(np.float64(r[name][i]))
        if "bias" in r:
            b = np.zeros(n)
            for e in range(r["bias_rows"][i], r["bias_rows"][i + 1]):
                if 0 <= r["bias_ids"][e] < n:
                    b[r["bias_ids"][e]] = r["bias"][e]
            y += b
            mag += np.abs(b)
        if "allowed" in r:
            bits = (r["allowed"][i].view(np.uint32)[np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1
            y[bits == 0] = -np.inf
        tol[i] = 5 * U * mag
    return out, tol


def apply(gpu, x, r, in_place=False):
    xd = dev(x)
    out = xd if in_place else torch.empty_like(xd)
    gpu.process_logits(xd, out, **{k: dev(v) for k, v in r.items()})
    return host(out)


def check(got, want, tol):
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine].astype(np.float32))
    assert np.isfinite(got[fine]).all() and (np.abs(got[fine] - want[fine]) <= tol[fine]).all()


def rules(rng, rows, n, width, biases):
    lens = rng.integers(0, width + 1, rows).astype(np.int32)
    counts = rng.integers(0, biases + 1, rows)
    total = int(counts.sum())
    return {"history": (rng.random((rows, width)) ** 3 * (n + 2) - 1).astype(np.int32), "history_lens": lens,
            "prompt_lens": (lens * rng.random(rows)).astype(np.int32),
            "repetition": (0.5 + rng.random(rows)).astype(np.float32),
            "frequency": rng.standard_normal(rows).astype(np.float32),
            "presence": rng.standard_normal(rows).astype(np.float32),
            "bias_rows": np.concatenate([[0], np.cumsum(counts)]).astype(np.int32),
            "bias_ids": rng.integers(-1, n + 1, total).astype(np.int32),
            "bias": (rng.standard_normal(total) * 5).astype(np.float32),
            "allowed": rng.integers(-2 ** 31, 2 ** 31, (rows, (n + 31) // 32 + 1)).astype(np.int32)}


GROUPS = [("history", "repetition"), ("history", "history_lens", "prompt_lens", "frequency"),
          ("history", "history_lens", "presence"), ("bias_rows", "bias_ids", "bias"), ("allowed",), (),
          ("history", "history_lens", "prompt_lens", "repetition", "frequency", "presence", "bias_rows", "bias_ids",
           "bias", "allowed")]


@pytest.mark.parametrize("rows,n,width,biases", [(1, 1, 1, 1), (3, 31, 5, 9), (2, 33, 300, 3), (5, 1000, 40, 20),
                                                 (2, 50257, 300, 40), (3, 8193, 9000, 300), (2, 4096, 0, 1),
                                                 (1, 151936, 4001, 300), (70, 4099, 7, 2),
                                                 # more than 2^21 logits: the larger blocks
                                                 (520, 4099, 30, 4), (16, 131075, 5001, 40)])
@pytest.mark.parametrize("group", range(len(GROUPS)))
def test_matches_definition(gpu, rows, n, width, biases, group):
    rng = np.random.default_rng(n + group)
    x = (rng.standard_normal((rows, n)) * 4).astype(np.float32)
    r = {k: v for k, v in rules(rng, rows, n, width, biases).items() if k in GROUPS[group]}
    want, tol = definition(x, r)
    check(apply(gpu, x, r), want, tol)
    check(apply(gpu, x, r, in_place=True), want, tol)


def test_last_of_an_ids_biases_counts(gpu):
    n = 100
    ids = np.array([5, 7, 5, 5, 7, 99] * 200 + [5], np.int32)
    bias = np.arange(len(ids), dtype=np.float32)
    x = np.zeros((2, n), np.float32)
    r = {"bias_rows": np.array([0, len(ids), len(ids)], np.int32), "bias_ids": ids, "bias": bias}
    got = apply(gpu, x, r)
    assert got[0, 5] == len(ids) - 1 and got[0, 7] == len(ids) - 3 and got[0, 99] == len(ids) - 2
    assert np.count_nonzero(got) == 3


def test_a_mask_that_allows_nothing(gpu):
    x = np.array([[1.0, np.nan, np.inf] * 50] * 2, np.float32)
    r = {"allowed": np.array([[0] * 5, [-1] * 5], np.int32)}
    got = apply(gpu, x, r)
    assert (got[0] == -np.inf).all()
    np.testing.assert_array_equal(got[1], x[1])
    tok = torch.empty(1, dtype=torch.int32, device="cuda")
    gpu.argmax(dev(got[:1]), tok)
    assert host(tok)[0] == 0


def test_infinite_and_nan_logits(gpu):
    x = np.array([[np.inf, -np.inf, np.nan, 0.0, -0.0, 3e38, -3e38, 1e-45]], np.float32)
    r = {"history": np.arange(8, dtype=np.int32)[None], "repetition": np.array([2.0], np.float32),
         "presence": np.array([0.5], np.float32)}
    got = apply(gpu, x, r)[0]
    assert got[0] == np.inf and got[1] == -np.inf and np.isnan(got[2])
    assert (got[3:5] == -0.5).all() and got[5] == np.float32(1.5e38) and got[6] == -np.inf and got[7] == -0.5


def test_captured_rules_follow_their_arrays(gpu):
    rng = np.random.default_rng(5)
    rows, n = 4, 5003
    x = (rng.standard_normal((rows, n)) * 4).astype(np.float32)
    r = rules(rng, rows, n, 50, 10)
    d = {k: dev(v) for k, v in r.items()}
    xd = dev(x)
    out = torch.empty_like(xd)
    gpu.process_logits(xd, out, **d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gpu.process_logits(xd, out, **d)
    for i in range(3):
        r["history"] = (rng.random((rows, 50)) * n).astype(np.int32)
        r["history_lens"] = rng.integers(0, 51, rows).astype(np.int32)
        for k in ("history", "history_lens"):
            d[k].copy_(dev(r[k]))
        out.fill_(9.0)
        torch.cuda.synchronize()
        g.replay()
        want, tol = definition(x, r)
        check(host(out), want, tol)


def test_wrong_tensors_are_refused(gpu):
    x = torch.zeros((2, 64), device="cuda")
    i = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    f = torch.zeros(2, device="cuda")
    for r in (dict(history=i.long()), dict(history=i[:1]), dict(repetition=f[:1]), dict(repetition=f.double()),
              dict(history=i, history_lens=i), dict(bias=f), dict(allowed=i.float()), dict(presence=f.cpu())):
        with pytest.raises(ValueError):
            gpu.process_logits(x, x, **r)
    with pytest.raises(ValueError):
        gpu.process_logits(x, x[:1])
    with pytest.raises(gpu.HipError):
        gpu.process_logits(x, x, allowed=i[:, :1].contiguous())


@pytest.mark.parametrize("first,out_first", [(0, 1), (1, 1), (1, 2), (2, 0), (3, 2)])
@pytest.mark.parametrize("n", [5, 1023, 4099, 700001])
def test_rows_at_any_address(gpu, first, out_first, n):
    # rows of a larger tensor start at any multiple of 4 bytes, in and out each their own
    rng = np.random.default_rng(n + first)
    x = (rng.standard_normal((3, n)) * 4).astype(np.float32)
    r = rules(rng, 3, n, 37, 6)
    want, tol = definition(x, r)
    space = torch.zeros(3 * n + 8, device="cuda")
    xd = space[first:first + 3 * n].view(3, n)
    xd.copy_(dev(x))
    room = torch.full((3 * n + 8,), 55.0, device="cuda")
    gpu.process_logits(xd, room[out_first:out_first + 3 * n].view(3, n), **{k: dev(v) for k, v in r.items()})
    got = host(room)
    check(got[out_first:out_first + 3 * n].reshape(3, n), want, tol)
    assert (got[:out_first] == 55).all() and (got[out_first + 3 * n:] == 55).all()
