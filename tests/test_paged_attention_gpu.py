"""gorch_hip_paged_attention against its definition in 64 bits: both cache
types, head layouts, lengths from none to thousands of keys, page sizes that
end inside tiles, rows that see nothing, pages that do not exist, infinities
and NaN where no token looks, streams, graphs and offsets past 32 bits. The
tolerance is paged_case's, from the arithmetic."""
import numpy as np
import pytest
import torch

from tests.paged_case import Case, dev, host

pytestmark = pytest.mark.gpu

SENTINEL = 123.0


def attend(gpu, c, q, hq, causal=True, extra=0, **bounds):
    out = torch.full((c.tokens + extra, hq * c.hd), SENTINEL, device="cuda")
    qd = torch.zeros((c.tokens + extra, hq * c.hd), device="cuda")
    qd[:c.tokens] = dev(q.reshape(c.tokens, -1))
    kv, b = c.cache(gpu), c.batch(gpu, extra, **bounds)
    kv.attention(b, qd, out, causal=causal)
    got = host(out)
    assert (got[c.tokens:] == SENTINEL).all()
    return got[:c.tokens].reshape(c.tokens, hq, c.hd)


def queries(c, hq, scale=1.5):
    return (c.rng.standard_normal((c.tokens, hq, c.hd)) * scale).astype(np.float32)


def check(got, want, tol):
    assert np.isfinite(got).all()
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), f"{(off > 0).sum()} values off, the worst {off.max()} beyond its bound"


LAYOUTS = [(16, 8, 128), (14, 2, 64), (12, 12, 64), (8, 1, 256), (6, 2, 96), (20, 1, 80), (3, 3, 16), (40, 2, 48)]
SHAPES = [[(1, 1)], [(333, 1)], [(0, 0), (5, 1), (0, 0), (33, 2), (16, 16), (0, 0)],
          [(130, 130), (300, 17), (64, 64), (1, 1), (257, 33)], [(2, 5), (0, 3), (40, 1), (7, 7)],
          [(70, 1)] * 9 + [(129, 40)]]


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_matches_definition(gpu, dtype, hq, hkv, hd, shape):
    seqs = SHAPES[shape]
    c = Case(dtype, hkv, hd, (16, 24, 1, 32, 100, 7)[shape], seqs, seed=shape)
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    bounds = dict(max_new=max(n for _, n in seqs), max_kv=max(n for n, _ in seqs)) if shape % 2 else {}
    check(attend(gpu, c, q, hq, extra=3, **bounds), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,hd,seqs", [
    (4, 2, 128, [(5000, 1)]), (4, 2, 64, [(4111, 3), (130, 1)]), (7, 1, 64, [(3000, 20), (1, 1), (2048, 1)]),
    (2, 1, 128, [(1500, 300), (2100, 2)]), (8, 1, 256, [(1025, 9)])])
def test_long_caches(gpu, dtype, hq, hkv, hd, seqs):
    c = Case(dtype, hkv, hd, 16, seqs, seed=hd)
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    for bounds in ({}, dict(max_new=max(n for _, n in seqs), max_kv=max(n for n, _ in seqs)), dict(max_kv=6000)):
        check(attend(gpu, c, q, hq, **bounds), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_not_causal(gpu, dtype):
    c = Case(dtype, 2, 64, 16, [(37, 20), (200, 3), (0, 2)], seed=5)
    q = queries(c, 4)
    want, tol = c.attention(q, 4, causal=False)
    check(attend(gpu, c, q, 4, causal=False), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_max_kv_cuts_what_is_seen(gpu, dtype):
    c = Case(dtype, 2, 64, 16, [(300, 50), (90, 1)], seed=6)
    q = queries(c, 4)
    want, tol = c.attention(q, 4, limit=77)
    check(attend(gpu, c, q, 4, max_kv=77), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_keys_on_no_page_are_not_seen(gpu, dtype):
    c = Case(dtype, 2, 64, 16, [(300, 40), (200, 1), (40, 3), (100, 100)], seed=7)
    q = queries(c, 4)
    c.table[0, 3], c.table[0, 18], c.table[1, 0], c.table[3, 6] = -1, c.pages, 1 << 30, -(1 << 31)
    c.table[2, :] = -5  # no page at all: zeros
    want, tol = c.attention(q, 4)
    got = attend(gpu, c, q, 4)
    check(got, want, tol)
    assert (got[c.cu[2]:c.cu[3]] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,hd,length,n", [(4, 2, 64, 90, 20), (16, 8, 128, 300, 200), (2, 1, 256, 40, 40)])
def test_nonfinite_keys_and_values_stay_with_who_sees_them(gpu, dtype, hq, hkv, hd, length, n):
    # infinities and NaN in the keys and values of later tokens of a chunk
    # change nothing for earlier tokens; who sees an infinite value gets it
    c = Case(dtype, hkv, hd, 16, [(length, n), (50, 1)], seed=8)
    q = queries(c, hq)
    first = length - n // 2
    pools = [(c.v, 0x7f80 if dtype == "bf16" else 0x7f, 3), (c.k, 0x7fc0 if dtype == "bf16" else 0xff, 9)]
    for pool, code, later in pools:
        pool[c.slot(0, min(first + later, length - 1))][:, 5] = code
    want, tol = c.attention(q, hq)
    got = attend(gpu, c, q, hq)
    bad_from = n - n // 2 + 3  # the first token that sees the value
    check(got[:bad_from], want[:bad_from], tol[:bad_from])
    check(got[n:], want[n:], tol[n:])
    k_from = min(n - n // 2 + 9, n - 1)
    assert not np.isfinite(got[bad_from:n, :, 5]).any()
    np.testing.assert_array_equal(np.isnan(got[bad_from:k_from]), np.isnan(want[bad_from:k_from]))
    np.testing.assert_array_equal(np.isinf(got[bad_from:k_from]), np.isinf(want[bad_from:k_from]))
    assert np.isnan(got[k_from:n]).all()


def test_a_query_of_nan_stays_a_row(gpu):
    c = Case("bf16", 2, 64, 16, [(60, 30)], seed=9)
    q = queries(c, 4)
    want, tol = c.attention(q, 4)
    q[7, 1, 3], q[9, 2, 0] = np.nan, np.inf
    got = attend(gpu, c, q, 4)
    assert np.isnan(got[7, 1]).all() and np.isnan(got[9, 2]).all()
    got[7, 1], got[9, 2] = want[7, 1], want[9, 2]
    check(got, want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_large_scores(gpu, dtype):
    # one key far above the others, and weights that underflow
    c = Case(dtype, 2, 64, 16, [(500, 3), (700, 1), (33, 33)], seed=10)
    q = queries(c, 4, 60.0)
    want, tol = c.attention(q, 4)
    check(attend(gpu, c, q, 4), want, tol)


@pytest.mark.parametrize("seqs,bounds", [([(700, 1), (30, 1)], dict(max_new=1)), ([(2500, 64), (90, 1)], {})])
def test_runs_agree_bit_for_bit(gpu, seqs, bounds):
    c = Case("bf16", 2, 128, 16, seqs, seed=11)
    q = queries(c, 4)
    a = attend(gpu, c, q, 4, **bounds)
    for _ in range(2):
        assert np.array_equal(a, attend(gpu, c, q, 4, **bounds))


def test_offsets_past_32_bits(gpu):
    # pools of 5 GiB, the sequence in their last pages
    hkv, page, hd = 8, 64, 128
    pages = (5 << 30) // (hkv * page * hd)
    c = Case("e4m3", hkv, hd, page, [(200, 3)], seed=12, spare=0)
    k, v = (torch.zeros((pages, hkv, page, hd), dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros((pages, hkv, page), device="cuda") for _ in "kv")
    for big, small in ((k, c.k), (v, c.v), (ks, c.ks), (vs, c.vs)):
        big[-c.pages:] = dev(small)
    kv = gpu.PagedKV(k, v, ks, vs)
    b = gpu.PagedBatch(dev(c.cu), dev(c.lens), dev(c.table + np.int32(pages - c.pages)), c.tokens)
    q = queries(c, 16)
    out = torch.empty((3, 16 * hd), device="cuda")
    kv.attention(b, dev(q.reshape(3, -1)), out)
    want, tol = c.attention(q, 16)
    check(host(out).reshape(3, 16, hd), want, tol)
    ko, vo = (torch.empty((3, hkv * hd), device="cuda") for _ in "kv")
    kv.read(b, ko, vo)
    assert np.array_equal(host(vo), c.rows("v", 0)[0][-3:].reshape(3, -1).astype(np.float32))
    assert np.array_equal(host(ko), c.rows("k", 0)[0][-3:].reshape(3, -1).astype(np.float32))


def test_streams_do_not_share(gpu):
    # two calls at once on two streams, each with its own workspace
    cs = [Case("bf16", 2, 64, 16, [(1800, 1), (900, 1)], seed=20 + i) for i in range(2)]
    qs = [queries(c, 4) for c in cs]
    made = [(c.cache(gpu), c.batch(gpu, max_new=1, max_kv=1800), dev(q.reshape(c.tokens, -1)),
             torch.empty((c.tokens, 256), device="cuda")) for c, q in zip(cs, qs)]
    ws = [kv.workspace(b, 4) for kv, b, _, _ in made]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (kv, b, q, out), w, s in zip(made, ws, streams):
            with torch.cuda.stream(s):
                kv.attention(b, q, out, ws=w)
    for c, q, (_, _, _, out) in zip(cs, qs, made):
        want, tol = c.attention(q, 4)
        check(host(out).reshape(c.tokens, 4, 64), want, tol)


def test_captured_step_follows_the_batch(gpu):
    # a captured call reads lengths and pages when it is replayed
    c = Case("e4m3", 2, 64, 16, [(640, 1), (500, 1), (33, 1)], seed=13)
    q = queries(c, 4)
    kv, b = c.cache(gpu), c.batch(gpu, max_new=1, max_kv=640)
    qd, out = dev(q.reshape(3, -1)), torch.empty((3, 256), device="cuda")
    ws = kv.workspace(b, 4)
    kv.attention(b, qd, out, ws=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.attention(b, qd, out, ws=ws)
    for lens in ([640, 500, 33], [5, 499, 1], [0, 17, 32], [639, 320, 30]):
        c.lens[:] = lens
        c.seqs = [(n, 1) for n in lens]
        b.t[1].copy_(dev(c.lens))
        torch.cuda.synchronize()
        for _ in range(2):
            out.fill_(SENTINEL)
            g.replay()
            want, tol = c.attention(q, 4)
            check(host(out).reshape(3, 4, 64), want, tol)


def test_captured_mixed_step_follows_the_batch(gpu):
    # prompts beside single tokens: both kernels, split, and their join in one graph
    c = Case("bf16", 2, 128, 16, [(900, 1), (1200, 150), (640, 1), (333, 60)], seed=16)
    hq = 4
    q = queries(c, hq)
    kv, b = c.cache(gpu), c.batch(gpu, max_new=150, max_kv=1200)
    assert gpu.kernel_choice("paged_attention", c.tokens, 4, hq, 2, 128, 150, 1200).endswith("+many split")
    qd, out = dev(q.reshape(c.tokens, -1)), torch.empty((c.tokens, hq * 128), device="cuda")
    ws = kv.workspace(b, hq)
    kv.attention(b, qd, out, ws=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.attention(b, qd, out, ws=ws)
    for seqs in ([(900, 1), (1200, 150), (640, 1), (333, 60)], [(700, 60), (40, 1), (1, 1), (150, 150)],
                 [(0, 0), (1199, 3), (639, 130), (1, 1)]):
        c.seqs, c.lens[:], c.cu[1:] = seqs, [n for n, _ in seqs], np.cumsum([n for _, n in seqs])
        live = c.cu[-1]
        b.t[0].copy_(dev(c.cu))
        b.t[1].copy_(dev(c.lens))
        torch.cuda.synchronize()
        want, tol = c.attention(q, hq)
        for _ in range(2):
            out.fill_(SENTINEL)
            ws.fill_(0xff)  # nothing is taken from an earlier call's sums
            g.replay()
            got = host(out).reshape(-1, hq, 128)
            check(got[:live], want[:live], tol[:live])
            assert (got[live:] == SENTINEL).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,hd,seqs", [
    # key ranges of the kernel for many rows, each width of its heads, whole and in part
    (2, 1, 256, [(700, 90)]), (2, 1, 208, [(700, 90), (300, 1)]), (3, 1, 112, [(900, 70)]), (2, 2, 32, [(900, 70)]),
    # tiles of 4 and 16 rows, split
    (4, 2, 192, [(1500, 1), (1100, 2)]), (7, 1, 96, [(1500, 1)]), (16, 1, 256, [(1500, 1), (3, 1)]),
    (5, 1, 32, [(1500, 3)]), (1, 1, 16, [(1500, 9)]),
    # both kinds of rows: one split, the other, both; two tiles of single rows; heads that fill more than two
    (4, 4, 64, [(100, 1)] * 3 + [(700, 400)]), (2, 1, 128, [(4000, 2), (90, 90)]), (20, 1, 80, [(1500, 1), (900, 70)]),
    (40, 1, 64, [(300, 1), (70, 1), (900, 2)])])
def test_splits(gpu, dtype, hq, hkv, hd, seqs):
    c = Case(dtype, hkv, hd, 24, seqs, seed=hd + hq)
    bounds = dict(max_new=max(n for _, n in seqs), max_kv=max(n for n, _ in seqs))
    assert "split" in gpu.kernel_choice("paged_attention", c.tokens, len(seqs), hq, hkv, hd, *bounds.values())
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    check(attend(gpu, c, q, hq, **bounds), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("count,bounds", [(70, {}), (70, dict(max_new=1, max_kv=500)), (1100, dict(max_new=1)), (4200, {})])
def test_many_sequences(gpu, dtype, count, bounds):
    # a search of one, two and three steps for a token's sequence; more blocks than run at once
    rng = np.random.default_rng(count)
    single = "max_new" in bounds
    seqs = [(int(rng.integers(0, 40)), 1 if single else int(rng.integers(0, 3))) for _ in range(count)]
    seqs[3], seqs[-2] = (500, 1), ((40, 1) if single else (90, 60))
    c = Case(dtype, 1, 32, 16, seqs, seed=count)
    q = queries(c, 2)
    want, tol = c.attention(q, 2)
    check(attend(gpu, c, q, 2, extra=1, **bounds), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_a_shared_prefix(gpu, dtype):
    # the same pages in several sequences, and valid pages named past a sequence's last position
    c = Case(dtype, 2, 64, 16, [(200, 1), (170, 4), (230, 70), (40, 1)], seed=17)
    c.table[1, :5], c.table[2, :7] = c.table[0, :5], c.table[0, :7]
    c.table[c.table >= c.pages] = c.table[0, 0]
    q = queries(c, 4)
    want, tol = c.attention(q, 4)
    for bounds in ({}, dict(max_new=70, max_kv=230), dict(max_kv=4000)):
        check(attend(gpu, c, q, 4, **bounds), want, tol)


@pytest.mark.parametrize("n", [1, 40])
def test_no_pages_at_all(gpu, n):
    c = Case("bf16", 1, 64, 16, [(n, n), (0, 0)], seed=18)
    kv, b = c.cache(gpu), gpu.PagedBatch(dev(c.cu), dev(c.lens), torch.empty((2, 0), dtype=torch.int32, device="cuda"), n)
    out, rows = torch.full((n, 128), SENTINEL, device="cuda"), torch.full((n, 64), SENTINEL, device="cuda")
    kv.attention(b, dev(queries(c, 2).reshape(n, -1)), out)
    kv.read(b, rows, None)
    assert (host(out) == 0).all() and (host(rows) == SENTINEL).all()


@pytest.mark.parametrize("length,n", [(70, 1), (900, 2), (60, 50), (900, 50)])
def test_infinite_values_of_both_signs(gpu, length, n):
    # column 2: +inf, 3: -inf, 4: both, 5: NaN, in keys that all see
    c = Case("bf16", 1, 64, 16, [(length, n)], seed=19)
    for p, col, code in ((3, 2, 0x7f80), (4, 3, 0xff80), (5, 4, 0x7f80), (9, 4, 0xff80), (2, 5, 0xffc1)):
        c.v[c.slot(0, p)][:, col] = code
    q = queries(c, 2, 0.1)
    with np.errstate(invalid="ignore"):
        want, tol = c.attention(q, 2)
    got = attend(gpu, c, q, 2)
    assert (got[-1, :, 2] == np.inf).all() and (got[-1, :, 3] == -np.inf).all() and np.isnan(got[-1, :, 4:6]).all()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)])
    check(got[fine], want[fine], tol[fine])


def test_small_workspace_is_refused(gpu):
    c = Case("bf16", 1, 128, 16, [(5000, 1)], seed=14)
    kv, b = c.cache(gpu), c.batch(gpu, max_new=1, max_kv=5000)
    q, out = dev(queries(c, 2).reshape(1, -1)), torch.empty((1, 256), device="cuda")
    ws = kv.workspace(b, 2)
    if ws is not None:
        with pytest.raises(gpu.HipError) as e:
            kv.attention(b, q, out, ws=ws[:-16])
        assert e.value.rc == 2


def test_wrong_tensors_are_refused(gpu):
    c = Case("bf16", 2, 64, 16, [(20, 2)], seed=15)
    kv, b = c.cache(gpu), c.batch(gpu)
    q, out = dev(queries(c, 4).reshape(2, -1)), torch.empty((2, 256), device="cuda")
    for bad in (lambda: kv.attention(b, q[:1], out[:1]), lambda: kv.attention(b, q.double(), out),
                lambda: kv.attention(b, q, out[:, :128]), lambda: kv.attention(b, q.cpu(), out),
                lambda: kv.attention(b, q[:, :100].contiguous(), out), lambda: kv.read(b, out, None),
                lambda: gpu.PagedBatch(dev(c.cu).long(), dev(c.lens), dev(c.table), 2),
                lambda: gpu.PagedBatch(dev(c.cu)[:2], dev(np.array([1, 2], np.int32)), dev(c.table), 2)):
        with pytest.raises(ValueError):
            bad()
