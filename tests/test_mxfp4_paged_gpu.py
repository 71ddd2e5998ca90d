"""The paged cache in MXFP4: gorch_hip_paged_append, gorch_hip_paged_read and
gorch_hip_paged_attention against their definitions in 64 bits, with the head
layouts, lengths, pages and masks of the other cache types' tests."""
import numpy as np
import pytest
import torch

from tests.mx_case import MxCase, encode, half_step, spread, values
from tests.paged_case import dev, host
from tests.test_paged_append_gpu import LAYOUTS, SENTINEL, append, finished
from tests.test_paged_attention_gpu import SHAPES, attend, check, queries

pytestmark = pytest.mark.gpu


def check_append(c, hq, x, params, q_out, pools, scales, neox=0, skipped=lambda s, p: False, with_q=True):
    gq, gk, cos, sin = params
    hkv, hd = c.hkv, c.hd
    touched = np.zeros((c.pages, c.page), bool)
    for s, (length, n) in enumerate(c.seqs):
        for i in range(n):
            t, p = c.cu[s] + i, length - n + i
            if p < 0 or skipped(s, p):
                if with_q:
                    assert (q_out[t] == SENTINEL).all()
                continue
            at = c.slot(s, p)
            touched[at[0], at[2]] = True
            rows = x[t].reshape(-1, hd)
            co, si = (None, None) if cos is None else (cos[p:p + 1], sin[p:p + 1])
            if with_q:
                q, qt = finished(rows[None, :hq], gq, 1e-6, co, si, neox)
                assert (np.abs(q_out[t].reshape(1, hq, hd) - q) <= qt).all()
            k, kt = (y[0] for y in finished(rows[None, hq:hq + hkv], gk, 1e-6, co, si, neox))
            codes, scale = encode(rows[hq + hkv:])
            np.testing.assert_array_equal(pools[1][at], codes)
            np.testing.assert_array_equal(scales[1][at], scale)
            # a finished key is within kt of k: its scale that of some value there, its codes half a step from it
            kt = kt * 1.01
            low, high = (encode(np.maximum(np.abs(k) + d * kt, 0))[1] for d in (-1, 1))
            got = scales[0][at]
            assert ((low <= got) & (got <= high)).all()
            held, step = values(pools[0][at], got), spread(got, hd)
            assert (np.abs(held - k) <= kt + half_step(np.abs(k) + kt, step)).all()
    for got, was in zip(pools + scales, (c.k, c.v, c.ks, c.vs)):
        for page in range(c.pages):
            keep = ~touched[page]
            assert np.array_equal(got[page][:, keep], was[page][:, keep])


@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("norm,rope,neox", [(True, True, 0), (False, True, 1), (True, False, 0), (False, False, 0),
                                            (True, True, 1)])
def test_append_matches_definition(gpu, hq, hkv, hd, norm, rope, neox):
    c = MxCase(hkv, hd, 24, [(0, 0), (40, 7), (1, 1), (0, 0), (130, 30), (25, 25)], seed=hd + neox, fill=False)
    check_append(c, hq, *append(gpu, c, hq, norm, rope, neox, fused=norm), neox=neox)


@pytest.mark.parametrize("seqs,bounds", [([(777, 1)], dict(max_new=1)), ([(9 + i, 1) for i in range(100)], {}),
                                         ([(1000, 1000), (3, 3)], {}), ([(i % 3, i % 3) for i in range(300)], dict(max_new=2))])
def test_append_batches(gpu, seqs, bounds):
    c = MxCase(2, 64, 16, seqs, seed=3, fill=False)
    check_append(c, 4, *append(gpu, c, 4, True, True, extra=5, **bounds))


def test_append_without_q_or_place(gpu):
    c = MxCase(2, 80, 16, [(40, 9)], seed=4, fill=False)
    check_append(c, 4, *append(gpu, c, 4, True, True, with_q=False), with_q=False)
    c = MxCase(2, 64, 16, [(60, 20), (3, 9)], seed=5, fill=False)
    c.table[0, 2] = -1
    check_append(c, 4, *append(gpu, c, 4, True, True, rope_rows=55),
                 skipped=lambda s, p: (s == 0 and 32 <= p < 48) or p >= 55)


def test_append_of_extremes(gpu):
    c = MxCase(1, 64, 16, [(5, 5)], seed=6, fill=False)
    x = np.zeros((5, 3 * 64), np.float32)
    x[0, 64:128], x[1, 64:] = 1e-35, -0.0
    x[2, 70], x[2, 150] = np.inf, np.nan
    x[3, 64:] = 3e38
    x[4, 64:] = np.linspace(-7, 7, 128)
    kv, b = c.cache(gpu), c.batch(gpu)
    heads = gpu.GQA(dict(dim=64, num_q=1, num_kv=1, head_dim=64))
    q, k, v = dev(x).split([64, 64, 64], 1)
    kv.append(b, heads, None, k, v, None)
    ko, vo = (torch.full((5, 64), SENTINEL, device="cuda") for _ in "kv")
    kv.read(b, ko, vo)
    for got, y in ((ko, x[:, 64:128]), (vo, x[:, 128:])):
        np.testing.assert_array_equal(host(got), values(*encode(y)).astype(np.float32))


@pytest.mark.parametrize("hkv,hd", [(8, 128), (2, 64), (1, 256), (2, 96), (1, 80), (3, 16), (2, 48), (4, 128), (6, 64)])
@pytest.mark.parametrize("seqs", [[(40, 7), (0, 0), (130, 130)], [(3000, 2990), (2500, 2500)]])
def test_read_is_exact(gpu, hkv, hd, seqs):
    c = MxCase(hkv, hd, 24, seqs, seed=hd)
    c.table[0, 0] = -1
    kv, b = c.cache(gpu), c.batch(gpu, 4)
    outs = [torch.full((c.tokens + 4, hkv * hd), SENTINEL, device="cuda") for _ in "kv"]
    kv.read(b, *outs)
    one = torch.full((c.tokens + 4, hkv * hd), SENTINEL, device="cuda")
    kv.read(b, None, one)
    assert torch.equal(one, outs[1])
    for which, out in zip("kv", outs):
        out = host(out)
        assert (out[c.tokens:] == SENTINEL).all()
        for s, (length, n) in enumerate(seqs):
            rows, ok = c.rows(which, s)
            for i in range(n):
                want = rows[length - n + i].reshape(-1) if ok[length - n + i] else SENTINEL
                assert np.array_equal(out[c.cu[s] + i].astype(np.float64), np.broadcast_to(want, hkv * hd))


@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_matches_definition(gpu, hq, hkv, hd, shape):
    seqs = SHAPES[shape]
    c = MxCase(hkv, hd, (16, 24, 1, 32, 100, 7)[shape], seqs, seed=shape)
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    bounds = dict(max_new=max(n for _, n in seqs), max_kv=max(n for n, _ in seqs)) if shape % 2 else {}
    check(attend(gpu, c, q, hq, extra=3, **bounds), want, tol)


@pytest.mark.parametrize("hq,hkv,hd,seqs", [
    (4, 2, 128, [(5000, 1)]), (4, 2, 64, [(4111, 3), (130, 1)]), (7, 1, 64, [(3000, 20), (1, 1), (2048, 1)]),
    (2, 1, 128, [(1500, 300), (2100, 2)]), (8, 1, 256, [(1025, 9)])])
def test_long_caches(gpu, hq, hkv, hd, seqs):
    c = MxCase(hkv, hd, 16, seqs, seed=hd)
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    for bounds in ({}, dict(max_new=max(n for _, n in seqs), max_kv=max(n for n, _ in seqs)), dict(max_kv=6000)):
        check(attend(gpu, c, q, hq, **bounds), want, tol)


def test_not_causal_cut_and_on_no_page(gpu):
    c = MxCase(2, 64, 16, [(37, 20), (200, 3), (0, 2)], seed=5)
    q = queries(c, 4)
    check(attend(gpu, c, q, 4, causal=False), *c.attention(q, 4, causal=False))
    c = MxCase(2, 64, 16, [(300, 50), (90, 1)], seed=6)
    q = queries(c, 4)
    check(attend(gpu, c, q, 4, max_kv=77), *c.attention(q, 4, limit=77))
    c = MxCase(2, 64, 16, [(300, 40), (200, 1), (40, 3), (100, 100)], seed=7)
    q = queries(c, 4)
    c.table[0, 3], c.table[0, 18], c.table[1, 0], c.table[3, 6] = -1, c.pages, 1 << 30, -(1 << 31)
    c.table[2, :] = -5  # no page at all: zeros
    got = attend(gpu, c, q, 4)
    check(got, *c.attention(q, 4))
    assert (got[c.cu[2]:c.cu[3]] == 0).all()


@pytest.mark.parametrize("hq,hkv,hd,length,n", [(4, 2, 64, 90, 20), (16, 8, 128, 300, 200), (2, 1, 256, 40, 40),
                                                (2, 1, 80, 70, 5)])
def test_nan_keys_and_values_stay_with_who_sees_them(gpu, hq, hkv, hd, length, n):
    c = MxCase(hkv, hd, 16, [(length, n), (50, 1)], seed=8)
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    g = c.vs.shape[-1] - 1  # the last group of columns
    at_v, at_k = length - n + n // 2, length - 2
    c.vs[c.slot(0, at_v)][:, g] = 255
    c.ks[c.slot(0, at_k)][:, 0] = 255
    got = attend(gpu, c, q, hq)
    v_from, k_from = n // 2, n - 2  # the first rows that see them
    check(got[:v_from], want[:v_from], tol[:v_from])
    check(got[n:], want[n:], tol[n:])
    check(got[v_from:k_from][..., :32 * g], want[v_from:k_from][..., :32 * g], tol[v_from:k_from][..., :32 * g])
    assert np.isnan(got[v_from:n, :, 32 * g:]).all()
    assert np.isnan(got[k_from:n]).all()


@pytest.mark.parametrize("hq,hkv,hd,length,n", [(4, 2, 64, 90, 20), (4, 2, 128, 300, 200), (2, 1, 256, 40, 40),
                                                (2, 1, 80, 70, 5), (32, 4, 64, 100, 3)])
def test_infinite_values_stay_in_their_columns(gpu, hq, hkv, hd, length, n):
    # 4 * 2^126 and 2 * 2^127 are past f32; their groups' other codes, and the rows before them, are not
    c = MxCase(hkv, hd, 16, [(length, n), (50, 1)], seed=14)
    q = queries(c, hq) / 8  # (weights that do not vanish)
    g = c.vs.shape[-1] - 1
    at = [length - n + n // 2, length - n // 3 - 1]
    for p, scale, code in ((at[0], 253, 0x6f), (at[1], 254, 0x34)):
        c.v[c.slot(0, p)][:, 16 * g:] = 0  # the group is zeros but for two columns
        c.v[c.slot(0, p)][:, 16 * g + 2] = code
        c.vs[c.slot(0, p)][:, g] = scale
    got = attend(gpu, c, q, hq)
    # without what is infinite (0x34: 2 * 2^127 is, 1.5 * 2^127 is not; 0x6f: -6 and 4, times 2^126)
    for p, scale, code in ((at[0], 253, 0), (at[1], 254, 0x30)):
        c.v[c.slot(0, p)][:, 16 * g:] = 0
        c.v[c.slot(0, p)][:, 16 * g + 2] = code
        c.vs[c.slot(0, p)][:, g] = scale
    want, tol = c.attention(q, hq)
    first, second = (p - (length - n) for p in at)
    if first == second:
        first = n  # (3 rows: the later write is the only one)
    a, b = 32 * g + 4, 32 * g + 5
    for r in range(n):
        row = np.ones(hd, bool)
        row[a], row[b] = r < min(first, second), r < first
        check(got[r][:, row], want[r][:, row], tol[r][:, row])
        if r >= min(first, second):
            is_a = np.isposinf if r < first else (np.isneginf if r < second else np.isnan)
            assert is_a(got[r, :, a]).all()
        if r >= first:
            assert np.isposinf(got[r, :, b]).all()
    check(got[n:], want[n:], tol[n:])


def test_large_magnitudes(gpu):
    # scales at the ends of f32's range where their products stay inside it, and scale 0, whose values count as zeros
    c = MxCase(1, 64, 16, [(100, 1), (90, 60)], seed=9)
    c.ks[:] = np.where(c.ks == 255, 255, 60)
    c.vs[:] = np.where(c.vs == 255, 255, 230)
    c.vs[c.slot(0, 7)] = 0
    c.vs[c.slot(1, 7)] = 1
    q = queries(c, 2) * np.float32(2.0 ** 60)
    check(attend(gpu, c, q, 2), *c.attention(q, 2))


@pytest.mark.parametrize("seqs,bounds", [([(600, 1), (31, 1)], dict(max_new=1, max_kv=640)), ([(700, 90), (5, 1)], {})])
def test_captured_with_lengths_that_change(gpu, seqs, bounds):
    c = MxCase(2, 128, 16, seqs, seed=10)
    q = queries(c, 4)
    kv, b = c.cache(gpu), c.batch(gpu, **bounds)
    ws = kv.workspace(b, 4)
    qd, out = dev(q.reshape(c.tokens, -1)), torch.zeros((c.tokens, 4 * 128), device="cuda")
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        kv.attention(b, qd, out, ws=ws)
    first = c.lens.copy()
    for less in (0, 9, 3):
        c.lens = first - np.array([less, 0], np.int32)
        c.seqs = [(int(n), m) for n, (_, m) in zip(c.lens, seqs)]
        b.t[1].copy_(dev(c.lens))
        out.fill_(5)
        graph.replay()
        want, tol = c.attention(q, 4)
        check(host(out).reshape(want.shape), want, tol)
        again = torch.empty_like(out)
        kv.attention(b, qd, again)
        assert torch.equal(again, out)


def test_append_then_attend_then_read(gpu):
    # the operators as a step uses them: a fused q/k/v Linear in four bits, its rows into the pages, attention, the
    # output projection in four bits added to the residual stream
    from tests.test_mxfp4_linear_gpu import expected, weight

    hq, hkv, hd, dim = 4, 2, 64, 128
    seqs = [(40, 6), (129, 1), (9, 9)]
    c = MxCase(hkv, hd, 16, seqs, seed=11)
    rng, T = c.rng, c.tokens
    wq, wo = weight(rng, (hq + 2 * hkv) * hd, dim), weight(rng, dim, hq * hd)
    x = rng.standard_normal((T, dim)).astype(np.float32)
    qkv, q_out, out = (torch.zeros((T, n), device="cuda") for n in ((hq + 2 * hkv) * hd, hq * hd, hq * hd))
    stream = dev(x)
    cos, sin = gpu.rope_tables(hd, 256, 1e6)
    heads = gpu.GQA(dict(dim=dim, num_q=hq, num_kv=hkv, head_dim=hd, rope=True, rope_cos=cos, rope_sin=sin, rope_max_seq=256))
    kv, b = c.cache(gpu), c.batch(gpu, max_new=9, max_kv=160)
    gpu.linear_mxfp4(stream, gpu.pack_mxfp4(*map(dev, wq)), qkv.shape[1], None, qkv)
    q, k, v = qkv.split([hq * hd, hkv * hd, hkv * hd], 1)
    kv.append(b, heads, q, k, v, q_out)
    kv.attention(b, q_out, out)
    gpu.linear_mxfp4(out, gpu.pack_mxfp4(*map(dev, wo)), dim, None, stream, residual=stream)
    ko, vo = (torch.zeros((T, hkv * hd), device="cuda") for _ in "kv")
    kv.read(b, ko, vo)
    # each against what went into it
    check(host(qkv), *expected(x, *wq))
    np.testing.assert_array_equal(host(vo).reshape(T, hkv, hd), values(*encode(host(v).reshape(T, hkv, hd))))
    c.k, c.v, c.ks, c.vs = (host(t) for t in (kv.k, kv.v, kv.k_scale, kv.v_scale))
    want, tol = c.attention(host(q_out).reshape(T, hq, hd), hq)
    check(host(out).reshape(T, hq, hd), want, tol)
    check(host(stream), *expected(host(out), *wo, residual=x))


def test_on_another_stream(gpu):
    c = MxCase(2, 64, 16, [(600, 1), (90, 40)], seed=12)
    q = queries(c, 4)
    kv, b = c.cache(gpu), c.batch(gpu)
    qd, out = dev(q.reshape(c.tokens, -1)), torch.zeros((c.tokens, 256), device="cuda")
    ko, vo = (torch.zeros((c.tokens, 128), device="cuda") for _ in "kv")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv.attention(b, qd, out)
        kv.read(b, ko, vo)
    side.synchronize()
    want, tol = c.attention(q, 4)
    check(host(out).reshape(want.shape), want, tol)
    for got, which in ((ko, "k"), (vo, "v")):
        rows = np.concatenate([c.rows(which, s)[0][n - m:] for s, (n, m) in enumerate(c.seqs)])
        np.testing.assert_array_equal(host(got).reshape(rows.shape), rows.astype(np.float32))


def test_refusals(gpu):
    k = torch.zeros((4, 2, 16, 32), dtype=torch.uint8, device="cuda")
    s = torch.zeros((4, 2, 16, 2), dtype=torch.uint8, device="cuda")
    gpu.PagedKV(k, k, s, s)
    for bad in (s[..., :1], s.int(), s.cpu(), torch.zeros((4, 2, 16), dtype=torch.uint8, device="cuda")):
        with pytest.raises((ValueError, TypeError)):
            gpu.PagedKV(k, k, s, bad)
    with pytest.raises(ValueError):
        gpu.PagedKV(k, k, s)
    with pytest.raises(ValueError):
        gpu.PagedKV.new(4, 16, 2, 64, "fp4")
    c = MxCase(2, 64, 16, [(5, 1)])
    kv, b = c.cache(gpu), c.batch(gpu)
    apart = torch.zeros(kv.k_scale.numel() + 2, dtype=torch.uint8, device="cuda")[2:].view(kv.k_scale.shape)
    with pytest.raises(Exception, match="4-byte"):
        gpu.PagedKV(kv.k, kv.v, apart, kv.v_scale).read(b, torch.zeros((1, 128), device="cuda"), None)


def test_pools_past_32_bits(gpu):
    # the same pages behind 2^32 bytes of codes: the same bits
    off = (1 << 26) // (8 * 16) + 3
    results = []
    for base in (0, off):
        c = MxCase(8, 128, 16, [(100, 1), (60, 40), (700, 2)], seed=13)
        q, k, v = (dev(c.rng.standard_normal((c.tokens, n * 128)).astype(np.float32)) for n in (16, 8, 8))
        pools = []
        for pool in (c.k, c.v, c.ks, c.vs):
            big = torch.zeros((base + c.pages,) + pool.shape[1:], dtype=torch.uint8, device="cuda")
            big[base:] = dev(pool)
            pools.append(big)
        c.table += base
        kv, b = gpu.PagedKV(*pools), c.batch(gpu)
        heads = gpu.GQA(dict(dim=2048, num_q=16, num_kv=8, head_dim=128))
        out, q_out = torch.zeros_like(q), torch.zeros_like(q)
        ko, vo = torch.zeros_like(k), torch.zeros_like(v)
        kv.append(b, heads, q, k, v, q_out)
        kv.attention(b, q_out, out)
        kv.read(b, ko, vo)
        results.append([host(t) for t in (out, ko, vo)] + [host(p[base:]) for p in pools])
        assert base == 0 or not any(p[:64].any() or p[base - 64:base].any() for p in pools)
        del kv, pools
    assert np.isfinite(results[0][0]).all() and results[0][0].any()
    for small, large in zip(*results):
        np.testing.assert_array_equal(small, large)


@pytest.mark.parametrize("hq,n,down", [(2, 1, False), (2, 1, True), (14, 1, False), (2, 200, False), (2, 200, True)])
def test_scores_that_rise_or_fall(gpu, hq, n, down):
    # from 2^-6 to some 60, or back: the running maximum moves by a little, then by a lot, or never again
    c = MxCase(2 if hq == 2 else 1, 64, 16, [(800, n), (30, 1)], seed=15)
    for p in range(800):
        k = c.slot(0, 799 - p if down else p)
        c.k[k] = (c.k[k] & 0x33) | 0x22  # 1 or 1.5
        c.ks[k] = 115 + p // 64
    q = np.abs(queries(c, hq)) + np.float32(0.5)
    check(attend(gpu, c, q, hq), *c.attention(q, hq))


@pytest.mark.parametrize("hq,hkv,hd,n", [(2, 1, 64, 1), (16, 8, 128, 1), (4, 1, 80, 1), (14, 2, 64, 1), (2, 1, 64, 200),
                                         (2, 1, 256, 90), (2, 1, 96, 200)])
def test_values_whose_weighted_sum_stays_in_f32(gpu, hq, hkv, hd, n):
    # the last keys outweigh the first ones by less than 2^8, and all 400 values add up to less than 2^127: weights above
    # 1 would carry the sums of a wave's keys past f32 (a page of many slots, so that one range of keys has them all)
    c = MxCase(hkv, hd, 32768, [(400, n), (30, 1)], seed=16)
    c.vs[:] = np.where(c.vs == 255, 255, 242)
    c.v &= 0x77  # positive, up to 6 * 2^115
    for p in range(400):
        k = c.slot(0, p)
        c.k[k], c.ks[k] = 0, 127
        c.k[k][:, 0] = 2 if p >= 128 else 0  # column 0: 1, or nothing
    q = np.zeros((c.tokens, hq, hd), np.float32)
    q[..., 0] = 5 * np.sqrt(hd)
    check(attend(gpu, c, q, hq, causal=False, max_new=n), *c.attention(q, hq, causal=False))


@pytest.mark.parametrize("hq,hkv,hd,n", [(2, 1, 64, 1), (16, 8, 128, 1), (2, 1, 80, 1), (14, 2, 64, 1), (2, 1, 256, 1), (2, 1, 64, 40),
                                         (8, 1, 256, 10), (6, 2, 96, 20)])
def test_values_of_the_smallest_scales(gpu, hq, hkv, hd, n):
    # byte 0 is 2^-127 here too; an output is a mean of 40 such values, whose weighted sum (weights of 2^-8) is held to
    # 2^-149 a product or addition: 2^-141 in the output, three times 40
    c = MxCase(hkv, hd, 16, [(40, n), (1, 1)], seed=17)
    c.vs[:] = np.where(c.vs == 255, 255, c.rng.integers(0, 3, c.vs.shape))
    c.k[:], c.ks[:] = 0, np.where(c.ks == 255, 255, 127)
    q = queries(c, hq)
    want, _ = c.attention(q, hq, causal=False)
    got = attend(gpu, c, q, hq, causal=False, max_new=n)
    assert (np.abs(want) > 2.0 ** -132).mean() > 0.8
    assert (np.abs(got - want) <= 120 * 2.0 ** -141).all()
