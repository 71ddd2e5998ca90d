"""gorch_hip_paged_append and gorch_hip_paged_read against their definitions
in 64 bits: norms and rotations of both pairings, head layouts, fused and
separate projections, both cache types, tokens without a place, and what must
stay as it was."""
import numpy as np
import pytest
import torch

from tests.paged_case import E4M3, Case, dev, host

pytestmark = pytest.mark.gpu

SENTINEL = 77.0
U = 2.0 ** -24  # half a step of f32


def tables(hd, rows, rng):
    a = rng.uniform(0, 6.28, (rows, hd // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def finished(x, gain, eps, cos, sin, neox):
    """x [n, heads, hd] f32 -> norm and rotation in 64 bits, and the bound of
    the f32 result: with a norm, the reciprocal root and two products round
    (3 U, 4 with the f64 statistics' own last places); the rotation rounds two
    products and a sum (each of the two terms twice: 2 U of their magnitudes)."""
    y = x.astype(np.float64)
    tol = np.zeros_like(y)
    if gain is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * gain.astype(np.float64)
        tol = 4 * U * np.abs(y)
    if cos is not None:
        c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
        half = x.shape[-1] // 2
        a, b = (np.s_[..., 0::2], np.s_[..., 1::2]) if neox else (np.s_[..., :half], np.s_[..., half:])
        z, t = np.empty_like(y), np.empty_like(y)
        z[a], z[b] = y[a] * c - y[b] * s, y[a] * s + y[b] * c
        t[a] = (tol[a] + 2 * U * np.abs(y[a])) * np.abs(c) + (tol[b] + 2 * U * np.abs(y[b])) * np.abs(s)
        t[b] = (tol[a] + 2 * U * np.abs(y[a])) * np.abs(s) + (tol[b] + 2 * U * np.abs(y[b])) * np.abs(c)
        y, tol = z, t
    return y, tol


def append(gpu, c, hq, norm, rope, neox=0, fused=True, rope_rows=None, in_place=False, with_q=True, extra=0, **bounds):
    """Runs an append of random rows; returns (x, params, q_out, k, v, ks, vs)."""
    T, hd, hkv = c.tokens + extra, c.hd, c.hkv
    widths = [hq * hd, hkv * hd, hkv * hd]
    x = (c.rng.standard_normal((T, sum(widths))) * np.exp(c.rng.standard_normal((T, 1)))).astype(np.float32)
    most = int(max(c.lens, default=1)) if rope_rows is None else rope_rows
    gq, gk = ((1 + 0.3 * c.rng.standard_normal(hd)).astype(np.float32) for _ in "qk")
    cos, sin = tables(hd, max(most, 1), c.rng)
    w = dict(dim=8, num_q=hq, num_kv=hkv, head_dim=hd, norm_eps=1e-6, rope_neox=neox)
    if norm:
        w.update(q_norm=gq, k_norm=gk)
    if rope:
        w.update(rope=True, rope_cos=dev(cos), rope_sin=dev(sin), rope_max_seq=max(most, 1))
    heads = gpu.GQA(w)
    if fused:
        q, k, v = dev(x).split(widths, 1)
    else:
        q, k, v = (t.contiguous() for t in dev(x).split(widths, 1))
    q_out = q if in_place else torch.full((T, hq * hd), SENTINEL, device="cuda")
    kv, b = c.cache(gpu), c.batch(gpu, extra, **bounds)
    kv.append(b, heads, q if with_q else None, k, v, q_out if with_q else None)
    pools = [host(p.view(torch.int16).view(torch.uint16) if p.dtype == torch.bfloat16 else p) for p in (kv.k, kv.v)]
    pools = [p.view(np.uint16) if c.dtype == "bf16" else p.view(np.uint8) for p in pools]
    scales = [None, None] if c.dtype == "bf16" else [host(kv.k_scale), host(kv.v_scale)]
    return x, (gq if norm else None, gk if norm else None, cos if rope else None, sin if rope else None), \
        host(q_out), pools, scales


def check(c, hq, x, params, q_out, pools, scales, neox=0, skipped=lambda s, p: False, with_q=True):
    gq, gk, cos, sin = params
    hkv, hd = c.hkv, c.hd
    want_pools = [c.k.copy(), c.v.copy()]
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
            q, qt = finished(rows[None, :hq], gq, 1e-6, co, si, neox)
            k, kt = finished(rows[None, hq:hq + hkv], gk, 1e-6, co, si, neox)
            v, vt = rows[None, hq + hkv:].astype(np.float64), np.zeros((1, hkv, hd))
            if with_q:
                assert (np.abs(q_out[t].reshape(1, hq, hd) - q) <= qt).all()
            for j, (y, yt) in enumerate(((k[0], kt[0]), (v[0], vt[0]))):
                got = pools[j][at]
                if c.dtype == "bf16":
                    g = (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
                    # half a bf16 step of the value, 2^-8, and where the f32 value stood
                    assert (np.abs(g - y) <= yt * 1.01 + 2.0 ** -8 * np.abs(y)).all()
                else:
                    sc = scales[j][at].astype(np.float64)
                    amax = np.abs(y).max(-1)
                    assert (np.abs(sc - amax / 448) <= (yt.max(-1) + 2 * U * amax) / 448).all()
                    # half an e4m3 step: 2^-4 of the value, or 2^-10 scales below the normal range; the
                    # quotient's own roundings move the value by 4 U at most
                    g = E4M3[got] * sc[:, None]
                    assert (np.abs(g - y) <= 1.01 * yt + 4 * U * amax[:, None] +
                            np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * sc[:, None])).all()
    # everything else is as it was
    for got, was in zip(pools, want_pools):
        for page in range(c.pages):
            keep = ~touched[page]
            assert np.array_equal(got[page][:, keep], was[page][:, keep])


LAYOUTS = [(16, 8, 128), (14, 2, 64), (12, 12, 64), (8, 1, 256), (6, 2, 96), (20, 1, 80), (3, 3, 16), (40, 2, 48)]


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("norm,rope,neox", [(True, True, 0), (False, True, 1), (True, False, 0), (False, False, 0),
                                            (True, True, 1)])
def test_append_matches_definition(gpu, dtype, hq, hkv, hd, norm, rope, neox):
    c = Case(dtype, hkv, hd, 24, [(0, 0), (40, 7), (1, 1), (0, 0), (130, 30), (25, 25)], seed=hd + neox, fill=False)
    check(c, hq, *append(gpu, c, hq, norm, rope, neox, fused=norm), neox=neox)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("seqs,bounds", [([(777, 1)], dict(max_new=1)), ([(9 + i, 1) for i in range(100)], dict(max_new=1)),
                                         ([(9 + i, 1) for i in range(100)], {}), ([(1000, 1000), (3, 3)], {}),
                                         ([(i % 3, i % 3) for i in range(300)], dict(max_new=2)),
                                         # max_new is a bound that the kernels do not rely on
                                         ([(5, 2), (4, 0), (9, 1), (8, 1)], dict(max_new=1))])
def test_append_batches(gpu, dtype, seqs, bounds):
    c = Case(dtype, 2, 64, 16, seqs, seed=3, fill=False)
    check(c, 4, *append(gpu, c, 4, True, True, extra=5, **bounds))


def test_append_without_q(gpu):
    c = Case("bf16", 2, 64, 16, [(40, 9)], seed=4, fill=False)
    check(c, 4, *append(gpu, c, 4, True, True, with_q=False), with_q=False)


@pytest.mark.parametrize("neox", [0, 1])
def test_append_q_in_place(gpu, neox):
    c = Case("bf16", 2, 128, 16, [(40, 9)], seed=4, fill=False)
    check(c, 4, *append(gpu, c, 4, True, True, neox, fused=False, in_place=True), neox=neox)


def test_tokens_without_a_place_are_skipped(gpu):
    # a negative position, one past max_kv, one past the RoPE tables, and bad pages
    c = Case("e4m3", 2, 64, 16, [(3, 5), (60, 20), (100, 70), (30, 30)], seed=5, fill=False)
    c.table[2, 4], c.table[2, 5], c.table[3, 0] = -1, c.pages, 1 << 30
    none = lambda s, p: p >= 90 or p >= 95 or not 0 <= c.table[s, p // 16] < c.pages  # noqa: E731
    check(c, 4, *append(gpu, c, 4, True, True, rope_rows=95, max_kv=90), skipped=none)
    c = Case("bf16", 2, 64, 16, [(100, 70)], seed=6, fill=False)
    check(c, 4, *append(gpu, c, 4, True, True, rope_rows=80), skipped=lambda s, p: p >= 80)


def test_quantised_rows_of_odd_values(gpu):
    # zeros, tiny rows, infinities, NaN, the largest and subnormal values
    c = Case("e4m3", 1, 64, 16, [(8, 8)], seed=7, fill=False)
    x = np.zeros((8, 128), np.float32)
    x[1, :64] = 1e-38
    x[2, 5], x[2, 6] = np.inf, 1.0
    x[3, 5], x[3, 6] = np.nan, 1.0
    x[4, :64] = 3e38
    x[5, 0], x[5, 1] = -448.0, 0.013671875  # 7 / 512: a subnormal code's value
    x[6, 0], x[6, 1:4] = 1.0, [2.0 ** -18, 2.0 ** -20, -2.0 ** -17]
    x[7, :64] = -1e-30
    kv, b = c.cache(gpu), c.batch(gpu)
    k, v = (t.contiguous() for t in dev(x).split([64, 64], 1))
    heads = gpu.GQA(dict(dim=8, num_q=1, num_kv=1, head_dim=64))
    kv.append(b, heads, None, k, v, None)
    ko, vo = (torch.empty((8, 64), device="cuda") for _ in "kv")
    kv.read(b, ko, vo)
    got = host(ko)
    assert (got[0] == 0).all() and (got[1] == 0).all() and (host(vo) == 0).all()
    assert np.isnan(got[2]).all()
    assert np.isnan(got[3, 5]) and abs(got[3, 6] - 1) <= 2 * U and (got[3, 7:] == 0).all()
    np.testing.assert_allclose(got[4], 3e38, rtol=4 * U)
    np.testing.assert_allclose(got[5, :2], x[5, :2], rtol=4 * U)
    np.testing.assert_allclose(got[6, :4], [1, 2.0 ** -18, 0, -2.0 ** -17], rtol=0, atol=2.0 ** -10 / 448 + 4 * U)
    np.testing.assert_allclose(got[7], -1e-30, rtol=4 * U)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hkv,hd,page", [(8, 128, 16), (2, 64, 7), (1, 256, 64), (5, 48, 1), (25, 64, 32)])
def test_read_is_the_cache(gpu, dtype, hkv, hd, page):
    # every value bit for bit (a code times its scale, rounded once)
    c = Case(dtype, hkv, hd, page, [(33, 33), (0, 0), (100, 20), (1, 1), (2, 5)], seed=8)
    c.table[2, -1 if page > 64 else c.table[2].shape[0] - 1] = c.table[2, -1]
    last = (100 - 1) // page
    c.table[2, last] = -3
    kv, b = c.cache(gpu), c.batch(gpu, 2)
    outs = [torch.full((c.tokens + 2, hkv * hd), SENTINEL, device="cuda") for _ in "kv"]
    kv.read(b, *outs)
    want = [np.full((c.tokens + 2, hkv * hd), SENTINEL, np.float32) for _ in "kv"]
    for s, (length, n) in enumerate(c.seqs):
        for i in range(n):
            p = length - n + i
            for w, name in zip(want, "kv"):
                r = c.row(name, s, p) if p >= 0 else None
                if r is not None:
                    w[c.cu[s] + i] = r.astype(np.float32).reshape(-1)
    assert np.array_equal(host(outs[0]), want[0]) and np.array_equal(host(outs[1]), want[1])
    only = torch.full_like(outs[0], SENTINEL)
    kv.read(b, None, only)
    assert np.array_equal(host(only), want[1])
    kv.read(b, only, None)
    assert np.array_equal(host(only), want[0])


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_read_of_many_tokens(gpu, dtype):
    # more tokens than the small blocks take, none of some sequences, an end inside a block
    c = Case(dtype, 1, 32, 16, [(3001, 3001), (0, 0), (1500, 1210), (2, 1)], seed=9)
    kv, b = c.cache(gpu), c.batch(gpu, 1)
    outs = [torch.full((c.tokens + 1, 32), SENTINEL, device="cuda") for _ in "kv"]
    kv.read(b, *outs)
    for out, name in zip(outs, "kv"):
        got = host(out)
        want = np.concatenate([c.rows(name, s)[0][length - n:] for s, (length, n) in enumerate(c.seqs) if n])
        assert np.array_equal(got[:c.tokens], want.reshape(c.tokens, 32).astype(np.float32))
        assert (got[c.tokens:] == SENTINEL).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_serving_step(gpu, dtype):
    """One layer of a serving step from the framework's own pieces: a fused QKV Linear, append, attention, the Wo
    Linear, logits under their rules and a token drawn, for a prompt's chunks and then single tokens; the attention
    checked against the same rows in the contiguous f32 cache of what the pages hold, and the pages against the
    read-back."""
    import math

    rng = np.random.default_rng(3)
    hq, hkv, hd, dim, vocab, page = 4, 2, 64, 256, 1000, 16
    width = (hq + 2 * hkv) * hd
    wqkv, wo, wlm = (dev((rng.standard_normal(s) / 16).astype(np.float32)).bfloat16().view(torch.int16)
                     for s in ((width, dim), (dim, hq * hd), (vocab, dim)))
    cos, sin = gpu.rope_tables(hd, 256, 10000.0)
    heads = gpu.GQA(dict(dim=dim, num_q=hq, num_kv=hkv, head_dim=hd, rope=True, rope_cos=cos, rope_sin=sin,
                         rope_max_seq=256))
    kv = gpu.PagedKV.new(40, page, hkv, hd, dtype)
    table = dev(rng.permutation(40)[:32].reshape(2, 16).astype(np.int32))
    lens = np.zeros(2, np.int32)
    spoken = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    for step, new in enumerate([(37, 90), (40, 1), (1, 1), (1, 1)]):
        lens += np.array(new, np.int32)
        T = sum(new)
        b = gpu.PagedBatch(dev(np.cumsum([0, *new]).astype(np.int32)), dev(lens), table, T, max_new=max(new),
                           max_kv=int(lens.max()))
        x = dev(rng.standard_normal((T, dim)).astype(np.float32))
        qkv = torch.empty((T, width), device="cuda")
        gpu.linear_bf16(x, wqkv, None, qkv)
        q, k, v = qkv.split([hq * hd, hkv * hd, hkv * hd], 1)
        q_out, out, y = (torch.empty((T, w), device="cuda") for w in (hq * hd, hq * hd, dim))
        kv.append(b, heads, q, k, v, q_out)
        kv.attention(b, q_out, out)
        # the whole cache read back, into the contiguous form
        whole = gpu.PagedBatch(dev(np.cumsum([0, *lens]).astype(np.int32)), dev(lens), table, int(lens.sum()))
        kc, vc = (torch.empty((int(lens.sum()), hkv * hd), device="cuda") for _ in "kv")
        kv.read(whole, kc, vc)
        at = row = 0
        for s, n in enumerate(new):
            L = int(lens[s])
            ref = torch.empty((n, hq * hd), device="cuda")
            gpu.gqa_attention_cached(q_out[row:row + n].contiguous(), kc[at:at + L].contiguous(),
                                     vc[at:at + L].contiguous(), ref, 1, n, L - n, hq, hkv, hd, L)
            # both follow the same definition in f32; scores of a few units
            assert (out[row:row + n] - ref).abs().max().item() <= 2.0 ** -16 * vc.abs().max().item()
            at, row = at + L, row + n
        gpu.linear_bf16(out, wo, None, y, residual=x)
        ends = torch.tensor([new[0] - 1, T - 1], device="cuda")
        logits = torch.empty((2, vocab), device="cuda")
        gpu.linear_bf16(y[ends].contiguous(), wlm, None, logits)
        allowed = torch.zeros((2, math.ceil(vocab / 32)), dtype=torch.int32, device="cuda")
        allowed[:, 3] = 0x0ff0
        gpu.process_logits(logits, logits, history=spoken, repetition=torch.full((2,), 1e6, device="cuda"),
                           allowed=allowed)
        tok = torch.empty(2, dtype=torch.int32, device="cuda")
        gpu.sample(logits, 0.7, 4, 0.0, torch.full((2,), 0.3, dtype=torch.float64, device="cuda"), tok)
        got = host(tok)
        assert ((got >= 100) & (got < 108)).all()
        spoken[:, step] = tok
