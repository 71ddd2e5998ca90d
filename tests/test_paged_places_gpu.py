"""Where gorch_hip_paged_append writes: the scales of slots that no token has
stay as they were, and a pool past 32-bit offsets gets what a small one gets."""
import numpy as np
import pytest
import torch

from tests.paged_case import Case, dev, host
from tests.test_paged_append_gpu import append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 64), (8, 1, 256), (6, 2, 96), (3, 3, 16)])
def test_append_leaves_the_other_scales(gpu, hq, hkv, hd):
    # tokens at negative positions, past max_kv, past the RoPE tables and on no page write nothing, scales included
    c = Case("e4m3", hkv, hd, 16, [(3, 5), (0, 0), (60, 20), (100, 70), (30, 30)], seed=hd)
    for scales in (c.ks, c.vs):  # every slot has one to lose, NaN where no token is
        scales[np.isfinite(scales)] = 5.0
    c.table[3, 2], c.table[3, 3], c.table[4, 0] = -1, c.pages, 1 << 30
    _, _, _, pools, scales = append(gpu, c, hq, True, True, extra=2, rope_rows=85, max_kv=90)
    written = np.zeros((c.pages, c.page), bool)
    for s, (length, n) in enumerate(c.seqs):
        for p in range(max(length - n, 0), min(length, 85)):
            page = c.table[s, p // 16]
            if 0 <= page < c.pages:
                written[page, p % 16] = True
    for got, was in zip(scales, (c.ks, c.vs)):
        got, was = (np.moveaxis(x.view(np.uint32), 1, 2) for x in (got, was))
        assert np.array_equal(got[~written], was[~written])
        assert (got[written] != was[written]).any(-1).all()
    for got, was in zip(pools, (c.k, c.v)):
        assert np.array_equal(np.moveaxis(got, 1, 2)[~written], np.moveaxis(was, 1, 2)[~written])


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_append_past_32_bits(gpu, dtype):
    # the last pages of a pool of 5 * 2^30 elements hold what a small pool holds
    hq, hkv, page, hd = 16, 8, 64, 128
    pages = (5 << 30) // (hkv * page * hd)
    c = Case(dtype, hkv, hd, page, [(200, 70), (5, 1)], seed=21, spare=0)
    x = dev(c.rng.standard_normal((c.tokens, (hq + 2 * hkv) * hd)).astype(np.float32))
    q, k, v = x.split([hq * hd, hkv * hd, hkv * hd], 1)
    heads = gpu.GQA(dict(dim=8, num_q=hq, num_kv=hkv, head_dim=hd))
    small = c.cache(gpu)
    outs = [torch.full((c.tokens, hq * hd), 7.0, device="cuda") for _ in "ab"]
    small.append(c.batch(gpu), heads, q, k, v, outs[0])
    kind = torch.int16 if dtype == "bf16" else torch.uint8
    pools = [torch.zeros((pages, hkv, page, hd), dtype=kind, device="cuda") for _ in "kv"]
    scales = [None if dtype == "bf16" else torch.zeros((pages, hkv, page), device="cuda") for _ in "kv"]
    olds = (small.k, small.v, small.k_scale, small.v_scale)
    for big, was in zip((*pools, *scales), (c.k, c.v, c.ks, c.vs)):
        if big is not None:
            big[-c.pages:] = dev(was.view(np.int16) if was.dtype == np.uint16 else was)
    b = gpu.PagedBatch(dev(c.cu), dev(c.lens), dev(c.table + np.int32(pages - c.pages)), c.tokens)
    gpu.PagedKV(*pools, *scales).append(b, heads, q, k, v, outs[1])
    assert torch.equal(*outs)
    for big, want in zip((*pools, *scales), olds):
        if big is not None:
            got, want = (host(t.contiguous().view(torch.uint8)) for t in (big[-c.pages:], want))
            assert np.array_equal(got, want)
            assert not big[:-c.pages].any().item()
