"""gorch_hip_paged_read in all the forms that it chooses by a token's columns and
the number of tokens, in each cache type: 32, 64, 128 or 256 lanes a token, one
token or four in turn."""
import numpy as np
import pytest
import torch

from tests.mx_case import values
from tests.paged_case import E4M3, dev, host

pytestmark = pytest.mark.gpu

SENTINEL = 123.0


def pool(rng, dtype, shape):
    """Codes, scales (or None) and values in f32 of a pool [pages, KV heads, page size, columns]."""
    if dtype == "bf16":
        bits = (rng.standard_normal(shape).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
        return bits.view(np.int16), None, (bits.astype(np.uint32) << 16).view(np.float32)
    if dtype == "e4m3":
        codes = rng.integers(0, 127, shape).astype(np.uint8) + rng.integers(0, 2, shape).astype(np.uint8) * np.uint8(128)
        scales = np.exp2(rng.integers(-9, 3, shape[:3])).astype(np.float32)
        return codes, scales, (E4M3[codes] * scales[..., None]).astype(np.float32)
    codes = rng.integers(0, 256, shape[:3] + (shape[3] // 2,)).astype(np.uint8)
    scales = rng.integers(0, 250, shape[:3] + (-(-shape[3] // 32),)).astype(np.uint8)
    return codes, scales, values(codes, scales).astype(np.float32)


# tokens from which four are taken in turn: 2^15 / (lanes / 32); fewer than 32 lanes' columns take 64 up to 4,096 tokens
@pytest.mark.parametrize("dtype", ["bf16", "e4m3", "mxfp4"])
@pytest.mark.parametrize("hkv,hd,four", [(1, 32, 32768), (3, 16, 32768), (1, 128, 32768), (2, 80, 16384), (2, 128, 16384),
                                         (3, 112, 8192), (4, 128, 8192), (8, 128, 4096), (9, 128, 4096)])
def test_many_tokens(gpu, dtype, hkv, hd, four):
    rng = np.random.default_rng(hd)
    page, pages = 24, 700
    k, v = pool(rng, dtype, (pages, hkv, page, hd)), pool(rng, dtype, (pages, hkv, page, hd))
    kv = gpu.PagedKV(*(dev(t) if t is not None else None for t in (k[0], v[0], k[1], v[1])))
    # one token short of four in turn, then the fewest of them and some more: no tokens of some sequences, an end inside a
    # block, pages that many sequences share, some that do not exist, rows behind the last sequence
    for tokens in (four - 1, four, four + 8 * page + 5):
        new = [tokens // 3, 0, 1, tokens // 2, 0]
        new += [tokens - sum(new)]
        lens = [n + (0 if i % 2 else 37) for i, n in enumerate(new)]
        table = rng.integers(0, pages, (len(new), -(-max(lens) // page))).astype(np.int32)
        table[0, 2], table[3, 1], table[5, 0] = -1, pages, -(1 << 31)
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        b = gpu.PagedBatch(dev(cu), dev(np.array(lens, np.int32)), dev(table), tokens + 3)
        outs = [torch.full((tokens + 3, hkv * hd), SENTINEL, device="cuda") for _ in "kv"]
        kv.read(b, *outs)
        seq = np.repeat(np.arange(len(new)), new)
        pos = np.array(lens)[seq] - np.array(new)[seq] + np.arange(tokens) - cu[seq]
        at = table[seq, pos // page]
        there = (at >= 0) & (at < pages)
        assert not there.all()
        for out, (_, _, held) in zip(outs, (k, v)):
            want = np.full((tokens + 3, hkv, hd), SENTINEL, np.float32)
            want[:tokens][there] = held[at[there], :, pos[there] % page]
            np.testing.assert_array_equal(host(out).reshape(want.shape), want)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3", "mxfp4"])
@pytest.mark.parametrize("hkv,hd", [(1, 32), (2, 64), (2, 128), (4, 128), (8, 128)])
@pytest.mark.parametrize("tokens", [1, 3, 4096, 4097])
def test_few_tokens(gpu, dtype, hkv, hd, tokens):
    rng = np.random.default_rng(tokens)
    page, pages = 16, 300
    k, v = pool(rng, dtype, (pages, hkv, page, hd)), pool(rng, dtype, (pages, hkv, page, hd))
    kv = gpu.PagedKV(*(dev(t) if t is not None else None for t in (k[0], v[0], k[1], v[1])))
    table = rng.integers(0, pages, (1, -(-(tokens + 5) // page))).astype(np.int32)
    b = gpu.PagedBatch(dev(np.array([0, tokens], np.int32)), dev(np.array([tokens + 5], np.int32)), dev(table), tokens)
    only = torch.full((tokens, hkv * hd), SENTINEL, device="cuda")
    kv.read(b, None, only)
    pos = np.arange(5, tokens + 5)
    np.testing.assert_array_equal(host(only).reshape(tokens, hkv, hd), v[2][table[0, pos // page], :, pos % page])
