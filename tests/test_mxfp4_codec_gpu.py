"""gorch_hip_mxfp4_encode, gorch_hip_mxfp4_decode and gorch_hip_pack_mxfp4
against the format's definition: every bit, since nothing but a rounding to the
nearest of eight codes happens."""
import numpy as np
import pytest
import torch

from tests.mx_case import encode, unpack, values
from tests.paged_case import dev, host

pytestmark = pytest.mark.gpu


def rows(rng, n, cols, bf16):
    x = (rng.standard_normal((n, cols)) * np.exp(2 * rng.standard_normal((n, 1)))).astype(np.float32)
    # values that lie on the border between two codes, and on that between two scales
    x[::3] = rng.integers(-28, 29, x[::3].shape) * np.float32(0.25)
    if bf16:
        x = (x.view(np.uint32) & 0xffff0000).view(np.float32)
    return x


def run(gpu, x, bf16=False, apart=0):
    n, cols = x.shape
    kind = torch.bfloat16 if bf16 else torch.float32
    wide = torch.zeros((n, cols + apart), dtype=kind, device="cuda")
    wide[:, :cols] = dev(x).to(kind)
    codes = torch.full((n, cols // 2), 0xee, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, -(-cols // 32)), 0xee, dtype=torch.uint8, device="cuda")
    gpu.mxfp4_encode(wide[:, :cols], codes, scales)
    back = torch.full((n, cols + apart), 9.0, dtype=kind, device="cuda")
    gpu.mxfp4_decode(codes, scales, back[:, :cols])
    back = host(back.float())
    assert (back[:, cols:] == 9).all()
    return host(codes), host(scales), back[:, :cols]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,cols,apart", [(1, 8, 0), (1, 32, 0), (3, 16, 0), (5, 40, 0), (33, 1000, 0), (17, 96, 8),
                                          (64, 1024, 0), (7, 2048, 64), (1000, 24, 0), (2, 100000, 0)])
def test_codec_is_exact(gpu, bf16, n, cols, apart):
    x = rows(np.random.default_rng(n + cols), n, cols, bf16)
    codes, scales, back = run(gpu, x, bf16, apart)
    want_codes, want_scales = encode(x)
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want_codes)
    np.testing.assert_array_equal(back.astype(np.float64), values(codes, scales))


def test_no_value_moves_more_than_half_a_step(gpu):
    x = rows(np.random.default_rng(0), 50, 320, False)
    _, scales, back = run(gpu, x)
    step = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, 1)
    a = np.abs(x.astype(np.float64))
    assert (a <= 7 * step).all()
    half = step * np.where(a <= 2 * step, 0.25, np.where(a <= 4 * step, 0.5, 1.0))
    assert (np.abs(back - x.astype(np.float64)) <= half).all()


def test_every_code_and_scale_decodes(gpu):
    codes = np.tile(np.arange(256, dtype=np.uint8)[:16] * 17, (256, 1))
    codes[:, 1::2] ^= 0x5a
    scales = np.arange(256, dtype=np.uint8)[:, None]
    out = torch.empty((256, 32), device="cuda")
    gpu.mxfp4_decode(dev(codes), dev(scales), out)
    with np.errstate(over="ignore"):
        want = values(codes, scales).astype(np.float32)  # (6 * 2^127 is past f32)
    np.testing.assert_array_equal(host(out), want)


def test_extremes(gpu):
    x = np.zeros((12, 64), np.float32)
    x[1, 3], x[2, 40], x[3, 5] = np.inf, np.nan, -np.inf
    x[4] = 3.4028235e38
    x[5] = 1e-38
    x[6, 7] = -1e-45
    x[7] = np.float32(2.0 ** -100)
    x[8] = np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    x[9, :32] = -0.0
    x[10, 0], x[10, 1] = 7.0, np.float32(2.0 ** -20)
    x[11, 0], x[11, 1] = np.nextafter(np.float32(7), np.float32(8)), -0.75
    codes, scales, back = run(gpu, x)
    want_codes, want_scales = encode(x)
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want_codes)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(back, values(codes, scales).astype(np.float32))
    assert np.isnan(back[1, :32]).all() and (back[1, 32:] == 0).all()


def test_empty_and_wide(gpu):
    for shape in ((0, 32), (3, 0)):
        x = torch.empty(shape, device="cuda")
        codes = torch.empty((shape[0], shape[1] // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((shape[0], shape[1] // 32), dtype=torch.uint8, device="cuda")
        gpu.mxfp4_encode(x, codes, scales)
        gpu.mxfp4_decode(codes, scales, x)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [1 << 20, (1 << 20) + 8])
def test_offsets_past_32_bits(gpu, bf16, cols):
    # bytes, and of the bf16 rows elements too, past 2^32
    n = 4100
    x = torch.zeros((n, cols), dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    rng = np.random.default_rng(1)
    some = {r: rows(rng, 1, cols, bf16)[0] for r in (0, 2047, 4096, n - 1)}
    for r, v in some.items():
        x[r] = dev(v).to(x.dtype)
    codes = torch.full((n, cols // 2), 7, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, -(-cols // 32)), 7, dtype=torch.uint8, device="cuda")
    gpu.mxfp4_encode(x, codes, scales)
    x.fill_(3)
    gpu.mxfp4_decode(codes, scales, x)
    for r, v in some.items():
        want_codes, want_scales = encode(v[None])
        np.testing.assert_array_equal(host(codes[r]), want_codes[0])
        np.testing.assert_array_equal(host(scales[r]), want_scales[0])
        np.testing.assert_array_equal(host(x[r].float()), values(want_codes, want_scales)[0].astype(np.float32))
    assert int(codes.count_nonzero(dim=1).count_nonzero()) <= len(some)  # the other rows are zeros


@pytest.mark.parametrize("N,K", [(1, 8), (16, 128), (17, 136), (50, 1600), (33, 520), (5, 4864)])
def test_pack_holds_every_code_once(gpu, N, K):
    rng = np.random.default_rng(N)
    codes = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    scales = rng.integers(0, 255, (N, -(-K // 32))).astype(np.uint8)
    got = host(gpu.pack_mxfp4(dev(codes), dev(scales)))
    nt, nk = -(-N // 16), -(-K // 128)
    nq = -(-nk // 4)
    c = np.zeros((16 * nt, 128 * nk), np.uint8)
    c[:N, :K] = unpack(codes)
    c = (c[:, 0::2] | c[:, 1::2] << 4).reshape(nt, 16, nk, 4, 16)  # tile, row, column tile, group, byte
    s = np.zeros((16 * nt, 16 * nq), np.uint8)
    s[:N, :scales.shape[1]] = scales
    s = s.reshape(nt, 16, nq, 4, 4)  # tile, row, word, column tile of it, group
    np.testing.assert_array_equal(got[:nt * nk * 1024], c.transpose(0, 2, 3, 1, 4).ravel())
    np.testing.assert_array_equal(got[nt * nk * 1024:], s.transpose(0, 2, 4, 1, 3).ravel())


def test_on_another_stream_and_captured(gpu):
    x = rows(np.random.default_rng(5), 40, 520, False)
    xd, back = dev(x), torch.zeros((40, 520), device="cuda")
    codes, scales = (torch.zeros((40, n), dtype=torch.uint8, device="cuda") for n in (260, 17))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        gpu.mxfp4_encode(xd, codes, scales)
        gpu.mxfp4_decode(codes, scales, back)
    for turn in range(3):
        y = np.roll(x, turn, 0)
        xd.copy_(dev(y))
        back.zero_()
        graph.replay()
        np.testing.assert_array_equal(host(back).astype(np.float64), values(*encode(y)))


def test_refusals(gpu):
    x = torch.zeros((4, 64), device="cuda")
    codes, scales = (torch.zeros((4, n), dtype=torch.uint8, device="cuda") for n in (32, 2))
    for call in (lambda *a: gpu.mxfp4_encode(*a), lambda v, c, s: gpu.mxfp4_decode(c, s, v)):
        call(x, codes, scales)
        for bad in ((x.half(), codes, scales), (x.cpu(), codes, scales), (x[:, ::2], codes[:, :16], scales[:, :1]),
                    (x[0], codes, scales), (x, codes[:, :31], scales), (x, codes, scales[:, :1]), (x, codes.int(), scales),
                    (x, codes, scales.cpu()), (x[:1].expand(4, 64), codes, scales)):
            with pytest.raises((ValueError, TypeError)):
                call(*bad)
        with pytest.raises(Exception, match="multiple of 8"):
            call(x[:, :60], codes[:, :30].contiguous(), scales)
