"""CPU-only checks of the four-bit operators' refusals and sizes: every
argument check comes before any device work, so fake pointers reach it."""
import ctypes as C

import pytest

from gorch_amd import hip
from tests.test_paged_args import FAKE, ODD, append, attend, batch, cache, heads, read

L = hip.lib


def encode(x=FAKE, bf16=0, stride=64, codes=FAKE, scales=FAKE, rows=4, cols=64):
    return L().gorch_hip_mxfp4_encode(None, x, bf16, stride, codes, scales, rows, cols)


def decode(x=FAKE, bf16=0, stride=64, codes=FAKE, scales=FAKE, rows=4, cols=64):
    return L().gorch_hip_mxfp4_decode(None, codes, scales, x, bf16, stride, rows, cols)


BAD_CODEC = [(dict(rows=-1), 2), (dict(cols=-8), 2), (dict(cols=1 << 31), 2), (dict(x=None), 2), (dict(codes=None), 2),
             (dict(scales=None), 2), (dict(stride=56), 2), (dict(stride=-64), 2), (dict(cols=60), 1), (dict(cols=4), 1),
             (dict(x=ODD), 1), (dict(codes=FAKE + 2), 1), (dict(stride=66), 1), (dict(stride=68, bf16=1), 1),
             (dict(rows=1 << 36), 1)]


@pytest.mark.parametrize("call,name", [(encode, "mxfp4_encode"), (decode, "mxfp4_decode")])
@pytest.mark.parametrize("over,rc", BAD_CODEC)
def test_codec_refusals(call, name, over, rc):
    assert call(**over) == rc and name in hip.last_error()


@pytest.mark.parametrize("call", [encode, decode])
def test_codec_of_nothing(call):
    assert call(rows=0, x=None, codes=None, scales=None) == 0
    assert call(cols=0, stride=0, x=None, codes=None, scales=None) == 0


@pytest.mark.parametrize("over,rc", [(dict(N=-1), 2), (dict(K=-8), 2), (dict(codes=None), 2), (dict(scales=None), 2),
                                     (dict(Wp=None), 2), (dict(K=12), 1), (dict(codes=FAKE + 2), 1), (dict(Wp=FAKE + 8), 1),
                                     (dict(N=1 << 20), 1)])
def test_pack_refusals(over, rc):
    a = dict(codes=FAKE, scales=FAKE, Wp=FAKE, N=16, K=64)
    a.update(over)
    assert L().gorch_hip_pack_mxfp4(None, *a.values()) == rc and "pack_mxfp4" in hip.last_error()


def test_packed_bytes():
    size = L().gorch_hip_packed_mxfp4_bytes
    assert size(0, 64) == size(64, 0) == size(-1, 64) == 0
    assert size(1, 8) == size(16, 128) == 1024 + 256
    assert size(17, 128) == 2 * (1024 + 256)
    assert size(16, 1600) == 13 * 1024 + 4 * 256
    assert size(1 << 19, 16640) == (1 << 15) * (130 * 1024 + 33 * 256)


def linear(x=FAKE, Wp=FAKE, bias=None, residual=None, y=FAKE + 64, M=4, N=16, K=64, epi=0, ws=None, n=0):
    return L().gorch_hip_linear_mxfp4(None, x, Wp, bias, residual, y, M, N, K, epi, ws, n)


@pytest.mark.parametrize("over,rc", [(dict(M=-1), 2), (dict(N=-1), 2), (dict(K=-8), 2), (dict(K=0), 2), (dict(x=None), 2),
                                     (dict(Wp=None), 2), (dict(y=None), 2), (dict(y=FAKE), 2), (dict(epi=2), 2),
                                     (dict(K=20), 1), (dict(x=ODD), 1), (dict(Wp=FAKE + 8), 1), (dict(M=17), 2),
                                     (dict(M=17, ws=FAKE, n=8), 2), (dict(M=17, ws=None, n=1 << 30), 2),
                                     (dict(M=17, ws=FAKE + 8, n=1 << 30), 1), (dict(M=(1 << 20) + 1), 1),
                                     (dict(N=1 << 20), 1), (dict(K=(1 << 24) + 8), 1)])
def test_linear_refusals(over, rc):
    assert linear(**over) == rc and "linear_mxfp4" in hip.last_error()


def test_linear_of_nothing_and_workspaces():
    assert linear(M=0, x=None, Wp=None, y=None) == 0 and linear(N=0, x=None, Wp=None, y=None) == 0
    size = L().gorch_hip_linear_mxfp4_workspace_size
    assert size(0, 16, 64) == size(-1, 16, 64) == size(16, 0, 64) == size(17, 16, 0) == 0
    assert size(1, 4096, 1024) == 0 and size(1, 16, 8192) > 0 and size(17, 16, 128) > 0 and size(2000, 16, 4096) >= 125 * 32 * 7680


MX = dict(dtype=2, k_scale=FAKE, v_scale=FAKE)


@pytest.mark.parametrize("over,rc", [(dict(k_scale=None), 2), (dict(v_scale=None), 2), (dict(head_dim=72), 1),
                                     (dict(head_dim=272), 1), (dict(k=ODD), 1), (dict(k_scale=FAKE + 2), 1),
                                     (dict(v_scale=FAKE + 1), 1), (dict(dtype=3), 2), (dict(dtype=-1), 2)])
def test_cache_refusals(over, rc):
    kv, b = cache(**{**MX, **over}), batch()
    w = heads(head_dim=kv.head_dim, num_kv=kv.num_kv)
    assert attend(kv, b) == rc and "paged_attention" in hip.last_error()
    assert append(kv, b, w) == rc and "paged_append" in hip.last_error()
    assert read(kv, b) == rc and "paged_read" in hip.last_error()


def test_an_empty_batch_is_nothing():
    kv = cache(**MX)
    for over in (dict(tokens=0), dict(seqs=0)):
        assert attend(kv, batch(**over)) == 0 and append(kv, batch(**over), heads()) == 0 and read(kv, batch(**over)) == 0


def test_attention_workspace_is_checked():
    kv, b = cache(**MX, num_pages=1 << 20), batch(tokens=1, seqs=1, max_pages=4096, max_new=1)
    need = L().gorch_hip_paged_attention_workspace_size(C.byref(kv), C.byref(b), 4)
    assert need > 0
    assert attend(kv, b, ws=FAKE, n=need - 1) == 2 and attend(kv, b, ws=None, n=need) == 2
    assert attend(kv, b, ws=FAKE + 8, n=need) == 1


@pytest.mark.parametrize("head_dim", [17, 33, 49, 127])
def test_new_pools_of_an_odd_head_are_refused(head_dim):
    # (half of it rounded down would be the pools of another head)
    with pytest.raises(ValueError, match="even"):
        hip.PagedKV.new(4, 16, 2, head_dim, "mxfp4")
