"""CPU-only checks of the paged cache's and the logits rules' refusals: every
argument check comes before any device work, so fake pointers reach it."""
import ctypes as C

import pytest

from gorch_amd import hip

FAKE, ODD = 0x10000, 0x10004


def cache(**over):
    s = hip._PagedKVC(hip.KV_BF16, 8, 16, 2, 64, FAKE, FAKE, None, None)
    for k, v in over.items():
        setattr(s, k, v)
    return s


def batch(**over):
    s = hip._PagedBatchC(4, 2, 4, 0, 0, FAKE, FAKE, FAKE)
    for k, v in over.items():
        setattr(s, k, v)
    return s


def heads(**over):
    s = hip._GQAW()
    s.num_q, s.num_kv, s.head_dim, s.norm_eps = 4, 2, 64, 1e-6
    for k, v in over.items():
        setattr(s, k, v)
    return s


def attend(kv, b, q=FAKE, num_q=4, out=FAKE, ws=None, n=0):
    return hip.lib().gorch_hip_paged_attention(None, C.byref(kv), C.byref(b), q, num_q, out, 1, ws, n)


def append(kv, b, w, q=FAKE, qs=256, k=FAKE, ks=128, v=FAKE, vs=128, out=FAKE + 64):
    return hip.lib().gorch_hip_paged_append(None, C.byref(kv), C.byref(b), C.byref(w), q, qs, k, ks, v, vs, out)


def read(kv, b, ko=FAKE, vo=FAKE):
    return hip.lib().gorch_hip_paged_read(None, C.byref(kv), C.byref(b), ko, vo)


BAD_CACHE = [(dict(dtype=7), 2), (dict(num_pages=0), 2), (dict(page_size=0), 2), (dict(num_kv=-1), 2),
             (dict(head_dim=0), 2), (dict(head_dim=72), 1), (dict(head_dim=272), 1), (dict(k=None), 2),
             (dict(v=None), 2), (dict(k=ODD), 1), (dict(v=ODD), 1), (dict(dtype=1), 2),
             (dict(dtype=1, k_scale=FAKE), 2), (dict(num_kv=1 << 16), 1)]
BAD_BATCH = [(dict(tokens=-1), 2), (dict(seqs=-1), 2), (dict(max_pages=-1), 2), (dict(max_new=-1), 2),
             (dict(max_kv=-1), 2), (dict(cu_seqlens=None), 2), (dict(kv_lens=None), 2), (dict(page_table=None), 2),
             (dict(max_pages=1 << 27), 2), (dict(max_pages=0x7fff001), 2),
             (dict(tokens=1 << 24), 1)]


@pytest.mark.parametrize("over,rc", BAD_CACHE)
def test_bad_cache_is_refused(over, rc):
    kv, b = cache(**over), batch()
    w = heads(head_dim=kv.head_dim, num_kv=kv.num_kv)
    assert attend(kv, b) == rc and "paged_attention" in hip.last_error()
    assert append(kv, b, w) == rc and "paged_append" in hip.last_error()
    assert read(kv, b) == rc and "paged_read" in hip.last_error()


@pytest.mark.parametrize("over,rc", BAD_BATCH)
def test_bad_batch_is_refused(over, rc):
    kv, b = cache(), batch(**over)
    assert attend(kv, b) == rc
    assert append(kv, b, heads()) == rc
    assert read(kv, b) == rc
    assert hip.lib().gorch_hip_paged_attention_workspace_size(C.byref(kv), C.byref(b), 4) == 0 or rc != 2


def test_null_structs_are_refused():
    L = hip.lib()
    kv, b = cache(), batch()
    assert L.gorch_hip_paged_attention(None, None, C.byref(b), FAKE, 4, FAKE, 1, None, 0) == 2
    assert L.gorch_hip_paged_attention(None, C.byref(kv), None, FAKE, 4, FAKE, 1, None, 0) == 2
    assert L.gorch_hip_paged_append(None, C.byref(kv), C.byref(b), None, None, 0, FAKE, 128, FAKE, 128, None) == 2
    assert L.gorch_hip_paged_attention_workspace_size(None, C.byref(b), 4) == 0
    assert L.gorch_hip_process_logits(None, None, FAKE, FAKE, 1, 8) == 2


def test_attention_arguments():
    kv, b = cache(), batch()
    assert attend(kv, b, num_q=3) == 2 and attend(kv, b, num_q=0) == 2
    assert attend(kv, b, q=None) == 2 and attend(kv, b, out=None) == 2
    assert attend(kv, b, q=ODD) == 1 and attend(kv, b, out=ODD) == 1


def test_append_arguments():
    kv, b = cache(), batch()
    assert append(kv, b, heads(num_kv=4)) == 2 and append(kv, b, heads(head_dim=128)) == 2
    assert append(kv, b, heads(num_q=3)) == 2
    assert append(kv, b, heads(), q=None) == 2 and append(kv, b, heads(), out=None) == 2
    assert append(kv, b, heads(), k=None) == 2 and append(kv, b, heads(), v=None) == 2
    assert append(kv, b, heads(), ks=127) == 2 and append(kv, b, heads(), qs=128) == 2
    assert append(kv, b, heads(), ks=129) == 1 and append(kv, b, heads(), k=ODD) == 1
    assert append(kv, b, heads(rope_cos=FAKE)) == 2
    assert append(kv, b, heads(rope_cos=FAKE, rope_sin=ODD)) == 1
    # q may be its own output only where its rows lie together
    assert append(kv, b, heads(), qs=512, out=FAKE) == 2


def test_nothing_to_do_is_no_work():
    for b in (batch(tokens=0), batch(seqs=0), batch(tokens=0, cu_seqlens=None, kv_lens=None, page_table=None)):
        assert attend(cache(), b) == 0 and append(cache(), b, heads()) == 0 and read(cache(), b) == 0
    assert read(cache(), batch(), None, None) == 0
    r = hip._LogitsRulesC()
    assert hip.lib().gorch_hip_process_logits(None, C.byref(r), None, None, 0, 8) == 0
    assert hip.lib().gorch_hip_process_logits(None, C.byref(r), None, None, 4, 0) == 0


@pytest.mark.parametrize("over,rows,n,rc", [
    ({}, -1, 8, 2), ({}, 1, -8, 2), (dict(history=FAKE, history_stride=-1), 1, 8, 2), (dict(biases=-1), 1, 8, 2),
    (dict(biases=2, bias=FAKE, bias_ids=FAKE), 1, 8, 2), (dict(biases=2, bias=FAKE, bias_rows=FAKE), 1, 8, 2),
    (dict(biases=2, bias_rows=FAKE, bias_ids=FAKE), 1, 8, 2), (dict(allowed=FAKE, allowed_stride=1), 1, 33, 2),
    ({}, 65536, 8, 1)])
def test_bad_logits_rules_are_refused(over, rows, n, rc):
    r = hip._LogitsRulesC()
    for k, v in over.items():
        setattr(r, k, v)
    assert hip.lib().gorch_hip_process_logits(None, C.byref(r), FAKE, FAKE, rows, n) == rc
    assert hip.lib().gorch_hip_process_logits(None, C.byref(r), None, FAKE, max(rows, 1), max(n, 1)) != 0


def test_cpu_tensors_are_refused():
    import torch

    with pytest.raises(ValueError):
        hip._p(torch.zeros(4))
    with pytest.raises((ValueError, RuntimeError, AssertionError)):
        hip.PagedKV(torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        hip.PagedKV(torch.zeros((2, 2, 16, 64)), torch.zeros((2, 2, 16, 64)))
    with pytest.raises(ValueError):
        hip.PagedKV(torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16),
                    torch.zeros((2, 2, 16)), torch.zeros((2, 2, 16)))


def test_too_many_heads_are_refused():
    w = heads(num_q=1 << 16)
    assert append(cache(), batch(), w, qs=1 << 23) == 1 and "num_q" in hip.last_error()
    assert append(cache(), batch(tokens=0), w) == 1


def test_workspace_of_a_long_prompt_beside_single_tokens_stays_small():
    # 64 key ranges for the 7 single tokens' rows alone
    n = hip.lib().gorch_hip_paged_attention_workspace_size(
        C.byref(cache(num_kv=8, head_dim=128)), C.byref(batch(tokens=8199, seqs=8, max_pages=8192)), 32)
    assert 64 * 7 * 32 * 130 * 4 <= n < 32 << 20


def test_too_large_a_launch_is_refused():
    # 2^24 sequences of a token or less, 1 KV head: one launch has fewer blocks
    kv, b = cache(num_kv=1), batch(tokens=16, seqs=1 << 25, max_new=1)
    assert attend(kv, b, num_q=4, ws=FAKE, n=1 << 60) == 1 and "too many" in hip.last_error()
    assert attend(cache(num_kv=8), batch(tokens=1 << 20), num_q=512) == 1


@pytest.mark.parametrize("dims,name", [
    # 2 heads per KV head: a conversation's step short and long, many of them, prompts, a chunk, a mixed batch
    # (4 prompts may all be short ones: 32 tiles of few rows, split)
    ((1, 1, 16, 8, 128, 1, 60), "few4"), ((1, 1, 16, 8, 128, 1, 777), "few4 split"),
    ((64, 64, 16, 8, 128, 1, 8192), "few4 split"), ((4096, 4096, 16, 8, 128, 1, 4096), "few4"),
    ((8192, 4, 16, 8, 128, 2048, 2048), "few4+many split"), ((2048, 1, 16, 8, 128, 2048, 16384), "many split"),
    ((600, 27, 16, 8, 128, 500, 4000), "few4+many split"),
    # 7 heads per KV head, 16 draft rows, one KV head for all
    ((3, 3, 14, 2, 64, 1, 32749), "few16 split"), ((64, 16, 16, 8, 128, 4, 2000), "few16 split"),
    ((80, 16, 16, 8, 128, 5, 2000), "few16 split"), ((4, 4, 32, 1, 128, 1, 200), "few16 split"),
    ((2, 1, 16, 8, 128, 0, 100), "few4"), ((60, 9, 40, 1, 64, 20, 90), "many"), ((100, 1, 16, 8, 128, 0, 100), "many")])
def test_kernel_choice(dims, name):
    assert hip.kernel_choice("paged_attention", *dims) == name


def test_kernel_choice_of_nothing():
    for dims in ((0, 1, 16, 8, 128, 1, 60), (1, 0, 16, 8, 128, 1, 60), (1, 1, 15, 8, 128, 1, 60),
                 (1, 1, 16, 8, 72, 1, 60), (1, 1, 16, 0, 128, 1, 60), (1 << 24, 1, 16, 8, 128, 1, 60)):
        assert hip.kernel_choice("paged_attention", *dims) is None
