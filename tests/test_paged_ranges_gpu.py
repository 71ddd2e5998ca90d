"""gorch_hip_paged_attention's key ranges: more blocks than run at once, the last
ranges first; large batches of single tokens with one long sequence;
workspaces made for smaller bounds."""
import numpy as np
import pytest
import torch

from tests.paged_case import Case, dev, host
from tests.test_paged_attention_gpu import attend, check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,hd,count,new", [(2, 1, 64, 64, 1), (7, 1, 32, 64, 1), (4, 2, 128, 32, 2), (2, 1, 256, 400, 1)])
def test_last_ranges_first(gpu, dtype, hq, hkv, hd, count, new):
    # two long conversations among short ones: 64 (sequence, KV head) tiles in 16 ranges of 256 keys, 400 in two of
    # 2,048: more blocks than run at once
    rng = np.random.default_rng(hd)
    seqs = [(int(rng.integers(new, 60)), int(rng.integers(0, new + 1))) for _ in range(count)]
    seqs[7], seqs[-1] = (4096, new), (900, new)
    c = Case(dtype, hkv, hd, 16, seqs, seed=hd)
    bounds = dict(max_new=new, max_kv=4096)
    assert "split" in gpu.kernel_choice("paged_attention", c.tokens + 1, count, hq, hkv, hd, *bounds.values())
    q = queries(c, hq)
    want, tol = c.attention(q, hq)
    check(attend(gpu, c, q, hq, extra=1, **bounds), want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("count", [255, 256])
def test_large_decode_batches(gpu, dtype, count):
    # on both sides of 2,048 (sequence, KV head) tiles, one long conversation among short ones
    rng = np.random.default_rng(count)
    seqs = [(int(rng.integers(1, 12)), 1) for _ in range(count)]
    seqs[100] = (4500, 1)
    c = Case(dtype, 8, 16, 16, seqs, seed=count)
    q = queries(c, 16)
    want, tol = c.attention(q, 16)
    bounds = dict(max_new=1, max_kv=4500)
    check(attend(gpu, c, q, 16, **bounds), want, tol)


def test_a_workspace_of_smaller_bounds_is_refused(gpu):
    c = Case("bf16", 1, 128, 16, [(5000, 1)], seed=14)
    kv, b, short = c.cache(gpu), c.batch(gpu, max_new=1, max_kv=5000), c.batch(gpu, max_new=1, max_kv=1000)
    q, out = dev(queries(c, 2).reshape(1, -1)), torch.full((1, 256), 9.0, device="cuda")
    ws, small = kv.workspace(b, 2), kv.workspace(short, 2)
    assert ws is not None and small is not None and small.numel() < ws.numel()
    for bad in (ws[:-16], small):
        with pytest.raises(gpu.HipError) as e:
            kv.attention(b, q, out, ws=bad)
        assert e.value.rc == 2 and "workspace" in str(e.value)
    assert (host(out) == 9).all()
    kv.attention(b, q, out, ws=ws)
    assert np.isfinite(host(out)).all() and not (host(out) == 9).any()
