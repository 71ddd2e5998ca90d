"""CPU-only checks of what gorch_hip_paged_attention plans at the ends of its
ranges, by its workspace and its choice of kernels."""
import ctypes as C

import pytest

from gorch_amd import hip

FAKE = 0x10000


def workspace(tokens, num_q, num_kv=8, hd=16, seqs=1, max_new=0, max_kv=256):
    kv = hip._PagedKVC(hip.KV_BF16, 8, 16, num_kv, hd, FAKE, FAKE, None, None)
    b = hip._PagedBatchC(tokens, seqs, -(-max_kv // 16), max_new, max_kv, FAKE, FAKE, FAKE)
    return hip.lib().gorch_hip_paged_attention_workspace_size(C.byref(kv), C.byref(b), num_q)


@pytest.mark.parametrize("max_new", [1, 64])
@pytest.mark.parametrize("seqs", [1, 3])
def test_no_ranges_where_their_join_would_leave_a_launch(max_new, seqs):
    # a join is a wave a (token, head) row, and a launch has less than 2^32 threads. Rows of no sequence count: most
    # of these are some, so that few blocks have work and the keys of those would be split
    for tokens in (1 << 20, 1 << 22, (1 << 23) - 1):
        assert workspace(tokens, 32, max_new=max_new, seqs=seqs) == 0
        name = hip.kernel_choice("paged_attention", tokens, seqs, 32, 8, 16, max_new, 256)
        assert name is not None and "split" not in name
    assert workspace(1 << 19, 32, max_new=max_new, seqs=seqs) > 0
