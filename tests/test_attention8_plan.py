"""What a launch of attention over 8-bit pages is divided into, through the C ABI and on the host."""
import ctypes as C

import pytest
from test_decoding_refusals import attn, pages8, seqs

from rust_interference_engine_amd import _lib


def workspace(n_head, n_kv, hd, max_len, n_seq=1, max_new=1, n_rows=None, ty=1):
    pg = pages8(head_dim=hd, n_kv=n_kv, slot_stride=hd, head_stride=16 * hd, page_stride=16 * hd * n_kv, table_cols=1 << 16)
    at = attn(n_head=n_head, q_head_stride=hd, out_head_stride=hd, q_row_stride=hd * n_head, out_row_stride=hd * n_head)
    return _lib.lib().rie_hip_k_paged_attention8_ws(C.byref(pg), C.byref(seqs(n_seq=n_seq, n_rows=n_rows or n_seq * max_new, max_new=max_new, max_len=max_len)), ty, C.byref(at))


@pytest.mark.parametrize("n_head,n_kv,hd", [(3, 1, 64), (7, 1, 64), (1, 1, 96), (15, 5, 64), (5, 1, 32), (9, 1, 128), (25, 1, 256)])
def test_partial_results_lie_at_multiples_of_16_bytes(n_head, n_kv, hd):
    """each is 16-byte vectors of a group's rows and two floats of each row; odd numbers of rows and of parts"""
    R = n_head // n_kv
    part = -(-R * (hd + 2) * 4 // 16) * 16
    seen = set()
    for n_seq in (1, 3, 5):
        for max_len in range(1000, 20000, 500):
            n = workspace(n_head, n_kv, hd, max_len, n_seq)
            assert n % (part * n_kv) == 0, (n_seq, max_len, n)
            seen.add(n // (part * n_kv) % 2)
    assert seen == {0, 1}
