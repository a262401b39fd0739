"""What a launch of attention over 8-bit pages is divided into, through the C ABI and on the host."""
import ctypes as C
import os
import subprocess

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


CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust_interference_engine_amd", "csrc")
CODE = f'''#include "{CSRC}/serve_index.hpp"
using namespace rie;
extern "C" int waves(int n_rows, int n_seq, int max_new, int G, int n_kv, int hd) {{ return tile8_wave_count(n_rows, n_seq, max_new, G, n_kv, hd); }}
extern "C" long blocks(int n_rows, int n_seq, int G, int M) {{ return block_count(n_rows, n_seq, G, M); }}
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan8")
    (d / "s.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True)
    so = C.CDLL(str(d / "s.so"))
    so.blocks.restype = C.c_long
    return so


def test_a_launch_of_tiles_has_under_2_to_the_32_threads(plan):
    """a workgroup for each block of rows and KV head, at the largest numbers that the library takes"""
    for n_seq, n_rows, G, n_kv in (((1 << 23) - 1, 300, 1, 1), (1 << 23, 300, 1, 1), ((1 << 24) - 5, 300, 1, 1), ((1 << 20) - 4, 300, 1, 16), (1, (1 << 26) - 4, 1, 1), (1 << 20, 1 << 20, 2, 8),
                                   (1, 1 << 20, 32, 32), (4095, 300, 1, 4095), (1 << 12, 1 << 14, 1, 3900)):
        assert (n_seq + n_rows * G // 128) * n_kv < 1 << 24
        for hd in (32, 64, 96, 128, 256):
            w = plan.waves(n_rows, n_seq, n_rows, G, n_kv, hd)
            assert w in (4, 8) and plan.blocks(n_rows, n_seq, G, 32 * w) * n_kv * 64 * w < 1 << 32, (n_seq, n_rows, G, n_kv, hd)
    assert plan.waves(509 * 13, 13, 509, 4, 8, 128) == 8 and plan.waves(4000, 4, 1000, 4, 8, 256) == 4 and plan.waves(100, 13, 30, 4, 8, 128) == 4
