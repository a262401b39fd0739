"""Whether two sets of strided rows share memory (csrc/serve_index.hpp), compiled for the host, against sets of bytes; and
the rotary calls that are refused for it."""
import ctypes
import os
import random
import subprocess

import pytest
from test_decoding_refusals import P, ROT, V, rotary

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust_interference_engine_amd", "csrc")
CODE = f'''#include "{CSRC}/serve_index.hpp"
using namespace rie;
extern "C" int overlap(const long *a, const long *b) {{
    auto rows = [](const long *x) {{ return RowsAt{{(const void *)x[0], x[1], x[2], x[3], x[4], x[5]}}; }};
    return rows_overlap(rows(a), rows(b));
}}
'''


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "s.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True)
    so = ctypes.CDLL(str(d / "s.so"))
    return lambda a, b: bool(so.overlap((ctypes.c_long * 6)(*a), (ctypes.c_long * 6)(*b)))


def bytes_of(x):
    p, n, row, heads, head, width = x
    return {p + i * row + j * head + e for i in range(n) for j in range(heads) for e in range(width)}


@pytest.mark.parametrize("seed", range(40))
def test_against_sets_of_bytes(overlap, seed):
    r = random.Random(seed)
    seen = set()
    for _ in range(200):
        width = r.choice([1, 2, 4, 8])
        row, head = r.randint(0, 60), r.randint(0, 40)
        a = (1000, r.randint(1, 6), row, r.randint(1, 5), head, width)
        same = r.random() < 0.7
        b = (1000 + r.choice([0, width, row, head, -row, r.randint(-200, 200), row * 6]), r.randint(1, 6), row if same else r.randint(0, 60), r.randint(1, 5), head if same else r.randint(0, 40),
             r.choice([width, 2 * width]))
        want = bool(bytes_of(a) & bytes_of(b))
        assert overlap(a, b) == overlap(b, a) == want, (a, b)
        seen.add(want)
    assert seen == {False, True}


def test_layouts_that_programs_have(overlap):
    n, hd = (1 << 26) - 4, 128
    row = 48 * hd
    q, k = (P, n, row, 32, hd, hd), (P + 32 * hd, n, row, 8, hd, hd)
    assert not overlap(q, k)  # a fused projection
    assert not overlap((P, n, row, 8, 2 * hd, hd), (P + hd, n, row, 8, 2 * hd, hd))  # heads in turns
    assert overlap(q, (P + 31 * hd, n, row, 8, hd, hd)) and overlap(q, (P + 32 * hd + 1, n, row, 16, hd, hd))  # the next row's first head
    assert not overlap((P, 1000, hd, 32, 1000 * hd, hd), (P + 32000 * hd, 1000, hd, 8, 1000 * hd, hd))  # heads first, one behind the other
    assert not overlap((P, 5000, 4096, 1, 0, 4096), (P + 5000 * 4096, 5000, 1024, 1, 0, 1024))
    far = 1 << 42
    assert not overlap((P, n, far, 4096, 1 << 30, 2048), (P + (1 << 29), n, far, 4096, 1 << 30, 2048))
    assert overlap((P, n, far, 4096, 1 << 30, 2048), (P + (n - 5) * far + (4095 << 30) + 2047, n, far, 1, 0, 2))
    assert overlap((P, 1 << 20, 7, 1 << 12, 11, 1), (P + 5, 1 << 20, 13, 1 << 12, 17, 1))


@pytest.mark.parametrize("kw,text", [
    (dict(), "q_out and k_out"), (dict(q_out=P, k_out=P), "q_out and k_out"), (dict(k_out=V + 2 * 255), "q_out and k_out"), (dict(k_out=V + 2 * (7 * 256 + 250)), "q_out and k_out"),
    (dict(q_out=P + 2, n_k=0, k=0, k_out=0), "q and q_out"), (dict(q_out=V - 2, q=V, k_out=V + (1 << 20)), "q and q_out"), (dict(k=V + 64, k_out=V + (1 << 20)), "q_out and k "),
    (dict(q=V + (1 << 20) + 2, k_out=V + (1 << 20)), "k_out and q "), (dict(q_out=P, k_out=V, k=P + 2 * 100), "q_out and k "), (dict(dst_ty=0, k_out=V + 4 * 8 * 256 - 4), "q_out and k_out"),
])
def test_rotary_to_memory_that_overlaps(kw, text):
    rc, m = rotary(**kw)
    assert rc == -5 and text in m and "share memory" in m, (rc, m)


@pytest.mark.parametrize("kw", [
    dict(k_out=V + (1 << 20)), dict(q=P, q_out=P, q_row_stride=512, q_out_row_stride=512, k=P + 2 * 256, k_out=P + 2 * 256, k_row_stride=512, k_out_row_stride=512),
    dict(q_row_stride=384, k=P + 2 * 256, k_row_stride=384, q_out_row_stride=384, k_out=V + 2 * 256, k_out_row_stride=384),
    dict(q_out_head_stride=128, q_out_row_stride=512, k_out=V + 2 * 64, k_out_head_stride=128, k_out_row_stride=512), dict(dst_ty=0, k_out=V + 4 * 8 * 256),
    dict(q=P, k=P, q_row_stride=0, q_head_stride=0, k_out=V + (1 << 20)), dict(n_q=0, q=0, q_out=0), dict(n_k=0, k=0, k_out=0),
])
def test_rotary_to_memory_that_does_not(kw):
    rc, m = rotary(**kw)
    assert rc == -5 and "share" not in m and "stride" not in m, (rc, m)  # made-up pointers, or no GPU at all
    assert ROT["n_rows"] == 8
