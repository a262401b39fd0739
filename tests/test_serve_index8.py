"""Which blocks of an 8-bit cache new tokens are written to (csrc/serve_index.hpp), compiled for the host: every block has
an id of its own, whatever the device memory holds."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust_interference_engine_amd", "csrc")
CODE = f'''#include "{CSRC}/serve_index.hpp"
using namespace rie;
extern "C" {{
int id(int start, int i, int shift) {{ return append8_id(start, i, shift); }}
long count(int rows, int seqs, int shift) {{ return append8_count(rows, seqs, shift); }}
}}
'''


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("serve8")
    (d / "s.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True)
    so = ctypes.CDLL(str(d / "s.so"))
    so.count.restype = ctypes.c_long
    return so


@pytest.mark.parametrize("shift", [4, 5, 8, 12])
def test_ids_cover_every_block_that_a_sequence_can_touch(lib, shift):
    r = random.Random(shift)
    block = 1 << shift
    for _ in range(300):
        lens = [r.choice([0, 0, 1, 2, block - 1, block, block + 1, r.randint(0, 5 * block)]) for _ in range(r.randint(1, 40))]
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        ids = [lib.id(s, i, shift) for i, s in enumerate(starts)]
        assert ids[0] == 0 and ids[-1] <= lib.count(starts[-1], len(lens), shift)
        for i, n in enumerate(lens):
            for pos0 in (0, 1, block - 1, r.randrange(block)):
                touched = 0 if n == 0 else (pos0 + n - 1 >> shift) - (pos0 >> shift) + 1
                assert ids[i + 1] - ids[i] >= touched


def test_ids_rise_and_stay_below_the_count_at_the_limits(lib):
    for shift in (4, 12):
        for rows, seqs in (((1 << 26) - 4, 1), ((1 << 26) - 4, 1 << 12), (1, (1 << 24) - 1), (1 << 20, 1 << 20)):
            assert lib.id(0, 0, shift) == 0 < lib.id(rows, seqs, shift) <= lib.count(rows, seqs, shift) < 1 << 31
