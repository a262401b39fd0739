"""More of csrc on the host: sequences whose length passes what their table can address (serve_index.hpp), inline assembly."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust_interference_engine_amd", "csrc")
CODE = f'''#include "{CSRC}/serve_index.hpp"
using namespace rie;
extern "C" {{
void view(int s, int e, int len, int n_rows, int cap, int *o) {{ SeqView v = seq_view(s, e, len, n_rows, cap); o[0] = v.n_new; o[1] = v.len; o[2] = v.pos0(); }}
void range(int n_new, int len, int cap, int t0, int t1, int window, int KT, int *o) {{
    SeqView v = seq_view(0, n_new, len, n_new, cap); KeyRange r = key_range(v, t0, t1, window);
    o[0] = r.lo; o[1] = r.hi; o[2] = first_tile(r, KT); o[3] = tile_count(r, KT); }}
}}
'''


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plans")
    (d / "p.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o", str(d / "p.so"), str(d / "p.cpp")], check=True)
    return ctypes.CDLL(str(d / "p.so"))


def out(n):
    return (ctypes.c_int * n)()


def test_positions_come_from_the_length_that_the_memory_holds(lib):
    o = out(3)
    for cap in (16, 32, 2 ** 30):
        for n in (0, 1, 10, 1000):
            for length in (0, 1, 31, 32, 33, 37, 5000, 2 ** 30, 2 ** 30 + 5, 2 ** 31 - 1):
                lib.view(0, n, length, 1000, cap, o)
                assert list(o) == [n, min(length, cap), length - n]


def test_key_ranges_end_with_the_table(lib):
    o = out(4)
    r = random.Random(3)
    for _ in range(6000):
        cap = 16 * r.randint(1, 10)
        n, length = r.randint(1, 50), r.choice([r.randint(0, 200), r.randint(cap, cap + 60), 2 ** 31 - 1])
        t0 = r.randrange(n)
        t1 = r.randrange(t0, n)
        window = r.choice([0, 1, 2, 30, 500, 2 ** 30, 2 ** 31 - 1])
        KT = r.choice([32, 64, 128])
        seen = set()
        for t in range(t0, t1 + 1):
            p = length - n + t
            seen |= set(range(max(0, p - window + 1) if window else 0, min(p, cap - 1) + 1))
        lib.range(n, length, cap, t0, t1, window, KT, o)
        lo, hi, first, tiles = o
        assert 0 <= lo <= hi <= cap
        if not seen:
            assert lo == hi and tiles == 0
            continue
        assert (lo, hi) == (min(seen), max(seen) + 1)
        assert first * KT <= lo and (first + tiles) * KT >= hi and (first + tiles - 1) * KT < hi


def test_inline_assembly_names_the_registers_it_writes():
    """m0 is the compiler's too: a block that writes it says so"""
    found = 0
    for folder in (CSRC, os.path.join(CSRC, "kernels")):
        for name in sorted(os.listdir(folder)):
            if not name.endswith((".hip", ".hpp")):
                continue
            with open(os.path.join(folder, name)) as f:
                text = f.read()
            for at in [i for i in range(len(text)) if text.startswith("s_mov_b32 m0", i)]:
                block = text[at:text.index(";\n", at)]
                assert '"m0"' in block.rsplit(":", 1)[1], (name, block)
                found += 1
    assert found
