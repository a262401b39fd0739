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
int few(int paged, int max_new, int G) {{ return few_row_blocks(paged, max_new, G); }}
int splits(int nt, int C, int S) {{ return split_count(nt, C, S); }}
void tiles(long wgs, int slots, int tiles, double tile_us, double part_us, int most, int *o) {{
    SplitPlan p = tile_plan(wgs, slots, tiles, tile_us, part_us, most); o[0] = p.C; o[1] = p.S; }}
}}
'''


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plans")
    (d / "p.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o", str(d / "p.so"), str(d / "p.cpp")], check=True)
    so = ctypes.CDLL(str(d / "p.so"))
    so.tiles.argtypes = [ctypes.c_long] + [ctypes.c_int] * 2 + [ctypes.c_double] * 2 + [ctypes.c_int, ctypes.c_void_p]
    return so


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


def test_which_kernel_takes_a_launch(lib):
    for max_new, G, want in [(1, 1, 1), (1, 16, 1), (4, 4, 1), (16, 1, 1), (1, 17, 2), (17, 1, 2), (5, 4, 2), (4, 8, 2), (8, 4, 2), (32, 1, 2), (1, 32, 2),
                             (33, 1, 0), (1, 33, 0), (3, 11, 0), (5, 8, 0), (2 ** 30, 4096, 0)]:
        assert lib.few(1, max_new, G) == want and lib.few(0, max_new, G) == 0


def test_splits_of_tiles_take_every_tile_once_and_fit_the_partials(lib):
    o = out(2)
    for wgs in (1, 2, 5, 63, 123, 255, 488, 511, 512, 1023, 100000):
        for slots in (256, 512):
            for tiles in (0, 1, 2, 3, 7, 8, 33, 64, 127, 129, 1000, 2 ** 24):
                for tile_us, part_us in ((2.0, 0.0), (2.0, 4.0), (0.5, 0.01), (2.0, 1e6)):
                    lib.tiles(wgs, slots, tiles, tile_us, part_us, 128, o)
                    C, Sn = o
                    assert 1 <= Sn <= 128 and C >= 1 and C * Sn >= tiles and (Sn == 1 or C * (Sn - 1) < tiles)
                    assert Sn == 1 or wgs < slots  # with every slot taken nothing is won
                    assert Sn == 1 or tiles * tile_us > Sn * part_us  # the partials cost less than the tiles they share out
                    for nt in (0, 1, C - 1, C, C + 1, tiles, 3 * tiles + 1):
                        ns = lib.splits(nt, C, Sn)
                        assert 1 <= ns <= Sn
                        ends = [min((s + 1) * C, nt) if s < ns - 1 else nt for s in range(ns)]
                        assert all(e > s * C for s, e in enumerate(ends)) or nt == 0
    lib.tiles(1, 512, 1000, 2.0, 0.01, 128, o)
    assert o[1] > 16  # one workgroup over a long cache is split


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
