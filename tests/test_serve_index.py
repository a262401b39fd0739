"""Where a serving batch's rows, positions, blocks and splits lie (csrc/serve_index.hpp), compiled for the host: every
index stays inside what it indexes, whatever the device memory holds."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust_interference_engine_amd", "csrc")
CODE = f'''#include "{CSRC}/serve_index.hpp"
using namespace rie;
extern "C" {{
void view(int s, int e, int len, int n_rows, int cap, int *o) {{ SeqView v = seq_view(s, e, len, n_rows, cap); o[0] = v.row0; o[1] = v.n_new; o[2] = v.len; }}
int base(int start, int i, int G, int M) {{ return block_base(start, i, G, M); }}
long count(int rows, int seqs, int G, int M) {{ return block_count(rows, seqs, G, M); }}
void range(int n_new, int len, int t0, int t1, int window, int KT, int *o) {{
    SeqView v{{0, n_new, len}}; KeyRange r = key_range(v, t0, t1, window);
    o[0] = r.lo; o[1] = r.hi; o[2] = first_tile(r, KT); o[3] = tile_count(r, KT); }}
int splits(int nt, int C, int S) {{ return split_count(nt, C, S); }}
void plan(long wgs, int tiles, int want, int least, int most, int *o) {{ SplitPlan p = split_plan(wgs, tiles, want, least, most); o[0] = p.C; o[1] = p.S; }}
}}
'''


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("serve")
    (d / "s.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True)
    so = ctypes.CDLL(str(d / "s.so"))
    so.count.restype = ctypes.c_long
    so.count.argtypes = [ctypes.c_int] * 4
    so.plan.argtypes = [ctypes.c_long] + [ctypes.c_int] * 4 + [ctypes.c_void_p]
    return so


def out(n):
    return (ctypes.c_int * n)()


ODD = [-2 ** 31, -7, -1, 0, 1, 5, 16, 17, 1000, 2 ** 30, 2 ** 31 - 1]


@pytest.mark.parametrize("n_rows,cap", [(1, 16), (16, 16), (100, 1600), (2 ** 30, 2 ** 30)])
def test_a_view_lies_inside_the_rows_and_positions_whatever_the_memory_holds(lib, n_rows, cap):
    o = out(3)
    for s in ODD:
        for e in ODD:
            for n in ODD:
                lib.view(s, e, n, n_rows, cap, o)
                row0, new, length = o
                assert 0 <= row0 <= n_rows and 0 <= new and row0 + new <= n_rows and 0 <= length <= cap
                if 0 <= s <= e <= n_rows and 0 <= n <= cap:
                    assert (row0, new, length) == (s, e - s, n)


def test_block_ids_cover_every_sequences_rows_once(lib):
    r = random.Random(1)
    for _ in range(300):
        G, M = r.choice([1, 3, 7, 8]), r.choice([16, 128])
        lens = [r.choice([0, 0, 1, 2, r.randint(0, 400)]) for _ in range(r.randint(1, 40))]
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        bases = [lib.base(s, i, G, M) for i, s in enumerate(starts)]
        for i, n in enumerate(lens):
            assert bases[i + 1] - bases[i] >= -(-n * G // M)
        assert bases[0] == 0 and bases[-1] == lib.count(starts[-1], len(lens), G, M)


def test_key_ranges_are_those_of_the_rule(lib):
    o = out(4)
    r = random.Random(2)
    for _ in range(4000):
        n, length = r.randint(1, 50), r.randint(0, 200)
        t0 = r.randrange(n)
        t1 = r.randrange(t0, n)
        window = r.choice([0, 1, 2, 30, 500, 2 ** 30])
        KT = r.choice([32, 64, 128])
        seen = [j for t in (t0, t1) for p in [length - n + t] if p >= 0 for j in (max(0, p - window + 1) if window else 0, p)]
        lib.range(n, length, t0, t1, window, KT, o)
        lo, hi, first, tiles = o
        if not seen:
            assert lo == hi == tiles == 0
            continue
        assert lo <= min(seen) and hi == max(seen) + 1 and hi <= length
        if length - n + t0 >= 0:
            assert lo == min(seen)
        assert first * KT <= lo and (first + tiles) * KT >= hi and (first + tiles - 1) * KT < hi


def test_splits_take_every_tile_once_and_fit_the_partials(lib):
    o = out(2)
    for wgs in (1, 2, 5, 63, 384, 511, 512, 1023, 1024, 100000):
        for tiles in (0, 1, 2, 3, 7, 8, 33, 64, 127, 1000, 2 ** 23):
            for want, least in ((1024, 1), (512, 4)):
                lib.plan(wgs, tiles, want, least, 64, o)
                C, Sn = o
                assert 1 <= Sn <= 64 and C >= 1 and (Sn == 1 or (C >= least and C * Sn >= tiles and C * (Sn - 1) < tiles and wgs < want))
                for nt in (0, 1, C - 1, C, C + 1, tiles, 3 * tiles + 1):
                    ns = lib.splits(nt, C, Sn)
                    assert 1 <= ns <= Sn
                    ends = [min((s + 1) * C, nt) if s < ns - 1 else nt for s in range(ns)]
                    assert all(e > s * C for s, e in enumerate(ends)) or nt == 0  # the last takes all that are left
