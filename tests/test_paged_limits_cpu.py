"""CPU: the paged attention's division of work (csrc/paged_split.h) up to the largest sizes that a call accepts, and the size query at and behind
them."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "scoreperformer_amd", "csrc")


def _host_check(tmp_path, source):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(source)
    subprocess.run([shutil.which("g++") or "c++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.returncode, r.stdout, r.stderr)


HEAD = r"""
#include "paged_split.h"
#include <cstdio>
#include <cstdlib>
#include <cmath>
#include <climits>
using namespace spn_paged;
#define NEED(c) do { if (!(c)) { std::printf("line %d: %s (R %d h %d kvh %d W %d shift %d esize %d)\n", __LINE__, #c, R, h, kvh, W, shift, esize); return 1; } } while (0)
static int lg(double hi) { return (int)std::exp2(std::log2(hi) * std::rand() / RAND_MAX); }     // 1 .. hi, evenly over the logarithm
"""

SPLIT = HEAD + r"""
static const int FIXED[][5] = {{4096, 256, 256, 262144, 12}, {512, 4095, 4095, 131072, 12}, {(1 << 21) - 1, 1, 1, 1, 12}, {1, (1 << 21) - 1, 1, 1, 3},
                               {1, 1, 1, (1 << 28) - 1, 3}, {1, 1, 1, (1 << 27) - 1, 4}, {8191, 256, 256, 262143, 3}, {1, 1, 1, (1 << 19) - 1, 12}};
int main() {
    int seen = 0;
    for (int it = 0; it < 400000 || seen < 50000; ++it) {
        int R = lg(2097152), kvh = lg(65536), h = kvh * lg(64), shift = 3 + std::rand() % 10, W = lg(268435456.0), esize = std::rand() % 2 ? 2 : 4;
        if (it < 16) { const int* f = FIXED[it / 2]; R = f[0]; h = f[1]; kvh = f[2]; W = f[3]; shift = f[4]; esize = it % 2 ? 2 : 4; }
        if (!sizes_ok(R, h, kvh, W, shift)) { NEED(it >= 16); continue; }
        ++seen;
        const Split s = split_of(R, h, kvh, W, shift, esize);
        const int tile = 64 / esize;
        const long cap = (long)W << shift, full = (cap + tile - 1) / tile, segments = (long)R * kvh * s.passes;
        NEED(s.passes >= 1 && s.rows >= 1 && s.rows <= HEADS && s.passes * HEADS >= h / kvh);
        NEED(s.max_tiles >= 1 && full <= INT_MAX);
        NEED(s.units >= 1 && s.units <= INT_MAX - 1 && segments <= (1 << 21));
        NEED(s.waves == 0 || s.units == segments);
        if (s.waves) { NEED(scratch_of(s, R) == 0); continue; }
        NEED(scratch_of(s, R) >= (size_t)s.units * s.rows * (HEAD + 2) * 4 && scratch_of(s, R) < (1ull << 40));
        // the parts of the batch fit the workspace, whatever the lengths: all full, all alike, one full among short ones
        for (int k = 0; k < 6; ++k) {
            const long some = k == 0 ? full : k == 1 ? 0 : k == 2 ? 1 : lg((double)full);
            const bool lone = k >= 4;                                       // only the first request is that long
            const long total = lone ? segments / R * (some + (R - 1)) : segments * some;
            const int most = most_of(total, s.max_tiles);
            NEED(most >= 1);
            const long parts = lone ? segments / R * (parts_of((int)some, most) + (long)(R - 1) * parts_of(1, most)) : segments * parts_of((int)some, most);
            NEED(parts >= segments && parts <= s.units);
            NEED(parts_of((int)some, most) == MAX_PARTS || (long)parts_of((int)some, most) * most >= some);
        }
    }
    std::puts("ok");
    return 0;
}
"""


def test_the_division_of_any_accepted_batch_fits_its_workspace(tmp_path):
    _host_check(tmp_path, SPLIT)


TILES = HEAD + r"""
int main() {
    const int R = 1, h = 1, kvh = 1, shift = 3, W = 1, esize = 2;
    for (int tile = 16; tile <= 32; tile *= 2)
        for (int it = 0; it < 1000000; ++it) {
            const int rows = it < 5000 ? it : it < 10000 ? INT_MAX - (it - 5000) : lg(2147483647.0);
            const int n = tiles_of(rows, tile);
            NEED(n >= 0 && (long)n * tile >= rows && (long)(n - 1) * tile < rows);
            for (int t = n - 1; t >= 0 && t >= n - 3; --t) {                                // the kernel asks for tiles that hold a row
                NEED(part_filled(t, tile, rows) == ((long)t * tile + tile > rows));
                NEED((long)t * tile + tile - 1 <= INT_MAX);                                 // every row number of the tile is an int
            }
        }
    std::puts("ok");
    return 0;
}
"""


def test_tiles_of_any_length(tmp_path):
    """Lengths up to 2^31 - 1: as many tiles as hold the rows, and the last one known as such."""
    _host_check(tmp_path, TILES)


INDEX = HEAD + r"""
int main() {
    const int R = 1, h = 1, kvh = 1, esize = 2;
    for (int it = 0; it < 2000000; ++it) {
        const int shift = 3 + std::rand() % 10, W = it % 3 ? lg(2147483647.0) : INT_MAX - std::rand() % 100;
        const int len = it % 5 ? lg(2147483647.0) : INT_MAX - std::rand() % 5000, fresh = lg(2147483647.0), width = INT_MAX;
        // a release walks the held pages 64 at a time: the walk's end stays an int for any width of the table
        const long held = pages_of(len, shift) < W ? pages_of(len, shift) : W;
        NEED(held >= 0 && held <= (1 << 28) && held + 64 <= INT_MAX);
        const int need = pages_needed(len, fresh, width, W, shift);
        NEED(need >= -1 && (need < 0 || pages_of(len, shift) + need <= W));
        NEED(need < 0 || pages_of((long)len + fresh, shift) == pages_of(len, shift) + need);
        if (((long)W << shift) >= (1L << 31)) continue;                                     // (refused by plan and attention)
        const int n = rows_of(len, W, shift);
        NEED(n <= len && n <= (long)W << shift && (n == 0 || ((n - 1) >> shift) < W));
        NEED(need < 0 || (long)len + fresh <= INT_MAX);                                     // the new length is an int
    }
    std::puts("ok");
    return 0;
}
"""


def test_index_arithmetic_at_the_widest_tables(tmp_path):
    """Tables of up to 2^31 - 1 entries a row: plan's counts, release's walk, the rows that the attention takes."""
    _host_check(tmp_path, INDEX)


QUERY = """
import ctypes, sys
lib = ctypes.CDLL(sys.argv[1])
f = lib.spn_paged_attn_workspace_bytes
f.restype = ctypes.c_size_t
for line in sys.stdin:
    print(f(*(ctypes.c_int(int(x)) for x in line.split())), flush=True)
"""


def _query(rows):
    """In a process of its own: a size query that faults is that process's end."""
    from scoreperformer_amd import build, lib
    build.build()
    r = subprocess.run([sys.executable, "-c", QUERY, lib.LIB_PATH], input="\n".join(" ".join(map(str, x)) for x in rows), capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-500:])
    return [int(x) for x in r.stdout.split()]


@pytest.mark.parametrize("dtype", [0, 1])
def test_the_size_query_answers_at_the_largest_accepted_sizes(dtype):
    """2^30 rows for each of 4096 x 256 segments; 4095 key heads; one table row of 2^31 - 8 rows."""
    got = _query([(4096, 256, 256, 262144, 4096, dtype), (512, 4095, 4095, 131072, 4096, dtype), (1, 1, 1, 2 ** 28 - 1, 8, dtype)])
    # a part for each segment twice over at most (8192 parts of full tables), 66 floats and a header each
    assert 0 < got[0] <= 2 * 2 ** 20 * (66 * 4 + 16) + 16 + 4096 * 4
    assert 0 < got[1] <= 2 * 512 * 4095 * (66 * 4 + 16) + 16 + 512 * 4
    assert 0 < got[2] <= (8192 + 1) * (66 * 4 + 16) + 16


def test_the_size_query_is_zero_for_sizes_that_the_call_refuses():
    big = 2 ** 31 - 1
    bad = [(0, 8, 1, 4, 16, 1), (1, 0, 1, 4, 16, 1), (1, 8, 0, 4, 16, 1), (1, 8, 3, 4, 16, 1), (1, 8, 1, 0, 16, 1), (1, 8, 1, 4, 12, 1), (1, 8, 1, 2 ** 28, 8, 1),
           (2 ** 20, 2, 1, 4, 16, 1), (big, big, big, big, 4096, 0), (2 ** 12, 8, 1, 2 ** 19, 16, 1), (1, 4096, 4096, 4, 4096, 1), (-1, -8, -1, -4, 16, 1)]
    assert _query(bad) == [0] * len(bad)
