"""The sums of enx_pages_grow (csrc/pages_want.h), compiled for the host, at sizes that no test's table has:
what the rows want, added up as the kernel does, 1024 rows at a time, and refused as soon as it passes the pool."""

import ctypes as C
import random
import subprocess

import pytest

from conftest import ROOT

SOURCE = """
#include "pages_want.h"
using namespace enx;
// 1: refused.  rows of (copy, fresh); at[i]: copies and pages before row i, at[n] all of them.
extern "C" int grow_sums(uint32_t n, const uint8_t* copy, const uint32_t* fresh, uint32_t pages, uint64_t* at) {
    unsigned long long run = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += 1024) {
        for (uint32_t i = i0; i < n && i < i0 + 1024; ++i) {
            at[2 * i] = want_copies(run), at[2 * i + 1] = want_pages(run);
            run += want_of(copy[i], fresh[i], pages);
        }
        if (want_pages(run) > pages) return 1;
    }
    at[2 * n] = want_copies(run), at[2 * n + 1] = want_pages(run);
    return 0;
}
"""


@pytest.fixture(scope="module")
def sums(tmp_path_factory):
    at = tmp_path_factory.mktemp("want")
    (at / "want.cc").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT / 'enargeia_b200' / 'csrc'}", str(at / "want.cc"),
                    "-o", str(at / "want.so")], check=True)
    fn = C.CDLL(str(at / "want.so")).grow_sums

    def call(rows, pages):
        n = len(rows)
        out = (C.c_uint64 * (2 * n + 2))()
        refused = fn(n, (C.c_uint8 * n)(*[c for c, _ in rows]), (C.c_uint32 * n)(*[f for _, f in rows]), pages, out)
        return None if refused else [(out[2 * i], out[2 * i + 1]) for i in range(n + 1)]

    return call


def expected(rows, pages):
    at, copies, total = [], 0, 0
    for c, f in rows:
        at.append((copies, total))
        copies, total = copies + c, total + c + f
    return at + [(copies, total)] if total <= pages else None


@pytest.mark.parametrize("rows,pages", [
    ([(0, 16384)] * 262144, 1 << 28),           # 2^32 pages: a 32-bit sum is back at 0
    ([(0, 16384)] * 262143 + [(1, 16390)], 64),
    ([(0, (1 << 31) - 1)] * 262144, 1 << 28),   # 2^49
    ([(1, 0)] * 262144, 1 << 28),               # every row copies
    ([(1, 1023)] * 262144, 1 << 28),            # the pool to the last page, and one more
    ([(1, 1023)] * 262143 + [(1, 1024)], 1 << 28),
    ([(0, 1 << 28)], 1 << 28), ([(1, 1 << 28)], 1 << 28), ([(0, 0)] * 5, 1), ([(0, 2)], 1), ([(0, 1)] * 1025, 1024),
])
def test_ends_of_the_range(sums, rows, pages):
    assert sums(rows, pages) == expected(rows, pages)


def test_random_rows(sums):
    rng = random.Random(5)
    for _ in range(200):
        n, pages = rng.randint(1, 3000), 1 << rng.randint(0, 28)
        rows = [(rng.randint(0, 1), rng.choice([0, 1, rng.randint(0, max(1, 2 * pages // n))])) for _ in range(n)]
        assert sums(rows, pages) == expected(rows, pages)
