"""The page operations' host twin keeps its own rules, and the C entry points refuse bad arguments
before any CUDA work."""

import ctypes as C
import random

import pytest

from pages_twin import Pages


def test_counts_follow_the_tables():
    rng = random.Random(5)
    p = Pages(12, 6, 60, 16)
    for _ in range(200):
        some = rng.sample(range(12), rng.randint(1, 12))
        p.grow(some, [rng.randint(0, 20) for _ in some])
        empty = [r for r in range(12) if not p.lengths[r]]
        if empty:
            p.fork([rng.choice([r for r in range(12) if r not in empty] or [0]) for _ in empty], empty)
        p.free(some, [rng.randint(0, 90) for _ in some])
        if rng.random() < 0.2:
            used = sum(n > 0 for n in p.refs)
            p.compact()
            assert all(n > 0 for n in p.refs[:used]) and not any(p.refs[used:])
        held = [q for r, row in enumerate(p.table) for q in row[: -(-p.lengths[r] // 16)]]
        assert all(p.refs[q] == held.count(q) for q in range(60))
        assert all(q == -1 for r, row in enumerate(p.table) for q in row[-(-p.lengths[r] // 16):])


@pytest.fixture(scope="module")
def lib():
    from enargeia_b200 import build, _lib

    build.build()
    return _lib.load()


def test_entry_points_refuse(lib):
    from enargeia_b200._lib import PagesDims

    p, good = C.c_void_p(16), PagesDims(4, 4, 8, 16)
    assert lib.enx_pages_free(None, p, p, p, p, 1, p, C.byref(good), None) == 1
    assert lib.enx_pages_free(p, p, p, None, p, 1, p, C.byref(good), None) == 1
    assert lib.enx_pages_free(p, p, p, p, p, 5, p, C.byref(good), None) == 3
    assert lib.enx_pages_free(p, p, p, None, None, 0, p, C.byref(good), None) == 0
    for bad in (PagesDims(0, 4, 8, 16), PagesDims((1 << 18) + 1, 4, 8, 16), PagesDims(4, 0, 8, 16), PagesDims(4, 4, 0, 16),
                PagesDims(4, 4, 8, 0), PagesDims(4, 1 << 20, 8, 1 << 12)):
        assert lib.enx_pages_fork(p, p, p, p, p, 1, p, C.byref(bad), None) == 3
    assert lib.enx_pages_grow(p, p, p, p, p, 1, p, None, p, C.byref(good), p, None) == 1
    assert lib.enx_pages_grow(p, p, p, p, p, 1, p, p, p, C.byref(good), C.c_void_p(20), None) == 1
    assert lib.enx_pages_compact(p, p, p, None, p, p, p, p, C.byref(good), p, None) == 1
    assert lib.enx_pages_copy(p, 1, 4, 24, p, 1, p, p, None) == 1
    assert lib.enx_pages_copy(C.c_void_p(8), 1, 4, 32, p, 1, p, p, None) == 1
    assert lib.enx_pages_copy(p, 0, 4, 32, p, 1, p, p, None) == 3
    assert lib.enx_pages_copy(p, 1, 4, 32, None, 0, p, p, None) == 0
    assert lib.enx_pages_workspace_bytes(4, 8) >= 4 * 8 * 4 + 4 * 8
