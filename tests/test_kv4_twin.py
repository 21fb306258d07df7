"""The 4-bit cache's host twin keeps its own rules, and the C entry points refuse bad arguments
before any CUDA work."""

import ctypes as C

import numpy as np
import pytest

import kv4_twin as twin


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_round_trip_error_is_half_a_step(hd):
    x = np.random.default_rng(hd).standard_normal((50, 2, hd)).astype(np.float32)
    c, s, o = twin.quantise(x)
    n, g = twin.groups(hd)
    # half a step, and what the rounding of scale (15 of it) and offset to f16 takes off the ends
    slack = s.astype(np.float64) * (0.5 + 15 * 2.0 ** -11) + np.abs(o.astype(np.float64)) * 2.0 ** -11
    err = np.abs(twin.values(c, s, o) - x).reshape(50, 2, n, g)
    assert (err <= slack[..., None]).all() and c.max() == 15 and c.min() == 0


def test_pool_rows_do_not_overlap():
    rng = np.random.default_rng(1)
    p = twin.Pool(2, 16, 3, 128)
    held = {}
    for page in range(2):
        for slot in rng.permutation(16):
            for which in range(2):
                q = twin.quantise(rng.standard_normal((3, 128)).astype(np.float32))
                p.put(page, slot, which, *q)
                held[page, slot, which] = twin.values(*q)
    assert all((p.get(*at) == x).all() for at, x in held.items())


@pytest.fixture(scope="module")
def lib():
    from enargeia_b200 import build, _lib

    build.build()
    return _lib.load()


def test_entry_points_refuse(lib):
    from enargeia_b200._lib import Kv4Dims

    p, st = C.c_void_p(256), (C.c_int64 * 4)(64, 64, 64, 64)
    good = (4, 4, 8, 16, 2, 64, 0, 0)

    def write(dims=good, k=p, pool=p, tokens=1):
        return lib.enx_kv4_write(k, p, st, tokens, pool, p, p, p, None, None, C.byref(Kv4Dims(*dims)), None)

    def attn(dims=good, q=p, heads=4, queries=1, batch=1, scale=0.125, ws=p):
        return lib.enx_attn_kv4(q, st, p, p, p, None, p, batch, queries, heads, scale, C.byref(Kv4Dims(*dims)), ws, None)

    assert write(tokens=0) == 0 and attn(batch=0) == 0 and attn(queries=0) == 0
    assert write(k=None) == 1 and write(pool=C.c_void_p(8)) == 1 and attn(q=None) == 1 and attn(ws=C.c_void_p(8)) == 1
    for at, bad, status in ((0, 0, 3), (1, 0, 3), (1, 1 << 28, 3), (2, 0, 3), (3, 8, 1), (3, 24, 1), (4, 0, 3), (5, 96, 1), (5, 0, 1),
                            (6, 3, 1)):
        dims = good[:at] + (bad,) + good[at + 1:]
        assert write(dims) == status and attn(dims) == status, (at, bad)
    assert attn(heads=3) == 1 and attn(heads=0) == 1 and attn(scale=0.0) == 1 and attn(scale=float("nan")) == 1
    assert attn(batch=5) == 3 and attn(queries=1 << 17) == 3
    assert lib.enx_attn_kv4_workspace_bytes(256, 64) < 64 << 20


def test_the_bounded_writer_refuses(lib):
    from enargeia_b200._lib import Kv4Dims

    p, st = C.c_void_p(256), (C.c_int64 * 4)(64, 64, 64, 64)

    def write(dims=(4, 4, 8, 16, 2, 64, 0, 0), k=p, lengths=p, tokens=1):
        return lib.enx_kv4_write_held(k, p, st, tokens, p, p, lengths, p, p, None, None, C.byref(Kv4Dims(*dims)), None)

    assert write(tokens=0, lengths=None) == 0
    assert write(lengths=None) == 1 and write(k=None) == 1 and write((4, 4, 8, 24, 2, 64, 0, 0)) == 1
    assert b"enx_kv4_write_held" in lib.enx_last_error()
