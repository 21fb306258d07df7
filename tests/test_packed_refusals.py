"""enx_attn_packed refuses bad arguments before any CUDA work."""

import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from enargeia_b200 import build, _lib

    build.build()
    return _lib.load()


def test_entry_point_refuses(lib):
    p = C.c_void_p(256)
    good = dict(q=p, k=p, v=p, out=p, strides=(256, 64, 128, 64, 128, 64, 256, 64), offsets=p, seqs=1, tokens=9, heads=4, kv_heads=2,
                head_dim=64, dtype=1, scale=0.125)

    def call(**change):
        a = {**good, **change}
        strides = (C.c_int64 * 8)(*a["strides"])
        return lib.enx_attn_packed(a["q"], a["k"], a["v"], a["out"], strides, a["offsets"], a["seqs"], a["tokens"], a["heads"],
                                   a["kv_heads"], a["head_dim"], a["dtype"], a["scale"], None)

    assert call(seqs=0) == 0 and call(tokens=0) == 0
    for change in (dict(dtype=0), dict(dtype=3), dict(head_dim=0), dict(head_dim=60), dict(head_dim=136), dict(kv_heads=0), dict(heads=0),
                   dict(heads=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(q=None), dict(offsets=None),
                   dict(out=C.c_void_p(264)), dict(v=C.c_void_p(2)), dict(strides=(256, 64, 128, 64, 128, 68, 256, 64)),
                   dict(strides=(250, 64, 128, 64, 128, 64, 256, 64))):
        assert call(**change) == 1, change
    for change in (dict(heads=65536, kv_heads=1), dict(tokens=(1 << 24) + 1), dict(seqs=65537),
                   dict(strides=(0, 64, 128, 64, 128, 64, 256, 64)), dict(strides=(256, 64, 128, -64, 128, 64, 256, 64))):
        assert call(**change) == 3, change
