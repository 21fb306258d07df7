"""The paged 4-bit cache (enx_kv4_write, enx_attn_kv4) against its host twin in 64 bits.

What the cache holds is compared bit for bit.  Attention's bound is that of the twin (f32 sums); for
16-bit rows each weight is rounded to f16 too (2^-11), and every output to its type (half a step)."""

import math

import numpy as np
import pytest
import torch

import kv4_twin as twin
from enargeia_b200 import kernels as K
from enargeia_b200._lib import EnxError

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def rows(rng, shape, dtype):
    x = rng.standard_normal(shape) + 1.5 * rng.standard_normal(shape[-2:])
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


def tables(rng, lengths, page, spare=2, width=None):
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare)
    t = np.full((len(lengths), width or max(1, max(need))), -1, np.int64)
    at = 0
    for r, n in enumerate(need):
        t[r, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kv,hd,page", [(2, 64, 16), (2, 32, 64), (1, 128, 32), (3, 128, 128), (5, 64, 128)])
def test_write_is_the_twin_bit_for_bit(gpu, dtype, kv, hd, page):
    rng = np.random.default_rng(kv * hd + page)
    lengths = [1, 37, 2 * page, 3]
    table, pages = tables(rng, lengths, page)
    k, v = rows(rng, (sum(lengths), kv, hd), dtype), rows(rng, (sum(lengths), kv, hd), dtype)
    k[0] = 0.25  # a group of one value
    k[1, 0, :] = torch.arange(hd, device="cuda").to(dtype) % 16  # codes on the borders and exactly on the grid
    k[2, 0, :] = torch.arange(hd, device="cuda").to(dtype) % 31 / 2
    v[1] *= 1e-7  # scales below the normal f16 numbers
    v[3] *= 1e4 if dtype == F16 else 1e7  # and above them
    v[4, 0, 5], k[5, 0, 3] = math.nan, math.inf
    seqs = np.repeat(np.arange(4), lengths)
    positions = np.concatenate([np.arange(n) for n in lengths])
    order = rng.permutation(len(seqs))  # tokens in any order
    pool = torch.full((pages, K.kv4_page_bytes(page, kv, hd)), 0xAB, dtype=torch.uint8, device="cuda")
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    K.kv4_write(k, v, pool, i32(table), i32(seqs[order]), i32(positions[order]), page, ko, vo)
    want = twin.Pool(pages, page, kv, hd, 0xAB)
    for which, (x, back) in enumerate(((k, ko), (v, vo))):
        c, s, o = twin.quantise(x.float().cpu().numpy())
        for i, j in enumerate(order):
            want.put(table[seqs[j], positions[j] // page], positions[j] % page, which, c[i], s[i], o[i])
        held = torch.from_numpy(twin.values(c, s, o).astype(np.float32)).to(dtype)
        assert torch.equal(back.cpu().nan_to_num(7.0, 8.0, 9.0), held.nan_to_num(7.0, 8.0, 9.0))
    got = pool.cpu().numpy()
    nan = 0x7E  # any NaN pattern is one: both sides use the quiet one
    assert (got == want.bytes).all(), nan


def test_write_strides_and_passed_over_tokens(gpu):
    rng = np.random.default_rng(9)
    kv, hd, page = 2, 64, 32
    wide = rows(rng, (12, 3 * kv + 1, hd + 1), F16)
    k, v = wide[:, 1:1 + kv, 1:], wide[:, 3:3 + 2 * kv:2, :hd]  # odd starts and strides
    table = i32([[1, 99], [2, -1]])
    seqs = i32([0, 1, 2, -1, 0, 0, 0, 1, 1, 0, 1, 1])
    positions = i32([0, 5, 1, 1, -1, 64, 33, 33, 6, 31, 0, 31])
    good = [0, 1, 8, 9, 10, 11]  # rows, positions and pages that exist
    pool = torch.zeros(3, K.kv4_page_bytes(page, kv, hd), dtype=torch.uint8, device="cuda")
    ko, vo = torch.full((12, kv, hd), 3.0, dtype=F16, device="cuda"), torch.full((12, kv, hd), 4.0, dtype=F16, device="cuda")
    K.kv4_write(k, v, pool, table, seqs, positions, page, ko, vo)
    want = twin.Pool(3, page, kv, hd)
    for i in good:
        for which, x in enumerate((k, v)):
            want.put(int(table[seqs[i], positions[i] // page]), int(positions[i]) % page, which,
                     *twin.quantise(x[i].float().cpu().numpy()))
    assert (pool.cpu().numpy() == want.bytes).all()
    skipped = [i for i in range(12) if i not in good]
    assert (ko[skipped] == 3).all() and (vo[skipped] == 4).all()
    K.kv4_write(k[:0], v[:0], pool, table, seqs[:0], positions[:0], page)


def cache(rng, lengths, kv, hd, page, spare=2, width=None):
    """A twin pool whose unused bytes are NaN parameters, its table, and K and V per sequence."""
    table, pages = tables(rng, lengths, page, spare, width)
    pool = twin.Pool(pages, page, kv, hd, 0xFF)
    ks, vs = [], []
    for r, n in enumerate(lengths):
        for which, kept in ((0, ks), (1, vs)):
            x = (rng.standard_normal((n, kv, hd)) + rng.standard_normal((kv, hd))).astype(np.float32)
            c, s, o = twin.quantise(x)
            for i in range(n):
                pool.put(table[r, i // page], i % page, which, c[i], s[i], o[i])
            kept.append((twin.values(c, s, o), twin.magnitudes(c, s, o)))
    return table, pool, ks, vs


def check(q, out, lengths, ks, vs, scale, order=None):
    queries = q.shape[1]
    half = torch.finfo(out.dtype).eps / 2
    for b in range(q.shape[0]):
        r = b if order is None else order[b]
        want, bound = twin.attention(q[b].double().cpu().numpy(), ks[r][0], vs[r][0], scale, queries, ks[r][1], vs[r][1],
                                     0.0 if out.dtype == F32 else 2.0 ** -11)
        got = out[b].double().cpu().numpy()
        off = np.abs(got - want) - (bound * (1 + half) + half * np.abs(want))
        assert np.isfinite(got).all() and (off <= 1e-30).all(), (b, float(off.max()))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,hd,page,queries", [(14, 2, 64, 16, 1), (4, 2, 32, 32, 1), (4, 1, 128, 64, 1),
                                                      (16, 1, 128, 128, 1), (3, 3, 64, 32, 1), (14, 2, 64, 64, 4),
                                                      (6, 2, 32, 16, 7), (10, 2, 128, 16, 3), (9, 1, 64, 128, 2)])
def test_attention(gpu, heads, kv, hd, page, queries, dtype):
    rng = np.random.default_rng(heads * hd + page)
    lengths = [0, 1, 2, 15, 16, 17, 127, 128, 129, 300, 513]
    table, pool, ks, vs = cache(rng, lengths, kv, hd, page)
    q = torch.from_numpy(rng.standard_normal((len(lengths), queries, heads, hd)).astype(np.float32)).to(dtype).cuda()
    out = torch.full_like(q, 7.0)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(lengths), out, kv, page)
    check(q, out, lengths, ks, vs, hd ** -0.5)


def test_one_long_sequence_is_shared_by_many_blocks(gpu):
    rng = np.random.default_rng(3)
    lengths = [9000, 5, 4097]
    table, pool, ks, vs = cache(rng, lengths, 1, 64, 64)
    q = torch.from_numpy(rng.standard_normal((3, 1, 5, 64)).astype(np.float32)).cuda()
    outs = []
    for _ in range(3):
        out = torch.full_like(q, 7.0)
        K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(lengths), out, 1, 64)
        outs.append(out)
    check(q, outs[0], lengths, ks, vs, 0.125)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dtype", [F32, F16])
def test_rising_scores_and_wild_scales(gpu, dtype):
    """Scores that climb along the sequence move the softmax's reference many times; V's scales span
    the f16 range; one row dominates."""
    rng = np.random.default_rng(4)
    n, hd, page = 700, 64, 16
    table, pool, ks, vs = cache(rng, [n], 1, hd, page)
    k = (rng.standard_normal((n, 1, hd)) * 0.1 + np.linspace(-3, 3, n)[:, None, None]).astype(np.float32)
    v = (rng.standard_normal((n, 1, hd)) * 10.0 ** rng.uniform(-5, 3, (n, 1, 1))).astype(np.float32)
    for which, x, kept in ((0, k, ks), (1, v, vs)):
        c, s, o = twin.quantise(x)
        for i in range(n):
            pool.put(table[0, i // page], i % page, which, c[i], s[i], o[i])
        kept[0] = (twin.values(c, s, o), twin.magnitudes(c, s, o))
    q = torch.from_numpy(np.abs(rng.standard_normal((1, 1, 6, hd))).astype(np.float32)).to(dtype).cuda()
    q[0, 0, 1] *= -1
    q[0, 0, 2] = 0
    q[0, 0, 3] *= 1e-3
    q[0, 0, 4, 1:] = 0
    out = torch.empty_like(q)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32([n]), out, 1, page, scale=0.3)
    check(q, out, [n], ks, vs, 0.3)


@pytest.mark.parametrize("dtype,queries", [(F32, 1), (BF16, 2)])
def test_more_sequences_than_threads_of_a_block(gpu, dtype, queries):
    rng = np.random.default_rng(14)
    lengths = [int(v) for v in rng.integers(0, 70, 300)]
    lengths[:3], lengths[250] = [0, 0, 0], 700
    table, pool, ks, vs = cache(rng, lengths, 1, 64, 16)
    q = torch.from_numpy(rng.standard_normal((300, queries, 3, 64)).astype(np.float32)).to(dtype).cuda()
    out = torch.full_like(q, 7.0)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(lengths), out, 1, 16)
    check(q, out, lengths, ks, vs, 0.125)


def test_padded_batch_strides_and_three_axes(gpu):
    rng = np.random.default_rng(5)
    lengths = [40, 0, 200]
    table, pool, ks, vs = cache(rng, lengths, 2, 64, 32, width=9)
    order = [2, -1, 0, 1, 3, 2]  # a row twice, none, one outside the table
    wide = torch.from_numpy(rng.standard_normal((6, 20, 65)).astype(np.float32)).cuda()
    q = wide[:, 3:17, 1:]
    out = torch.full((6, 14, 64), 7.0, device="cuda")
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(lengths), out, 2, 32, seqs=i32(order))
    assert (out[1] == 7).all() and (out[4] == 7).all() and (out[3] == 0).all()
    for b in (0, 2, 5):
        check(q[b:b + 1, None], out[b:b + 1, None], lengths, ks, vs, 0.125, [order[b]])


def test_pages_outside_the_pool_poison_their_sequence(gpu):
    rng = np.random.default_rng(6)
    table, pool, ks, vs = cache(rng, [50, 50, 50], 1, 64, 16)
    table[0, 3], table[2, 0] = pool.bytes.shape[0], -1
    q = torch.from_numpy(rng.standard_normal((3, 1, 2, 64)).astype(np.float32)).cuda()
    out = torch.zeros_like(q)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32([50, 50, 50]), out, 1, 16)
    assert out[0].isnan().all() and out[2].isnan().all()
    check(q[1:2], out[1:2], [50], ks[1:2], vs[1:2], 0.125)
    # lengths outside the table are cut to it
    out.zero_()
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32([-3, 1 << 30, 50]), out, 1, 16)
    assert (out[0] == 0).all()


def test_a_page_whose_values_are_not_finite(gpu):
    """NaN in a token that a query does not see leaves it alone, and reaches those that see it."""
    rng = np.random.default_rng(7)
    table, pool, ks, vs = cache(rng, [20], 1, 64, 16)
    bad = np.full((1, 64), np.nan, np.float32)
    pool.put(table[0, 19 // 16], 19 % 16, 1, *twin.quantise(bad))
    q = torch.from_numpy(rng.standard_normal((1, 2, 2, 64)).astype(np.float32)).cuda()
    out = torch.zeros_like(q)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32([20]), out, 1, 16)
    assert out[0, 1].isnan().all()
    # (the twin's weights of unseen tokens are absent, not zero)
    want, bound = twin.attention(q[0].double().cpu().numpy(), ks[0][0], vs[0][0], 0.125, 2, ks[0][1], vs[0][1])
    assert (np.abs(out[0, 0].cpu().numpy() - want[0]) <= bound[0] + 2.0 ** -24 * np.abs(want[0])).all()


def test_write_grow_attend_in_one_captured_step(gpu):
    """A decode step as a server runs it: room for a token, its write and the attention over it,
    captured once and replayed, with rows forked from one prompt."""
    rng = np.random.default_rng(8)
    heads, kv, hd, page, n = 4, 2, 32, 16, 21
    table, lengths = i32(np.full((3, 4), -1)), i32([0, 0, 0])
    refs, status, count = i32([0] * 12), i32([0]), i32([0, 0])
    pool = torch.full((1, 12, K.kv4_page_bytes(page, kv, hd)), 0xFF, dtype=torch.uint8, device="cuda")
    pairs = i32([[0, 0]] * 3)
    prompt_k, prompt_v = rows(rng, (n, kv, hd), F32), rows(rng, (n, kv, hd), F32)
    K.pages_grow(table, lengths, refs, i32([0]), i32([n]), pairs, count, status, page)
    K.kv4_write(prompt_k, prompt_v, pool[0], table, i32([0] * n), i32(np.arange(n)), page)
    K.pages_fork(table, lengths, refs, i32([0, 0]), i32([1, 2]), status, page)
    every, one = i32([0, 1, 2]), i32([1, 1, 1])
    step_k, step_v = torch.zeros(3, kv, hd, device="cuda"), torch.zeros(3, kv, hd, device="cuda")
    q, out = torch.zeros(3, heads, hd, device="cuda"), torch.zeros(3, heads, hd, device="cuda")
    ws = torch.empty(K._lib.load().enx_attn_kv4_workspace_bytes(3, hd), dtype=torch.uint8, device="cuda")
    ps = torch.empty(K._lib.load().enx_pages_workspace_bytes(3, 12), dtype=torch.uint8, device="cuda")

    def step():
        at = lengths.clone()
        K.pages_grow(table, lengths, refs, every, one, pairs, count, status, page, ps)
        K.pages_copy(pool, pairs, count, status)
        K.kv4_write(step_k, step_v, pool[0], table, every, at, page)
        K.attn_kv4(q, pool[0], table, lengths, out, kv, page, workspace=ws)

    saved = [x.clone() for x in (table, lengths, refs, pool)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x, y in zip((table, lengths, refs, pool), saved):
        x.copy_(y)

    def held(x):
        c = twin.quantise(x.cpu().numpy())
        return np.stack([twin.values(*c), twin.magnitudes(*c)])

    k, v = [held(prompt_k)] * 3, [held(prompt_v)] * 3
    for turn in range(14):
        for x in (step_k, step_v, q):
            x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        graph.replay()
        k = [np.concatenate([k[b], held(step_k[b:b + 1])], 1) for b in range(3)]
        v = [np.concatenate([v[b], held(step_v[b:b + 1])], 1) for b in range(3)]
        check(q[:, None], out[:, None], None, k, v, hd ** -0.5)
    assert status.item() == 0 and lengths.tolist() == [35, 35, 35] and sorted(refs.tolist()) == [0] * 5 + [1] * 6 + [3]
    K.raw_check()


def test_a_workspace_is_taken_on_the_stream_of_the_call(gpu):
    """A block that the current stream has just given back, and still works on, is not this call's
    workspace on another stream."""
    rng = np.random.default_rng(17)
    table, pool, ks, vs = cache(rng, [2000], 1, 64, 64)
    q = torch.from_numpy(rng.standard_normal((1, 1, 4, 64)).astype(np.float32)).cuda()
    dev, out, t, n = torch.from_numpy(pool.bytes).cuda(), torch.zeros_like(q), i32(table), i32([2000])
    side, size = torch.cuda.Stream(), K._lib.load().enx_attn_kv4_workspace_bytes(1, 64)
    torch.cuda.synchronize()
    busy = torch.empty(size, dtype=torch.uint8, device="cuda")
    at = busy.data_ptr()
    torch.cuda._sleep(20_000_000)
    busy.fill_(0xFF)  # queued behind the sleep
    del busy
    ws = K._enough(None, size, q, side)
    assert ws.data_ptr() != at
    del ws
    K.attn_kv4(q, dev, t, n, out, 1, 64, stream=side)
    torch.cuda.synchronize()
    check(q, out, [2000], ks, vs, 0.125)


def test_nothing_cached_yet_and_in_place_write(gpu):
    rng = np.random.default_rng(15)
    q = torch.from_numpy(rng.standard_normal((5, 1, 4, 64)).astype(np.float32)).cuda()
    out = torch.full_like(q, 7.0)
    pool = torch.full((3, K.kv4_page_bytes(16, 2, 64)), 0xFF, dtype=torch.uint8, device="cuda")
    K.attn_kv4(q, pool, i32(np.full((5, 3), -1)), i32([0] * 5), out, 2, 16)
    assert (out == 0).all()
    k, v = rows(rng, (7, 2, 64), F16), rows(rng, (7, 2, 64), F16)
    want = [twin.values(*twin.quantise(x.float().cpu().numpy())).astype(np.float16) for x in (k, v)]
    K.kv4_write(k, v, pool, i32([[1]]), i32([0] * 7), i32(np.arange(7)), 16, k, v)  # the values replace their source
    assert (k.cpu().numpy() == want[0]).all() and (v.cpu().numpy() == want[1]).all()


def test_two_calls_at_once(gpu):
    rng = np.random.default_rng(16)
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for n in ([3000, 17, 900], [64] * 40):
        table, pool, ks, vs = cache(rng, n, 1, 64, 32)
        q = torch.from_numpy(rng.standard_normal((len(n), 1, 5, 64)).astype(np.float32)).cuda()
        work.append((q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(n), torch.zeros_like(q), n, ks, vs))
    torch.cuda.synchronize()
    for _ in range(5):
        for side, (q, pool, table, lengths, out, *_) in zip(sides, work):
            K.attn_kv4(q, pool, table, lengths, out, 1, 32, stream=side)
    torch.cuda.synchronize()
    for q, _, _, _, out, n, ks, vs in work:
        check(q, out, n, ks, vs, 0.125)


def test_another_stream(gpu):
    rng = np.random.default_rng(11)
    table, pool, ks, vs = cache(rng, [400, 90], 1, 64, 64)
    q = torch.from_numpy(rng.standard_normal((2, 1, 4, 64)).astype(np.float32)).cuda()
    dev, out, t, n = torch.from_numpy(pool.bytes).cuda(), torch.zeros_like(q), i32(table), i32([400, 90])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    K.attn_kv4(q, dev, t, n, out, 1, 64, stream=side)
    side.synchronize()
    check(q, out, [400, 90], ks, vs, 0.125)


def test_a_cache_behind_32_bits(gpu):
    pages, kv, hd, page = 30000, 8, 128, 128
    pool = torch.empty(pages, K.kv4_page_bytes(page, kv, hd), dtype=torch.uint8, device="cuda")  # 4.4 GB
    rng = np.random.default_rng(12)
    n = 130
    k, v = rows(rng, (n, kv, hd), BF16), rows(rng, (n, kv, hd), BF16)
    table = i32([[pages - 1, pages - 2]])
    K.kv4_write(k, v, pool, table, i32([0] * n), i32(np.arange(n)), page)
    q = rows(rng, (1, 1, 16, hd), BF16)
    out = torch.zeros_like(q)
    K.attn_kv4(q, pool, table, i32([n]), out, kv, page)
    held = []
    for x in (k, v):
        c, s, o = twin.quantise(x.float().cpu().numpy())
        held.append((twin.values(c, s, o), twin.magnitudes(c, s, o)))
    check(q, out, [n], held[:1], held[1:], hd ** -0.5)


def test_a_wait_that_gives_up_is_reported(gpu):
    rng = np.random.default_rng(13)
    table, pool, ks, vs = cache(rng, [600], 1, 64, 64)
    q = torch.from_numpy(rng.standard_normal((1, 1, 4, 64)).astype(np.float32)).cuda()
    dev, out, t, n = torch.from_numpy(pool.bytes).cuda(), torch.zeros_like(q), i32(table), i32([600])
    K.raw_check()
    try:
        K.set_wait_limit(1)  # one poll, which may be enough or not
        K.attn_kv4(q, dev, t, n, out, 1, 64)
        try:
            K.raw_check()
            check(q, out, [600], ks, vs, 0.125)
        except EnxError as e:
            assert e.status == 5
    finally:
        K.set_wait_limit(0)
    K.attn_kv4(q, dev, t, n, out, 1, 64)
    K.raw_check()
    check(q, out, [600], ks, vs, 0.125)


def test_refused_arguments(gpu):
    q = torch.zeros(2, 1, 4, 64, device="cuda")
    pool = torch.zeros(3, K.kv4_page_bytes(16, 2, 64), dtype=torch.uint8, device="cuda")
    t, n = i32([[0], [1]]), i32([1, 1])
    ok = dict(q=q, pool=pool, table=t, lengths=n, out=torch.zeros_like(q), kv_heads=2, page_tokens=16)
    K.attn_kv4(**ok)
    for bad in (dict(q=q.double(), out=q.double()), dict(out=torch.zeros_like(q).half()), dict(pool=pool[:, :-16].contiguous()),
                dict(table=t.long()), dict(lengths=i32([1])), dict(seqs=i32([0])), dict(page_tokens=8), dict(kv_heads=3),
                dict(scale=0.0), dict(scale=math.nan), dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), dict(q=q.cpu()), dict(table=t[:1]),
                dict(out=torch.zeros(2 * 4 * 64 + 1, device="cuda")[1:].view(2, 1, 4, 64))):
        with pytest.raises((ValueError, EnxError)):
            K.attn_kv4(**{**ok, **bad})
    k = torch.zeros(2, 2, 64, device="cuda")
    good = dict(k=k, v=k, pool=pool, table=t, seqs=n, positions=n, page_tokens=16)
    for bad in (dict(v=k.half()), dict(seqs=n[:1]), dict(positions=n.float()), dict(k_out=k.half()), dict(v_out=k[:1]),
                dict(k=k[:, :, :63], v=k[:, :, :63]), dict(pool=pool[None]), dict(k_out=torch.zeros(2, 64, 2, device="cuda").mT)):
        with pytest.raises((ValueError, EnxError)):
            K.kv4_write(**{**good, **bad})


def uneven(case, rng, n, hd):
    """(K, V, q [2 heads, hd]) where V's scales lie up to eight powers of ten apart, between tokens that
    one head or the other weighs, or between the groups of a row.  q is positive for head 0 and negative for head 1."""
    q = np.abs(rng.standard_normal((2, hd))) + 0.1
    q[1] *= -1
    k, v = 0.1 * rng.standard_normal((n, 1, hd)), rng.standard_normal((n, 1, hd))
    away = 60 / (np.abs(q).sum(1).min() * hd ** -0.5)  # K of one sign and this size: scores of about +-60
    if case == "early":
        v *= 3e-5
        k[5], v[5] = -away, 5e8 * v[5]
    elif case == "late":
        v *= 3e-5
        k[n - 9], v[n - 9] = -away, 5e8 * v[n - 9]
    elif case == "groups":  # of hd 128: the first half of a row large, the other small
        v[..., :64] *= 3e3
        v[..., 64:] *= 3e-4
    elif case == "rising":  # scores rise for head 0 as the scales fall, and fall for head 1
        k += np.linspace(-away, away, n)[:, None, None]
        v *= 10.0 ** np.linspace(3.5, -3.5, n)[:, None, None]
    elif case == "sink":  # the first token has nearly all the weight and a value near nothing
        k[0], v[0] = away / 6, 1e-5 * v[0]
    elif case == "zero":
        k[0], v[0] = away / 6, 0
    elif case == "flat":  # groups of one value, whose scale is 0
        v[:n // 2] = v[:n // 2, :, :1]
    elif case == "steep":  # (their bound says nothing: the result has to be finite)
        k, v = 1e5 * k, 1e4 * v
    return k.astype(np.float32), v.astype(np.float32), q.astype(np.float32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,queries", [(32, 1), (64, 1), (128, 1), (64, 6), (128, 6)])
@pytest.mark.parametrize("case", ["early", "late", "groups", "rising", "sink", "zero", "flat", "steep"])
def test_scales_far_apart_cost_a_row_nothing(gpu, case, hd, queries, dtype):
    """A value's weight keeps its bits whatever the scale of tokens that this row, or this group of 64 dims,
    gives no weight to."""
    rng = np.random.default_rng(hd + queries)
    n, page = 1500, 32
    table, pool, ks, vs = cache(rng, [n], 1, hd, page)
    k, v, q = uneven(case, rng, n, hd)
    for which, x, kept in ((0, k, ks), (1, v, vs)):
        c, s, o = twin.quantise(x)
        for i in range(n):
            pool.put(table[0, i // page], i % page, which, c[i], s[i], o[i])
        kept[0] = (twin.values(c, s, o), twin.magnitudes(c, s, o))
    q = torch.from_numpy(np.broadcast_to(q, (1, queries, 2, hd)).copy()).to(dtype).cuda()
    out = torch.empty_like(q)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32([n]), out, 1, page)
    check(q, out, [n], ks, vs, hd ** -0.5)
    assert K.raw_check() is None


def test_a_refused_grow_writes_nothing(gpu):
    """A row cut into the middle of a page that it shares, and no page left to copy it to: the other
    holder's tokens stay as they are, in a captured step whose host does not look at the status."""
    rng = np.random.default_rng(18)
    kv, hd, page = 2, 64, 16
    table, lengths = i32(np.full((4, 4), -1)), i32([0] * 4)
    refs, status, count, pairs = i32([0] * 4), i32([0]), i32([0, 0]), i32([[0, 0]] * 4)
    pool = torch.zeros(1, 4, K.kv4_page_bytes(page, kv, hd), dtype=torch.uint8, device="cuda")
    k, v = rows(rng, (32, kv, hd), F16), rows(rng, (32, kv, hd), F16)
    K.pages_grow(table, lengths, refs, i32([0, 2]), i32([32, 16]), pairs, count, status, page)
    K.kv4_write(k, v, pool[0], table, i32([0] * 32), i32(np.arange(32)), page, lengths=lengths)
    K.pages_fork(table, lengths, refs, i32([0]), i32([1]), status, page)
    K.pages_free(table, lengths, refs, i32([1]), i32([20]), status, page)
    ko, vo = torch.full((2, kv, hd), 3.0, dtype=F16, device="cuda"), torch.full((2, kv, hd), 4.0, dtype=F16, device="cuda")
    # row 1 wants a copy of its last page, row 3 (empty) a page: one is left
    which, one = i32([1, 3]), i32([1, 1])
    ps = torch.empty(K._lib.load().enx_pages_workspace_bytes(4, 4), dtype=torch.uint8, device="cuda")

    def step():
        at = lengths[which.long()]
        K.pages_grow(table, lengths, refs, which, one, pairs, count, status, page, ps)
        K.pages_copy(pool, pairs, count, status)
        K.kv4_write(k[:2], v[:2], pool[0], table, which, at, page, ko, vo, lengths=lengths)

    state = [x.clone() for x in (table, lengths, refs, pool)]
    step()
    assert status.item() == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip((table, lengths, refs, pool), state))
    assert (ko == 3).all() and (vo == 4).all()
    # with a page given back the same graph writes both
    K.pages_free(table, lengths, refs, i32([2]), i32([0]), status, page)
    status.zero_()
    graph.replay()
    assert status.item() == 0 and lengths.tolist() == [32, 21, 0, 1]
    want = twin.Pool(4, page, kv, hd)
    want.bytes[:] = state[3][0].cpu().numpy()
    t = table.tolist()
    assert t[1][1] not in t[0] and t[3][0] not in t[0] + t[1]
    want.bytes[t[1][1]] = want.bytes[t[0][1]]
    for i, (page_no, slot) in enumerate(((t[1][1], 4), (t[3][0], 0))):
        for part, x in enumerate((k, v)):
            want.put(page_no, slot, part, *twin.quantise(x[i].float().cpu().numpy()))
    assert (pool[0].cpu().numpy() == want.bytes).all()
    for part, back in enumerate((ko, vo)):
        x = (k, v)[part][:2].float().cpu().numpy()
        assert (back.cpu().numpy() == twin.values(*twin.quantise(x)).astype(np.float16)).all()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_lengths_bound_what_is_written(gpu, dtype):
    """Positions at and past the row's length, of rows of length zero and below, are passed over."""
    rng = np.random.default_rng(19)
    kv, hd, page = 1, 32, 16
    table, lengths = i32([[0, 1], [2, 3], [4, 5]]), i32([17, 0, -4])
    seqs, positions = i32([0, 0, 0, 1, 2, 0, 3, -1]), i32([16, 17, 31, 0, 0, 0, 0, 0])
    k, v = rows(rng, (8, kv, hd), dtype), rows(rng, (8, kv, hd), dtype)
    pool = torch.zeros(6, K.kv4_page_bytes(page, kv, hd), dtype=torch.uint8, device="cuda")
    K.kv4_write(k, v, pool, table, seqs, positions, page, lengths=lengths)
    want = twin.Pool(6, page, kv, hd)
    for i, (at, slot) in ((0, (1, 0)), (5, (0, 0))):
        for part, x in enumerate((k, v)):
            want.put(at, slot, part, *twin.quantise(x[i].float().cpu().numpy()))
    assert (pool.cpu().numpy() == want.bytes).all()
    for bad in (i32([1, 1]), lengths.long(), lengths.cpu()):
        with pytest.raises(ValueError):
            K.kv4_write(k, v, pool, table, seqs, positions, page, lengths=bad)


@pytest.mark.parametrize("hd", [32, 128])
def test_values_at_the_end_of_f16_stay_finite(gpu, hd):
    """15 steps of a rounded scale may pass 65504, which f16 rows read back as 65504."""
    k = torch.linspace(0, 65504, hd, device="cuda").half().repeat(3, 2, 1)
    v = -k
    k[1, 0] -= 30000
    k[2], v[2] = torch.linspace(-65504, 65504, hd, device="cuda").half(), 1.0
    pool = torch.zeros(1, K.kv4_page_bytes(16, 2, hd), dtype=torch.uint8, device="cuda")
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    K.kv4_write(k, v, pool, i32([[0]]), i32([0, 0, 0]), i32([0, 1, 2]), 16, ko, vo)
    past = 0
    for x, back in ((k, ko), (v, vo)):
        held = twin.values(*twin.quantise(x.float().cpu().numpy()))
        past += int((held > 65504).sum())
        assert (back.cpu().numpy() == np.minimum(held, 65504.0).astype(np.float16)).all()
    assert past > 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_a_token_with_all_the_weight_comes_back_rounded_once(gpu, hd, dtype):
    """Its weight is 1, and scale, code and offset are exact: what is left of the bound is the f32 sum of the
    two terms (2^-22 of their sizes: f32 rows split them at code 8) and the output's own half step."""
    rng = np.random.default_rng(hd)
    lengths = [1] * 40 + [70] * 10
    table, pool, ks, vs = cache(rng, lengths, 1, hd, 16)
    q = np.abs(rng.standard_normal((50, 1, 4, hd))).astype(np.float32) + 0.2
    for r in range(40, 50):  # one token far above the others, anywhere
        at = int(rng.integers(70))
        c, s, o = twin.quantise(np.full((1, hd), 60 * hd ** -0.5, np.float32))
        pool.put(table[r, at // 16], at % 16, 0, c, s, o)
        c, s, o = twin.quantise((rng.standard_normal((1, hd)) * 3).astype(np.float32))
        pool.put(table[r, at // 16], at % 16, 1, c, s, o)
        vs[r] = (twin.values(c, s, o)[None], twin.magnitudes(c, s, o)[None])
    q = torch.from_numpy(q).to(dtype).cuda()
    out = torch.empty_like(q)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(lengths), out, 1, 16, scale=1.0)
    half = torch.finfo(dtype).eps / 2
    for r in range(50):
        value, size = vs[r][0][0, 0], vs[r][1][0, 0]
        off = np.abs(out[r, 0].double().cpu().numpy() - value) - (half * np.abs(value) * (1 + 2.0 ** -11) + 2.0 ** -22 * size)
        assert (off <= 0).all(), (r, float(off.max()))


@pytest.mark.parametrize("heads,kv,hd,queries", [(14, 2, 64, 1), (4, 2, 32, 1), (16, 2, 128, 1), (14, 2, 64, 3), (16, 2, 128, 4)])
def test_f16_rows_lose_no_more_than_the_outputs_rounding(gpu, heads, kv, hd, queries):
    """f16 rows are held to the bound of f32 rows (`weight` 0: no further rounding of the weights) and half a step
    of the output.  Small scores, so that the bound's share of them is small too."""
    rng = np.random.default_rng(hd + queries)
    lengths = [4, 5, 7, 9, 17, 33, 60, 64, 65, 130, 300]
    table, pool, ks, vs = cache(rng, lengths, kv, hd, 32)
    q = torch.from_numpy(0.05 * rng.standard_normal((len(lengths), queries, heads, hd)).astype(np.float32)).half().cuda()
    out = torch.empty_like(q)
    K.attn_kv4(q, torch.from_numpy(pool.bytes).cuda(), i32(table), i32(lengths), out, kv, 32)
    half = torch.finfo(F16).eps / 2
    for b in range(len(lengths)):
        want, bound = twin.attention(q[b].double().cpu().numpy(), ks[b][0], vs[b][0], hd ** -0.5, queries, ks[b][1], vs[b][1])
        off = np.abs(out[b].double().cpu().numpy() - want) - (bound * (1 + half) + half * np.abs(want) + 2.0 ** -25)
        assert (off <= 0).all(), (b, float(off.max()))
