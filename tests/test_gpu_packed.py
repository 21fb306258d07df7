"""enx_attn_packed against attention in 64 bits on the same 16-bit inputs.

Bound: scores are f32 sums of hd products of 16-bit values, exact products, each of hd/16 + 1
accumulations cut at 2^-22 of the largest partial sum, at most Q = scale * sum |q k|: 2^-18 Q with
hd 128; a weight is off by a factor exp(2 * 2^-18 Q) and by 7.6e-5 (the cubic of some exponentials, 7.5e-5,
and f32 roundings), which acts above and below the quotient, and its rounding to 16 bits is half a step (weights below f16's normal numbers: 2^-25 of the largest, times the keys).
Outputs are rounded once more, half a step."""

import math

import pytest
import torch

from enargeia_b200 import kernels as K
from enargeia_b200._lib import EnxError

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(lengths, heads, kv, hd, dtype, seed=0, spare=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = sum(lengths) + spare
    q = torch.randn(t, heads, hd, generator=gen, device="cuda").to(dtype)
    k = (torch.randn(t, kv, hd, generator=gen, device="cuda") + torch.randn(kv, hd, generator=gen, device="cuda")).to(dtype)
    v = (torch.randn(t, kv, hd, generator=gen, device="cuda") + 0.3 * torch.randn(kv, hd, generator=gen, device="cuda")).to(dtype)
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda")


def reference(q, k, v, scale):
    """(out, bound) of one prompt, q [n, heads, hd], in f64."""
    n, heads, hd = q.shape
    g = heads // k.shape[1]
    half = torch.finfo(q.dtype).eps / 2
    outs, bounds = [], []
    for h in range(heads):
        qq, kk, vv = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        s = (qq @ kk.T) * scale
        seen = torch.tril(torch.ones(n, n, dtype=torch.bool, device=q.device))
        s = s.masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1)
        big = ((qq.abs() @ kk.abs().T) * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
        outs.append(p @ vv)
        rel = 2 * torch.expm1(2.0 ** -17 * big) + 2 * 7.6e-5 + half
        tiny = p.amax(-1, keepdim=True) * 2.0 ** -25 * (seen.double() @ vv.abs())
        bounds.append(rel * (p @ vv.abs()) + tiny)
    return torch.stack(outs, 1), torch.stack(bounds, 1)


def check(out, q, k, v, ends, scale=None):
    half = torch.finfo(q.dtype).eps / 2
    ends = ends.tolist()
    for a, b in zip(ends, ends[1:]):
        if b > a:
            want, bound = reference(q[a:b], k[a:b], v[a:b], q.shape[-1] ** -0.5 if scale is None else scale)
            got = out[a:b].double()
            off = (got - want).abs() - (bound * (1 + half) + half * want.abs() + 2.0 ** -25)
            assert got.isfinite().all() and float(off.max()) <= 0, (a, b, float(off.max()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (4, 2, 32), (4, 1, 128), (2, 2, 8), (3, 1, 72), (5, 5, 120)])
def test_lengths_around_the_tiles(gpu, heads, kv, hd, dtype):
    lengths = [1, 0, 2, 127, 128, 129, 255, 256, 257, 0, 383, 385, 600, 31]
    q, k, v, ends = make(lengths, heads, kv, hd, dtype, hd)
    out = torch.full_like(q, 7.0)
    K.attn_packed(q, k, v, out, ends)
    K.raw_check()
    check(out, q, k, v, ends)


@pytest.mark.parametrize("hd,dtype", [(64, F16), (128, BF16)])
def test_a_long_prompt(gpu, hd, dtype):
    q, k, v, ends = make([4100, 70, 2900], 2, 1, hd, dtype, 3)
    out = torch.full_like(q, 7.0)
    K.attn_packed(q, k, v, out, ends)
    check(out, q, k, v, ends)
    again = torch.zeros_like(q)
    K.attn_packed(q, k, v, again, ends)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_that_climb(gpu, dtype):
    """The running reference moves at every tile; large scores, both signs, a row of zeros."""
    q, k, v, ends = make([1000], 4, 1, 64, dtype, 4)
    ramp = torch.linspace(-2, 2, 1000, device="cuda")[:, None, None]
    k = (0.05 * k + ramp).to(dtype)
    q = q.abs()
    q[:, 1] *= -1
    q[:, 2] = 0
    q[:, 3] *= 0.01
    out = torch.empty_like(q)
    K.attn_packed(q, k, v, out, ends, scale=0.25)
    check(out, q, k, v, ends, 0.25)


def test_side_by_side_projection_and_rows_of_no_prompt(gpu):
    heads, kv, hd = 6, 2, 64
    lengths = [200, 77]
    q, k, v, ends = make(lengths, heads, kv, hd, F16, 5, spare=40)
    t = q.shape[0]
    qkv = torch.empty(t, heads + 2 * kv, hd, dtype=F16, device="cuda")
    qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:] = q, k, v
    # heads outside, tokens inside, and rows before the first prompt
    wide = torch.full((heads, t, hd + 8), 7.0, dtype=F16, device="cuda")
    out = wide[:, :, 8:].transpose(0, 1)
    ends = ends + 13
    K.attn_packed(qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], out, ends)
    check(out, q, k, v, ends)
    assert (out[:13] == 7).all() and (out[290:] == 7).all() and (wide[:, :, :8] == 7).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("hd,dtype", [(64, F16), (128, BF16)])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, bad, hd, dtype):
    lengths = [130, 300, 40]
    q, k, v, ends = make(lengths, 2, 1, hd, dtype, 6)
    clean = torch.empty_like(q)
    K.attn_packed(q, k, v, clean, ends)
    # behind one prompt's end lies the next one's start
    v2, k2 = v.clone(), k.clone()
    v2[130 + 200, 0, 3] = bad  # token 200 of the second prompt
    k2[130 + 280] = bad        # all of token 280's key
    v2[430:] = bad             # the whole third prompt
    out = torch.empty_like(q)
    K.attn_packed(q, k2, v2, out, ends)
    assert torch.equal(out[:130], clean[:130])
    second, was = out[130:430], clean[130:430]
    assert torch.equal(second[:200], was[:200])
    cols = [i for i in range(hd) if i != 3]
    assert torch.equal(second[200:280][:, :, cols], was[200:280][:, :, cols])
    hit = second[200:280, :, 3]
    assert hit.isnan().all() if math.isnan(bad) else (hit == bad).all()
    if math.isnan(bad):
        assert second[280:].isnan().all() and out[430:].isnan().all()


def test_infinite_values_of_both_signs(gpu):
    q, k, v, ends = make([100], 1, 1, 64, F16, 7)
    v[10, 0, 0], v[20, 0, 0] = math.inf, -math.inf
    out = torch.empty_like(q)
    K.attn_packed(q, k, v, out, ends)
    assert out[:10].isfinite().all() and (out[10:20, 0, 0] == math.inf).all() and out[20:, 0, 0].isnan().all()
    assert out[:, :, 1:].isfinite().all()


def test_nothing_to_do(gpu):
    q, k, v, ends = make([5], 2, 1, 64, F16)
    out = torch.full_like(q, 7.0)
    K.attn_packed(q, k, v, out, ends[:1])
    K.attn_packed(q[:0], k[:0], v[:0], out[:0], torch.zeros(3, dtype=torch.int32, device="cuda"))
    K.attn_packed(q, k, v, out, torch.zeros(4, dtype=torch.int32, device="cuda"))
    # offsets outside the tensor, or falling, are cut to it
    K.attn_packed(q, k, v, out, torch.tensor([-9, -1, 0], dtype=torch.int32, device="cuda"))
    assert (out == 7).all()
    K.attn_packed(q, k, v, out, torch.tensor([0, 900], dtype=torch.int32, device="cuda"))
    check(out, q, k, v, ends)


@pytest.mark.parametrize("t,heads,kv", [(1, 1, 1), (1, 4, 2), (3, 1, 1)])
def test_the_smallest_tensors(gpu, t, heads, kv):
    """Axes of one entry have no step of their own."""
    q, k, v, ends = make([t], heads, kv, 64, BF16, 14)
    out = torch.full_like(q, 7.0)
    K.attn_packed(q, k, v, out, ends)
    check(out, q, k, v, ends)


def test_two_calls_at_once(gpu):
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = [make([900, 40, 300], 6, 2, hd, F16, 15 + hd) for hd in (64, 128)]
    outs = [torch.zeros_like(w[0]) for w in work]
    torch.cuda.synchronize()
    for _ in range(5):
        for side, (q, k, v, ends), out in zip(sides, work, outs):
            K.attn_packed(q, k, v, out, ends, stream=side)
    torch.cuda.synchronize()
    K.raw_check()
    for (q, k, v, ends), out in zip(work, outs):
        check(out, q, k, v, ends)


def test_captured_on_another_stream(gpu):
    q, k, v, ends = make([300, 500], 4, 2, 64, BF16, 8)
    out = torch.zeros_like(q)
    K.attn_packed(q, k, v, out, ends)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        K.attn_packed(q, k, v, out, ends)
    for seed in range(3):
        nq, nk, nv, _ = make([300, 500], 4, 2, 64, BF16, 20 + seed)
        for x, y in ((q, nq), (k, nk), (v, nv)):
            x.copy_(y)
        ends.copy_(torch.tensor([0, 100 * seed + 50, 800], dtype=torch.int32))
        graph.replay()
        check(out, q, k, v, ends)
    direct = torch.zeros_like(out)
    side.wait_stream(torch.cuda.current_stream())
    K.attn_packed(q, k, v, direct, ends, stream=side)
    side.synchronize()
    assert torch.equal(direct, out)


def test_offsets_behind_32_bits(gpu):
    """Rows whose elements lie past 2^32 bytes and 2^31 elements of their tensor."""
    t, heads, hd = 1 << 20, 17, 128
    q = torch.empty(t, heads, hd, dtype=BF16, device="cuda")  # 4.6 GB
    out = torch.empty_like(q)
    a, n = t - 300, 300
    gen = torch.Generator(device="cuda").manual_seed(9)
    q[a:] = torch.randn(n, heads, hd, generator=gen, device="cuda").to(BF16)
    k = q[:, :1]
    K.attn_packed(q, k, k, out, torch.tensor([a, t], dtype=torch.int32, device="cuda"))
    check(out[a:], q[a:], k[a:], k[a:], torch.tensor([0, n]))


def test_prompt_then_pages_then_decode(gpu):
    """A prompt is written to the 4-bit cache, attends what the cache holds of it, and its last token's
    result is what a decode step over the cache gives for the same query."""
    heads, kv, hd, page = 14, 2, 64, 64
    lengths = [200, 64, 333]
    q, k, v, ends = make(lengths, heads, kv, hd, F16, 10)
    dev = q.device
    i32 = dict(dtype=torch.int32, device=dev)
    table, held, refs = torch.full((3, 8), -1, **i32), torch.zeros(3, **i32), torch.zeros(20, **i32)
    pairs, count, status = torch.zeros(3, 2, **i32), torch.zeros(2, **i32), torch.zeros(1, **i32)
    rows = torch.arange(3, **i32)
    K.pages_grow(table, held, refs, rows, torch.tensor(lengths, **i32), pairs, count, status, page)
    seqs = torch.repeat_interleave(rows, torch.tensor(lengths, device=dev)).int()
    positions = (torch.arange(sum(lengths), **i32) - ends[:-1].repeat_interleave(torch.tensor(lengths, device=dev))).int()
    pool = torch.zeros(20, K.kv4_page_bytes(page, kv, hd), dtype=torch.uint8, device=dev)
    kk, vv, out = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q)
    K.kv4_write(k, v, pool, table, seqs, positions, page, kk, vv)
    K.attn_packed(q, kk, vv, out, ends)
    check(out, q, kk, vv, ends)
    last = (ends[1:] - 1).long()
    step = torch.empty(3, heads, hd, dtype=F16, device=dev)
    K.attn_kv4(q[last], pool, table, held, step, kv, page)
    # two roundings of the values to f16 (2^-11) and of weights (2^-11) apart, each way
    far = (step.double() - out[last].double()).abs()
    assert float((far - 2.0 ** -9 * vv.double().abs().amax()).max()) <= 0 and status.item() == 0


def test_a_wait_that_gives_up_is_reported(gpu):
    q, k, v, ends = make([700, 90], 3, 1, 64, F16, 12)
    out = torch.empty_like(q)
    K.raw_check()
    try:
        K.set_wait_limit(1)  # one poll, which may be enough or not
        K.attn_packed(q, k, v, out, ends)
        try:
            K.raw_check()
            check(out, q, k, v, ends)
        except EnxError as e:
            assert e.status == 5
    finally:
        K.set_wait_limit(0)
    K.attn_packed(q, k, v, out, ends)
    K.raw_check()
    check(out, q, k, v, ends)


@pytest.mark.parametrize("prompts", [33, 300])
def test_many_prompts(gpu, prompts):
    """More than a warp of prompts, of all lengths, and empty ones between them."""
    lengths = [(7 * i * i + 3 * i) % 290 for i in range(prompts)]
    q, k, v, ends = make(lengths, 4, 2, 32, BF16, 13)
    out = torch.full_like(q, 7.0)
    K.attn_packed(q, k, v, out, ends)
    K.raw_check()
    check(out, q, k, v, ends)


def test_refused_arguments(gpu):
    q, k, v, ends = make([9], 4, 2, 64, F16)
    ok = dict(q=q, k=k, v=v, out=torch.empty_like(q), offsets=ends)
    odd = torch.empty(9, 4, 68, dtype=F16, device="cuda")
    for bad in (dict(q=q.float(), k=k.float(), v=v.float(), out=q.float()), dict(out=q[:8]), dict(k=k[:8]), dict(v=v.bfloat16()),
                dict(offsets=ends.long()), dict(offsets=ends[:0]), dict(k=k[:, :, :56], v=v[:, :, :56]), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.nan), dict(q=odd[:, :, :64]), dict(q=odd[:, :, 4:]), dict(offsets=ends.cpu()),
                dict(k=k[:, :1].expand(9, 3, 64), v=v[:, :1].expand(9, 3, 64)), dict(k=k[:1].expand(9, 2, 64)),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises((ValueError, EnxError)):
            K.attn_packed(**{**ok, **bad})
    wide = torch.empty(9, 2, 136, dtype=F16, device="cuda")
    with pytest.raises(EnxError):
        K.attn_packed(wide, wide, wide, torch.empty_like(wide), ends)
    thin = torch.empty(9, 2, 12, dtype=F16, device="cuda")
    with pytest.raises(EnxError):
        K.attn_packed(thin, thin, thin, torch.empty_like(thin), ends)


@pytest.mark.parametrize("hd,dtype,big", [(128, BF16, 3e38), (128, BF16, 1e30), (72, BF16, 3e38), (64, BF16, 3e38), (128, F16, 6e4),
                                          (64, F16, 6e4)])
def test_large_values_that_a_row_does_not_see_do_not_reach_it(gpu, hd, dtype, big):
    """Finite ones: a weight of what a row does not see is zero, not merely small."""
    lengths = [130, 300, 40]
    q, k, v, ends = make(lengths, 2, 1, hd, dtype, 16, spare=90)
    clean = torch.empty_like(q)
    K.attn_packed(q, k, v, clean, ends)
    signs = 1 - 2 * (torch.arange(v.numel(), device="cuda").reshape(v.shape) % 3 % 2)
    loud = (big * signs).to(dtype)
    v2, k2, q2 = v.clone(), k.clone(), q.clone()
    v2[130 + 200:430], k2[130 + 200:430] = loud[330:430], loud[330:430]  # the second prompt's later tokens, its diagonal tiles
    v2[430:], k2[430:], q2[430:] = loud[430:], loud[430:], loud[430:]    # the third prompt, and rows of none
    out = torch.empty_like(q)
    K.attn_packed(q2, k2, v2, out, ends)
    assert torch.equal(out[:130], clean[:130]) and torch.equal(out[130:330], clean[130:330])
    # every token's own successor is loud: what a row sees of the rest of its tile is what it saw before
    for at in (1, 5, 63, 64, 127):
        v2, k2 = v.clone(), k.clone()
        v2[130 + at:430] = loud[130 + at:430]
        K.attn_packed(q, k2, v2, out, ends)
        assert torch.equal(out[130:130 + at], clean[130:130 + at]), at


@pytest.mark.parametrize("hd,dtype,big", [(128, BF16, 3e38), (64, BF16, 3e38), (128, F16, 6e4)])
def test_a_weight_that_underflows_is_zero(gpu, hd, dtype, big):
    """Four tokens lie some 500 below the others in the exponent of two: whatever they hold, they add nothing."""
    q, k, v, ends = make([400], 2, 1, hd, dtype, 17)
    q = q.abs()
    k[:4] = -45 * 128 / hd
    quiet, loud = torch.empty_like(q), torch.empty_like(q)
    v[:4] = 0
    K.attn_packed(q, k, v, quiet, ends)
    v[:4] = big
    K.attn_packed(q, k, v, loud, ends)
    assert torch.equal(quiet[4:], loud[4:]) and (loud[0] == v[0]).all()


def test_waits_that_run_out_raise_the_error(gpu):
    """An item of 512 key tiles takes most of a millisecond, and its output waits for all of it: one poll is
    not enough.  The status says so, and the next call is whole again."""
    q, k, v, ends = make([1 << 16], 1, 1, 64, BF16, 18)
    out = torch.empty_like(q)
    K.raw_check()
    try:
        K.set_wait_limit(1)
        K.attn_packed(q, k, v, out, ends)
        with pytest.raises(EnxError) as e:
            K.raw_check()
        assert e.value.status == 5 and "enx_attn_packed" in str(e.value)
        K.raw_check()  # read and cleared
    finally:
        K.set_wait_limit(0)
    q, k, v, ends = make([700, 90], 1, 1, 64, BF16, 19)
    out = torch.empty_like(q)
    K.attn_packed(q, k, v, out, ends)
    K.raw_check()
    check(out, q, k, v, ends)
