"""Cases that measure the paged 4-bit KV cache and the packed prompt attention.

Four operators, reached through `enargeia_b200.kernels`:

  kv4_write   quantises new K and V rows to 4 bits and puts them into their pages;
  attn_kv4    attention of one or a few new tokens per sequence over such a cache;
  attn_packed causal attention over whole prompts, packed one behind another;
  pages_*     freeing, forking, growing, compacting and copying the pages of a cache.

`run` computes them in elementary torch operations where `own` is false, and calls the
framework where it is true.  A page holds `page` tokens of every kv head; the bytes of one head
of a page are its K codes [page][hd/2], K parameters [page][groups] (f16 scale, f16 offset), then
the same for V.  A group is min(64, hd) neighbouring elements of one token's head; a code c stands
for scale * c + offset, two codes to a byte, the even element in the low half.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ---- cases ----------------------------------------------------------------------------------


def _attn_kv4(name, batch, longest, heads, kv, hd, dtype, page, queries=1):
    return {"name": name, "op": "attn_kv4", "batch": batch, "longest": longest, "heads": heads, "kv": kv, "hd": hd,
            "dtype": dtype, "page": page, "queries": queries}


def _write(name, seqs, longest, kv, hd, dtype, page):
    return {"name": name, "op": "kv4_write", "seqs": seqs, "longest": longest, "kv": kv, "hd": hd, "dtype": dtype, "page": page}


def _packed(name, seqs, longest, heads, kv, hd, dtype):
    return {"name": name, "op": "attn_packed", "seqs": seqs, "longest": longest, "heads": heads, "kv": kv, "hd": hd, "dtype": dtype}


def _turn(name, prompts, samples, longest, page, layers, page_bytes):
    return {"name": name, "op": "pages_turn", "prompts": prompts, "samples": samples, "longest": longest, "page": page,
            "layers": layers, "page_bytes": page_bytes}


def _compact(name, seqs, longest, page, layers, page_bytes, pages):
    return {"name": name, "op": "pages_compact", "seqs": seqs, "longest": longest, "page": page, "layers": layers,
            "page_bytes": page_bytes, "pages": pages}


def listed():
    return [
        # the first decoded token behind a 32-id prompt, one user: latency alone
        _attn_kv4("kv4 one short", 1, 33, 14, 2, 64, "f32", 16),
        # batched decode of 256 sequences on their way to context 2048, one layer
        _attn_kv4("kv4 batch 256", 256, 2048, 14, 2, 64, "f32", 64),
        # a few users with long documents, wider heads
        _attn_kv4("kv4 long", 4, 131072, 32, 8, 128, "bf16", 64),
        # four drafted tokens of each sequence verified in one call
        _attn_kv4("kv4 verify 4", 24, 5000, 14, 2, 64, "f16", 32, 4),
        # one decode step's rows of 256 sequences
        _write("write step", 256, 1, 2, 64, "f32", 64),
        # the rows of prompts that were just prefilled
        _write("write prompts", 19, 4100, 8, 128, "bf16", 64),
        # a handful of chat turns
        _packed("packed short", 6, 130, 14, 2, 64, "f16"),
        # a prefill batch of prompts up to the 2048-token context
        _packed("packed prompts", 16, 2048, 14, 2, 64, "f16"),
        # long documents, wider heads
        _packed("packed long", 3, 12001, 32, 8, 128, "bf16"),
        # one prompt's four samples replaced by four new ones
        _turn("turn four samples", 1, 4, 300, 16, 24, 2304),
        # eight samples of each of 64 prompts replaced
        _turn("turn many samples", 64, 8, 2047, 64, 24, 9216),
        # a fragmented pool closed up so that its upper part can be given back
        _compact("compact pool", 192, 1600, 64, 24, 9216, 4800),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["attn_kv4", "kv4_write", "attn_packed", "pages_turn", "pages_compact"])
    heads, kv, hd = rng.choice([(14, 2, 64), (4, 2, 32), (32, 8, 128), (8, 8, 64), (16, 1, 128), (12, 4, 64), (10, 2, 128)])
    page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["f32", "f16", "bf16"])
    if op == "attn_kv4":
        longest = _log(rng, 1, 131072)
        batch = _log(rng, 1, min(256, max(1, (1 << 29) // (longest * kv * hd))))
        queries = rng.choice([1, 1, 1, 2, 3, 5, 8])
        return {k: v for k, v in _attn_kv4("", batch, longest, heads, kv, hd, dtype, page, queries).items() if k != "name"}
    if op == "kv4_write":
        longest = _log(rng, 1, 8192)
        seqs = _log(rng, 1, max(1, min(256, 40000 * 1024 // (longest * kv * hd))))
        return {k: v for k, v in _write("", seqs, longest, kv, hd, dtype, page).items() if k != "name"}
    if op == "attn_packed":
        longest = _log(rng, 1, 12001)
        seqs = _log(rng, 1, max(1, min(64, 2 * 12001 ** 2 * 32 * 128 // (longest ** 2 * heads * hd), 30000 // longest)))
        return {k: v for k, v in _packed("", seqs, longest, heads, kv, hd, rng.choice(["f16", "bf16"])).items() if k != "name"}
    page_bytes, layers = page * kv * (hd + 8 * max(1, hd // 64)), rng.choice([2, 4, 24])
    if op == "pages_turn":
        longest, samples = _log(rng, 1, 4096), _log(rng, 1, 8)
        prompts = _log(rng, 1, max(1, min(64, (220 << 20) // (layers * page_bytes * samples))))
        while prompts > 1 and layers * page_bytes * prompts * (longest // page + 2 + samples) > 2 << 30:
            prompts //= 2
        longest = max(1, min(longest, (2 << 30) // (layers * page_bytes) * page // (2 * prompts) - page * (samples + 2)))
        return {k: v for k, v in _turn("", prompts, samples, longest, page, layers, page_bytes).items() if k != "name"}
    pages = max(16, min(_log(rng, 16, 16384), (900 << 20) // (layers * page_bytes)))
    seqs = _log(rng, 1, min(192, pages // 2))
    longest = max(1, int(pages * rng.uniform(0.3, 0.9) / seqs)) * page
    return {k: v for k, v in _compact("", seqs, longest, page, layers, page_bytes, pages).items() if k != "name"}


# ---- inputs ---------------------------------------------------------------------------------


def _sizes(case):
    """The case's sizes as numbers."""
    return [v if isinstance(v, int) else sum(map(ord, v)) for k, v in sorted(case.items()) if k != "name"]


def _rng(case, seed):
    """A host generator and a device one, both from the case's sizes and the seed."""
    host = np.random.default_rng([int(seed)] + _sizes(case))
    dev = torch.Generator(device=DEV)
    dev.manual_seed(int(host.integers(1 << 62)))
    return host, dev


def _lengths(case, count):
    """`count` lengths up to the case's longest, which one of them has: the same ones for every
    seed (in another order), so that a case is one amount of work."""
    n = np.random.default_rng(_sizes(case)).integers(1, case["longest"] + 1, count).astype(np.int64)
    n[0] = case["longest"]
    if "pages" in case:  # no more than the pool holds
        n = np.minimum(n, case["pages"] // count * case["page"])
    return n


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(DEV)


def _tables(host, lengths, page, spare=0, width=None):
    """A page table with every sequence's pages drawn without order from a pool."""
    need = -(-lengths // page)
    width = int(max(1, need.max())) if width is None else width
    total = int(need.sum())
    order = host.permutation(total + spare)[:total]
    table = np.full((len(lengths), width), -1, np.int64)
    table[np.arange(width) < need[:, None]] = order
    return table, total + spare


def _rows(shape, dtype, gen, channel):
    """Activations as attention sees them: unit noise about a mean that each channel has."""
    x = torch.randn(shape, generator=gen, device=DEV)
    return (x + channel).to(dtype)


def prepare(case, seed):
    host, gen = _rng(case, seed)
    s = {"case": dict(case)}
    op = case["op"]
    if op in ("pages_turn", "pages_compact"):
        return _prepare_pages(case, host, gen, s)
    kv, hd, dt = case["kv"], case["hd"], TYPES[case["dtype"]]
    channel_k = 1.5 * torch.randn(kv, hd, generator=gen, device=DEV)
    channel_v = 0.3 * torch.randn(kv, hd, generator=gen, device=DEV)
    if op == "attn_packed":
        n = host.permutation(_lengths(case, case["seqs"]))
        t = int(n.sum())
        s["offsets"] = _i32(np.concatenate([[0], np.cumsum(n)]))
        s["lengths"] = [int(v) for v in n]  # the program that packed the prompts knows them
        # q, k and v as one projection leaves them: side by side in each token's row
        heads = case["heads"]
        qkv = torch.empty(t, heads + 2 * kv, hd, dtype=dt, device=DEV)
        qkv[:, :heads] = _rows((t, heads, hd), dt, gen, 0.0)
        qkv[:, heads:heads + kv] = _rows((t, kv, hd), dt, gen, channel_k)
        qkv[:, heads + kv:] = _rows((t, kv, hd), dt, gen, channel_v)
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        s["out"] = torch.zeros(t, heads, hd, dtype=dt, device=DEV)
        return s
    page = case["page"]
    if op == "kv4_write":
        n = _lengths(case, case["seqs"])
        before = 2 * n % (3 * page)  # what the sequences hold already
        order = host.permutation(len(n))
        n, before = n[order], before[order]
        table, pages = _tables(host, n + before, page, spare=3)
        t = int(n.sum())
        s["table"] = _i32(table)
        s["seqs"] = _i32(np.repeat(np.arange(case["seqs"]), n))
        s["positions"] = _i32(np.concatenate([b + np.arange(m) for b, m in zip(before, n)]))
        s["k"] = _rows((t, kv, hd), dt, gen, channel_k)
        s["v"] = _rows((t, kv, hd), dt, gen, channel_v)
        s["pool"] = torch.zeros(pages, page * kv * (hd + 8 * max(1, hd // 64)), dtype=torch.uint8, device=DEV)
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    n = host.permutation(_lengths(case, case["batch"]))
    table, pages = _tables(host, n, page, spare=3)
    s["table"], s["lengths"] = _i32(table), _i32(n)
    s["pool"] = torch.empty(pages, page * kv * (hd + 8 * max(1, hd // 64)), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (page * kv * hd))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        k = _rows((b - a, page, kv, hd), torch.float32, gen, channel_k)
        v = _rows((b - a, page, kv, hd), torch.float32, gen, channel_v)
        s["pool"][a:b] = torch.cat([*_packed_rows(k), *_packed_rows(v)], dim=-1).reshape(b - a, -1)
    s["q"] = _rows((case["batch"], case["queries"], case["heads"], hd), dt, gen, 0.0)
    s["out"] = torch.zeros_like(s["q"])
    return s


def _prepare_pages(case, host, gen, s):
    page = case["page"]
    if case["op"] == "pages_turn":
        n = host.permutation(_lengths(case, case["prompts"]))
        forks = np.repeat(np.arange(case["prompts"]), case["samples"])  # the sample rows' prompts
        total = int((-(-n // page)).sum())
        pages = 2 * total + 2 * len(forks) + 8
        width = -(-int(n.max()) // page) + 2
        table = np.full((len(n) + len(forks), width), -1, np.int64)
        held = np.arange(width) < (-(-n // page))[:, None]
        table[:len(n)][held] = host.permutation(pages)[:total]
        refs = np.bincount(table[table >= 0], minlength=pages)
        # the samples of the turn before: they share their prompt's full pages and own the rest
        free = iter(np.flatnonzero(refs == 0))
        lengths = np.concatenate([n, n[forks] + 1])
        for i, p in enumerate(forks):
            full = int(n[p]) // page
            table[len(n) + i, :full] = table[p, :full]
            refs[table[p, :full]] += 1
            own_page = next(free)
            table[len(n) + i, full] = own_page
            refs[own_page] = 1
        s["src"] = _i32(forks)
        s["dst"] = _i32(len(n) + np.arange(len(forks)))
        s["keep"] = torch.zeros(len(forks), dtype=torch.int32, device=DEV)
        s["add"] = torch.ones(len(forks), dtype=torch.int32, device=DEV)
        s["pairs"] = torch.full((len(forks), 2), -1, dtype=torch.int32, device=DEV)
    else:
        pages = case["pages"]
        n = host.permutation(_lengths(case, case["seqs"]))
        table, _ = _tables(host, n, page, spare=pages - int((-(-n // page)).sum()))
        lengths = n
        refs = np.bincount(table[table >= 0], minlength=pages)
        s["pairs"] = torch.full((pages, 2), -1, dtype=torch.int32, device=DEV)
        s["table_out"], s["refs_out"] = _i32(np.full_like(table, -1)), _i32(np.zeros(pages))
    s["table"], s["lengths"], s["refs"] = _i32(table), _i32(lengths), _i32(refs)
    s["count"] = torch.zeros(2, dtype=torch.int32, device=DEV)
    s["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    s["pool"] = torch.randint(0, 256, (case["layers"], pages, case["page_bytes"]), generator=gen, device=DEV, dtype=torch.uint8)
    return s


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    return _own(s) if own else PLAIN[s["case"]["op"]](s)


def _own(s):
    from enargeia_b200 import kernels as K

    c = s["case"]
    if c["op"] == "attn_kv4":
        K.attn_kv4(s["q"], s["pool"], s["table"], s["lengths"], s["out"], c["kv"], c["page"])
        return s["out"]
    if c["op"] == "kv4_write":
        K.kv4_write(s["k"], s["v"], s["pool"], s["table"], s["seqs"], s["positions"], c["page"], s["k_out"], s["v_out"])
        return {"pool": s["pool"], "k": s["k_out"], "v": s["v_out"]}
    if c["op"] == "attn_packed":
        K.attn_packed(s["q"], s["k"], s["v"], s["out"], s["offsets"])
        return s["out"]
    if c["op"] == "pages_turn":
        K.pages_free(s["table"], s["lengths"], s["refs"], s["dst"], s["keep"], s["status"], c["page"])
        K.pages_fork(s["table"], s["lengths"], s["refs"], s["src"], s["dst"], s["status"], c["page"])
        K.pages_grow(s["table"], s["lengths"], s["refs"], s["dst"], s["add"], s["pairs"], s["count"], s["status"], c["page"])
        K.pages_copy(s["pool"], s["pairs"], s["count"], s["status"])
        return _page_outputs(s, s["table"], s["refs"])
    K.pages_compact(s["table"], s["lengths"], s["refs"], s["table_out"], s["refs_out"], s["pairs"], s["count"], s["status"],
                    c["page"])
    K.pages_copy(s["pool"], s["pairs"], s["count"], s["status"])
    return _page_outputs(s, s["table_out"], s["refs_out"])


def _page_outputs(s, table, refs):
    return {"table": table, "lengths": s["lengths"], "refs": refs, "pairs": s["pairs"], "count": s["count"],
            "status": s["status"], "pool": s["pool"]}


# ---- plain forms ----------------------------------------------------------------------------


def _quantise(x):
    """(codes, scales, offsets) of x [..., hd], in 16-bit parameters per group.  In 64 bits, which
    settle on which side of a border a value lies."""
    g = min(64, x.shape[-1])
    x = x.unflatten(-1, (x.shape[-1] // g, g)).double()
    low, high = x.amin(-1), x.amax(-1)
    # (a tensor of fifteens: torch turns the division by a number into a product)
    scale = ((high - low) / torch.full_like(high, 15.0)).clamp(max=65504.0).float().half()
    offset = low.clamp(-65504.0, 65504.0).float().half()
    wide = scale.double()[..., None]
    codes = torch.where(wide > 0, ((x - offset.double()[..., None]) / wide).round_().clamp_(0, 15), torch.zeros_like(x))
    return codes.float(), scale, offset


def _packed_rows(x):
    """The bytes of x [pages, page, kv, hd]: codes and parameters, [pages, kv, bytes] each."""
    codes, scale, offset = _quantise(x)
    c = codes.flatten(-2).to(torch.uint8)
    c = (c[..., 0::2] | (c[..., 1::2] << 4)).transpose(1, 2).flatten(2)
    p = torch.stack([scale, offset], -1).transpose(1, 2).contiguous().view(torch.uint8).flatten(2)
    return c.contiguous(), p


def _values(codes, params, hd):
    """f32 [..., hd] of code bytes [..., hd/2] and their parameters' bytes [..., groups*4]."""
    p = params.contiguous().view(torch.float16).unflatten(-1, (-1, 2)).float()
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (p.shape[-2], -1))
    return (c * p[..., :1] + p[..., 1:]).flatten(-2)


def _sections(pool, kv, page, hd):
    """K codes, K parameters, V codes, V parameters of pages [..., bytes]: [..., kv, page, bytes] each."""
    groups = max(1, hd // 64)
    b = pool.unflatten(-1, (kv, -1))
    sizes = [page * hd // 2, page * groups * 4] * 2
    return [x.unflatten(-1, (page, -1)) for x in b.split(sizes, dim=-1)]


def _plain_attn_kv4(s):
    c = s["case"]
    kv, hd, page, heads = c["kv"], c["hd"], c["page"], c["heads"]
    b, queries = s["q"].shape[:2]
    kc, kp, vc, vp = _sections(s["pool"][s["table"].clamp(min=0).long()], kv, page, hd)
    # [b, pages, kv, page, hd] -> [b, kv, tokens, hd]
    k = _values(kc, kp, hd).transpose(1, 2).flatten(2, 3)
    v = _values(vc, vp, hd).transpose(1, 2).flatten(2, 3)
    at = torch.arange(k.shape[2], device=DEV)
    n = s["lengths"].long()[:, None]
    v = torch.where((at < n)[:, None, :, None], v, torch.zeros_like(v))
    q = s["q"].float().unflatten(2, (kv, heads // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, kv, q*g, hd]
    scores = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    last = n - queries + torch.arange(queries, device=DEV)  # [b, q]: the position of each query
    seen = (at <= last[..., None]).repeat_interleave(heads // kv, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    s["out"].copy_(out.unflatten(2, (queries, heads // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3))
    return s["out"]


def _plain_kv4_write(s):
    c = s["case"]
    kv, hd, page = c["kv"], c["hd"], c["page"]
    where = s["table"].long()[s["seqs"].long(), (s["positions"] // page).long()]
    slot = (s["positions"] % page).long()
    sections = _sections(s["pool"], kv, page, hd)
    for x, back, codes_at, params_at in ((s["k"], s["k_out"], 0, 1), (s["v"], s["v_out"], 2, 3)):
        codes, scale, offset = _quantise(x)
        back.copy_((codes * scale.float()[..., None] + offset.float()[..., None]).flatten(-2))
        u = codes.flatten(-2).to(torch.uint8)
        sections[codes_at][where, :, slot] = u[..., 0::2] | (u[..., 1::2] << 4)
        sections[params_at][where, :, slot] = torch.stack([scale, offset], -1).view(torch.uint8).flatten(-2)
    return {"pool": s["pool"], "k": s["k_out"], "v": s["v_out"]}


def _plain_attn_packed(s):
    c = s["case"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    begin = 0
    for n in s["lengths"]:  # the prompts have nothing to do with one another
        rows = slice(begin, begin + n)
        q = s["q"][rows].float().unflatten(1, (kv, heads // kv)).permute(1, 2, 0, 3)  # [kv, g, n, hd]
        k = s["k"][rows].float().permute(1, 2, 0)[:, None]
        v = s["v"][rows].float().permute(1, 0, 2)[:, None]
        e = torch.matmul(q, k).div_(math.sqrt(hd))
        at = torch.arange(n, device=DEV)
        e.masked_fill_(at[None, :] > at[:, None], -math.inf)
        e.sub_(e.amax(-1, keepdim=True)).exp_()
        out = torch.matmul(e, v).div_(e.sum(-1, keepdim=True))
        s["out"][rows] = out.permute(2, 0, 1, 3).flatten(1, 2).to(s["out"].dtype)
        begin += n
    return s["out"]


def _held(lengths, page, width):
    """Which entries of each row's table hold a page, for those lengths."""
    return torch.arange(width, device=DEV) < ((lengths.long() + page - 1) // page)[:, None]


def _plain_pages_turn(s):
    page, table, lengths, refs = s["case"]["page"], s["table"], s["lengths"], s["refs"]
    src, dst, width = s["src"].long(), s["dst"].long(), table.shape[1]
    one = torch.ones((), dtype=torch.int32, device=DEV)
    # free what the rows hold behind `keep`
    kept = torch.minimum(lengths[dst], s["keep"])
    gone = _held(lengths[dst], page, width) & ~_held(kept, page, width)
    rows = table[dst]
    refs.index_put_((rows[gone].long(),), -one, accumulate=True)
    table[dst] = rows.masked_fill(gone, -1)
    lengths[dst] = kept
    # fork: the same pages, held once more
    held = _held(lengths[src], page, width)
    table[dst] = torch.where(held, table[src], torch.full_like(table[dst], -1))
    refs.index_put_((table[src][held].long(),), one, accumulate=True)
    lengths[dst] = lengths[src]
    # grow: a shared page that is partly filled is copied before it is written (all its writers
    # copy it unless nobody else holds it: then the first of them keeps it), then new pages
    old, new = lengths[dst], lengths[dst] + s["add"]
    partial = (old % page != 0) & (s["add"] > 0)
    last = table[dst, (old // page).long().clamp(max=width - 1)].long()
    last = torch.where(partial, last, torch.zeros_like(last))
    writers = torch.bincount(last[partial], minlength=refs.numel())
    order = torch.arange(len(dst), device=DEV)
    first = torch.full((refs.numel(),), len(dst), device=DEV).scatter_reduce(0, last[partial], order[partial], "amin")
    copy = partial & ~((writers[last] == refs[last]) & (first[last] == order))
    fresh = _held(new, page, width) & ~_held(old, page, width)
    wanted = torch.cat([copy[:, None], fresh], 1)
    free = torch.nonzero(refs == 0).flatten()[: int(wanted.sum())].int()
    got = torch.full_like(wanted, -1, dtype=torch.int32)
    got[wanted] = free
    refs[free.long()] = 1
    refs.index_put_((last[copy],), -one, accumulate=True)
    table[dst] = torch.where(fresh, got[:, 1:], table[dst])
    table[dst[copy], (old // page).long()[copy]] = got[copy, 0]
    lengths[dst] = new
    made = torch.stack([last[copy].int(), got[copy, 0]], 1)
    s["pairs"][: len(made)] = made
    s["count"].copy_(torch.stack([copy.sum(), wanted.sum()]))
    s["pool"][:, made[:, 1].long()] = s["pool"][:, made[:, 0].long()]
    return _page_outputs(s, table, refs)


def _plain_pages_compact(s):
    page, table, refs = s["case"]["page"], s["table"], s["refs"]
    live = refs > 0
    total = live.sum()
    below = torch.arange(len(refs), device=DEV) < total
    holes, movers = torch.nonzero(~live & below).flatten(), torch.nonzero(live & ~below).flatten()
    to = torch.arange(len(refs), dtype=torch.int32, device=DEV)
    to[movers] = holes.int()
    held = _held(s["lengths"], page, table.shape[1])
    s["table_out"].copy_(torch.where(held, to[table.clamp(min=0).long()], torch.full_like(table, -1)))
    s["refs_out"].zero_()
    s["refs_out"][to[live].long()] = refs[live]
    s["pairs"][: len(movers)] = torch.stack([movers, holes], 1).int()
    s["count"][0] = len(movers)
    s["count"][1] = total
    s["pool"][:, holes] = s["pool"][:, movers]
    return _page_outputs(s, s["table_out"], s["refs_out"])


PLAIN = {"attn_kv4": _plain_attn_kv4, "kv4_write": _plain_kv4_write, "attn_packed": _plain_attn_packed,
         "pages_turn": _plain_pages_turn, "pages_compact": _plain_pages_compact}


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    op = case["op"]
    n = _lengths(case, case.get("batch") or case.get("seqs") or case["prompts"])
    if op in ("pages_turn", "pages_compact"):
        used = -(-n // case["page"])
        if op == "pages_turn":
            # each sample's rows and counts go down and up again; its partly filled page is copied
            table = 12 * int(used.sum()) * case["samples"]
            copied = int((n % case["page"] != 0).sum()) * case["samples"]
        else:
            # counts and tables once in and out; of the pages in use, those that lie above their number move
            table = 8 * (case["pages"] + int(used.sum()))
            copied = int(used.sum()) * (1 - int(used.sum()) / case["pages"])
        return {"bytes": table + 2 * copied * case["layers"] * case["page_bytes"], "flops": 0}
    kv, hd, tokens = case["kv"], case["hd"], int(n.sum())
    size = 4 if case["dtype"] == "f32" else 2
    held = kv * (hd + 8 * max(1, hd // 64))  # a token's K and V in the cache
    if op == "kv4_write":  # rows and where they go in, the cache's bytes and the values they stand for out
        return {"bytes": tokens * (4 * kv * hd * size + held + 8), "flops": 0}
    heads = case["heads"]
    if op == "attn_packed":
        return {"bytes": tokens * 2 * hd * size * (heads + kv), "flops": int((n * (n + 1)).sum()) * 2 * heads * hd}
    queries = case["queries"]
    return {"bytes": tokens * held + 2 * len(n) * queries * heads * hd * size, "flops": 4 * tokens * queries * heads * hd}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    op = case["op"]
    if op in ("pages_turn", "pages_compact"):
        return None  # whole numbers: the plain form is their definition
    s = prepare(case, seed)
    if op == "kv4_write":
        return {"pool": None, "k": _exact_round_trip(s["k"]), "v": _exact_round_trip(s["v"])}
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    share = heads // kv
    if op == "attn_packed":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        ends = s["offsets"].tolist()
        for a, b in zip(ends, ends[1:]):
            for h in range(heads):
                k, v = s["k"][a:b, h // share].double(), s["v"][a:b, h // share].double()
                for i in range(a, b, 4096):
                    j = min(b, i + 4096)
                    w = (s["q"][i:j, h].double() @ k[: j - a].T) * hd ** -0.5
                    w += torch.full_like(w, -math.inf).triu_(i - a + 1)
                    out[i:j, h] = torch.softmax(w, -1) @ v[: j - a]
        return out
    page = case["page"]
    groups, g = max(1, hd // 64), min(64, hd)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    piece = page * (hd // 2 + 4 * groups)
    for b, n in enumerate(s["lengths"].tolist()):
        used = s["pool"][s["table"][b, : -(-n // page)].long()].reshape(-1, kv, 2, piece)
        for h in range(kv):
            kvs = []
            for which in range(2):
                raw = used[:, h, which]
                code = raw[:, : page * hd // 2].reshape(-1, hd // 2, 1)
                nibble = torch.cat([code % 16, torch.div(code, 16, rounding_mode="floor")], -1).reshape(-1, groups, g).double()
                par = raw[:, page * hd // 2:].contiguous().view(torch.float16).reshape(-1, groups, 2).double()
                kvs.append((nibble * par[..., 0:1] + par[..., 1:2]).reshape(-1, hd)[:n])
            for j in range(case["queries"]):
                m = n - case["queries"] + j + 1
                if m > 0:
                    q = s["q"][b, j, h * share:(h + 1) * share].double()
                    out[b, j, h * share:(h + 1) * share] = torch.softmax((q @ kvs[0][:m].T) * hd ** -0.5, -1) @ kvs[1][:m]
    return out


def _exact_round_trip(x):
    d = x.double()
    g = min(64, d.shape[-1])
    d = d.reshape(*d.shape[:-1], -1, g)
    low, high = d.min(-1, keepdim=True).values, d.max(-1, keepdim=True).values
    scale = ((high - low) / torch.full_like(low, 15)).to(torch.float32).to(torch.float16).double()
    offset = low.to(torch.float16).double()
    steps = torch.round((d - offset) / scale.clamp(min=1e-30)).clamp(0, 15)
    return (steps * scale + offset).reshape(x.shape)
