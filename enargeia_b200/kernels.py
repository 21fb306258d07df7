"""The raw kernel entry points of libenx, over torch CUDA tensors.

Each function mirrors one WGSL dispatch of the reference (inputs, output, dims) and calls the
C ABI directly.  torch is only the allocator and stream provider here.
"""

from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from ._lib import AttnDecodeDims, EmbeddingDims, Kv4Dims, MatmulQ4Dims, PagesDims, SampleDims, SamplingRow, call


def _ptr(t: Optional[torch.Tensor]):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return C.c_void_p(t.data_ptr())


def _stream(stream=None):
    s = torch.cuda.current_stream() if stream is None else stream
    return C.c_void_p(s.cuda_stream)


def _u32(t: torch.Tensor):
    # int32 storage reinterpreted as u32 on the device side
    if t.dtype not in (torch.int32, torch.uint32):
        raise ValueError("packed words must be int32/uint32 tensors")
    return _ptr(t)


def matmul_q4(x, packed, scales, zeros, bias, out, m, n, k, out_stride=None, out_offset=0, stream=None):
    """matmul_q4_decode / matmul_q4_prefill (src/kernels/matmul_q4.ts:50-64)."""
    d = MatmulQ4Dims(m, n, k, 1 if bias is not None else 0, 64, k // 64, n if out_stride is None else out_stride,
                     out_offset, min(n, 65535), 0, 0, 0)
    call("enx_matmul_q4", _ptr(x), _u32(packed), _ptr(scales), _u32(zeros), _ptr(bias), _ptr(out), C.byref(d),
         _stream(stream))
    return out


def set_wait_limit(spins: int, device: int = 0) -> None:
    """Polls a bounded device wait makes before it gives up (0: the default)."""
    call("enx_set_wait_limit", device, spins)


def raw_check():
    """Synchronise the device and raise if a bounded wait of the raw tensor-core GEMM gave up."""
    call("enx_raw_check")


def lm_head_q8(x, packed, scales, zeros, out, rows, hidden, row_begin=0, out_offset=0, stream=None):
    """lm_head_q8 (src/kernels/embedding_variants.ts:135-180)."""
    d = EmbeddingDims(1, hidden, row_begin, rows, 64, hidden // 64, 0, out_offset, min(rows, 65535), 0, 0, 0)
    call("enx_lm_head_q8", _ptr(x), _u32(packed), _ptr(scales), _u32(zeros), _ptr(out), C.byref(d), _stream(stream))
    return out


def embed_gather_q8(ids, packed, scales, zeros, out, hidden, row_begin, row_count, stream=None):
    """embed_gather_q8 (src/kernels/embedding_variants.ts:100-130)."""
    d = EmbeddingDims(ids.numel(), hidden, row_begin, row_count, 64, hidden // 64, 0, 0, 0, 0, 0, 0)
    call("enx_embed_gather_q8", _u32(ids), _u32(packed), _ptr(scales), _u32(zeros), _ptr(out), C.byref(d),
         _stream(stream))
    return out


def sample(logits, history, out, temperature, top_p, repetition_penalty, random, stream=None):
    """sample (src/kernels/sample.wgsl): in-place penalty on `logits`, one id to out[0]."""
    d = SampleDims(logits.numel(), 0 if history is None else history.numel(), temperature, top_p,
                   repetition_penalty, random, 0, 0)
    call("enx_sample", _ptr(logits), None if history is None or history.numel() == 0 else _u32(history), _u32(out),
         C.byref(d), None, _stream(stream))
    return out


def sample_batched(logits, history, history_length, rows, out, stream=None):
    """Rows of logits [B, V]; history [B, stride] (u32); history_length [B]; rows: a CUDA byte
    tensor of B SamplingRow structs (see `sampling_rows`)."""
    B, V = logits.shape
    call("enx_sample_batched", _ptr(logits), V, B, _u32(history), history.shape[1], _u32(history_length),
         _ptr(rows), _u32(out), _stream(stream))
    return out


def sampling_rows(params, device="cuda") -> torch.Tensor:
    """[(temperature, top_p, repetition_penalty, random), ...] -> device bytes of SamplingRow."""
    arr = (SamplingRow * len(params))(*[SamplingRow(*p) for p in params])
    host = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8)
    return host.to(device)


def attn_decode(q, k_cache, v_cache, out, position, heads, kv_heads, head_dim, workspace=None, stream=None):
    d = AttnDecodeDims(position, heads, kv_heads, head_dim, 0, kv_heads * head_dim, 0, 0)
    if workspace is None:
        n = _lib.load().enx_attn_decode_workspace_bytes(position + 1, heads, head_dim)
        workspace = torch.empty(n, dtype=torch.uint8, device=q.device)
    call("enx_attn_decode", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), C.byref(d), _ptr(workspace),
         _stream(stream))
    return out


def attn_prefill(q, k_cache, v_cache, out, queries, begin, heads, kv_heads, head_dim, workspace=None, stream=None):
    if workspace is None:
        n = _lib.load().enx_attn_prefill_workspace_bytes(queries, begin + queries, heads, head_dim)
        workspace = torch.empty(n, dtype=torch.uint8, device=q.device)
    call("enx_attn_prefill", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), queries, begin, heads, kv_heads,
         head_dim, _ptr(workspace), _stream(stream))
    return out


def rmsnorm(x, w, out, seq, features, eps=1e-6, stream=None):
    call("enx_rmsnorm", _ptr(x), _ptr(w), _ptr(out), seq, features, eps, _stream(stream))
    return out


def rope(x, out, cos_t, sin_t, seq, heads, head_dim, pos0=0, out_offset=0, stream=None):
    call("enx_rope", _ptr(x), _ptr(out), _ptr(cos_t), _ptr(sin_t), seq, heads, head_dim, pos0, out_offset,
         _stream(stream))
    return out


def cache_pack(src, dst, count, dst_offset=0, stream=None):
    call("enx_cache_pack", _ptr(src), _ptr(dst), count, dst_offset, _stream(stream))
    return dst


def silu_mul(g, u, out, stream=None):
    call("enx_silu_mul", _ptr(g), _ptr(u), _ptr(out), g.numel(), _stream(stream))
    return out


def add(a, b, out, stream=None):
    call("enx_add", _ptr(a), _ptr(b), _ptr(out), a.numel(), _stream(stream))
    return out


# ---- pages of a shared key/value cache -----------------------------------------------------------
#
# These calls take a few microseconds on the GPU, so their checks are kept short: one look at each
# tensor, and argument blocks that only depend on sizes are made once per sizes.

_INT32 = torch.int32


def _ints(t: torch.Tensor, n: int) -> int:
    """Address of a contiguous int32 CUDA tensor of n entries."""
    if t.dtype is not _INT32 or t.numel() != n or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"expected a contiguous int32 CUDA tensor of {n} entries, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


#: The current device and the current stream's handle, without the objects around them.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call_on(tensors, stream, name: str, *args) -> None:
    """`call` with the stream appended, on the device that all the tensors (None: absent) are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"expected all tensors on one device, got {tensors[0].device} and {t.device}")
    if index < 0:
        raise ValueError("expected CUDA tensors")
    if index != _current_device():
        with torch.cuda.device(index):
            return call(name, *args, _raw_stream(index) if stream is None else stream.cuda_stream)
    call(name, *args, _raw_stream(index) if stream is None else stream.cuda_stream)


def _enough(workspace: Optional[torch.Tensor], nbytes: int, like: torch.Tensor, stream) -> torch.Tensor:
    """The caller's workspace, or one for this call from the memory of the stream that it runs on (the
    allocator orders a block's users by the stream that it was taken on)."""
    if workspace is None:
        if stream is None:
            return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
        with torch.cuda.stream(stream):
            return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    if workspace.numel() * workspace.element_size() < nbytes or not workspace.is_contiguous() or not workspace.is_cuda:
        raise ValueError(f"the workspace has to have {nbytes} contiguous bytes on the device")
    return workspace


@lru_cache(maxsize=256)
def _pages_block(rows, width, pages, page_tokens):
    """(argument block, workspace bytes) of the page calls."""
    return C.byref(PagesDims(rows, width, pages, page_tokens)), _lib.load().enx_pages_workspace_bytes(rows, pages)


def pages_free(table, lengths, refs, rows, keep, status, page_tokens, stream=None):
    """Rows `rows` of the page table keep their first `keep` tokens; the pages behind lose a holder.

    table int32 [rows, width], lengths int32 [rows], refs int32 [pages] (holders of each page) and
    status int32 [1] (error bits of include/enx.h, added to) are the cache's state; lists are int32."""
    r, w = table.shape
    n, p = rows.numel(), refs.numel()
    _call_on((table, lengths, refs, rows, keep, status), stream, "enx_pages_free", _ints(table, r * w), _ints(lengths, r),
             _ints(refs, p), _ints(rows, n), _ints(keep, n), n, _ints(status, 1), _pages_block(r, w, p, page_tokens)[0])


def pages_fork(table, lengths, refs, src, dst, status, page_tokens, stream=None):
    """Empty rows `dst` become further holders of the pages of rows `src`."""
    r, w = table.shape
    n, p = dst.numel(), refs.numel()
    _call_on((table, lengths, refs, src, dst, status), stream, "enx_pages_fork", _ints(table, r * w), _ints(lengths, r),
             _ints(refs, p), _ints(src, n), _ints(dst, n), n, _ints(status, 1), _pages_block(r, w, p, page_tokens)[0])


def pages_grow(table, lengths, refs, rows, add, pairs, count, status, page_tokens, workspace=None, stream=None):
    """Room for `add` more tokens in rows `rows`; pairs int32 [n, 2] and count int32 [2] say which
    pages to copy before they are written (`pages_copy`) and how many pages were taken."""
    r, w = table.shape
    n, p = rows.numel(), refs.numel()
    if pairs.numel() < 2 * n:
        raise ValueError(f"pairs has to have {n} rows")
    block, nbytes = _pages_block(r, w, p, page_tokens)
    ws = _enough(workspace, nbytes, table, stream)
    _call_on((table, lengths, refs, rows, add, pairs, count, status, ws), stream, "enx_pages_grow", _ints(table, r * w),
             _ints(lengths, r), _ints(refs, p), _ints(rows, n), _ints(add, n), n, _ints(pairs, pairs.shape[0] * 2), _ints(count, 2),
             _ints(status, 1), block, ws.data_ptr())


def pages_compact(table, lengths, refs, table_out, refs_out, pairs, count, status, page_tokens, workspace=None,
                  stream=None):
    """Closes the used pages up to the front: the table and the counts under the new numbers, pairs
    int32 [pages, 2] of pages to copy, count = (pairs, pages in use)."""
    r, w = table.shape
    p = refs.numel()
    if pairs.numel() < 2 * p or table_out.shape != table.shape:
        raise ValueError(f"pairs has to have {p} rows, and table_out the table's shape")
    block, nbytes = _pages_block(r, w, p, page_tokens)
    ws = _enough(workspace, nbytes, table, stream)
    _call_on((table, lengths, refs, table_out, refs_out, pairs, count, status, ws), stream, "enx_pages_compact",
             _ints(table, r * w), _ints(lengths, r), _ints(refs, p), _ints(table_out, r * w), _ints(refs_out, p),
             _ints(pairs, pairs.shape[0] * 2), _ints(count, 2), _ints(status, 1), block, ws.data_ptr())


def pages_copy(pool, pairs, count, status, stream=None):
    """Copies page pairs[i, 0] onto page pairs[i, 1] in every layer of pool uint8 [layers, pages,
    page bytes], for the first count[0] pairs."""
    layers, pages, nbytes = pool.shape
    if pool.dtype is not torch.uint8:
        raise ValueError("expected a uint8 pool [layers, pages, page bytes]")
    n = pairs.shape[0]
    _call_on((pool, pairs, count, status), stream, "enx_pages_copy", _ptr(pool), layers, pages, nbytes, _ints(pairs, 2 * n), n,
             _ints(count, count.numel()), _ints(status, 1))


# ---- a paged cache held in 4 bits, and attention over it ---------------------------------------------

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def kv4_page_bytes(page_tokens: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of a page of the 4-bit cache (one layer): codes and parameters of K and V."""
    return page_tokens * kv_heads * (head_dim + 8 * max(1, head_dim // 64))


@lru_cache(maxsize=256)
def _kv4_block(rows, width, pages, nbytes, page_tokens, kv_heads, head_dim, dtype):
    """The argument block of the 4-bit cache's calls."""
    if dtype not in _DTYPES:
        raise ValueError(f"expected float32, float16 or bfloat16, got {dtype}")
    if nbytes != kv4_page_bytes(page_tokens, kv_heads, head_dim):
        raise ValueError(f"a page has {kv4_page_bytes(page_tokens, kv_heads, head_dim)} bytes, the pool's {nbytes}")
    return C.byref(Kv4Dims(rows, width, pages, page_tokens, kv_heads, head_dim, _DTYPES[dtype], 0))


@lru_cache(maxsize=256)
def _strides(*elements):
    return (C.c_int64 * len(elements))(*elements)


@lru_cache(maxsize=64)
def _attn_kv4_bytes(batch, head_dim):
    return _lib.load().enx_attn_kv4_workspace_bytes(batch, head_dim)


def _rows_of(t: torch.Tensor) -> int:
    """Address of a CUDA tensor whose last axis is contiguous (its other strides go with the call)."""
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("the last axis has to be contiguous")
    return t.data_ptr()


def _pool_of(pool: torch.Tensor):
    """(pages, page bytes) of one layer's pool."""
    if pool.dtype is not torch.uint8 or pool.dim() != 2:
        raise ValueError("expected one layer's uint8 pool [pages, page bytes]")
    return pool.shape


def kv4_write(k, v, pool, table, seqs, positions, page_tokens, k_out=None, v_out=None, stream=None, lengths=None):
    """Quantises k and v [tokens, kv_heads, head_dim] into the 4-bit cache: token i to position
    positions[i] of table row seqs[i] (int32; a negative position is passed over).  k_out and v_out,
    if given, receive the values that the cache now holds.  With lengths (int32 [rows]) a position at or
    past its row's length is passed over too: nothing is written where `pages_grow` was refused."""
    shape = k.shape
    tokens, kv_heads, hd = shape
    if v.shape != shape or v.dtype is not k.dtype:
        raise ValueError("k and v have to have one shape and type")
    for o in (k_out, v_out):
        if o is not None and (o.shape != shape or o.dtype is not k.dtype):
            raise ValueError("k_out and v_out have to have the shape and type of k")
    r, w = table.shape
    pages, nbytes = _pool_of(pool)
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    held = () if lengths is None else (_ints(lengths, r),)
    _call_on((k, v, pool, table, seqs, positions, k_out, v_out, lengths), stream, "enx_kv4_write_held" if held else "enx_kv4_write",
             _rows_of(k), _rows_of(v), _strides(k0, k1, v0, v1), tokens, _ptr(pool), _ints(table, r * w), *held, _ints(seqs, tokens),
             _ints(positions, tokens), _ptr(k_out), _ptr(v_out), _kv4_block(r, w, pages, nbytes, page_tokens, kv_heads, hd, k.dtype))


def attn_kv4(q, pool, table, lengths, out, kv_heads, page_tokens, seqs=None, scale=None, workspace=None, stream=None):
    """Attention of each sequence's newest tokens over its 4-bit cache: q and out [batch, queries,
    heads, head_dim] or [batch, heads, head_dim]; sequence b is table row seqs[b] (or b), and
    lengths[row] counts its tokens, the queries' own included."""
    shape = q.shape
    if shape != out.shape or q.dtype is not out.dtype:
        raise ValueError("q and out have to have one shape and type")
    if len(shape) == 3:
        batch, heads, hd = shape
        queries, (s0, s2, _) = 1, q.stride()
        s1 = 0
    else:
        batch, queries, heads, hd = shape
        s0, s1, s2, _ = q.stride()
    r, w = table.shape
    pages, nbytes = _pool_of(pool)
    ws = _enough(workspace, _attn_kv4_bytes(batch, hd), q, stream)
    _call_on((q, pool, table, lengths, out, seqs, ws), stream, "enx_attn_kv4", _rows_of(q), _strides(s0, s1, s2), _ptr(pool),
             _ints(table, r * w), _ints(lengths, r), None if seqs is None else _ints(seqs, batch), _ptr(out), batch, queries, heads,
             hd ** -0.5 if scale is None else scale, _kv4_block(r, w, pages, nbytes, page_tokens, kv_heads, hd, q.dtype),
             ws.data_ptr())
    return out


def attn_packed(q, k, v, out, offsets, scale=None, stream=None):
    """Causal attention over prompts packed one behind another: q and out [tokens, heads, head_dim], k
    and v [tokens, kv_heads, head_dim], float16 or bfloat16, any strides whose rows start on 16 bytes;
    prompt s has rows offsets[s] to offsets[s + 1] - 1 (int32 on the device)."""
    tokens, heads, hd = q.shape
    kv_heads = k.shape[1]
    if q.dtype is not torch.float16 and q.dtype is not torch.bfloat16:
        raise ValueError(f"expected float16 or bfloat16, got {q.dtype}")
    if out.shape != q.shape or k.shape != (tokens, kv_heads, hd) or v.shape != k.shape:
        raise ValueError("q and out have to have one shape, and k and v one with the same tokens and head_dim")
    if not (q.dtype is k.dtype is v.dtype is out.dtype):
        raise ValueError("q, k, v and out have to have one type")
    n = offsets.numel()
    if n < 1:
        raise ValueError("offsets has an entry more than there are prompts")
    (q0, q1, _), (k0, k1, _), (v0, v1, _), (o0, o1, _) = q.stride(), k.stride(), v.stride(), out.stride()
    _call_on((q, k, v, out, offsets), stream, "enx_attn_packed", _rows_of(q), _rows_of(k), _rows_of(v), _rows_of(out),
             _strides(q0, q1, k0, k1, v0, v1, o0, o1), _ints(offsets, n), n - 1, tokens, heads, kv_heads, hd, _DTYPES[q.dtype],
             hd ** -0.5 if scale is None else scale)
    return out


def to_device_u32(a) -> torch.Tensor:
    """numpy uint32 -> CUDA int32 tensor with the same bits."""
    import numpy as np

    return torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).cuda()
