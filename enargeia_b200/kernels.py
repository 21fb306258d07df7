"""The raw kernel entry points of libenx, over torch CUDA tensors.

Each function mirrors one WGSL dispatch of the reference (inputs, output, dims) and calls the
C ABI directly.  torch is only the allocator and stream provider here.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import AttnDecodeDims, EmbeddingDims, MatmulQ4Dims, PagesDims, SampleDims, SamplingRow, call


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


def _i32(t: torch.Tensor, *shape) -> C.c_void_p:
    """Pointer of a contiguous int32 CUDA tensor, of this shape (None: any size there)."""
    if t.dtype != torch.int32:
        raise ValueError("expected an int32 tensor")
    if len(shape) != t.dim() or any(w is not None and w != g for w, g in zip(shape, t.shape)):
        raise ValueError(f"expected an int32 tensor of shape {shape}, got {tuple(t.shape)}")
    return _ptr(t)


def _call_on(first: torch.Tensor, others, name: str, *args, stream=None) -> None:
    """`call` with the stream appended, on the device that all the tensors have to be on."""
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"expected all tensors on {device}, got one on {t.device}")
    if device.index == torch.cuda.current_device():
        call(name, *args, _stream(stream))
    else:
        with torch.cuda.device(device):
            call(name, *args, _stream(stream))


def _scratch(nbytes: int, like: torch.Tensor, stream=None) -> torch.Tensor:
    """A workspace for one call: its memory is not handed out again before the call is done."""
    if stream is None or like.device.index != torch.cuda.current_device():
        with torch.cuda.device(like.device):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    else:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    if stream is not None:
        ws.record_stream(stream)
    return ws


def _enough(workspace: Optional[torch.Tensor], nbytes: int, like: torch.Tensor, stream) -> torch.Tensor:
    if workspace is None:
        return _scratch(nbytes, like, stream)
    if workspace.numel() * workspace.element_size() < nbytes:
        raise ValueError(f"the workspace has to have {nbytes} bytes")
    return workspace


def _pages_dims(table, lengths, refs, status, page_tokens):
    rows, width = table.shape
    return (_i32(table, None, None), _i32(lengths, rows), _i32(refs, None), _i32(status, 1),
            PagesDims(rows, width, refs.numel(), page_tokens))


def pages_free(table, lengths, refs, rows, keep, status, page_tokens, stream=None):
    """Rows `rows` of the page table keep their first `keep` tokens; the pages behind lose a holder.

    table int32 [rows, width], lengths int32 [rows], refs int32 [pages] (holders of each page) and
    status int32 [1] (error bits of include/enx.h, added to) are the cache's state; lists are int32."""
    t, l, r, st, d = _pages_dims(table, lengths, refs, status, page_tokens)
    n = rows.numel()
    _call_on(table, (lengths, refs, rows, keep, status), "enx_pages_free", t, l, r, _i32(rows, n), _i32(keep, n), n, st,
             C.byref(d), stream=stream)


def pages_fork(table, lengths, refs, src, dst, status, page_tokens, stream=None):
    """Empty rows `dst` become further holders of the pages of rows `src`."""
    t, l, r, st, d = _pages_dims(table, lengths, refs, status, page_tokens)
    n = dst.numel()
    _call_on(table, (lengths, refs, src, dst, status), "enx_pages_fork", t, l, r, _i32(src, n), _i32(dst, n), n, st,
             C.byref(d), stream=stream)


def pages_grow(table, lengths, refs, rows, add, pairs, count, status, page_tokens, workspace=None, stream=None):
    """Room for `add` more tokens in rows `rows`; pairs int32 [n, 2] and count int32 [2] say which
    pages to copy before they are written (`pages_copy`) and how many pages were taken."""
    t, l, r, st, d = _pages_dims(table, lengths, refs, status, page_tokens)
    n = rows.numel()
    if pairs.shape[0] < n:
        raise ValueError(f"pairs has to have {n} rows")
    ws = _enough(workspace, _lib.load().enx_pages_workspace_bytes(d.rows, d.pages), table, stream)
    _call_on(table, (lengths, refs, rows, add, pairs, count, status, ws), "enx_pages_grow", t, l, r, _i32(rows, n),
             _i32(add, n), n, _i32(pairs, None, 2), _i32(count, 2), st, C.byref(d), _ptr(ws), stream=stream)


def pages_compact(table, lengths, refs, table_out, refs_out, pairs, count, status, page_tokens, workspace=None,
                  stream=None):
    """Closes the used pages up to the front: the table and the counts under the new numbers, pairs
    int32 [pages, 2] of pages to copy, count = (pairs, pages in use)."""
    t, l, r, st, d = _pages_dims(table, lengths, refs, status, page_tokens)
    if pairs.shape[0] < d.pages:
        raise ValueError(f"pairs has to have {d.pages} rows")
    ws = _enough(workspace, _lib.load().enx_pages_workspace_bytes(d.rows, d.pages), table, stream)
    _call_on(table, (lengths, refs, table_out, refs_out, pairs, count, status, ws), "enx_pages_compact", t, l, r,
             _i32(table_out, d.rows, d.width), _i32(refs_out, d.pages), _i32(pairs, None, 2), _i32(count, 2), st,
             C.byref(d), _ptr(ws), stream=stream)


def pages_copy(pool, pairs, count, status, stream=None):
    """Copies page pairs[i, 0] onto page pairs[i, 1] in every layer of pool uint8 [layers, pages,
    page bytes], for the first count[0] pairs."""
    if pool.dtype != torch.uint8 or pool.dim() != 3:
        raise ValueError("expected a uint8 pool [layers, pages, page bytes]")
    layers, pages, nbytes = pool.shape
    _call_on(pool, (pairs, count, status), "enx_pages_copy", _ptr(pool), layers, pages, nbytes, _i32(pairs, None, 2),
             pairs.shape[0], _i32(count, None), _i32(status, 1), stream=stream)


def to_device_u32(a) -> torch.Tensor:
    """numpy uint32 -> CUDA int32 tensor with the same bits."""
    import numpy as np

    return torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).cuda()
