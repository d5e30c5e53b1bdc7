"""Attention over the paged KV cache on the library's own kernels: a sliding
window with sinks, and a prefix that a whole batch shares.

The cache layout is that of ``attention.allocate_kv_cache``: position ``j`` of a
sequence lies in slot ``table[j // block_size] * block_size + j % block_size``.
Both functions take the sequences' lengths as device tensors, allocate their
output and workspace from torch's allocator on the stream they run on, never
synchronise, and can be captured in a CUDA graph.  Queries are ragged: sequence
``s`` owns the tokens ``cu_seqlens_q[s] : cu_seqlens_q[s + 1]`` and its last one
is at position ``context_lens[s] - 1``; without ``cu_seqlens_q`` every sequence
has one token (decode).  A query that sees nothing gets zeros.
"""
from __future__ import annotations

import ctypes
import struct

from . import _lib
from .device import dtype_code, require_cuda

# _lib.AttentionArgs field by field (packing is far cheaper than ctypes fields)
_ARGS = struct.Struct("@Q2q2Q3qQ2q3Q8qQQ5if")
assert _ARGS.size == ctypes.sizeof(_lib.AttentionArgs)
_AS_POINTER = ctypes.POINTER(_lib.AttentionArgs)


def _tensors(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, out):
    torch = require_cuda()
    if q.dim() != 3 or k_cache.dim() != 3:
        raise ValueError("q is [tokens, heads, head_dim], the caches [slots, kv_heads, head_dim]")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("the caches must have one shape and one layout")
    if not q.dtype == k_cache.dtype == v_cache.dtype:
        raise ValueError("q and the caches must have one dtype")
    if q.shape[2] != k_cache.shape[2]:
        raise ValueError(f"q has head_dim {q.shape[2]}, the caches {k_cache.shape[2]}")
    if q.stride(2) != 1 or k_cache.stride(2) != 1:
        raise ValueError("a head's elements must be adjacent")
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or \
            block_tables.stride(1) != 1:
        raise ValueError("block_tables must be an int32 [sequences, blocks] tensor with "
                         "adjacent entries")
    seqs = block_tables.shape[0]
    for t, n, what in ((context_lens, seqs, "context_lens"),
                       (cu_seqlens_q, seqs + 1, "cu_seqlens_q")):
        if t is not None and (t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous()):
            raise ValueError(f"{what} must be a contiguous int32 tensor of {n} entries")
    if cu_seqlens_q is None and q.shape[0] != seqs:
        raise ValueError(f"{q.shape[0]} tokens of {seqs} sequences need cu_seqlens_q")
    index = q.get_device()
    for t in (q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, out):
        if t is not None and (t.get_device() != index or index < 0):
            raise ValueError("all tensors must be on one CUDA device")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1
                            or out.stride(1) != out.shape[2]):
        raise ValueError("out must have q's shape and dtype and adjacent heads")
    return torch


def _attend(entry, what, q, k_cache, v_cache, block_tables, context_lens, block_size, window,
            sinks, prefix_len, cu_seqlens_q, max_query_len, max_context_len, scale, out, stream):
    torch = _tensors(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, out)
    if q.get_device() != torch.cuda.current_device():
        with torch.cuda.device(q.get_device()):
            return _attend(entry, what, q, k_cache, v_cache, block_tables, context_lens,
                           block_size, window, sinks, prefix_len, cu_seqlens_q, max_query_len,
                           max_context_len, scale, out, stream)
    if stream is not None and stream != torch.cuda.current_stream():
        with torch.cuda.stream(stream):   # output and workspace belong to that stream
            return _attend(entry, what, q, k_cache, v_cache, block_tables, context_lens,
                           block_size, window, sinks, prefix_len, cu_seqlens_q, max_query_len,
                           max_context_len, scale, out, None)
    tokens, heads, head_dim = q.shape
    slots, kv_heads, _ = k_cache.shape
    seqs, width = block_tables.shape
    if out is None:
        out = torch.empty((tokens, heads, head_dim), dtype=q.dtype, device=q.device)
    if scale is None:
        scale = head_dim ** -0.5
    lib = _lib.lib()

    def pack(workspace, nbytes):
        return _ARGS.pack(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            slots, k_cache.stride(0), k_cache.stride(1), block_tables.data_ptr(),
            block_tables.stride(0), width, context_lens.data_ptr(),
            cu_seqlens_q.data_ptr() if cu_seqlens_q is not None else 0, out.data_ptr(),
            out.stride(0), tokens, seqs, max_query_len, max_context_len, window, sinks,
            prefix_len, workspace, nbytes, dtype_code(q.dtype), heads, kv_heads, head_dim,
            block_size, scale)

    try:
        args = pack(0, 0)
    except struct.error as exc:
        raise ValueError(f"{what}: {exc}") from exc
    need = lib.ie_attention_workspace_size(ctypes.cast(args, _AS_POINTER))
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        args = pack(workspace.data_ptr(), need)
    _lib.check(entry(lib)(ctypes.cast(args, _AS_POINTER), _lib.stream_ptr()), what)
    return out


def window_attention(q, k_cache, v_cache, block_tables, context_lens, block_size: int, *,
                     window: int = 0, sinks: int = 0, cu_seqlens_q=None, max_query_len: int = 0,
                     max_context_len: int = 0, scale: float | None = None, out=None,
                     stream=None):
    """Causal attention in which the query at position ``p`` sees key ``j <= p`` iff
    ``j > p - window`` or ``j < sinks`` (``window=0``: every ``j <= p``).

    q: ``[tokens, heads, head_dim]`` (bf16 / f16 / f32).  block_tables: int32
    ``[sequences, blocks]``; an entry outside the cache (-1: the page was given
    back) hides its keys.  context_lens: int32 ``[sequences]``; cu_seqlens_q:
    int32 ``[sequences + 1]``.  ``max_query_len`` and ``max_context_len`` are the
    longest of the batch and size the launch (0: not known).  Returns a tensor
    like q.  bf16 / f16 with heads of 64 or 128 elements and 16-byte aligned
    rows run on the tensor cores.
    """
    return _attend(lambda lib: lib.ie_window_attention, "window_attention", q, k_cache, v_cache,
                   block_tables, context_lens, block_size, window, sinks, 0, cu_seqlens_q,
                   max_query_len, max_context_len, scale, out, stream)


def shared_prefix_attention(q, k_cache, v_cache, block_tables, context_lens, prefix_len: int,
                            block_size: int, *, cu_seqlens_q=None, max_query_len: int = 0,
                            max_context_len: int = 0, scale: float | None = None, out=None,
                            stream=None):
    """Causal attention of sequences that begin with the same ``prefix_len`` tokens:
    the prefix is read once for the whole batch, through the first row of
    ``block_tables``, and the keys from ``prefix_len`` on through each
    sequence's own row.  A sequence shorter than the prefix sees its part of
    it.  The other arguments are those of ``window_attention``."""
    return _attend(lambda lib: lib.ie_shared_prefix_attention, "shared_prefix_attention", q,
                   k_cache, v_cache, block_tables, context_lens, block_size, 0, 0, prefix_len,
                   cu_seqlens_q, max_query_len, max_context_len, scale, out, stream)
