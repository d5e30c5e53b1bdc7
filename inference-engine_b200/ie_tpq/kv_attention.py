"""Attention over the paged KV cache on the library's own kernels: a sliding
window with sinks, and a prefix that a whole batch shares.

The cache layout is that of ``attention.allocate_kv_cache``: position ``j`` of a
sequence lies in slot ``table[j // block_size] * block_size + j % block_size``.
Both functions take the sequences' lengths as device tensors, allocate their
output and workspace from torch's allocator on the stream they run on, never
synchronise, and can be captured in a CUDA graph.  Queries are ragged: sequence
``s`` owns the tokens ``cu_seqlens_q[s] : cu_seqlens_q[s + 1]`` and its last one
is at position ``context_lens[s] - 1``; without ``cu_seqlens_q`` every sequence
has one token (decode).  A query that sees nothing gets zeros, and so does a token
that ``cu_seqlens_q`` gives to no sequence (the end of a padded batch).
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .device import require_cuda

# _lib.AttentionArgs field by field (packing is far cheaper than ctypes fields)
_ARGS = struct.Struct("@Q2q2Q3qQ2q3Q8q5if")
assert _ARGS.size == ctypes.sizeof(_lib.AttentionArgs)

_DTYPES = {torch.bfloat16: _lib.IE_DT_BF16, torch.float16: _lib.IE_DT_F16,
           torch.float32: _lib.IE_DT_F32}
_ENTRIES: dict = {}


def _entry(name: str):
    """The library's function taking the packed arguments as bytes."""
    if name not in _ENTRIES:
        require_cuda()
        lib = _lib.lib()
        fn = lib[name]     # an object of its own: the declared prototype stays
        fn.restype = getattr(lib, name).restype
        fn.argtypes = [ctypes.c_char_p, *getattr(lib, name).argtypes[1:]]
        _ENTRIES[name] = fn
    return _ENTRIES[name]


def _attend(name, q, k_cache, v_cache, block_tables, context_lens, block_size, window, sinks,
            prefix_len, cu_seqlens_q, max_query_len, max_context_len, scale, out, stream):
    entry = _entry(name)
    # ---- the tensors: shapes, types, layouts, one device
    q_shape, q_stride = q.shape, q.stride()
    k_shape, k_stride = k_cache.shape, k_cache.stride()
    if len(q_shape) != 3 or len(k_shape) != 3:
        raise ValueError("q is [tokens, heads, head_dim], the caches [slots, kv_heads, head_dim]")
    if v_cache.shape != k_shape or v_cache.stride() != k_stride:
        raise ValueError("the caches must have one shape and one layout")
    dtype = q.dtype
    if k_cache.dtype != dtype or v_cache.dtype != dtype or dtype not in _DTYPES:
        raise ValueError("q and the caches must have one dtype: bfloat16, float16 or float32")
    tokens, heads, head_dim = q_shape
    if head_dim != k_shape[2]:
        raise ValueError(f"q has head_dim {head_dim}, the caches {k_shape[2]}")
    if q_stride[2] != 1 or k_stride[2] != 1:
        raise ValueError("a head's elements must be adjacent")
    t_shape, t_stride = block_tables.shape, block_tables.stride()
    if len(t_shape) != 2 or block_tables.dtype != torch.int32 or t_stride[1] != 1:
        raise ValueError("block_tables must be an int32 [sequences, blocks] tensor with "
                         "adjacent entries")
    seqs, width = t_shape
    if context_lens.dtype != torch.int32 or context_lens.numel() != seqs or \
            not context_lens.is_contiguous():
        raise ValueError(f"context_lens must be a contiguous int32 tensor of {seqs} entries")
    index = q.get_device()
    if not (index == k_cache.get_device() == v_cache.get_device() == block_tables.get_device()
            == context_lens.get_device() and index >= 0):
        raise ValueError("all tensors must be on one CUDA device")
    cu = 0
    if cu_seqlens_q is None:
        if tokens != seqs:
            raise ValueError(f"{tokens} tokens of {seqs} sequences need cu_seqlens_q")
    else:
        if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_q.numel() != seqs + 1 or \
                not cu_seqlens_q.is_contiguous() or cu_seqlens_q.get_device() != index:
            raise ValueError(f"cu_seqlens_q must be a contiguous int32 tensor of {seqs + 1} "
                             "entries on the same device")
        cu = cu_seqlens_q.data_ptr()
    if out is not None and (out.shape != q_shape or out.dtype != dtype or out.stride(2) != 1
                            or out.stride(1) != head_dim or out.get_device() != index):
        raise ValueError("out must have q's shape, dtype and device, and adjacent heads")

    # ---- the device and stream: output and workspace belong to them
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _attend(name, q, k_cache, v_cache, block_tables, context_lens, block_size,
                           window, sinks, prefix_len, cu_seqlens_q, max_query_len,
                           max_context_len, scale, out, stream)
    if stream is not None and stream != torch.cuda.current_stream():
        with torch.cuda.stream(stream):
            return _attend(name, q, k_cache, v_cache, block_tables, context_lens, block_size,
                           window, sinks, prefix_len, cu_seqlens_q, max_query_len,
                           max_context_len, scale, out, None)

    if out is None:
        out = q.new_empty(tokens, heads, head_dim)
    try:
        args = _ARGS.pack(
            q.data_ptr(), q_stride[0], q_stride[1], k_cache.data_ptr(), v_cache.data_ptr(),
            k_shape[0], k_stride[0], k_stride[1], block_tables.data_ptr(), t_stride[0], width,
            context_lens.data_ptr(), cu, out.data_ptr(), out.stride(0), tokens, seqs,
            max_query_len, max_context_len, window, sinks, prefix_len, _DTYPES[dtype], heads,
            k_shape[1], head_dim, block_size, head_dim ** -0.5 if scale is None else scale)
    except struct.error as exc:
        raise ValueError(f"{name[3:]}: {exc}") from exc
    need = _entry("ie_attention_workspace_size")(args)
    workspace = q.new_empty(need, dtype=torch.uint8) if need else None
    code = entry(args, workspace.data_ptr() if need else None, need, _lib.stream_ptr())
    if code:
        _lib.check(code, name[3:])
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
    longest of the batch and size the launch (0: not known).  ``scale`` (positive;
    by default ``head_dim ** -0.5``) multiplies the scores.  Returns a tensor
    like q.  bf16 / f16 with heads of 64 or 128 elements and 16-byte aligned
    rows run on the tensor cores.
    """
    return _attend("ie_window_attention", q, k_cache, v_cache, block_tables, context_lens,
                   block_size, window, sinks, 0, cu_seqlens_q, max_query_len, max_context_len,
                   scale, out, stream)


def shared_prefix_attention(q, k_cache, v_cache, block_tables, context_lens, prefix_len: int,
                            block_size: int, *, cu_seqlens_q=None, max_query_len: int = 0,
                            max_context_len: int = 0, scale: float | None = None, out=None,
                            stream=None):
    """Causal attention of sequences that begin with the same ``prefix_len`` tokens:
    the prefix is read through the first row of ``block_tables``, once for the
    whole batch (a short prefix of few sequences, and any prefix in f32 or with other head
    sizes than 64 and 128: by each, from L2), and the keys from ``prefix_len`` on through
    each sequence's own row.  A sequence shorter than the prefix sees its part of
    it.  The other arguments are those of ``window_attention``."""
    return _attend("ie_shared_prefix_attention", q, k_cache, v_cache, block_tables, context_lens,
                   block_size, 0, 0, prefix_len, cu_seqlens_q, max_query_len, max_context_len,
                   scale, out, stream)
