"""Log probabilities of given tokens, with the entropy and the best alternatives
of every row (``ie_token_logprobs``)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .device import require_cuda

_DTYPES = {torch.float32: _lib.IE_DT_F32, torch.bfloat16: _lib.IE_DT_BF16,
           torch.float16: _lib.IE_DT_F16}
_ENTRY = None      # the library's function, once a GPU has been seen


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor        # f32 [rows]
    entropy: torch.Tensor         # f32 [rows], nats
    top_logprobs: torch.Tensor    # f32 [rows, top], best first
    top_tokens: torch.Tensor      # int64 [rows, top], ties to the lower token


def token_logprobs(logits, tokens, top: int = 0, stream=None) -> TokenLogprobs:
    """``log softmax(logits)[r, tokens[r]]``, the rows' entropies and their ``top``
    (at most 64) largest log probabilities, in one pass over the logits.

    logits: CUDA ``[rows, vocab]`` (f32 / bf16 / f16), rows of any stride.  tokens:
    int64 ``[rows]``; one outside the vocabulary has log probability -inf.
    Logits of -inf (a vocabulary mask) are allowed; a row with a NaN or +inf, or
    with no logit above -inf, gives NaN.
    """
    global _ENTRY
    if _ENTRY is None:
        require_cuda()
        _ENTRY = _lib.lib().ie_token_logprobs
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("logits must be a row-contiguous 2-D tensor")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {logits.dtype}; expected float32, bfloat16 or float16")
    rows, vocab = shape
    if tokens.dtype != torch.long or tokens.dim() != 1 or tokens.shape[0] != rows or \
            not tokens.is_contiguous():
        raise ValueError("tokens must be a contiguous int64 tensor of one entry per row")
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index:
        raise ValueError("logits and tokens must be on one CUDA device")
    if not 0 <= top <= min(vocab, _lib.IE_LOGPROBS_MAX_TOP):
        raise ValueError(f"top={top} outside [0, min({_lib.IE_LOGPROBS_MAX_TOP}, {vocab})]")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top, stream)
    if stream is not None and stream != torch.cuda.current_stream():
        with torch.cuda.stream(stream):   # the outputs belong to that stream
            return token_logprobs(logits, tokens, top)
    logprobs = torch.empty(rows, dtype=torch.float32, device=logits.device)
    entropy = logprobs.new_empty(rows)
    top_logprobs = logprobs.new_empty(rows, top)
    top_tokens = tokens.new_empty(rows, top)
    code = _ENTRY(
        logits.data_ptr(), stride[0], _DTYPES[logits.dtype], rows, vocab,
        tokens.data_ptr(), top, logprobs.data_ptr(), entropy.data_ptr(),
        top_logprobs.data_ptr(), top_tokens.data_ptr(), _lib.stream_ptr())
    if code:
        _lib.check(code, "token_logprobs")
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)
