"""Log probabilities of given tokens, with entropy and top alternatives: what
a server returns beside its tokens, and what compressed caches are compared
with uncompressed ones by."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L

__all__ = ["TokenLogprobs", "token_logprobs"]

_MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """logprobs, entropy (rows,) fp32; top_ids (rows, top_k) int32 and
    top_logprobs (rows, top_k) fp32."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top_k: int = 0) -> TokenLogprobs:
    """Natural log probabilities under softmax(logits).

    logits (rows, vocab) fp32, fp16 or bf16, contiguous in vocab; targets
    (rows,) int64: a negative one (padding) gives 0, one past the vocabulary
    NaN. ``top_k`` <= 32 alternatives by value, equal ones by index; -1 and
    -inf past the vocabulary. Logits of -inf are impossible tokens; a row of
    nothing else gives -inf and entropy 0. A row with NaN or +inf gives NaN
    everywhere and ids of -1. There is no gradient: logits that want one are
    refused.
    """
    t = (L._fast or L.fast()).logprobs(logits, targets, top_k)
    if t is not None:
        return TokenLogprobs._make(t)
    if not (logits.is_cuda and targets.is_cuda):
        L.require_cuda(logits, targets)
    L.refuse_graph("token_logprobs", logits)
    if logits.dim() != 2 or not 0 < logits.size(1) < 2 ** 31:
        raise ValueError("logits must be (rows, vocab), vocab from 1 to 2^31 - 1")
    n, vocab = logits.shape
    row_stride, stride = logits.stride()
    if stride != 1 and vocab > 1:
        raise ValueError("logits must be contiguous in vocab")
    index = logits.get_device()
    if (targets.dtype is not torch.int64 or targets.dim() != 1 or targets.size(0) != n
            or targets.get_device() != index or not targets.is_contiguous()):
        raise ValueError("targets must be a contiguous int64 tensor with one element per row, on the logits' device")
    if not 0 <= top_k <= _MAX_TOP:
        raise ValueError(f"top_k must be in [0, {_MAX_TOP}], got {top_k}")
    dt = L.dtype_code(logits.dtype)
    out = torch.empty((2 + top_k) * n, dtype=torch.float32, device=logits.device)
    lp, ent, top = out.split_with_sizes((n, n, top_k * n))
    ids = torch.empty((n, top_k), dtype=torch.int32, device=logits.device)
    at = out.data_ptr()
    L.launch("ss_token_logprobs", index, logits.data_ptr(), dt, n, row_stride, vocab, targets.data_ptr(),
             top_k, at, at + 4 * n, ids.data_ptr(), at + 8 * n)
    return TokenLogprobs(lp, ent, ids, top.view(n, top_k))
