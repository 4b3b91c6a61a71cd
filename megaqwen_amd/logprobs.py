"""Log probabilities of given tokens, with the entropy of each row and its most likely tokens.

    r = token_logprobs(logits, tokens, top_k=5)
    r.logprobs, r.entropy                     # fp32, one per row of logits
    r.top_logprobs, r.top_tokens              # fp32 and int32 [..., 5], most likely first

One pass over the logits, none of it materialised as probabilities.  The compute is the
hand-written gfx950 kernel behind `mq_token_logprobs` (include/megaqwen_hip.h,
megaqwen_amd/csrc/logprobs.hip); there is no PyTorch fallback.
`megaqwen_amd.quality.decoder_logprobs` and `MegakernelDecoder.decode_step_with_logprobs` call it.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._launch import DTYPES, call, no_grad

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top_k: int = 0) -> TokenLogprobs:
    """Natural-log probabilities under softmax(logits [..., vocab]) (bf16, fp16 or fp32).

    logprobs [...]: of `tokens` [...] (int32 or int64); -inf for a token outside [0, vocab).
    entropy [...]: of the row's distribution.  top_logprobs, top_tokens [..., top_k]: the top_k (at
    most 32) most likely tokens; equal logits are ordered by the lower token.
    A row of -inf alone has no distribution: log probabilities -inf, entropy 0, tokens 0 ..
    top_k - 1.  A row that holds a NaN or +inf gives NaN."""
    dtype, dev, shape = DTYPES.get(logits.dtype), logits.get_device(), logits.shape
    if not logits.is_cuda:
        raise ValueError("token_logprobs expects CUDA tensors")
    if dtype is None:
        raise ValueError(f"token_logprobs only supports fp16/bf16/fp32, got {logits.dtype}")
    if not shape or shape[-1] < 1:
        raise ValueError(f"logits must be [..., vocab], got {tuple(shape)}")
    if tokens.get_device() != dev:
        raise ValueError(f"tokens is on {tokens.device}, logits on {logits.device}")
    wide = tokens.dtype == torch.int64
    if not wide and tokens.dtype != torch.int32:
        raise ValueError(f"tokens must be int32 or int64, got {tokens.dtype}")
    lead, vocab, top_k = (shape[0],) if len(shape) == 2 else tuple(shape[:-1]), shape[-1], int(top_k)
    if tokens.shape != lead:
        raise ValueError(f"Shape mismatch logits={tuple(shape)} tokens={tuple(tokens.shape)}")
    if not 0 <= top_k <= MAX_TOP_K or top_k > vocab:
        raise ValueError(f"top_k must be in [0, min({MAX_TOP_K}, vocab={vocab})], got {top_k}")
    if torch.is_grad_enabled():
        no_grad("token_logprobs", logits)
    if len(shape) != 2:
        logits = logits.reshape(-1, vocab)
    stride, step = logits.stride()
    if step != 1 and vocab > 1:
        logits = logits.contiguous()
        stride = vocab
    tokens = tokens.contiguous()
    rows = logits.shape[0]
    lp = logits.new_empty(lead, dtype=torch.float32)
    entropy = torch.empty_like(lp)
    top_lp = lp.new_empty((*lead, top_k))
    top_tok = torch.empty_like(top_lp, dtype=torch.int32)
    if rows:
        lib = _lib.load()
        # scratch of this call alone, in stream order
        size = lib.mq_token_logprobs_workspace_bytes(rows, vocab, top_k)
        ws = lp.new_empty(size // 4) if size else None
        call(lib.mq_token_logprobs, dev, logits.data_ptr(), stride, tokens.data_ptr(), wide, lp.data_ptr(),
             entropy.data_ptr(), top_lp.data_ptr() or None, top_tok.data_ptr() or None, rows, vocab, top_k, dtype,
             None if ws is None else ws.data_ptr(), size)
    return TokenLogprobs(lp, entropy, top_lp, top_tok)
