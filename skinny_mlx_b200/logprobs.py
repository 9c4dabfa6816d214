"""Log probabilities of tokens under a step's logits on B200, with entropy and alternatives.

The verify step's logits [rows, V] stay on the device: `token_logprobs` reads them once and returns, per
row, the log probability of a given token, the entropy of the distribution and the top_n most likely
tokens.  `spec.accept` is the argmax counterpart; `spec.greedy` and `spec.speculative` fill a `logprobs`
list with it."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_TOP = 32
MAX_VOCAB = 2**27
_TYPES = {torch.bfloat16: 0, torch.float32: 1}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # f32 [rows]: ln p of the given token
    entropy: torch.Tensor       # f32 [rows]: -sum p ln p, in nats
    top_logprobs: torch.Tensor  # f32 [rows, top_n], descending
    top_ids: torch.Tensor       # int32 [rows, top_n]


_ws_bytes: dict[tuple, int] = {}


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0) -> TokenLogprobs:
    """logits bf16 or f32 [rows, V] (unit column stride, rows may be further apart), tokens int32 or int64
    [rows] on the same device; top_n <= 32 alternatives (ties to the lowest index, a NaN above every number:
    the order of spec.accept).  No host synchronisation.

    A logit of -inf has probability 0; a row of nothing else has log probabilities -inf and entropy 0; a
    row with a NaN or +inf has NaN sums; a token outside [0, V), e.g. -1 for "none", has log probability
    -inf."""
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (no CPU fallback)")
    kind = _TYPES.get(logits.dtype)
    if kind is None or logits.dim() != 2:
        raise ValueError("logits must be a bf16 or f32 [rows, V] tensor")
    rows, v = logits.shape
    if not 1 <= v <= MAX_VOCAB or (v > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < v):
        raise ValueError(f"logits must have 1 to {MAX_VOCAB} columns, unit column stride and rows that do not overlap")
    if tokens.shape != (rows,) or tokens.dtype not in (torch.int32, torch.int64) or tokens.device != logits.device:
        raise ValueError(f"tokens must be int32 or int64 [{rows}] on the logits' device")
    if not 0 <= top_n <= min(MAX_TOP, v):
        raise ValueError(f"top_n must be in [0, {min(MAX_TOP, v)}]")
    dev = logits.device
    if tokens.dtype == torch.int64:  # ids beyond 32 bits are outside every vocabulary
        tokens = tokens.clamp(-1, 2**31 - 1).to(torch.int32)
    tokens = tokens.contiguous()
    lp = torch.empty(rows, dtype=torch.float32, device=dev)
    ent = torch.empty_like(lp)
    top = torch.empty(rows, top_n, dtype=torch.float32, device=dev)
    ids = torch.empty(rows, top_n, dtype=torch.int32, device=dev)
    if rows:
        key = (dev.index, rows, v, top_n)
        n = _ws_bytes.get(key)
        if n is None:
            with torch.cuda.device(dev):
                n = _ws_bytes[key] = int(_lib.lib().skinny_token_logprobs_workspace_bytes(rows, v, top_n))
        ws = torch.empty(n, dtype=torch.uint8, device=dev)  # scratch of this call alone
        _lib.launch("skinny_token_logprobs", dev.index, logits.data_ptr(), logits.stride(0), kind, rows, v,
                    tokens.data_ptr(), top_n, lp.data_ptr(), ent.data_ptr(), top.data_ptr(), ids.data_ptr(), ws.data_ptr(), n)
    return TokenLogprobs(lp, ent, top, ids)


__all__ = ["token_logprobs", "TokenLogprobs", "MAX_TOP", "MAX_VOCAB"]
