"""Log probabilities of given tokens, each position's entropy and its most likely tokens, in one pass over the logits.

    token_logprobs(logits, tokens, num_top, temperatures)    -> specdec_token_logprobs

Beside spec_sampler.probs_from_logits, which writes the whole [T, V] distribution: a server that answers with log
probabilities wants a few numbers for each emitted token.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from ._lib import DTYPE_CODES, Workspace, call_on, ptr, raw_stream, require_cuda, same_device

MAX_TOP = 32


@dataclass
class TokenLogprobs:
    logprobs: torch.Tensor       # [T] fp32, log p of the given token
    entropy: torch.Tensor        # [T] fp32, in nats
    top_ids: torch.Tensor        # [T, num_top] int64, the most likely tokens, likeliest first
    top_logprobs: torch.Tensor   # [T, num_top] fp32


def _err_word(device: torch.device) -> torch.Tensor:
    return Workspace.get(device, 256, name="logprobs")[:4].view(torch.int32)


def device_error(device: torch.device) -> int:
    """First error recorded on this device since the last reset (synchronises): 0 none, 8 a token id past the
    vocabulary (its log probability is NaN)."""
    return int(_err_word(device).item())


def reset_device_error(device: torch.device) -> None:
    _err_word(device).zero_()


@lru_cache(maxsize=4096)
def _workspace_bytes(index: int, T: int, V: int, dtype: int, num_top: int) -> int:
    with torch.cuda.device(index):
        return int(_lib.lib().specdec_logprobs_workspace_bytes(T, V, dtype, num_top))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, num_top: int = 0,
                   temperatures: torch.Tensor | None = None, *, workspace: str = "logprobs_parts") -> TokenLogprobs:
    """logits [T, V] (bf16, fp16 or fp32; rows may be strided), tokens [T] int64.  temperatures [T] fp32 > 0 (None: 1)
    divide the logits first.  num_top (0 to 32, at most V) alternatives a row: the largest logits, ties to the lowest
    index, NaN above every number.  Rows whose token is negative (padding) are not read: 0, 0, ids -1, 0.  A row with a
    NaN or +inf, or nothing but -inf, has NaN for every log probability and the entropy; a single -inf is a token of
    probability 0.  workspace: the name of the device workspace; calls that may run at the same time on different streams
    need different names."""
    index = logits.get_device()
    if not same_device(index, tokens, temperatures):
        require_cuda(logits, tokens, temperatures)
    if logits.dim() != 2 or logits.dtype not in DTYPE_CODES:
        raise ValueError(f"logits must be [T, V] bf16, fp16 or fp32 (got {logits.dtype} {tuple(logits.shape)})")
    T, V = logits.shape
    if tokens.shape != (T,):
        raise ValueError(f"tokens {tuple(tokens.shape)} for {T} rows of logits")
    if tokens.dtype.is_floating_point or tokens.dtype == torch.bool:
        raise ValueError(f"tokens must be integers (got {tokens.dtype})")
    if not 0 <= num_top <= min(MAX_TOP, V):
        raise ValueError(f"num_top {num_top}: 0 to {MAX_TOP} and at most the vocabulary")
    if temperatures is not None:
        if temperatures.shape != (T,):
            raise ValueError(f"temperatures {tuple(temperatures.shape)} for {T} rows of logits")
        temperatures = temperatures.to(torch.float32).contiguous()
    if T and (logits.stride(1) != 1 or (T > 1 and logits.stride(0) < V)):
        logits = logits.contiguous()
    stride = logits.stride(0) if T > 1 else V
    if tokens.dtype is not torch.int64 or not tokens.is_contiguous():
        tokens = tokens.to(torch.int64).contiguous()
    device = logits.device
    floats = torch.empty(T * (2 + num_top), dtype=torch.float32, device=device)      # one allocation for the three
    values, entropy, top = floats.split_with_sizes((T, T, T * num_top))
    out = TokenLogprobs(values, entropy, torch.empty(T, num_top, dtype=torch.int64, device=device), top.view(T, num_top))
    base, dtype = floats.data_ptr(), DTYPE_CODES[logits.dtype]
    ws_bytes = _workspace_bytes(index, T, V, dtype, num_top)
    call_on(index, _lib.lib().specdec_token_logprobs, logits.data_ptr(), dtype, T, V, stride, tokens.data_ptr(),
            ptr(temperatures), num_top, base, base + 4 * T, out.top_ids.data_ptr(), base + 8 * T,
            Workspace.address(index, ws_bytes, workspace), ws_bytes, Workspace.address(index, 256, "logprobs"),
            raw_stream(index))
    return out
