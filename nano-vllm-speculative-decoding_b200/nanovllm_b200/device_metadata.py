"""A verification round's metadata built on the GPU from the requests' lengths.

    verify_metadata(...)    batch_metadata.pack_verify_metadata and draft_placement (nanovllm/engine/batch_metadata.py:
                            121-181, speculative.py:514-527) in one launch, the blocks that a row lacks taken from a free
                            stack (scheduler.py:75-92)                                 -> specdec_verify_metadata_ex

The host form builds the arrays with numpy and copies them to the device three times a round; here the request state
stays on the GPU (lengths, last tokens, drafts, block tables, the free blocks), so a round's metadata costs one launch and
no host round trip.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._lib import Workspace, call_on, ptr, raw_stream, require_cuda, same_device
from .batch_metadata import packed_sizes


@dataclass
class DeviceRows:
    """The requests of a batch on the GPU: what verify_metadata reads of them, and the free blocks they grow into."""
    lengths: torch.Tensor        # [R] int64: tokens of each row, the last one included
    last_tokens: torch.Tensor    # [R] int64
    block_tables: torch.Tensor   # [R, W] int32
    num_blocks: torch.Tensor     # [R] int32: blocks each row holds
    free_blocks: torch.Tensor | None = None   # [capacity] int32 stack
    free_count: torch.Tensor | None = None    # [1] int32

    def advance(self, n_accept: torch.Tensor, tail: torch.Tensor, error: torch.Tensor) -> None:
        """A round's outcome: every row is longer by its accepted drafts and the tail token, which is its last now.
        Nothing changes where error, an int32 word on the device, is set."""
        done = error == 0
        self.lengths.add_((n_accept + 1) * done)
        self.last_tokens.copy_(torch.where(done, tail, self.last_tokens))


def _words(device: torch.device) -> torch.Tensor:
    """[error word, ticket] of this device."""
    return Workspace.get(device, 256, name="device_metadata")[:8].view(torch.int32)


def error_word(device: torch.device) -> torch.Tensor:
    """The int32 word that device_error reads, on the device."""
    return _words(device)[0]


def device_error(device: torch.device) -> int:
    """First error a verify_metadata call recorded on this device since the last reset (synchronises): 0 none, 6 the free
    blocks ran out, 7 row arguments out of range (a verified length outside 1..k+1, a length below 1, a table too narrow
    for the row, tokens that the padding rows cannot hold), 9 a block that a row needs, held or from the stack, has an id
    outside the cache.  A call that records one assigns nothing (num_blocks and free_count stay; after 9, block_tables may
    differ past num_blocks) and leaves every row empty: cumulative lengths 0, slots -1."""
    return int(_words(device)[0].item())


def reset_device_error(device: torch.device) -> None:
    _words(device)[0].zero_()


def _of(name: str, t: torch.Tensor | None, dtype: torch.dtype, shape: tuple) -> None:
    if t is not None and (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {shape} (got {t.dtype} {tuple(t.shape)})")


def verify_metadata(lengths: torch.Tensor, last_tokens: torch.Tensor, drafts: torch.Tensor,
                    verified_lens: torch.Tensor | None, block_tables: torch.Tensor, num_blocks: torch.Tensor,
                    free_blocks: torch.Tensor | None, free_count: torch.Tensor | None, *, block_size: int, num_rows: int,
                    num_tokens: int, pad_block_id: int, width: int, buf64: torch.Tensor, buf32: torch.Tensor,
                    cache_blocks: int | None = None) -> None:
    """Writes the metadata of verifying R rows into the packed buffers buf64 / buf32 (batch_metadata.packed_views of
    num_rows, num_tokens and width names their parts), the drafts placed among the input ids.

    lengths, last_tokens [R] int64: a row's token count (its last token included, whose K/V are not stored yet) and that
    token.  drafts [R, k] int64.  verified_lens [R] int64, 1..k+1 (None: k + 1 each); their sum and the tokens of the
    padding rows (at most k + 1 each) make num_tokens.  block_tables [R, W'] int32 and num_blocks [R] int32: the blocks a
    row holds, extended in place to what lengths - 1 + verified_lens tokens need with blocks from the top of the stack
    free_blocks[:free_count] (int32, free_count [1] int32, lowered in place), rows in order.  Both None: the rows must
    hold what they need.  cache_blocks: ids of the rows' blocks are below it (None: any whose slots fit 32 bits).  The row
    arguments may be empty (R = 0): all padding.  Calls on one device share an error word and
    a ticket: they must not overlap on the GPU."""
    index = buf64.get_device()
    if not same_device(index, lengths, last_tokens, drafts, verified_lens, block_tables, num_blocks, free_blocks,
                       free_count, buf32):
        require_cuda(buf64, lengths, last_tokens, drafts, verified_lens, block_tables, num_blocks, free_blocks, free_count,
                     buf32)
    if drafts.dim() != 2 or block_tables.dim() != 2:
        raise ValueError("drafts and block_tables must be 2-D")
    R, k = drafts.shape
    table_width = block_tables.shape[1]
    rows = (R,)
    _of("lengths", lengths, torch.int64, rows)
    _of("last_tokens", last_tokens, torch.int64, rows)
    _of("drafts", drafts, torch.int64, (R, k))
    _of("verified_lens", verified_lens, torch.int64, rows)
    _of("block_tables", block_tables, torch.int32, (R, table_width))
    _of("num_blocks", num_blocks, torch.int32, rows)
    if (free_blocks is None) != (free_count is None):
        raise ValueError("give free_blocks and free_count together")
    capacity = 0
    if free_blocks is not None:
        capacity = free_blocks.numel()
        _of("free_blocks", free_blocks, torch.int32, (capacity,))
        _of("free_count", free_count, torch.int32, (1,))
    if cache_blocks is not None and cache_blocks < 1:
        raise ValueError(f"cache_blocks {cache_blocks}: the cache's blocks, or None")
    n64, n32 = packed_sizes(num_rows, num_tokens, width)
    _of("buf64", buf64, torch.int64, (n64,))
    _of("buf32", buf32, torch.int32, (n32,))
    words = Workspace.address(index, 256, "device_metadata")       # [error word, ticket]
    call_on(index, _lib.lib().specdec_verify_metadata_ex, ptr(lengths), ptr(last_tokens), ptr(drafts), ptr(verified_lens), R,
            k, ptr(block_tables), table_width, ptr(num_blocks), ptr(free_blocks), ptr(free_count), capacity, block_size,
            num_rows, num_tokens, pad_block_id, width, buf64.data_ptr(), buf32.data_ptr(), words + 4, words,
            0 if cache_blocks is None else cache_blocks, raw_stream(index))
