"""Attention over an 8-bit paged K/V cache: e4m3 codes with one power-of-two fp32 scale per (group of slots, KV head).

    FP8Cache                    one layer's caches and scales, allocated together
    store_kvcache_fp8(...)      the store (attention.py:33-40 onto the 8-bit cache)   -> specdec_store_kvcache_fp8
    paged_attention_fp8(...)    verify and decode attention over it                   -> specdec_paged_attention_fp8
    AttentionFP8                attention.Attention on an FP8Cache, reading the same context

The cache halves the bytes that the attention of a long context reads, and the memory a token takes, next to the bf16
cache of nanovllm_b200.attention; the reference has no 8-bit cache.

Layout: k_cache / v_cache [blocks, Hkv, block_size, 128] float8_e4m3fn (a block's rows of one head lie together, so a
tile of the attention is one contiguous piece of memory), k_scale / v_scale [blocks, Hkv, block_size / group] fp32 with
group 16 or 32.  An element stands for its code times its group's scale.

What a store does to a group (16 or 32 consecutive slots of a block, one head):
  - a call that writes the group's first slot starts it: the scale is the smallest power of two 2^e (e >= -100) that
    brings the call's finite values in the group to at most 448, and the slots the call does not write stand for nothing
    until they are written;
  - any other call keeps the scale or, where its values need a larger one, raises it and requantises the group's other
    slots.  Slots past a sequence's end that were written by rejected drafts may keep a scale larger than needed until
    the group is started again.
Codes are rounded to nearest even; infinities become +-448 times the scale and NaN stays NaN.  A slot that a call names
twice holds its last token.  The scales must be positive (FP8Cache starts them at 1).

Shapes and limits of the attention are those of nanovllm_b200.attention: head_dim 128, GQA groups of 1, 2, 4 or 8, rows of
at most 32 / (H / Hkv) queries, block_size a multiple of 128.  A query that sees no key (a row with no context, or fewer
keys than queries) gives zeros.  A NaN among a row's stored values reaches all of the row's queries, those whose mask
leaves its key out too, as in the bf16 cache's attention (0 * NaN in the matrix product); a NaN key only those that see it.

Accuracy: the queries of a row that share a KV head share an exponent, the largest element's, and are exact to 2^-22 of that
element; probabilities are off by 2^-9 of themselves or 2^-30 of the largest one; sums are fp32.  The scales of a row's values
may be up to 2^110 apart (a group of zeros has 2^-100): further apart, keys with the smaller ones can go missing from the
softmax's sum.

Errors found on the device are in attention.device_error: 2 row metadata, 3 a slot past the cache, 5 a block id outside the
cache (read as block 0).
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from ._lib import Workspace, call_on, ptr, raw_stream, require_cuda, same_device
from .attention import _SPLIT_MIN_BYTES, CTAS_SHIFT, EARLY_LAUNCH, _output, given_as_is
from .context import get_context

HEAD_DIM = 128
MAX_STORE_TOKENS = 16384


@dataclass
class FP8Cache:
    """One layer's 8-bit cache: codes [blocks, Hkv, block_size, 128], scales [blocks, Hkv, block_size / group]."""
    k_cache: torch.Tensor
    v_cache: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def allocate(cls, num_blocks: int, block_size: int, num_kv_heads: int, device: torch.device, *,
                 group: int = 16) -> "FP8Cache":
        """A zeroed cache of num_blocks blocks whose scales are 1."""
        if group not in (16, 32) or block_size % group:
            raise ValueError(f"group {group}: 16 or 32 slots share a scale, a divisor of block_size {block_size}")
        shape = (num_blocks, num_kv_heads, block_size, HEAD_DIM)

        def codes():
            return torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

        def scales():
            return torch.ones(*shape[:2], block_size // group, dtype=torch.float32, device=device)

        return cls(codes(), codes(), scales(), scales())

    def dequantised(self) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V as fp32 [blocks, block_size, Hkv, 128], the layout of the bf16 caches (for inspection)."""
        def one(cache, scale):
            group = cache.shape[2] // scale.shape[2]
            return (cache.float() * scale.repeat_interleave(group, dim=2).unsqueeze(-1)).transpose(1, 2).contiguous()
        return one(self.k_cache, self.k_scale), one(self.v_cache, self.v_scale)


def _cache_geometry(k_cache, v_cache, k_scale, v_scale) -> tuple[int, int, int, int]:
    """(blocks, Hkv, block_size, group) of a checked cache."""
    if k_cache.dtype is not torch.float8_e4m3fn or v_cache.dtype is not torch.float8_e4m3fn:
        raise ValueError(f"the 8-bit caches are float8_e4m3fn (got {k_cache.dtype}, {v_cache.dtype})")
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
        raise ValueError("the scales are float32")
    shape, scale_shape = tuple(k_cache.shape), tuple(k_scale.shape)
    if len(shape) != 4 or shape[3] != HEAD_DIM or v_cache.shape != shape:
        raise ValueError(f"caches must be [blocks, Hkv, block_size, {HEAD_DIM}] of one shape "
                         f"(got {shape}, {tuple(v_cache.shape)})")
    blocks, kv_heads, block_size, _ = shape
    if (len(scale_shape) != 3 or v_scale.shape != scale_shape or scale_shape[:2] != shape[:2]
            or (scale_shape[2] * 16 != block_size and scale_shape[2] * 32 != block_size)):
        raise ValueError(f"scales must be [blocks, Hkv, block_size / 16 or / 32] of one shape "
                         f"(got {scale_shape}, {tuple(v_scale.shape)} for caches {shape})")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous()):
        raise ValueError("caches and scales must be contiguous")
    return blocks, kv_heads, block_size, block_size // scale_shape[2]


def _int32(t: torch.Tensor | None) -> torch.Tensor | None:
    """t as a contiguous int32 tensor (itself where it is one)."""
    if t is None or (t.dtype is torch.int32 and t.is_contiguous()):
        return t
    return t.to(torch.int32).contiguous()


@lru_cache(maxsize=4096)
def _workspace_bytes(index: int, R: int, kv_heads: int) -> int:
    with torch.cuda.device(index):
        need = int(_lib.lib().specdec_attention_workspace_bytes(R, kv_heads))
    if need < 0:
        raise _lib.SpecdecError(f"no attention workspace for {R} rows of {kv_heads} KV heads")
    return max(need, _SPLIT_MIN_BYTES)


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """key / value [N, Hkv, 128] bf16 rows (dense heads, rows may be strided) to slot_mapping [N] of the 8-bit caches,
    in any order; slot -1 skipped.  At most 16384 tokens a call."""
    index = key.get_device()
    if not same_device(index, value, k_cache, v_cache, k_scale, v_scale, slot_mapping):
        require_cuda(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    blocks, kv_heads, block_size, group = _cache_geometry(k_cache, v_cache, k_scale, v_scale)
    if key.dtype is not torch.bfloat16 or value.dtype is not torch.bfloat16:
        raise ValueError("the B200 K/V store takes bf16 keys and values")
    shape = tuple(key.shape)
    if len(shape) != 3 or shape[1:] != (kv_heads, HEAD_DIM) or value.shape != shape:
        raise ValueError(f"key and value must be [N, {kv_heads}, {HEAD_DIM}] (got {shape}, {tuple(value.shape)})")
    N = shape[0]
    ks, vs = key.stride(), value.stride()
    if N and (ks[2] != 1 or vs[2] != 1 or (kv_heads > 1 and (ks[1] != HEAD_DIM or vs[1] != HEAD_DIM))):
        raise ValueError("key and value rows must hold their heads densely")
    if slot_mapping.numel() != N:
        raise ValueError(f"{slot_mapping.numel()} slots for {N} tokens")
    slots = _int32(slot_mapping)
    one_row = kv_heads * HEAD_DIM                           # a single row's stride says nothing
    call_on(index, _lib.lib().specdec_store_kvcache_fp8, key.data_ptr(), ks[0] if N > 1 else one_row, value.data_ptr(),
            vs[0] if N > 1 else one_row,
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), slots.data_ptr(), N, kv_heads,
            HEAD_DIM, blocks, block_size, group, Workspace.address(index, 256, "attention"), raw_stream(index))


def paged_attention_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, block_tables: torch.Tensor, scale: float, *,
                        cu_seqlens_q: torch.Tensor | None = None, cu_seqlens_k: torch.Tensor | None = None,
                        max_seqlen_q: int | None = None, context_lens: torch.Tensor | None = None,
                        query_len_per_seq: int = 1, causal: bool = True, out: torch.Tensor | None = None,
                        early_launch: bool = False, max_ctas: int = 0, workspace: str = "attention_split"
                        ) -> torch.Tensor:
    """attention.paged_attention over the 8-bit caches: q [T, H, 128] bf16, varlen (cu_seqlens_q/k, max_seqlen_q) or
    decode (context_lens with query_len_per_seq queries a row).  Returns out [T, H, 128] bf16; rows of out behind the last
    sequence are left as they were.  early_launch, max_ctas and workspace as there."""
    index = q.get_device()
    if not same_device(index, k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens_q, cu_seqlens_k, context_lens):
        require_cuda(q, k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens_q, cu_seqlens_k, context_lens)
    blocks, kv_heads, block_size, group = _cache_geometry(k_cache, v_cache, k_scale, v_scale)
    shape = tuple(q.shape)
    if q.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != HEAD_DIM:
        raise ValueError(f"q must be bf16 [T, H, {HEAD_DIM}] (got {q.dtype} {shape})")
    T, H, D = shape
    if cu_seqlens_q is not None:
        if cu_seqlens_k is None or max_seqlen_q is None:
            raise ValueError("varlen attention needs cu_seqlens_k and max_seqlen_q")
        cq, ck, ctx = _int32(cu_seqlens_q), _int32(cu_seqlens_k), None
        R, q_per_seq, max_q = cq.numel() - 1, 0, int(max_seqlen_q)
        if ck.numel() != R + 1:
            raise ValueError(f"cu_seqlens_q of {R} rows, cu_seqlens_k of {ck.numel() - 1}")
    elif context_lens is not None:
        cq, ck, ctx = None, None, _int32(context_lens)
        R, q_per_seq, max_q = ctx.numel(), query_len_per_seq, query_len_per_seq
    else:
        raise ValueError("give cu_seqlens_q / cu_seqlens_k (varlen) or context_lens (decode)")
    tables = _int32(block_tables)
    if tables.dim() != 2 or tables.shape[0] != R:
        raise ValueError(f"block tables {tuple(tables.shape)} for {R} rows")
    if not 0 <= max_ctas <= 255:
        raise ValueError(f"max_ctas {max_ctas}: 0 (one CTA per SM) to 255")
    out = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else _output(out, shape, q.device)
    strides = q.stride()
    row_stride = strides[0] if T > 1 else H * D             # of one row it says nothing
    if strides[2] != 1 or (H > 1 and strides[1] != D) or row_stride % 8 or q.data_ptr() % 16:
        q, row_stride = q.clone(memory_format=torch.contiguous_format), H * D
    ws_bytes = _workspace_bytes(index, R, kv_heads)
    early_launch = early_launch and given_as_is((tables, block_tables), (cq, cu_seqlens_q), (ck, cu_seqlens_k),
                                                (ctx, context_lens))
    flags = (EARLY_LAUNCH if early_launch else 0) | (max_ctas << CTAS_SHIFT)
    call_on(index, _lib.lib().specdec_paged_attention_fp8, q.data_ptr(), T, row_stride, H, kv_heads, D,
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, block_size, group,
            ptr(cq), ptr(ck), ptr(ctx), q_per_seq, R, tables.data_ptr(), tables.shape[1], max_q, scale, causal,
            out.data_ptr(), out.stride(0) if T > 1 else H * D, Workspace.address(index, ws_bytes, workspace), ws_bytes,
            Workspace.address(index, 256, "attention"), flags, raw_stream(index))
    return out


class AttentionFP8(torch.nn.Module):
    """attention.Attention (attention.py:43-77) over an 8-bit cache: forward(q, k, v) stores k / v at the context's
    slot_mapping and attends by the paged branch that the context selects."""

    def __init__(self, num_heads, head_dim, scale, num_kv_heads):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.cache: FP8Cache | None = None

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor | None = None
                ) -> torch.Tensor:
        context, c = get_context(), self.cache
        if c is None:
            raise ValueError("bind an FP8Cache to .cache before the forward")
        store_kvcache_fp8(k.view(-1, self.num_kv_heads, self.head_dim), v.view(-1, self.num_kv_heads, self.head_dim),
                          c.k_cache, c.v_cache, c.k_scale, c.v_scale, context.slot_mapping)
        q = q.view(-1, self.num_heads, self.head_dim)
        if context.is_prefill:
            if context.block_tables is None:
                raise NotImplementedError("prefill without a block table is outside the B200 verify/accept path")
            where = dict(cu_seqlens_q=context.cu_seqlens_q, cu_seqlens_k=context.cu_seqlens_k,
                         max_seqlen_q=context.max_seqlen_q)
        else:
            where = dict(context_lens=context.context_lens, query_len_per_seq=context.query_len_per_seq,
                         causal=context.causal)
        return paged_attention_fp8(q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, context.block_tables, self.scale,
                                   out=out, **where)
