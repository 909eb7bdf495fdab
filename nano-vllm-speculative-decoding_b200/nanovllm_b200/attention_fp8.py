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
keys than queries) gives zeros.  Errors found on the device are in attention.device_error: 2 row metadata, 3 a slot past
the cache, 5 a block id outside the cache (read as block 0).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._lib import check, ptr, require_cuda, stream_of
from .attention import CTAS_SHIFT, EARLY_LAUNCH, _err_word, _output, _row_metadata, _split_workspace
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
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        raise ValueError(f"the 8-bit caches are float8_e4m3fn (got {k_cache.dtype}, {v_cache.dtype})")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise ValueError("the scales are float32")
    if k_cache.dim() != 4 or k_cache.shape[3] != HEAD_DIM or v_cache.shape != k_cache.shape:
        raise ValueError(f"caches must be [blocks, Hkv, block_size, {HEAD_DIM}] of one shape "
                         f"(got {tuple(k_cache.shape)}, {tuple(v_cache.shape)})")
    blocks, kv_heads, block_size, _ = k_cache.shape
    if (k_scale.dim() != 3 or v_scale.shape != k_scale.shape or k_scale.shape[:2] != (blocks, kv_heads)
            or k_scale.shape[2] * 16 not in (block_size, block_size // 2)):
        raise ValueError(f"scales must be [blocks, Hkv, block_size / 16 or / 32] of one shape "
                         f"(got {tuple(k_scale.shape)}, {tuple(v_scale.shape)} for caches {tuple(k_cache.shape)})")
    if not all(t.is_contiguous() for t in (k_cache, v_cache, k_scale, v_scale)):
        raise ValueError("caches and scales must be contiguous")
    return blocks, kv_heads, block_size, block_size // k_scale.shape[2]


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """key / value [N, Hkv, 128] bf16 rows (dense heads, rows may be strided) to slot_mapping [N] of the 8-bit caches,
    in any order; slot -1 skipped.  At most 16384 tokens a call."""
    device = require_cuda(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    blocks, kv_heads, block_size, group = _cache_geometry(k_cache, v_cache, k_scale, v_scale)
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise ValueError("the B200 K/V store takes bf16 keys and values")
    if key.dim() != 3 or key.shape[1:] != (kv_heads, HEAD_DIM) or value.shape != key.shape:
        raise ValueError(f"key and value must be [N, {kv_heads}, {HEAD_DIM}] (got {tuple(key.shape)}, "
                         f"{tuple(value.shape)})")
    N = key.shape[0]
    for t in (key, value):
        if N and (t.stride(2) != 1 or (kv_heads > 1 and t.stride(1) != HEAD_DIM)):
            raise ValueError("key and value rows must hold their heads densely")
    if slot_mapping.numel() != N:
        raise ValueError(f"{slot_mapping.numel()} slots for {N} tokens")
    slots = slot_mapping.to(torch.int32).contiguous()
    with torch.cuda.device(device):
        check(_lib.lib().specdec_store_kvcache_fp8(
            ptr(key), key.stride(0), ptr(value), value.stride(0), ptr(k_cache), ptr(v_cache), ptr(k_scale), ptr(v_scale),
            ptr(slots), N, kv_heads, HEAD_DIM, blocks, block_size, group, ptr(_err_word(device)), stream_of(device)))


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
    device = require_cuda(q, k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens_q, cu_seqlens_k, context_lens)
    blocks, kv_heads, block_size, group = _cache_geometry(k_cache, v_cache, k_scale, v_scale)
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be bf16 [T, H, {HEAD_DIM}] (got {q.dtype} {tuple(q.shape)})")
    if cu_seqlens_q is None and context_lens is None:
        raise ValueError("give cu_seqlens_q / cu_seqlens_k (varlen) or context_lens (decode)")
    if not 0 <= max_ctas <= 255:
        raise ValueError(f"max_ctas {max_ctas}: 0 (one CTA per SM) to 255")
    T, H, D = q.shape
    out = _output(out, q.shape, device)
    if q.stride(2) != 1 or q.stride(1) != D or q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
    tables, cq, ck, ctx, R, q_per_seq, max_q = _row_metadata(block_tables, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                                                              context_lens, query_len_per_seq)
    if tables.dim() != 2 or tables.shape[0] != R or (ck is not None and ck.numel() != R + 1):
        raise ValueError(f"block tables {tuple(tables.shape)} and lengths disagree on the {R} rows")
    ws = _split_workspace(device, R, kv_heads, workspace)
    flags = (EARLY_LAUNCH if early_launch else 0) | (max_ctas << CTAS_SHIFT)
    with torch.cuda.device(device):
        check(_lib.lib().specdec_paged_attention_fp8(
            ptr(q), T, q.stride(0), H, kv_heads, D, ptr(k_cache), ptr(v_cache), ptr(k_scale), ptr(v_scale), blocks,
            block_size, group, ptr(cq), ptr(ck), ptr(ctx), q_per_seq, R, ptr(tables), tables.shape[1], max_q, float(scale),
            int(causal), ptr(out), out.stride(0), ptr(ws), ws.numel(), ptr(_err_word(device)), flags,
            stream_of(device)))
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
