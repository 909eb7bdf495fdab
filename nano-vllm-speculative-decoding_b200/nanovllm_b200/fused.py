"""Fused elementwise kernels around the verify forward (libspecdec_b200.so), mirroring the reference layers:

    rmsnorm(x, weight, eps[, residual])     nanovllm/layers/layernorm.py:16-40  -> specdec_rmsnorm
    silu_and_mul(gate_up)                   nanovllm/layers/activation.py:8-11  -> specdec_silu_mul
    qk_norm_rope_store(...)                 nanovllm/models/qwen3.py:77-86 + attention.py:62-63
                                            (q_norm, k_norm, RoPE, store_kvcache in one launch) -> specdec_norm_rope_store
    qk_norm_rope(...)                       the same without the cache: q, k, v rows in token order
    slots_in_range(...)                     the slots of the tokens that qk_norm_rope writes, -1 for the others
    rope_cache(head_dim, max_position, base) nanovllm/layers/rotary_embedding.py:17-27 (the cos|sin table)
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import Workspace, check, ptr, require_cuda, stream_of


def err_word(device: torch.device) -> torch.Tensor:
    return Workspace.get(device, 256, name="fused")[:4].view(torch.int32)


def device_error(device: torch.device) -> int:
    """First error recorded on this device since the last reset by the kernels that share this word: those here, the Markov
    rows and the context store (synchronises): 0 none, 3 a slot past the cache, 4 a position outside the rotary table,
    others a bounded wait that gave up."""
    return int(err_word(device).item())


def reset_device_error(device: torch.device) -> None:
    err_word(device).zero_()


def rope_cache(head_dim: int, max_position: int, base: float, device: torch.device) -> torch.Tensor:
    """rotary_embedding.py:17-27: [max_position, head_dim] fp32 = cat(cos(t * inv_freq), sin(t * inv_freq))."""
    inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.float) / head_dim))
    t = torch.arange(max_position, dtype=torch.float)
    freqs = torch.einsum("i,j -> ij", t, inv_freq)
    return torch.cat((freqs.cos(), freqs.sin()), dim=-1).contiguous().to(device)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None, *,
            out: torch.Tensor | None = None):
    """layernorm.py:16-40: without residual returns norm(x); with it returns (norm(x + residual), x + residual)."""
    device = require_cuda(x, weight, residual)
    width = x.shape[-1]
    T = x.numel() // width
    x = x.contiguous()
    out = torch.empty_like(x) if out is None else out
    res_out = torch.empty_like(x) if residual is not None else None
    check(_lib.lib().specdec_rmsnorm(ptr(x), ptr(None if residual is None else residual.contiguous()), ptr(weight),
                                     ptr(out), ptr(res_out), T, width, float(eps), stream_of(device)))
    return out if residual is None else (out, res_out)


def silu_and_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """activation.py:8-11: silu(x) * y over the two halves of the last dim (fp32 math, one rounding)."""
    device = require_cuda(gate_up)
    two_i = gate_up.shape[-1]
    T = gate_up.numel() // two_i
    if out is None:
        out = torch.empty(*gate_up.shape[:-1], two_i // 2, dtype=gate_up.dtype, device=device)
    check(_lib.lib().specdec_silu_mul(ptr(gate_up.contiguous()), ptr(out), T, two_i // 2, stream_of(device)))
    return out


def qk_norm_rope_store(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, q_norm: torch.Tensor,
                       k_norm: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor,
                       slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, eps: float,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """The verify forward's qkv [T, (H + 2 Hkv) * 128] -> q [T, H, 128] (q_norm, RoPE); k_norm + RoPE'd K and V
    rows go straight to their slots of the layer's paged caches (slot -1 skipped).  A token whose position lies outside
    cos_sin is not stored and has a zero query (device_error 4)."""
    device = require_cuda(qkv, positions, slot_mapping, k_cache, v_cache)
    T = qkv.shape[0]
    head_dim = 128
    if q_out is None:
        q_out = torch.empty(T, num_heads, head_dim, dtype=qkv.dtype, device=device)
    num_slots = k_cache.numel() // (num_kv_heads * head_dim)
    check(_lib.lib().specdec_norm_rope_store(
        ptr(qkv), 0, qkv.stride(0), T, 1, num_heads, num_kv_heads, ptr(q_norm), ptr(k_norm), 0, ptr(cos_sin),
        cos_sin.shape[0], ptr(positions), ptr(slot_mapping), ptr(k_cache), ptr(v_cache), 0, num_slots, ptr(q_out),
        float(eps), ptr(err_word(device)), stream_of(device)))
    return q_out


def qk_norm_rope(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, q_norm: torch.Tensor, k_norm: torch.Tensor,
                 cos_sin: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor, eps: float
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """qk_norm_rope_store with the K and V rows kept in token order instead of a cache's slots (for a store of another
    format): q [T, H, 128], k and v [T, Hkv, 128].  rows: int32 0 .. T-1 on the device.  A token whose position lies outside
    cos_sin has a zero query, and its K and V rows left unwritten (error 4) as qk_norm_rope_store leaves its slot: store with
    slots_in_range."""
    k, v = (torch.empty(qkv.shape[0], num_kv_heads, 128, dtype=qkv.dtype, device=qkv.device) for _ in range(2))
    q = qk_norm_rope_store(qkv, num_heads, num_kv_heads, q_norm, k_norm, cos_sin, positions, rows, k, v, eps)
    return q, k, v


def slots_in_range(slot_mapping: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """slot_mapping with -1 for the tokens whose position lies outside cos_sin: qk_norm_rope writes no row for them, and
    what their slots would get (memory as it was found) could raise the scale of a group that holds other tokens."""
    return slot_mapping.masked_fill(positions.clamp(0, cos_sin.shape[0] - 1) != positions, -1)
