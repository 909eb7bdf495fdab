"""numpy restatement, in 64 bits, of the 8-bit paged K/V cache and the attention over it -- test infrastructure only.

An element stands for code * scale: codes e4m3 (sign, 4 exponent bits with bias 7, 3 mantissa bits, largest 448, no
infinities), one scale per (block, head, group of slots).  Values are held decoded, as float64.
"""
from __future__ import annotations

import numpy as np


def round_e4m3(x):
    """The e4m3 value nearest to x (ties to the even mantissa), saturating at 448, NaN kept."""
    x = np.asarray(x, dtype=np.float64)
    a = np.minimum(np.abs(x), 448.0)
    _, e = np.frexp(a)                                # a = m * 2^e, m in [0.5, 1)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)   # one unit of the last mantissa bit
    y = np.minimum(np.rint(a / step) * step, 448.0)
    return np.where(np.isnan(x), np.nan, np.copysign(y, x))


def scale_for(amax: float) -> float:
    """The smallest 2^e, e >= -100, with amax <= 448 * 2^e."""
    e = -100
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def store(x, codes, scales, slots, group: int) -> None:
    """One side (K or V) in place: x [N, Hkv, D] to slots of codes [blocks, Hkv, block_size, D] (decoded values) with
    scales [blocks, Hkv, block_size / group]."""
    blocks, heads, block_size, _ = codes.shape
    last = {}
    for t, slot in enumerate(np.asarray(slots).tolist()):
        if 0 <= slot < blocks * block_size:
            last[slot] = t                            # a slot given twice holds its last token
    groups: dict[int, dict[int, int]] = {}
    for slot, t in last.items():
        groups.setdefault(slot // group, {})[slot % group] = t
    for g, members in groups.items():
        block, j0 = g * group // block_size, g * group % block_size
        for h in range(heads):
            rows = np.stack([x[t, h] for t in members.values()]).astype(np.float64)
            finite = np.abs(rows[np.isfinite(rows)])
            wanted = scale_for(float(finite.max()) if finite.size else 0.0)
            old = float(scales[block, h, j0 // group])
            new = wanted if 0 in members else max(old, wanted)
            for o in range(group):
                at = codes[block, h, j0 + o]
                if o in members:
                    at[:] = round_e4m3(np.asarray(x[members[o], h], dtype=np.float64) / new)
                elif 0 not in members and new > old:
                    at[:] = round_e4m3(at * (old / new))
            scales[block, h, j0 // group] = new


def paged_attention(q, k, v, k_scale, v_scale, block_tables, q_starts, q_lens, k_lens, scale: float,
                    causal: bool = True):
    """q [T, H, D]; k / v codes [blocks, Hkv, block_size, D] decoded.  Per row r the queries q_starts[r] .. + q_lens[r]
    over its first k_lens[r] keys.  Returns (o, spread): o [T, H, D] in 64 bits (rows not covered 0) and what an error of
    one part in 2^9 of every probability and of 2^-16 of every score's absolute terms can move o by."""
    T, H, D = q.shape
    _, heads, block_size, _ = k.shape
    each, group = H // heads, block_size // k_scale.shape[2]
    out, spread = np.zeros((T, H, D)), np.zeros((T, H, D))
    for r in range(len(q_lens)):
        n, L, q0 = int(q_lens[r]), int(k_lens[r]), int(q_starts[r])
        pos = np.arange(L)
        block, j = np.asarray(block_tables[r])[pos // block_size], pos % block_size
        for h in range(heads):
            kk = k[block, h, j] * k_scale[block, h, j // group][:, None].astype(np.float64)
            vv = v[block, h, j] * v_scale[block, h, j // group][:, None].astype(np.float64)
            for p in range(n):
                seen = min(L, L - n + p + 1) if causal else L
                if seen <= 0:
                    continue
                qq = q[q0 + p, h * each:(h + 1) * each].astype(np.float64)
                s = qq @ kk[:seen].T * scale
                w = np.exp(s - s.max(axis=1, keepdims=True))
                w /= w.sum(axis=1, keepdims=True)
                terms = (np.abs(qq) @ np.abs(kk[:seen]).T * abs(scale)).max(axis=1, keepdims=True)
                out[q0 + p, h * each:(h + 1) * each] = w @ vv[:seen]
                spread[q0 + p, h * each:(h + 1) * each] = (2.0 ** -9 + 2.0 ** -16 * terms) * (w @ np.abs(vv[:seen]))
    return out, spread
