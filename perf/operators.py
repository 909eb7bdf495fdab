"""The verification round over an 8-bit paged cache, operator by operator: the cases, their inputs, and each operator in
its plain form (elementary torch operations) and as this package's kernels.

    store      K/V rows into the e4m3 paged cache, one power-of-two scale per (group of tokens, KV head)
    attention  verify / decode attention over that cache
    metadata   block tables, slot maps and the rest of a round's metadata from request lengths
    logprobs   log probabilities of given tokens, entropy and top alternatives from a round's logits

The cache is [blocks, KV heads, block size, 128] e4m3 with scales [blocks, KV heads, block size / group] fp32: an element
stands for its code times its group's scale.  A group's scale is 2^e, e the smallest with every finite magnitude of the
group's stored tokens at most 448 * 2^e (and e >= -100).  A call that writes a group's first slot starts the group: the
scale comes from that call's tokens alone.  Otherwise the scale never falls, and where it rises the group's other slots
are requantised.

Set `own` to True to run the kernels.
"""
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE_DIR = str(Path(__file__).resolve().parent.parent / "nano-vllm-speculative-decoding_b200")
if PACKAGE_DIR not in sys.path:
    sys.path.insert(0, PACKAGE_DIR)

HEAD_DIM = 128
E4M3_MAX = 448.0
MIN_EXPONENT = -100
NEG = float("-inf")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    base = dict(heads=32, kv=8, block=256, group=16, q=8)
    return [
        # one request decoding one token: the smallest call, all latency
        dict(name="store_decode_1", op="store", rows=1, tokens=1, ctx=1000, kv=8, block=256, group=16, pad=0),
        # the 512 tokens of a 64-row verification appended to ~1000-token contexts, groups begun mid-way
        dict(name="store_verify_64x8", op="store", rows=64, tokens=8, ctx=1000, kv=8, block=256, group=16, pad=0),
        # four prompts of 4000 tokens stored whole, with padding tokens behind them
        dict(name="store_prompt_4x4000", op="store", rows=4, tokens=4000, ctx=0, kv=8, block=256, group=16, pad=96),
        # one request decoding one token
        dict(base, name="attn_decode_1", op="attention", rows=1, q=1, lo=1000, hi=1000, varlen=False, causal=True),
        # the verify attention of 32 requests with contexts between 900 and 1100
        dict(base, name="attn_verify_32x1k", op="attention", rows=32, lo=900, hi=1100, varlen=True, causal=True),
        # a draft block's attention: 7 queries a row that all see each other, 64 rows at ~3000 tokens
        dict(base, name="attn_draft_64x3k", op="attention", rows=64, q=7, lo=2900, hi=3107, varlen=False, causal=False),
        # the longest contexts: 64 requests at ~16k tokens
        dict(base, name="attn_verify_64x16k", op="attention", rows=64, lo=16200, hi=16384, varlen=True, causal=True),
        # a round's metadata for 64 requests, and for 512 requests of very different lengths padded to 520 rows
        dict(name="meta_64", op="metadata", rows=64, slots=64, k=7, block=256, lo=900, hi=1100, width=17, full=True),
        dict(name="meta_512", op="metadata", rows=512, slots=520, k=7, block=256, lo=1, hi=16000, width=64, full=False),
        # one request's 8 verified positions, five alternatives
        dict(name="logp_8", op="logprobs", rows=8, vocab=151936, dtype="bf16", top=5, temps=False),
        # 64 requests x 8 positions, twenty alternatives
        dict(name="logp_512", op="logprobs", rows=512, vocab=151936, dtype="bf16", top=20, temps=False),
        # fp32 logits of an odd vocabulary, a temperature for each row, no alternatives
        dict(name="logp_288_fp32", op="logprobs", rows=288, vocab=50257, dtype="fp32", top=0, temps=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["store", "attention", "attention", "metadata", "logprobs"])
    if op == "store":
        rows = _log(rng, 1, 200)
        prompt = rng.random() < 0.4
        tokens = _log(rng, 2, max(2, 16000 // rows)) if prompt else rng.randint(1, 8)
        return dict(op=op, rows=rows, tokens=tokens, ctx=0 if prompt else _log(rng, 1, 2000), kv=rng.choice([1, 2, 4, 8]),
                    block=rng.choice([128, 256]), group=rng.choice([16, 16, 32]), pad=rng.randint(0, 40))
    if op == "attention":
        hi = _log(rng, 8, 16384)
        group = rng.choice([1, 2, 4, 4, 8])
        kv = rng.choice([1, 2, 4, 8])
        return dict(op=op, rows=_log(rng, 1, max(1, min(200, 800000 // hi))), q=rng.randint(1, min(8, 32 // group)),
                    lo=max(1, rng.randint(hi // 3, hi)), hi=hi, heads=kv * group, kv=kv, block=rng.choice([128, 256]),
                    group=rng.choice([16, 16, 32]), varlen=rng.random() < 0.6, causal=True if rng.random() < 0.8 else False)
    if op == "metadata":
        rows = _log(rng, 1, 512)
        block = rng.choice([128, 256])
        hi = _log(rng, 1, 16000)
        return dict(op=op, rows=rows, slots=rows + rng.randint(0, 8), k=rng.randint(1, 15), block=block, lo=1, hi=hi,
                    width=(hi + 15 + block - 1) // block + rng.randint(0, 9), full=rng.random() < 0.4)
    return dict(op=op, rows=_log(rng, 1, 512), vocab=_log(rng, 900, 151936), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                top=rng.choice([0, 1, 5, 8, 20, 32]), temps=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------ the inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _host(seed):
    return torch.Generator().manual_seed(int(seed) + 7)


def _quantise(x, group):
    """x [.., tokens, 128] -> codes e4m3 of the same shape and scales [.., tokens / group]; the groups whole."""
    *lead, n, d = x.shape
    g = x.float().view(*lead, n // group, group, d)
    scale = _scale_of(g.abs().amax(dim=(-1, -2)))
    return (g / scale[..., None, None]).view(*lead, n, d).to(torch.float8_e4m3fn), scale


def _scale_of(amax):
    """2^e, e the smallest with amax <= 448 * 2^e = 0.875 * 2^(e + 9)."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 9 + (m > 0.875)).clamp_min(MIN_EXPONENT), MIN_EXPONENT)
    return torch.ldexp(torch.ones_like(amax), e)


def _random_cache(blocks, case, g):
    """A filled cache: unit-variance rows times a magnitude of each (block, head), stored a few blocks at a time."""
    shape = (blocks, case["kv"], case["block"], HEAD_DIM)
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(*shape[:2], case["block"] // case["group"], dtype=torch.float32, device="cuda")
    step = 512
    for b in range(0, blocks, step):
        n = min(step, blocks - b)
        x = torch.randn(n, *shape[1:], device="cuda", generator=g)
        x *= torch.rand(n, case["kv"], 1, 1, device="cuda", generator=g) + 0.5
        codes[b:b + n], scales[b:b + n] = _quantise(x.bfloat16(), case["group"])
    return codes, scales


def _spread(lo, hi, rows, host):
    """Whole numbers spread evenly over lo..hi, one a row, in an order of the seed: their sum is the case's."""
    return torch.linspace(lo, hi, rows, dtype=torch.float64).round().long()[torch.randperm(rows, generator=host)]


def _permutation(blocks, host):
    return torch.randperm(blocks, generator=host).to(torch.int32)


def _tables(need, width, perm):
    """Block tables [rows, width] (int32, host): row r's first need[r] blocks, dealt in order from a permutation."""
    first = need.cumsum(0) - need
    j = torch.arange(width)
    held = j[None, :] < need[:, None]
    return torch.where(held, perm[(first[:, None] + j[None, :]).clamp_max(perm.numel() - 1)], torch.zeros((), dtype=torch.int32))


def prepare(case, seed):
    g, host = _generator(seed), _host(seed)
    state = {"store": _prepare_store, "attention": _prepare_attention, "metadata": _prepare_metadata,
             "logprobs": _prepare_logprobs}[case["op"]](case, g, host)
    state["op"] = case["op"]
    return state


def _prepare_store(case, g, host):
    R, n, kv, bs = case["rows"], case["tokens"], case["kv"], case["block"]
    start = torch.zeros(R, dtype=torch.int64)
    if case["ctx"]:
        start = _spread(max(1, case["ctx"] - 100), case["ctx"] + 100, R, host)
    need = (start + n + bs - 1) // bs
    blocks = int(need.sum()) + 1
    tables = _tables(need, int(need.max()), _permutation(blocks, host)).long()
    pos = start[:, None] + torch.arange(n)[None, :]
    slots = tables.gather(1, pos // bs) * bs + pos % bs
    slots = torch.cat([slots.reshape(-1), torch.full((case["pad"],), -1)]).to(torch.int32).cuda()
    N = slots.numel()
    # K and V as the qkv projection leaves them: rows of one matrix, a few with magnitudes above the others'
    kvs = torch.randn(N, 2 * kv * HEAD_DIM, device="cuda", generator=g)
    kvs *= torch.exp2(torch.randn(N, 1, device="cuda", generator=g))
    kvs = kvs.bfloat16()
    k_cache, k_scale = _random_cache(blocks, case, g)
    v_cache, v_scale = _random_cache(blocks, case, g)
    return dict(key=kvs[:, :kv * HEAD_DIM].view(N, kv, HEAD_DIM), value=kvs[:, kv * HEAD_DIM:].view(N, kv, HEAD_DIM),
                k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, slots=slots)


def _prepare_attention(case, g, host):
    R, bs = case["rows"], case["block"]
    k_lens = _spread(case["lo"], case["hi"], R, host)
    q_lens = torch.full((R,), case["q"], dtype=torch.int64)
    if case["varlen"]:
        q_lens = _spread(case["q"], 1, R, host)
    need = (k_lens + bs - 1) // bs
    width, blocks = int(need.max()), int(need.sum()) + 1
    T = int(q_lens.sum())
    # queries with a few directions of their own, so that some keys stand out as in a trained model
    q = torch.randn(T, case["heads"], HEAD_DIM, device="cuda", generator=g)
    q *= torch.exp2(torch.randn(1, case["heads"], HEAD_DIM, device="cuda", generator=g))
    k_cache, k_scale = _random_cache(blocks, case, g)
    v_cache, v_scale = _random_cache(blocks, case, g)
    zero = torch.zeros(1, dtype=torch.int64)
    return dict(q=q.bfloat16(), k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale,
                tables=_tables(need, width, _permutation(blocks, host)).cuda(), scale=HEAD_DIM ** -0.5, max_q=case["q"],
                varlen=case["varlen"], causal=case["causal"] or case["varlen"], context_lens=k_lens.to(torch.int32).cuda(),
                cu_q=torch.cat([zero, q_lens.cumsum(0)]).to(torch.int32).cuda(),
                cu_k=torch.cat([zero, k_lens.cumsum(0)]).to(torch.int32).cuda())


def _prepare_metadata(case, g, host):
    R, k, bs, W = case["rows"], case["k"], case["block"], case["width"]
    lengths = _spread(case["lo"], case["hi"], R, host)
    lens = torch.full((R,), k + 1) if case["full"] else _spread(1, k + 1, R, host)
    held = (lengths - 1 + bs - 1) // bs                     # blocks of the tokens already cached: the rest are assigned
    pool = int((lengths + k).max()) // bs * R + R + 8
    perm = _permutation(pool, host)
    tables = _tables(held, W, perm)
    used = int(held.sum())
    free = torch.cat([perm[used:], torch.full((used,), -1, dtype=torch.int32)])
    n_pad = (case["slots"] - R) * (k + 1)
    tokens = int(lens.sum()) + (n_pad - n_pad // 3 if n_pad else 0)
    vocab = 151936
    return dict(lengths=lengths.cuda(), verified_lens=lens.cuda(), tables=tables.cuda(),
                num_blocks=held.to(torch.int32).cuda(), free_blocks=free.cuda(),
                free_count=torch.tensor([pool - used], dtype=torch.int32).cuda(),
                last_tokens=torch.randint(vocab, (R,), device="cuda", generator=g),
                drafts=torch.randint(vocab, (R, k), device="cuda", generator=g),
                buf64=torch.zeros(2 * tokens, dtype=torch.int64, device="cuda"),
                buf32=torch.zeros(tokens + 2 * (case["slots"] + 1) + case["slots"] * W, dtype=torch.int32, device="cuda"),
                block_size=bs, num_tokens=tokens, num_rows=case["slots"], pad_block_id=pool, width=W)


def _prepare_logprobs(case, g, host):
    T, V = case["rows"], case["vocab"]
    logits = torch.empty(T, V, dtype=DTYPES[case["dtype"]], device="cuda")
    for t in range(0, T, 64):
        logits[t:t + 64] = torch.randn(min(64, T - t), V, device="cuda", generator=g) * 3
    # the tokens a round verifies: mostly likely ones, some unlikely; a padded batch's last rows have none
    tokens = torch.randint(V, (T,), device="cuda", generator=g)
    likely = logits.float().argmax(dim=-1)
    tokens = torch.where(torch.rand(T, device="cuda", generator=g) < 0.6, likely, tokens)
    if T >= 16:
        tokens[-(T // 16):] = -1
    temps = torch.rand(T, device="cuda", generator=g) * 1.5 + 0.25 if case["temps"] else None
    return dict(logits=logits, tokens=tokens, top=case["top"], temps=temps)


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"store": _store, "attention": _attention, "metadata": _metadata, "logprobs": _logprobs}[state["op"]](state)


def _store(s):
    if own:
        from nanovllm_b200.attention_fp8 import store_kvcache_fp8
        store_kvcache_fp8(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
    else:
        _plain_store(s["key"], s["k_cache"], s["k_scale"], s["slots"])
        _plain_store(s["value"], s["v_cache"], s["v_scale"], s["slots"])
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_store(x, cache, scales, slots):
    """In place, one side.  Every token works on its whole group; a group's tokens all write the same values."""
    blocks, kv, bs, d = cache.shape
    per_block = scales.shape[2]
    group = bs // per_block
    slot = slots.long()
    live = slot >= 0
    gid = torch.where(live, slot // group, blocks * per_block)               # padding tokens: a group past the cache
    amax = torch.zeros(blocks * per_block + 1, kv, device=x.device)
    amax.scatter_reduce_(0, gid[:, None].expand(-1, kv), x.float().abs().amax(dim=-1), "amax")
    started = torch.zeros(blocks * per_block + 1, dtype=torch.bool, device=x.device)
    started.index_fill_(0, torch.where(live & (slot % group == 0), gid, blocks * per_block), True)
    wanted = _scale_of(amax[gid])                                             # [N, kv]
    b, j = (gid // per_block).clamp_max(blocks - 1), gid % per_block
    old = scales[b, :, j]
    kept = ~started[gid][:, None]
    new = torch.where(kept, torch.maximum(old, wanted), wanted)
    inside = j[:, None] * group + torch.arange(group, device=x.device)[None, :]              # [N, group]
    before = cache.view(torch.uint8)[b[:, None], :, inside].view(torch.float8_e4m3fn).float()    # [N, group, kv, d]
    ratio = torch.where(kept & (new > old), old / new, torch.ones_like(new))
    moved = (before * ratio[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = (x.float() / new[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    # padding tokens rewrite nothing: they are sent where the first live token writes the same values
    at = torch.where(live, torch.arange(slot.numel(), device=x.device), live.int().argmax())
    cache.view(torch.uint8)[b[at][:, None], :, inside[at]] = moved[at].view(torch.uint8)
    scales[b[at], :, j[at]] = new[at]
    cache.view(torch.uint8)[b[at], :, (slot % bs)[at]] = codes[at].view(torch.uint8)


def _attention(s):
    if own:
        from nanovllm_b200.attention_fp8 import paged_attention_fp8
        where = (dict(cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"], max_seqlen_q=s["max_q"]) if s["varlen"] else
                 dict(context_lens=s["context_lens"], query_len_per_seq=s["max_q"], causal=s["causal"]))
        return paged_attention_fp8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"], s["scale"],
                                   **where)
    return _plain_attention(s, torch.float32).to(torch.bfloat16)


def _rows_of(s):
    """Each row's query and key counts, and each token's row and place in it."""
    cu = s["cu_q"].long()
    q_lens, k_lens = cu[1:] - cu[:-1], s["context_lens"].long()
    T = s["q"].shape[0]
    row = torch.repeat_interleave(torch.arange(q_lens.numel(), device=cu.device), q_lens, output_size=T)
    return q_lens, k_lens, row, torch.arange(T, device=cu.device) - cu[row]


def _plain_attention(s, dtype):
    T, H, d = s["q"].shape
    kv = s["k_cache"].shape[1]
    q_lens, k_lens, row, place = _rows_of(s)
    R, Q = q_lens.numel(), s["max_q"]
    q = torch.zeros(R, Q, H, d, dtype=dtype, device=s["q"].device)
    q[row, place] = s["q"].to(dtype)
    q = q.view(R, Q, kv, H // kv, d).permute(0, 2, 1, 3, 4).reshape(R, kv, Q * (H // kv), d)
    k = _dequantised(s["k_cache"], s["k_scale"], s["tables"], dtype)
    scores = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]                                  # [R, kv, Q * G, keys]
    del k
    keys = torch.arange(scores.shape[-1], device=q.device)
    last = k_lens[:, None].expand(R, Q)
    if s["causal"]:
        last = k_lens[:, None] - q_lens[:, None] + torch.arange(Q, device=q.device)[None, :] + 1
        last = torch.minimum(last, k_lens[:, None])
    seen = keys[None, None, :] < last[:, :, None]                                               # [R, Q, keys]
    seen = seen[:, None, :, None, :].expand(R, 1, Q, H // kv, -1).reshape(R, 1, Q * (H // kv), -1)
    scores = scores.masked_fill_(~seen, NEG)
    top = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(torch.where(top == NEG, torch.zeros_like(top), top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    v = _dequantised(s["v_cache"], s["v_scale"], s["tables"], dtype)
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(R, kv, Q, H // kv, d).permute(0, 2, 1, 3, 4).reshape(R, Q, H, d)
    return o[row, place]


def _dequantised(cache, scales, tables, dtype):
    """A row's blocks one after another: [R, kv, width * block, 128]."""
    R, W = tables.shape
    _, kv, bs, d = cache.shape
    t = tables.long()
    x = cache.view(torch.uint8)[t].view(torch.float8_e4m3fn).to(dtype).view(R, W, kv, scales.shape[2], -1, d)
    x *= scales[t].to(dtype)[..., None, None]
    return x.view(R, W, kv, bs, d).permute(0, 2, 1, 3, 4).reshape(R, kv, W * bs, d)


def _metadata(s):
    if own:
        from nanovllm_b200.device_metadata import verify_metadata
        verify_metadata(s["lengths"], s["last_tokens"], s["drafts"], s["verified_lens"], s["tables"], s["num_blocks"],
                        s["free_blocks"], s["free_count"], block_size=s["block_size"], num_rows=s["num_rows"],
                        num_tokens=s["num_tokens"], pad_block_id=s["pad_block_id"], width=s["width"], buf64=s["buf64"],
                        buf32=s["buf32"])
    else:
        _plain_metadata(s)
    return s["buf64"], s["buf32"], s["tables"], s["num_blocks"], s["free_count"]


def _plain_metadata(s):
    bs, W, T, S = s["block_size"], s["width"], s["num_tokens"], s["num_rows"]
    R, k = s["drafts"].shape
    dev = s["lengths"].device
    start, lens = s["lengths"] - 1, s["verified_lens"]
    # new blocks, from the top of the free stack in row order
    need = (start + lens + bs - 1) // bs
    new = (need - s["num_blocks"]).clamp_min(0)
    taken = new.cumsum(0) - new
    j = torch.arange(W, device=dev)[None, :]
    nth = taken[:, None] + j - s["num_blocks"][:, None]
    fresh = (j >= s["num_blocks"][:, None]) & (j < need[:, None])
    from_top = (s["free_count"].long() - 1 - nth).clamp(0, s["free_blocks"].numel() - 1)
    s["tables"].copy_(torch.where(fresh, s["free_blocks"][from_top], s["tables"]))
    s["free_count"].sub_(new.sum().to(torch.int32))
    s["num_blocks"].copy_(torch.maximum(s["num_blocks"], need.to(torch.int32)))
    # rows, then padding rows of at most k + 1 tokens
    left = (T - lens.sum()) - torch.arange(S - R, device=dev) * (k + 1)
    q_lens = torch.cat([lens, left.clamp(0, k + 1)])
    first = q_lens.cumsum(0) - q_lens
    row = torch.repeat_interleave(torch.arange(S, device=dev), q_lens, output_size=T)
    place = torch.arange(T, device=dev) - first[row]
    real = row < R
    r = row.clamp_max(R - 1)
    position = torch.where(real, start[r], torch.zeros_like(r)) + place
    ids = torch.where(place == 0, s["last_tokens"][r], s["drafts"][r, (place - 1).clamp(0, k - 1)])
    s["buf64"][:T] = torch.where(real, ids, torch.zeros_like(ids))
    s["buf64"][T:] = position
    block = s["tables"][r, torch.where(real, position // bs, torch.zeros_like(r))].long()
    s["buf32"][:T] = torch.where(real, block * bs + position % bs, -1).to(torch.int32)
    k_lens = torch.cat([start + lens, q_lens[R:]])
    at = T
    s["buf32"][at] = 0
    s["buf32"][at + 1:at + S + 1] = q_lens.cumsum(0).to(torch.int32)
    at += S + 1
    s["buf32"][at] = 0
    s["buf32"][at + 1:at + S + 1] = k_lens.cumsum(0).to(torch.int32)
    at += S + 1
    table = s["buf32"][at:].view(S, W)
    table.fill_(s["pad_block_id"])
    table[:R] = torch.where(j < s["num_blocks"][:, None], s["tables"], table[:R])


def _logprobs(s):
    if own:
        from nanovllm_b200.logprobs import token_logprobs
        got = token_logprobs(s["logits"], s["tokens"], s["top"], s["temps"])
        return got.logprobs, got.entropy, got.top_ids, got.top_logprobs
    return _plain_logprobs(s)


def _plain_logprobs(s):
    x = s["logits"].float()
    T, V = x.shape
    live = s["tokens"] >= 0
    if s["temps"] is not None:
        x = x / s["temps"][:, None]
    m = x.amax(dim=-1, keepdim=True)
    x = x - m
    e = x.exp()
    total = e.sum(dim=-1)
    log_total = total.log()
    lp = x.gather(1, s["tokens"].clamp_min(0)[:, None])[:, 0] - log_total
    entropy = log_total - (x * e).sum(dim=-1) / total
    del e
    # the largest logits, ties to the lowest index: one integer key orders by value, then by index from the end
    ids = torch.empty(T, 0, dtype=torch.int64, device=x.device)
    if s["top"]:
        bits = (s["logits"].float() + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = order * (1 << 32) + (V - 1 - torch.arange(V, device=x.device))
        ids = V - 1 - (key.topk(s["top"], dim=-1).values & 0xFFFFFFFF)
    top = x.gather(1, ids) - log_total[:, None]
    zero = torch.zeros_like(lp)
    return (torch.where(live, lp, zero), torch.where(live, entropy, zero), torch.where(live[:, None], ids, -1),
            torch.where(live[:, None], top, torch.zeros_like(top)))


# ------------------------------------------------------------------------------------------------------ the bounds
def work(case):
    """What a pass cannot do without: inputs read once, outputs written once."""
    op = case["op"]
    if op == "store":
        N = case["rows"] * case["tokens"]
        row = case["kv"] * HEAD_DIM
        groups = case["rows"] * (case["tokens"] // case["group"] + 1)
        return {"bytes": N * row * 2 * 3 + (N + case["pad"]) * 4 + groups * case["kv"] * 2 * 8, "flops": N * row * 2 * 3}
    if op == "attention":
        keys = case["rows"] * (case["lo"] + case["hi"]) / 2
        T = case["rows"] * ((case["q"] + 1) / 2 if case["varlen"] else case["q"])
        cache = keys * case["kv"] * 2 * (HEAD_DIM + 4 / case["group"])
        tables = case["rows"] * 4 * ((case["hi"] + case["block"] - 1) // case["block"] + 2)
        return {"bytes": cache + T * case["heads"] * HEAD_DIM * 4 + tables,
                "flops": 4.0 * keys * case["heads"] * HEAD_DIM * T / case["rows"]}
    if op == "metadata":
        T = case["slots"] * (case["k"] + 1)
        return {"bytes": case["rows"] * (8 * 3 + 8 * case["k"] + 8) + T * 20 + case["slots"] * (8 + 8 * case["width"]),
                "flops": T * 8}
    size = 4 if case["dtype"] == "fp32" else 2
    rows = case["rows"] - (case["rows"] // 16 if case["rows"] >= 16 else 0)
    n = rows * case["vocab"]
    return {"bytes": n * size + case["rows"] * (8 + 8 + 12 * case["top"]), "flops": n * 6}


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"store": _exact_store, "attention": _exact_attention, "metadata": _exact_metadata,
            "logprobs": _exact_logprobs}[case["op"]](case, state)


def _exact_store(case, s):
    """From the definition, group by group in integer order; codes before their rounding."""
    out = []
    slots = s["slots"].long()
    live = torch.nonzero(slots >= 0)[:, 0]
    slot = slots[live]
    group = case["group"]
    per_block = case["block"] // group
    groups, which = torch.unique(slot // group, return_inverse=True)
    begun = torch.zeros(groups.numel(), dtype=torch.bool, device=slot.device)
    begun[which[slot % group == 0]] = True
    for x, cache, scales in ((s["key"], s["k_cache"], s["k_scale"]), (s["value"], s["v_cache"], s["v_scale"])):
        x = x.double()[live]
        codes, steps = cache.double(), scales.double()
        most = torch.zeros(groups.numel(), case["kv"], dtype=torch.float64, device=x.device)
        most.index_reduce_(0, which, x.abs().amax(dim=-1), "amax")
        step = torch.full_like(most, 2.0 ** -100)
        for e in range(-100, 121):                       # the smallest power of two that holds the group
            step = torch.where(most > 448.0 * step, torch.full_like(most, 2.0 ** (e + 1)), step)
        b, j = groups // per_block, groups % per_block
        old = steps[b, :, j]
        new = torch.where(begun[:, None] | (step > old), step, old)
        span = j[:, None] * group + torch.arange(group, device=x.device)
        held = codes[b[:, None], :, span]
        shrink = torch.where(begun[:, None] | (new <= old), torch.ones_like(new), old / new)
        codes[b[:, None], :, span] = held * shrink[:, None, :, None]
        codes[slot // case["block"], :, slot % case["block"]] = x / new[which][..., None]
        steps[b, :, j] = new
        out.append((codes, steps))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attention(case, s):
    """Row by row in 64 bits."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu, lens = s["cu_q"].tolist(), s["context_lens"].tolist()
    heads_each = case["heads"] // case["kv"]
    for r, L in enumerate(lens):
        n = cu[r + 1] - cu[r]
        pages = s["tables"][r, :(L + case["block"] - 1) // case["block"]].long()

        def rows(cache, scales):
            step = scales[pages].double().repeat_interleave(case["group"], dim=2)
            x = cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * step[..., None]
            return x.transpose(0, 1).reshape(case["kv"], -1, HEAD_DIM)[:, :L]

        k, v = rows(s["k_cache"], s["k_scale"]), rows(s["v_cache"], s["v_scale"])
        q = s["q"][cu[r]:cu[r + 1]].double().view(n, case["kv"], heads_each, HEAD_DIM)
        x = torch.einsum("nhgd,hkd->hngk", q, k) / math.sqrt(HEAD_DIM)
        if s["causal"]:
            at, key = torch.arange(n, device="cuda"), torch.arange(L, device="cuda")
            x = x.masked_fill((key[None, :] > (L - n + at)[:, None])[None, :, None, :], NEG)
        seen = (x > NEG).any(dim=-1, keepdim=True)
        p = torch.where(seen, torch.softmax(x, dim=-1), torch.zeros_like(x))
        out[cu[r]:cu[r + 1]] = torch.einsum("hngk,hkd->nhgd", p, v).reshape(n, case["heads"], HEAD_DIM)
    return out


def _exact_metadata(case, s):
    return None      # whole numbers only


def _exact_logprobs(case, s):
    lp, entropy, top = [], [], []
    for t in range(0, case["rows"], 32):
        raw = s["logits"][t:t + 32].double()
        x = raw if s["temps"] is None else raw / s["temps"][t:t + 32].double()[:, None]
        p = torch.log_softmax(x, dim=-1)
        tok = s["tokens"][t:t + 32]
        live = tok >= 0
        lp.append(torch.where(live, p.gather(1, tok.clamp_min(0)[:, None])[:, 0], 0.0))
        entropy.append(torch.where(live, -(p.exp() * p).sum(dim=-1), 0.0))
        best = p.gather(1, raw.sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]])
        top.append(torch.where(live[:, None], best, torch.zeros_like(best)))
    return torch.cat(lp), torch.cat(entropy), None, torch.cat(top)
