"""The 8-bit paged K/V cache: the store (codes and scales equal to the 64-bit oracle's, bit for bit) and the attention
over it.

Tolerance of the attention, from its roundings: the output is rounded to bf16 once (2^-8 of the value), every
probability may be off by 2^-9 of itself before it multiplies its value row (it reaches the tensor core as the sum of
three 3-bit parts), and a score, summed in fp32 and taken through a 2^-22 exponential, by 2^-16 of its absolute terms
(128 products and their fp32 sum: at most 128 * 2^-24 = 2^-17 of them; the exponent's product and sum the rest).
oracle.fp8_cache.paged_attention returns the last two as `spread`, per output."""
import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def F():
    from nanovllm_b200 import attention, attention_fp8
    attention.reset_device_error(DEV)
    return attention_fp8


def device_error():
    from nanovllm_b200 import attention
    torch.cuda.synchronize()
    return attention.device_error(DEV)


# ---------------------------------------------------------------------------------------------- the store
def random_cache(F, blocks, block_size, heads, group, seed, stale_nan=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = F.FP8Cache.allocate(blocks, block_size, heads, DEV, group=group)
    for cache, scale in ((c.k_cache, c.k_scale), (c.v_cache, c.v_scale)):
        cache.copy_((torch.randn(cache.shape, device=DEV, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn))
        scale.copy_(torch.exp2(torch.randint(-9, -4, scale.shape, device=DEV, generator=g).float()))
        if stale_nan:
            cache.view(torch.uint8).fill_(0x7F)
    return c


def host(c):
    return [t.double().cpu().numpy() for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale)]


def rows(N, heads, seed, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, 2 * heads * 128 + 64, device=DEV, generator=g)
    x = (x * torch.exp2(spread * torch.randn(N, 1, device=DEV, generator=g))).bfloat16()
    return (x[:, 32:32 + heads * 128].view(N, heads, 128), x[:, 32 + heads * 128:32 + 2 * heads * 128].view(N, heads, 128))


def check_store(F, c, key, value, slots, group):
    want = host(c)
    for side, x in ((0, key), (1, value)):
        O.store(x.double().cpu().numpy(), want[side], want[2 + side], slots.cpu().numpy(), group)
    F.store_kvcache_fp8(key, value, c.k_cache, c.v_cache, c.k_scale, c.v_scale, slots)
    got = host(c)
    assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])
    assert np.array_equal(got[0], want[0], equal_nan=True) and np.array_equal(got[1], want[1], equal_nan=True)


@pytest.mark.parametrize("heads,block_size,group", [(8, 256, 16), (1, 128, 16), (3, 128, 32), (2, 32, 32), (8, 16, 16)])
@pytest.mark.parametrize("N", [1, 2, 7, 15, 16, 17, 33, 100])
def test_store_runs_of_slots(F, heads, block_size, group, N):
    """A run of consecutive slots from the middle of a group: groups raised, groups started, a partial one at the end."""
    blocks = (N + 40) // block_size + 2
    c = random_cache(F, blocks, block_size, heads, group, N)
    key, value = rows(N, heads, N + heads)
    check_store(F, c, key, value, torch.arange(N, device=DEV, dtype=torch.int32) + 5, group)
    assert device_error() == 0


@pytest.mark.parametrize("group", [16, 32])
def test_store_any_order_twice_given_and_padding(F, group):
    """Slots shuffled over many groups, with padding between, every fifth one given again later (its last token stays)."""
    c = random_cache(F, 6, 128, 4, group, 1)
    g = torch.Generator().manual_seed(2)
    slots = torch.randperm(6 * 128, generator=g)[:300].to(torch.int32)
    slots = torch.cat([slots, slots[::5], torch.full((30,), -1, dtype=torch.int32)])
    slots = slots[torch.randperm(slots.numel(), generator=g)].to(DEV)
    key, value = rows(slots.numel(), 4, 3)
    check_store(F, c, key, value, slots, group)
    assert device_error() == 0


@pytest.mark.parametrize("value", [0.0, -0.0, 1e-38, 2.0 ** -126, 2.0 ** -133, 1e-30, 448.0, 450.0, 3.38e38, float("inf"),
                                   float("-inf"), float("nan")])
def test_store_special_values(F, value):
    c = random_cache(F, 1, 128, 2, 16, 4)
    key, val = rows(3, 2, 5)
    key[1] = value                      # a whole row of it
    val[:, 1, 77] = value               # one element of each row
    check_store(F, c, key, val, torch.tensor([16, 17, 3], device=DEV, dtype=torch.int32), 16)


def test_store_keeps_nan_codes_through_a_raise(F):
    c = random_cache(F, 1, 128, 1, 16, 6, stale_nan=True)
    key, val = rows(1, 1, 7)
    check_store(F, c, key * 1000, val * 1000, torch.tensor([9], device=DEV, dtype=torch.int32), 16)


@pytest.mark.parametrize("old", [0.0, 2.0 ** -140, 0.3, 2.0 ** 100])
def test_store_over_scales_of_any_origin(F, old):
    """Scales that no store wrote: zero (never set), below the smallest, no power of two, huge."""
    c = random_cache(F, 1, 128, 2, 16, 8)
    if old == 0.3:                      # codes stay those of a product with 1 / old: values that divide exactly
        c.k_cache.zero_()
        c.v_cache.zero_()
    c.k_scale.fill_(old)
    c.v_scale.fill_(old)
    key, val = rows(2, 2, 9)
    key, val = key * 256, val * 256
    check_store(F, c, key, val, torch.tensor([18, 19], device=DEV, dtype=torch.int32), 16)


def test_store_prompt_of_the_most_tokens(F):
    N = 16384
    c = random_cache(F, 65, 256, 2, 16, 10)
    key, value = rows(N, 2, 11)
    slots = torch.arange(N, device=DEV, dtype=torch.int32) + 37
    check_store(F, c, key, value, slots, 16)
    with pytest.raises(Exception, match="at most 16384"):
        k2, v2 = rows(N + 1, 2, 12)
        F.store_kvcache_fp8(k2, v2, c.k_cache, c.v_cache, c.k_scale, c.v_scale,
                            torch.full((N + 1,), -1, device=DEV, dtype=torch.int32))


@pytest.mark.parametrize("N", [1184, 1185, 3333])
@pytest.mark.parametrize("heads,group", [(1, 16), (8, 16), (9, 16), (2, 32), (9, 32)])
def test_store_many_tokens_in_any_order(F, N, heads, group):
    """Around and above the count where a CTA takes many tokens: slots shuffled over blocks, a fifth given twice, padding
    between, slots past the cache, and a mapping that starts off a 16-byte boundary."""
    from nanovllm_b200 import attention
    block_size, blocks = 128, 40
    c = random_cache(F, blocks, block_size, heads, group, N)
    g = torch.Generator().manual_seed(N + heads)
    first = N * 7 // 10
    slots = torch.randperm(blocks * block_size, generator=g)[:first].to(torch.int32)
    again = slots[torch.randperm(first, generator=g)[:N // 5]]
    rest = torch.full((N - first - again.numel(),), -1, dtype=torch.int32)
    rest[::9] = blocks * block_size + 5
    slots = torch.cat([slots, again, rest])
    slots = slots[torch.randperm(N, generator=g)]
    mapping = torch.zeros(N + 1, dtype=torch.int32, device=DEV)
    mapping[1:] = slots
    key, value = rows(N, heads, N)
    check_store(F, c, key, value, mapping[1:], group)
    assert device_error() == 3
    attention.reset_device_error(DEV)


@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("heads", [1, 8, 9])
def test_store_runs_of_many_tokens(F, heads, group):
    """Prompts one after another and verified rows of 8, each from the middle of a group, 2,500 tokens in a call."""
    lens = [900, 1, 700, 17] + [8] * 110 + [2]
    blocks = 64
    c = random_cache(F, blocks, 128, heads, group, 19)
    slots, at = [], 5
    for n in lens:
        slots += list(range(at, at + n))
        at += n + 13
    assert at <= blocks * 128
    slots = torch.tensor(slots, dtype=torch.int32, device=DEV)
    key, value = rows(slots.numel(), heads, 20)
    check_store(F, c, key, value, slots, group)
    assert device_error() == 0


def test_store_rows_of_a_group_far_apart(F):
    """Sixteen passes over 200 groups, each pass one slot of every group in another order: a group's tokens lie in many CTAs, and
    group numbers 1024 apart (which the look over the slots does not tell apart at first) are all there."""
    groups = [i + 1024 * (i % 3) for i in range(200)]
    c = random_cache(F, 200, 256, 2, 16, 21)
    g = torch.Generator().manual_seed(3)
    slots = torch.cat([torch.tensor([16 * groups[j] + (o + j) % 16 for j in torch.randperm(200, generator=g).tolist()])
                       for o in range(16)]).to(torch.int32).to(DEV)
    key, value = rows(slots.numel(), 2, 22)
    check_store(F, c, key, value, slots, 16)
    assert device_error() == 0


def test_store_nothing(F):
    c = random_cache(F, 1, 128, 2, 16, 13)
    before = [t.clone() for t in (c.k_cache.view(torch.uint8), c.v_cache.view(torch.uint8), c.k_scale, c.v_scale)]
    for N in (0, 5):
        key, value = rows(N, 2, 14)
        F.store_kvcache_fp8(key, value, c.k_cache, c.v_cache, c.k_scale, c.v_scale,
                            torch.full((N,), -1, device=DEV, dtype=torch.int64))
    assert all(torch.equal(a, b) for a, b in zip(before, (c.k_cache.view(torch.uint8), c.v_cache.view(torch.uint8),
                                                          c.k_scale, c.v_scale)))


def test_store_skips_a_slot_past_the_cache(F):
    from nanovllm_b200 import attention
    c = random_cache(F, 2, 128, 2, 16, 15)
    key, value = rows(3, 2, 16)
    check_store(F, c, key, value, torch.tensor([256, 7, 2 ** 31 - 1], device=DEV, dtype=torch.int32), 16)
    assert device_error() == 3
    attention.reset_device_error(DEV)


def test_store_replays_in_a_graph_and_on_another_stream(F):
    c, d = random_cache(F, 3, 128, 4, 16, 17), random_cache(F, 3, 128, 4, 16, 17)
    key, value = rows(50, 4, 18)
    slots = torch.arange(50, device=DEV, dtype=torch.int32) + 100

    def go(x):
        F.store_kvcache_fp8(key, value, x.k_cache, x.v_cache, x.k_scale, x.v_scale, slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(random_cache(F, 3, 128, 4, 16, 17))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            go(c)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(2):
        key.mul_(3.0)
        slots.add_(20 * step)
        graph.replay()
        go(d)
        torch.cuda.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(host(c), host(d)))


# ---------------------------------------------------------------------------------------------- the attention
def case(F, q_lens, k_lens, H=32, heads=8, block_size=256, group=16, seed=0, sharp=1.0, spread=0.5, stale_nan=True):
    """Rows over a shuffled cache written by the store itself; what no row owns holds NaN codes and NaN scales."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [max(1, math.ceil(k / block_size)) for k in k_lens]
    blocks = sum(need) + 3
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = torch.full((len(k_lens), max(need)), perm[-1], dtype=torch.int32)
    c = F.FP8Cache.allocate(blocks, block_size, heads, DEV, group=group)
    if stale_nan:
        for t in (c.k_cache, c.v_cache):
            t.view(torch.uint8).fill_(0x7F)
        for t in (c.k_scale, c.v_scale):
            t.fill_(float("nan"))
    used = 0
    for r, (n, L) in enumerate(zip(need, k_lens)):
        tables[r, :n] = torch.tensor(perm[used:used + n], dtype=torch.int32)
        used += n
        for at in range(0, L, 16384):
            pos = torch.arange(at, min(L, at + 16384))
            slots = (tables[r, pos // block_size].long() * block_size + pos % block_size).to(torch.int32).to(DEV)
            x = torch.randn(2, len(pos), heads, 128, device=DEV, generator=g)
            x = (x * torch.exp2(spread * torch.randn(2, len(pos), heads, 1, device=DEV, generator=g))).bfloat16()
            F.store_kvcache_fp8(x[0], x[1], c.k_cache, c.v_cache, c.k_scale, c.v_scale, slots)
    T = sum(q_lens)
    q = (torch.randn(T, H, 128, device=DEV, generator=g) * sharp).bfloat16()
    cu = lambda lens: torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(c=c, q=q, tables=tables.to(DEV), q_lens=q_lens, k_lens=k_lens, cu_q=cu(q_lens), cu_k=cu(k_lens),
                ctx=torch.tensor(k_lens, dtype=torch.int32, device=DEV), scale=128 ** -0.5)


def attend(F, s, decode=False, **kw):
    c = s["c"]
    where = (dict(context_lens=s["ctx"], query_len_per_seq=s["q_lens"][0]) if decode else
             dict(cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"], max_seqlen_q=max(s["q_lens"])))
    return F.paged_attention_fp8(s["q"], c.k_cache, c.v_cache, c.k_scale, c.v_scale, s["tables"], s["scale"], **where, **kw)


def oracle(s, causal=True):
    k, v, ks, vs = host(s["c"])
    starts = np.concatenate([[0], np.cumsum(s["q_lens"])[:-1]])
    return O.paged_attention(s["q"].double().cpu().numpy(), k, v, ks, vs, s["tables"].cpu().numpy(), starts, s["q_lens"],
                             s["k_lens"], s["scale"], causal)


def agree(out, want, spread):
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - want) - (2.0 ** -8 * np.abs(want) + spread + 1e-30)
    assert over.max() <= 0, f"{(over > 0).sum()} of {over.size} past the bound, worst by {over.max():.3g}"


def check(F, s, decode=False, causal=True):
    out = attend(F, s, decode, **({"causal": causal} if decode else {}))
    assert device_error() == 0
    agree(out, *oracle(s, causal))
    return out


@pytest.mark.parametrize("k_lens", [[1, 2, 8], [15, 16, 17], [31, 32, 33], [127, 128, 129], [255, 256, 257],
                                    [383, 512, 640], [159, 160, 161], [223, 224, 225]])
def test_attention_ragged_rows(F, k_lens):
    check(F, case(F, [min(k, q) for k, q in zip(k_lens, [1, 5, 8])], k_lens, seed=sum(k_lens)))


@pytest.mark.parametrize("H,heads,q", [(8, 8, 8), (1, 1, 32), (16, 8, 16), (64, 8, 4), (32, 4, 1), (4, 1, 8), (24, 3, 3)])
@pytest.mark.parametrize("block_size,group", [(256, 16), (128, 32)])
def test_attention_head_layouts(F, H, heads, q, block_size, group):
    check(F, case(F, [q] * 3, [300, 129, 800], H=H, heads=heads, block_size=block_size, group=group, seed=H + q))


@pytest.mark.parametrize("causal", [False, True])
def test_attention_decode_branch(F, causal):
    check(F, case(F, [7] * 4, [7, 100, 300, 1000], seed=9), decode=True, causal=causal)


def test_attention_single_tokens(F):
    check(F, case(F, [1] * 5, [1, 40, 128, 1000, 3001], seed=10), decode=True)


def test_attention_verify_batch(F):
    """32 rows x 8 queries, 32 / 8 heads, contexts between 900 and 1100."""
    lens = np.random.default_rng(0).integers(900, 1101, size=32).tolist()
    check(F, case(F, [8] * 32, lens, seed=1))


@pytest.mark.parametrize("k_lens", [[20000], [9000, 3000, 40]])
def test_attention_long_rows(F, k_lens):
    check(F, case(F, [8] * len(k_lens), k_lens, H=8, heads=2, seed=len(k_lens)))


@pytest.fixture(scope="module")
def long_row(F):
    """262,144 zero keys but the first, which has a 1 in its first dim; values between 0.75 and 1.25."""
    n = 1 << 18
    c = F.FP8Cache.allocate(n // 256, 256, 1, DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    for at in range(0, n, 16384):
        k = torch.zeros(16384, 1, 128, device=DEV)
        k[0, 0, 0] = float(at == 0)
        v = 0.75 + 0.5 * torch.rand(k.shape, device=DEV, generator=g)
        F.store_kvcache_fp8(k.bfloat16(), v.bfloat16(), c.k_cache, c.v_cache, c.k_scale, c.v_scale,
                            torch.arange(at, at + 16384, dtype=torch.int32, device=DEV))
    return c, n


@pytest.mark.parametrize("spike", [11.0, 12.5, 13.0, 13.5, 14.0, 14.5, 15.0, 15.5, 16.0, 16.5, 17.0, 17.5, 18.0, 19.0, 20.0])
def test_attention_long_flat_tail_below_one_key(F, long_row, spike):
    """One key e^spike times as likely as each of 262,143 others, which are 1 to 80 % of the row together, in one piece (a CTA for
    the whole row keeps one running maximum): probabilities between 2^-16 and 2^-29 of the largest count as exactly as others."""
    c, n = long_row
    q = torch.zeros(1, 4, 128, device=DEV)
    q[:, :, 0] = spike
    s = dict(c=c, q=q.bfloat16(), tables=torch.arange(n // 256, dtype=torch.int32, device=DEV)[None], q_lens=[1], k_lens=[n],
             cu_q=torch.tensor([0, 1], dtype=torch.int32, device=DEV), cu_k=torch.tensor([0, n], dtype=torch.int32, device=DEV),
             scale=1.0)
    out = attend(F, s, max_ctas=1)
    want, spread = oracle(s)
    assert device_error() == 0
    agree(out, want, spread)


@pytest.mark.parametrize("sharp,spread", [(0.001, 0.5), (20.0, 0.5), (300.0, 2.0), (1.0, 6.0)])
def test_attention_flat_and_peaked(F, sharp, spread):
    """Scores from almost equal to far apart, groups of very different scales side by side."""
    check(F, case(F, [8, 3], [700, 2049], H=8, heads=2, seed=20, sharp=sharp, spread=spread))


@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1e6, 1e25])
def test_attention_queries_of_any_size(F, factor):
    """Tiny and huge queries against the softmax scale that undoes them: the same scores."""
    s = case(F, [5, 8], [400, 130], H=8, heads=2, seed=21)
    s["q"] = (s["q"].float() * factor).bfloat16()
    s["scale"] = s["scale"] / factor
    check(F, s)


def test_attention_queries_of_mixed_sizes(F):
    """Rows, heads and dims of a query of sizes up to 2^12 apart."""
    s = case(F, [8, 8], [400, 130], H=8, heads=2, seed=22)
    g = torch.Generator(device=DEV).manual_seed(1)
    s["q"] = (s["q"].float() * torch.exp2(torch.rand(s["q"].shape, device=DEV, generator=g) * -12)).bfloat16()
    check(F, s)


def test_attention_values_of_very_different_scales(F):
    """One key whose value is 2^30 times the others', and one group of zeros."""
    s = case(F, [4, 4], [300, 40], H=4, heads=1, seed=23)
    t = s["tables"].cpu()
    x = torch.randn(1, 1, 128, device=DEV).bfloat16()
    slot = lambda r, p: torch.tensor([int(t[r, p // 256]) * 256 + p % 256], dtype=torch.int32, device=DEV)  # noqa: E731
    c = s["c"]
    F.store_kvcache_fp8(x, x * 2.0 ** 30, c.k_cache, c.v_cache, c.k_scale, c.v_scale, slot(0, 100))
    z = torch.zeros(16, 1, 128, device=DEV).bfloat16()
    F.store_kvcache_fp8(z, z, c.k_cache, c.v_cache, c.k_scale, c.v_scale,
                        torch.cat([slot(1, p) for p in range(16, 32)]))
    check(F, s)


def test_attention_rows_that_see_nothing(F):
    """No context, and fewer keys than queries (causal): zeros; empty rows and rows behind the last one stay as they were."""
    s = case(F, [3, 2, 0, 8], [0, 1, 5, 4], seed=24)
    out = torch.full((15, 32, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    s["q"] = torch.cat([s["q"], s["q"][:2]])
    attend(F, s, out=out)
    assert device_error() == 0
    want, spread = oracle(s)
    agree(out[:13], want[:13], spread[:13])
    assert (out[:4] == 0).all() and (out[5:9] == 0).all() and (out[13:] == 7).all()
    everything = case(F, [4] * 3, [0, 0, 0], seed=25)
    assert (attend(F, everything, decode=True, causal=False) == 0).all() and device_error() == 0


def test_attention_strided_rows(F):
    """q and out with padded rows, views of larger tensors."""
    s = case(F, [8, 5], [600, 257], seed=26)
    want = attend(F, s)
    wide = torch.zeros(13, 40, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 4:36] = s["q"]
    out = torch.full((13, 48, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    attend(F, dict(s, q=wide[:, 4:36]), out=out[:, 8:40])
    assert torch.equal(out[:, 8:40], want) and (out[:, :8] == 3).all() and (out[:, 40:] == 3).all()


def test_one_row_of_any_stride(F):
    """The row stride of a single row (a slice of wider rows) says nothing: q, out, keys and values of an odd one; and a dense q
    at an address that is no multiple of 16 bytes is copied."""
    s = case(F, [1], [300], seed=40)
    want = attend(F, s)
    wide = torch.zeros(2, 32 * 128 + 4, dtype=torch.bfloat16, device=DEV)
    wide[:1, :4096] = s["q"].view(1, -1)
    q = wide.as_strided((1, 32, 128), (wide.stride(0), 128, 1))
    out = torch.zeros(8200, dtype=torch.bfloat16, device=DEV).as_strided((1, 32, 128), (4100, 128, 1))
    attend(F, dict(s, q=q), out=out)
    assert torch.equal(out, want)
    wide.view(-1)[4:4100] = s["q"].view(-1)
    assert torch.equal(attend(F, dict(s, q=wide.view(-1)[4:4100].view(1, 32, 128))), want)
    c = random_cache(F, 1, 128, 2, 16, 4)
    key = torch.randn(1, 258, device=DEV).bfloat16().as_strided((1, 2, 128), (257, 128, 1))
    check_store(F, c, key, key, torch.tensor([3], device=DEV, dtype=torch.int32), 16)
    assert device_error() == 0


def test_attention_is_the_same_every_time(F):
    lens = np.random.default_rng(5).integers(500, 3000, size=24).tolist()
    s = case(F, [8] * 24, lens, seed=31)
    first = check(F, s)
    for _ in range(3):
        assert torch.equal(attend(F, s), first)
    few = attend(F, s, max_ctas=3)
    assert device_error() == 0
    agree(few, *oracle(s))


def test_attention_in_graphs_and_on_another_stream(F):
    """A captured call replays with new queries, lengths and cache contents; two graphs share the workspace in turn."""
    s, t = case(F, [8] * 6, [900, 30, 260, 128, 2000, 511], seed=32), case(F, [4] * 3, [77, 1500, 256], seed=33)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [], []
    with torch.cuda.stream(side):
        for x in (s, t):
            attend(F, x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(attend(F, x))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(2):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, out in zip((s, t), outs):
            agree(out, *oracle(x))
            x["q"].mul_(-0.5)
        s["k_lens"] = [800, 31, 8, 127, 1999, 512]
        s["cu_k"].copy_(torch.tensor([0] + np.cumsum(s["k_lens"]).tolist(), dtype=torch.int32))
        # row 1 grows into slots that no store wrote: write them
        c = s["c"]
        x = torch.randn(1, 8, 128, device=DEV).bfloat16()
        for r, p in ((1, 30), (5, 511)):
            slot = s["tables"][r, p // 256] * 256 + p % 256
            F.store_kvcache_fp8(x, x, c.k_cache, c.v_cache, c.k_scale, c.v_scale, slot.view(1))
    assert device_error() == 0


@pytest.mark.parametrize("cache", ["e4m3", "bf16"])
def test_early_launch_only_on_metadata_given_as_int32(F, cache, monkeypatch):
    """An early launch reads the row metadata before the kernel in front of it has ended, so it must not follow a conversion
    of them: int64 (or strided) metadata launch in order.  The flags are those that reach the library."""
    from nanovllm_b200 import _lib, attention
    flags = []
    real = _lib.lib()

    class Recorder:
        def __getattr__(self, name):
            fn = getattr(real, name)
            if name not in ("specdec_paged_attention_fp8", "specdec_paged_attention_ex"):
                return fn
            return lambda *args: (flags.append(args[-2] & attention.EARLY_LAUNCH), fn(*args))[1]

    s = case(F, [3, 3], [300, 40], seed=41)
    k = torch.randn(s["c"].k_cache.shape[0], 256, 8, 128, device=DEV).bfloat16()

    def go(tables, **where):
        if cache == "e4m3":
            c = s["c"]
            return F.paged_attention_fp8(s["q"], c.k_cache, c.v_cache, c.k_scale, c.v_scale, tables, s["scale"],
                                         early_launch=True, **where)
        return attention.paged_attention(s["q"], k, k, tables, s["scale"], early_launch=True, **where)

    varlen = dict(cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"], max_seqlen_q=3)
    decode = dict(context_lens=s["ctx"], query_len_per_seq=3)
    wide = torch.stack([s["ctx"], s["ctx"]], dim=1)[:, 0]
    monkeypatch.setattr(_lib, "lib", lambda: Recorder())
    want = go(s["tables"], **varlen)
    outs = [go(s["tables"], **decode), go(s["tables"].long(), **varlen), go(s["tables"], **{**varlen, "cu_seqlens_q": s["cu_q"].long()}),
            go(s["tables"], **{**varlen, "cu_seqlens_k": s["cu_k"].long()}), go(s["tables"], **{**decode, "context_lens": wide}),
            go(s["tables"], **varlen, context_lens=wide)]
    monkeypatch.undo()
    assert flags == [1, 1, 0, 0, 0, 0, 1]
    assert all(torch.equal(o, want) for o in outs) and device_error() == 0


def test_attention_module_stores_then_attends(F):
    from nanovllm_b200.context import reset_context, set_context
    s = case(F, [8, 5], [600, 257], seed=34)
    layer = F.AttentionFP8(32, 128, s["scale"], 8)
    layer.cache = s["c"]
    t = s["tables"].cpu()
    slots = [int(t[r, p // 256]) * 256 + p % 256 for r, (n, L) in enumerate([(8, 600), (5, 257)]) for p in range(L - n, L)]
    k, v = rows(13, 8, 35)
    set_context(True, s["cu_q"], s["cu_k"], 8, 4096, torch.tensor(slots, dtype=torch.int32, device=DEV), None, s["tables"])
    want = host(s["c"])
    out = layer(s["q"].view(-1, 32 * 128), k, v)
    reset_context()
    for side, x in ((0, k), (1, v)):
        O.store(x.double().cpu().numpy(), want[side], want[2 + side], slots, 16)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(host(s["c"]), want))
    agree(out, *oracle(s))


def test_attention_reports_bad_rows_and_pages(F):
    from nanovllm_b200 import attention
    s = case(F, [8, 8], [100, 300], seed=36)
    s["cu_k"].copy_(torch.tensor([0, 100, 100 + 513], dtype=torch.int32))      # past the table: row 1 is not read
    out = attend(F, s, out=torch.full((16, 32, 128), 5.0, dtype=torch.bfloat16, device=DEV))
    assert device_error() == 2 and (out[8:] == 5).all()
    attention.reset_device_error(DEV)
    for bad in (s["c"].k_cache.shape[0], -1, 2 ** 30):
        b = case(F, [8, 8], [100, 300], seed=37, stale_nan=False)
        b["tables"][1, 1] = bad
        attend(F, b)
        assert device_error() == 5
        attention.reset_device_error(DEV)


def test_refusals(F):
    from nanovllm_b200._lib import SpecdecError
    s = case(F, [8], [100], seed=38)
    c = s["c"]
    with pytest.raises(SpecdecError, match="packed columns"):
        F.paged_attention_fp8(s["q"], c.k_cache, c.v_cache, c.k_scale, c.v_scale, s["tables"], 1.0, cu_seqlens_q=s["cu_q"],
                              cu_seqlens_k=s["cu_k"], max_seqlen_q=9)
    with pytest.raises(SpecdecError, match="group 3"):
        F.paged_attention_fp8(s["q"][:, :24].contiguous(), c.k_cache, c.v_cache, c.k_scale, c.v_scale, s["tables"], 1.0,
                              cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"], max_seqlen_q=1)
    d = F.FP8Cache.allocate(1, 64, 8, DEV)
    with pytest.raises(SpecdecError, match="multiple of 128"):
        F.paged_attention_fp8(s["q"], d.k_cache, d.v_cache, d.k_scale, d.v_scale, s["tables"], 1.0, context_lens=s["ctx"],
                              query_len_per_seq=8)
    assert device_error() == 0
