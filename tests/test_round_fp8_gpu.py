"""A verification round over the 8-bit cache, end to end: the metadata built on the GPU, the target's forward with the
8-bit store and attention, the acceptance, and the log probabilities of what was emitted.

The 8-bit values (4 significant bits times a power of two) are exact in bf16, so the bf16 target over the dequantised
cache computes the same function: its logits differ by the two attentions' roundings alone, held to the 1e-2 relative
Frobenius error that the forward's other tests allow."""
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from oracle import spec_sampler as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BS, K = 256, 7


def build(varlen):
    from nanovllm_b200.device_metadata import DeviceRows
    from nanovllm_b200.speculative import VerifyRound
    from nanovllm_b200.target import Qwen3Shape, Qwen3Target
    shape = Qwen3Shape(hidden=256, layers=2, heads=4, kv_heads=2, intermediate=512, vocab=1000, max_position=4096,
                       aux_layer_ids=(0, 1))
    lengths = [300, 17, 513, 256, 1]
    total = sum(math.ceil((n + 30) / BS) for n in lengths) + 3
    target = Qwen3Target(shape, DEV, total, BS, seed=5, init_scale=0.05, kv_dtype=torch.float8_e4m3fn)
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(0)).to(torch.int32)
    held = [math.ceil((n - 1) / BS) for n in lengths]
    W = 4
    tables = torch.zeros(len(lengths), W, dtype=torch.int32)
    used = 0
    for r, h in enumerate(held):
        tables[r, :h] = perm[used:used + h]
        used += h
    g = torch.Generator(device=DEV).manual_seed(2)
    from nanovllm_b200.attention_fp8 import store_kvcache_fp8
    for c in target.kv_fp8:                      # the context: every token before the last one
        for r, n in enumerate(lengths):
            pos = torch.arange(n - 1)
            slots = (tables[r, pos // BS] * BS + pos % BS).to(torch.int32).to(DEV)
            x = torch.randn(2, n - 1, shape.kv_heads, 128, device=DEV, generator=g).bfloat16()
            store_kvcache_fp8(x[0], x[1], c.k_cache, c.v_cache, c.k_scale, c.v_scale, slots)
    free = torch.cat([perm[used:], torch.zeros(used, dtype=torch.int32)]).to(DEV)
    rows = DeviceRows(torch.tensor(lengths, device=DEV), torch.tensor([n % 997 for n in lengths], device=DEV), tables.to(DEV),
                      torch.tensor(held, dtype=torch.int32, device=DEV), free,
                      torch.tensor([total - used], dtype=torch.int32, device=DEV))
    counts = dict(token_counts=[8, 16, 24, 32, 40], max_rows=16) if varlen else {}
    rnd = VerifyRound(target, K, () if varlen else [len(lengths)], W, **counts)
    return SimpleNamespace(shape=shape, target=target, rnd=rnd, rows=rows, lengths=lengths)


def host_rows(rows):
    from nanovllm_b200.batch_metadata import RowState
    held = rows.num_blocks.tolist()
    return [RowState(n, t, table[:h]) for n, t, table, h in zip(rows.lengths.tolist(), rows.last_tokens.tolist(),
                                                               rows.block_tables.tolist(), held)]


def bf16_logits(c, num_tokens):
    """The bf16 target's logits over the dequantised caches, storing nothing."""
    from nanovllm_b200.target import Qwen3Target
    b = c.target.graphs[num_tokens][1]
    plain = Qwen3Target(c.shape, DEV, c.target.num_blocks, BS, seed=5, init_scale=0.05)
    for layer, cache in enumerate(c.target.kv_fp8):
        for side, x in enumerate(cache.dequantised()):
            y = x.nan_to_num(0.0).bfloat16()
            assert torch.equal(y.float(), x.nan_to_num(0.0))          # exact
            plain.kv_cache[side, layer].copy_(y)
    hidden = plain.forward(b["input_ids"], b["positions"], torch.full_like(b["slot_mapping"], -1), b["cu_seqlens_q"],
                           b["cu_seqlens_k"], K + 1, b["block_tables"])
    return plain.compute_logits(hidden)


@pytest.mark.parametrize("varlen", [False, True])
def test_rounds_on_the_device(varlen):
    from nanovllm_b200 import attention, device_metadata, logprobs
    from nanovllm_b200 import spec_sampler as S
    attention.reset_device_error(DEV)
    c = build(varlen)
    R = len(c.lengths)
    samp = S.sampling_tensors([SimpleNamespace(temperature=1.0, top_k=0, top_p=1.0)] * R, DEV)
    gen = torch.Generator(device=DEV).manual_seed(7)
    for step in range(3):
        q = torch.softmax(torch.randn(R, K, c.shape.vocab, device=DEV, generator=gen) * 0.3, -1)
        drafts = S.sample(q, gen)
        lens = [K + 1] * R if not varlen else [1 + (3 * r + step) % (K + 1) for r in range(R)]
        device_lens = torch.tensor(lens, device=DEV) if varlen else None
        replay = torch.Generator(device=DEV)
        replay.set_state(gen.get_state())
        before = (c.rows.lengths.clone(), c.rows.last_tokens.clone())
        n_accept, tail, got = c.rnd.run_round_device(c.rows, drafts, q, samp, gen, device_lens, sum(lens) if varlen else None,
                                                     num_top=3)
        torch.cuda.synchronize()
        assert attention.device_error(DEV) == 0 and device_metadata.device_error(DEV) == 0 and logprobs.device_error(DEV) == 0
        num_tokens = c.rnd.graph_for(R, sum(lens))
        logits = c.rnd.logits(num_tokens)
        # the metadata: what the host packs for the same rows
        b = c.target.graphs[num_tokens][1]
        packed = (b["_packed64"].clone(), b["_packed32"].clone())
        want_logits = bf16_logits(c, num_tokens)[:sum(lens)].float()
        assert (logits.float() - want_logits).norm() <= 1e-2 * want_logits.norm()
        after = (c.rows.lengths.clone(), c.rows.last_tokens.clone())
        c.rows.lengths.copy_(before[0])
        c.rows.last_tokens.copy_(before[1])
        kept = logits.clone()
        assert c.rnd.load(host_rows(c.rows), lens if varlen else None) == num_tokens
        c.rnd.place_drafts(num_tokens, drafts)
        assert torch.equal(packed[0], b["_packed64"]) and torch.equal(packed[1], b["_packed32"])
        c.rows.lengths.copy_(after[0])
        c.rows.last_tokens.copy_(after[1])
        # the acceptance: the oracle's on these logits with the generator's draws
        u = torch.rand(R, K, device=DEV, generator=replay).cpu().numpy()
        noise = S.exponential_noise_(torch.empty(R, c.shape.vocab, device=DEV), replay).cpu().numpy()
        p = O.probs_from_logits(kept.float().cpu().numpy(), np.ones(sum(lens), np.float32))
        args = (q.cpu().numpy(), drafts.cpu().numpy(), np.array(lens), u, noise)
        want_n, want_tail = O.accept_random_varlen(p, *args)
        fine = ~O.near_tie_flags(p, *args)
        assert np.array_equal(n_accept.cpu().numpy()[fine], want_n[fine])
        assert np.array_equal(tail.cpu().numpy()[fine], want_tail[fine])
        # the requests have advanced, and the log probabilities are those of what they emitted
        assert torch.equal(after[0], before[0] + n_accept + 1) and torch.equal(after[1], tail)
        tokens = []
        for r in range(R):
            out = drafts[r, :int(n_accept[r])].tolist() + [int(tail[r])]
            tokens += out + [-1] * (lens[r] - len(out))
        want = OL.token_logprobs(kept.double().cpu().numpy(), tokens, 3)
        np.testing.assert_allclose(got.logprobs.cpu().numpy(), want[0], rtol=2.0 ** -21, atol=4e-6)
        np.testing.assert_allclose(got.entropy.cpu().numpy(), want[1], rtol=2.0 ** -21, atol=4e-6)
        assert np.array_equal(got.top_ids.cpu().numpy(), want[2])


@pytest.mark.parametrize("varlen", [False, True])
def test_host_and_device_rounds_agree(varlen):
    """The same requests through run_round (host metadata, one copy back) and run_round_device: the same tokens, and the
    same bytes in the caches, over rounds that cross block borders."""
    from nanovllm_b200 import spec_sampler as S
    host, dev = build(varlen), build(varlen)
    R = len(host.lengths)
    samp = S.sampling_tensors([SimpleNamespace(temperature=0.7, top_k=40, top_p=0.9)] * R, DEV)
    gens = [torch.Generator(device=DEV).manual_seed(3) for _ in range(2)]
    make = torch.Generator(device=DEV).manual_seed(4)
    for step in range(3):
        q = torch.softmax(torch.randn(R, K, host.shape.vocab, device=DEV, generator=make) * 0.3, -1)
        drafts = S.sample(q, make)
        lens = [1 + (5 * r + step) % (K + 1) for r in range(R)] if varlen else None
        # the host side's blocks: those the device takes from its stack, in its order
        have = host.rows.num_blocks.tolist()
        free = int(host.rows.free_count)
        for r, n in enumerate(host.rows.lengths.tolist()):
            need = math.ceil((n - 1 + (lens[r] if varlen else K + 1)) / BS)
            while have[r] < need:
                free -= 1
                host.rows.block_tables[r, have[r]] = host.rows.free_blocks[free]
                have[r] += 1
        host.rows.num_blocks.copy_(torch.tensor(have, dtype=torch.int32))
        host.rows.free_count.fill_(free)
        appended = host.rnd.run_round(host_rows(host.rows), drafts, q, samp, gens[0], lens)
        n_accept, tail, none = dev.rnd.run_round_device(dev.rows, drafts, q, samp, gens[1],
                                                        torch.tensor(lens, device=DEV) if varlen else None,
                                                        sum(lens) if varlen else None)
        assert none is None
        assert appended == [drafts[r, :a].tolist() + [t] for r, (a, t) in enumerate(zip(n_accept.tolist(), tail.tolist()))]
        host.rows.lengths.add_(torch.tensor([len(x) for x in appended], device=DEV))
        host.rows.last_tokens.copy_(torch.tensor([x[-1] for x in appended], device=DEV))
        for name in ("lengths", "last_tokens", "block_tables", "num_blocks", "free_count"):
            assert torch.equal(getattr(host.rows, name), getattr(dev.rows, name)), name
        for a, b in zip(host.target.kv_fp8, dev.target.kv_fp8):
            assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
            assert torch.equal(a.k_cache.view(torch.uint8), b.k_cache.view(torch.uint8))
            assert torch.equal(a.v_cache.view(torch.uint8), b.v_cache.view(torch.uint8))


def test_a_round_without_blocks_leaves_the_rows():
    from nanovllm_b200 import device_metadata, logprobs
    from nanovllm_b200 import spec_sampler as S
    c = build(True)
    device_metadata.reset_device_error(DEV)
    R = len(c.lengths)
    c.rows.lengths[3] = 510                               # one block held, 510 + 7 tokens need a third
    c.rows.free_count.zero_()
    rows = [t.clone() for t in (c.rows.lengths, c.rows.last_tokens, c.rows.block_tables, c.rows.num_blocks)]
    caches = [(l.k_cache.clone(), l.v_cache.clone()) for l in c.target.kv_fp8]
    drafts = torch.randint(c.shape.vocab, (R, K), device=DEV)
    samp = S.sampling_tensors([SimpleNamespace(temperature=0.0, top_k=0, top_p=1.0)] * R, DEV)
    lens = torch.full((R,), K + 1, device=DEV)
    try:
        c.rnd.run_round_device(c.rows, drafts, None, samp, None, lens, R * (K + 1), num_top=1)
        assert device_metadata.device_error(DEV) == 6
        after = (c.rows.lengths, c.rows.last_tokens, c.rows.block_tables, c.rows.num_blocks)
        assert all(torch.equal(x, y) for x, y in zip(rows, after))
        for (k, v), l in zip(caches, c.target.kv_fp8):
            assert torch.equal(k.view(torch.uint8), l.k_cache.view(torch.uint8))
            assert torch.equal(v.view(torch.uint8), l.v_cache.view(torch.uint8))
    finally:
        device_metadata.reset_device_error(DEV)
    # lengths of another sum than num_verified: more than the graph holds, and fewer (the rest is padding, but the
    # acceptance refuses them: the blocks are assigned, the rows stay)
    c.rows.free_count.fill_(3)
    try:
        c.rnd.run_round_device(c.rows, drafts, None, samp, None, lens, 3 * (K + 1), num_top=1)
        assert device_metadata.device_error(DEV) == 7
        assert all(torch.equal(x, y) for x, y in zip(rows, after))
        device_metadata.reset_device_error(DEV)
        # 6 tokens a row need 1 block for row 2, 2 for row 3 and 1 for row 4: 3 free ones are one short
        c.rnd.run_round_device(c.rows, drafts, None, samp, None, lens - 2, R * (K + 1), num_top=1)
        assert device_metadata.device_error(DEV) == 6
        assert all(torch.equal(x, y) for x, y in zip(rows, after))
        device_metadata.reset_device_error(DEV)
        c.rows.free_count.fill_(4)
        c.rnd.run_round_device(c.rows, drafts, None, samp, None, lens - 2, R * (K + 1), num_top=1)
        assert device_metadata.device_error(DEV) == 0 and int(c.rows.free_count) == 0 and int(S.status_word(DEV)) == 1
        assert all(torch.equal(x, y) for x, y in zip(rows[:2], after[:2]))
    finally:
        device_metadata.reset_device_error(DEV)
        logprobs.reset_device_error(DEV)


@pytest.mark.parametrize("where", ["table", "stack"])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 10 ** 6, 2 ** 30, 2 ** 24, "pad"])
def test_bad_block_ids_hold_the_rows(where, bad):
    """An id that the target's cache does not have, in a row's table or on the stack: error 9, nothing stored, no row
    moved."""
    from nanovllm_b200 import attention, device_metadata
    from nanovllm_b200 import spec_sampler as S
    c = build(False)
    R = len(c.lengths)
    samp = S.sampling_tensors([SimpleNamespace(temperature=0.0, top_k=0, top_p=1.0)] * R, DEV)
    drafts = torch.randint(c.shape.vocab, (R, K), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    bad = c.target.pad_block_id if bad == "pad" else bad
    if where == "table":
        c.rows.block_tables[2, 0] = bad
    else:
        c.rows.free_blocks[int(c.rows.free_count) - 1] = bad
    before = [t.clone() for t in (c.rows.lengths, c.rows.last_tokens, c.rows.num_blocks, c.rows.free_count)]
    caches = [(l.k_cache.view(torch.uint8).clone(), l.v_cache.view(torch.uint8).clone()) for l in c.target.kv_fp8]
    try:
        c.rnd.run_round_device(c.rows, drafts, None, samp)
        assert device_metadata.device_error(DEV) == 9 and attention.device_error(DEV) == 0
        after = (c.rows.lengths, c.rows.last_tokens, c.rows.num_blocks, c.rows.free_count)
        assert all(torch.equal(x, y) for x, y in zip(before, after))
        for (k, v), l in zip(caches, c.target.kv_fp8):
            assert torch.equal(k, l.k_cache.view(torch.uint8)) and torch.equal(v, l.v_cache.view(torch.uint8))
    finally:
        device_metadata.reset_device_error(DEV)
        attention.reset_device_error(DEV)


@pytest.mark.parametrize("module", ["attention", "fused"])
def test_errors_of_the_forward_hold_the_rows(module):
    """With an error word of the forward's kernels set, a round moves no row; after the reset it does."""
    import importlib
    from nanovllm_b200 import spec_sampler as S
    m = importlib.import_module(f"nanovllm_b200.{module}")
    assert m.device_error(DEV) == 0
    c = build(False)
    R = len(c.lengths)
    samp = S.sampling_tensors([SimpleNamespace(temperature=0.0, top_k=0, top_p=1.0)] * R, DEV)
    drafts = torch.randint(c.shape.vocab, (R, K), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    before = (c.rows.lengths.clone(), c.rows.last_tokens.clone())
    try:
        (m.error_word(DEV) if module == "attention" else m.err_word(DEV)).fill_(4)
        c.rnd.run_round_device(c.rows, drafts, None, samp)
        assert torch.equal(c.rows.lengths, before[0]) and torch.equal(c.rows.last_tokens, before[1])
    finally:
        m.reset_device_error(DEV)
    n_accept, tail, _ = c.rnd.run_round_device(c.rows, drafts, None, samp)
    assert torch.equal(c.rows.lengths, before[0] + n_accept + 1) and torch.equal(c.rows.last_tokens, tail)


def poison(value=1e30):
    """Freed memory that torch.empty hands out next holds large values, small and large blocks alike."""
    junk = [torch.full((n,), value, dtype=torch.bfloat16, device=DEV) for n in [2048] * 500 + [1 << 22] * 4]
    torch.cuda.synchronize()
    del junk


def test_tokens_past_the_last_position_store_nothing():
    """Rows 259 to 266 of a target whose rotary table ends at 264: the caches' bytes are those of a forward that gives the last
    three tokens no slot, group mates of theirs included (memory that the forward finds holds 1e30)."""
    from nanovllm_b200 import fused
    from nanovllm_b200.attention_fp8 import store_kvcache_fp8
    from nanovllm_b200.target import Qwen3Shape, Qwen3Target
    shape = Qwen3Shape(hidden=256, layers=2, heads=4, kv_heads=2, intermediate=512, vocab=1000, max_position=264)
    tables = torch.tensor([[1, 2]], dtype=torch.int32, device=DEV)
    ids = torch.arange(8, device=DEV)
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (8, 267))
    at = torch.arange(259, 267, device=DEV)
    slots = (tables[0, at // BS] * BS + at % BS).to(torch.int32)
    caches = []
    for given in (True, False):
        target = Qwen3Target(shape, DEV, 3, BS, seed=5, init_scale=0.05, kv_dtype=torch.float8_e4m3fn)
        g = torch.Generator(device=DEV).manual_seed(2)
        for c in target.kv_fp8:
            pos = torch.arange(259, device=DEV)
            x = torch.randn(2, 259, 2, 128, device=DEV, generator=g).bfloat16()
            store_kvcache_fp8(x[0], x[1], c.k_cache, c.v_cache, c.k_scale, c.v_scale,
                              (tables[0, pos // BS] * BS + pos % BS).to(torch.int32))
        poison()
        inside = at < 264
        target.forward(ids, at if given else torch.where(inside, at, 0),
                       slots if given else torch.where(inside, slots, -1).to(torch.int32), cu_q, cu_k, 8, tables)
        torch.cuda.synchronize()
        caches.append([t.clone() for c in target.kv_fp8 for t in (c.k_cache.view(torch.uint8), c.v_cache.view(torch.uint8),
                                                                  c.k_scale, c.v_scale)])
    code = fused.device_error(DEV)
    fused.reset_device_error(DEV)
    assert code == 4
    assert all(torch.equal(a, b) for a, b in zip(*caches))


def test_a_row_past_the_last_position_holds_the_rows():
    """A row whose drafts cross the rotary table's end (its tokens there are neither rotated nor stored): error 4."""
    from nanovllm_b200 import attention, device_metadata, fused
    from nanovllm_b200 import spec_sampler as S
    c = build(False)
    R = len(c.lengths)
    samp = S.sampling_tensors([SimpleNamespace(temperature=0.0, top_k=0, top_p=1.0)] * R, DEV)
    drafts = torch.randint(c.shape.vocab, (R, K), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    end = 513 + 3                             # row 2 verifies positions 512 to 519
    c.target.cos_sin = c.target.cos_sin[:end]
    c.target.graphs.clear()
    c.target.graph_pool = None
    from nanovllm_b200.speculative import VerifyRound
    rnd = VerifyRound(c.target, K, [R], 4)
    assert fused.device_error(DEV) == 0
    before = (c.rows.lengths.clone(), c.rows.last_tokens.clone())
    try:
        rnd.run_round_device(c.rows, drafts, None, samp)
        assert fused.device_error(DEV) == 4
        assert device_metadata.device_error(DEV) == 0 and attention.device_error(DEV) == 0
        assert torch.equal(c.rows.lengths, before[0]) and torch.equal(c.rows.last_tokens, before[1])
    finally:
        fused.reset_device_error(DEV)


def test_greedy_rounds_of_a_padded_batch():
    """Fewer rows than the graph has, all greedy: the emitted tokens follow the argmax of the round's own logits."""
    from nanovllm_b200 import device_metadata
    from nanovllm_b200 import spec_sampler as S
    c = build(True)
    R = len(c.lengths)
    samp = S.sampling_tensors([SimpleNamespace(temperature=0.0, top_k=0, top_p=1.0)] * R, DEV)
    drafts = torch.randint(c.shape.vocab, (R, K), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    lens = [1, 8, 3, 2, 5]
    before = c.rows.lengths.clone()
    n_accept, tail, got = c.rnd.run_round_device(c.rows, drafts, None, samp, None, torch.tensor(lens, device=DEV), sum(lens),
                                                 num_top=0)
    assert device_metadata.device_error(DEV) == 0
    logits = c.rnd.logits(c.rnd.graph_for(R, sum(lens))).float()
    at = 0
    for r, n in enumerate(lens):
        best = logits[at:at + n].argmax(-1).tolist()
        a = 0
        while a < n - 1 and best[a] == int(drafts[r, a]):
            a += 1
        assert (int(n_accept[r]), int(tail[r])) == (a, best[a])
        p = torch.log_softmax(logits[at + a].double(), -1)[best[a]]
        assert abs(float(got.logprobs[at + a]) - float(p)) <= 4e-6 + 2.0 ** -21 * abs(float(p))
        assert got.logprobs[at + a + 1:at + n].tolist() == [0.0] * (n - a - 1)
        at += n
    assert torch.equal(c.rows.lengths, before + n_accept + 1)


def test_refused_cache_types():
    from nanovllm_b200.target import Qwen3Shape, Qwen3Target
    shape = Qwen3Shape(hidden=256, layers=1, heads=4, kv_heads=2, intermediate=256, vocab=100, max_position=64)
    with pytest.raises(ValueError, match="kv_dtype"):
        Qwen3Target(shape, DEV, 1, kv_dtype=torch.float16)
