"""token_logprobs against the 64-bit oracle.

Tolerances: with d = (logit - max) / temperature, fp32 keeps d to 2^-23 of itself (a subtraction and a quotient or a
product: two roundings of 2^-24) and the exponential is good to 2^-21 of its value plus d's own error; a sum of V positive
terms in any order inside a row of partial sums of at most 2^12 steps is good to 2^-12, held here far below by the partial
sums' number, so log S is bounded by 2^-20 relative of S plus |d| terms: an absolute 4e-6 + 2^-21 |log p| covers it."""
import numpy as np
import pytest
import torch

from oracle import logprobs as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def P():
    from nanovllm_b200 import logprobs
    logprobs.reset_device_error(DEV)
    return logprobs


def logits_of(T, V, dtype, seed, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(T, V, device=DEV, generator=g) * scale).to(TYPES[dtype])


def check(P, logits, tokens, num_top, temps=None, error=0):
    got = P.token_logprobs(logits, tokens, num_top, temps)
    assert P.device_error(DEV) == error
    want = O.token_logprobs(logits.double().cpu().numpy(), tokens.cpu().numpy(), num_top,
                            None if temps is None else temps.double().cpu().numpy())
    lp, entropy, ids, top = (t.cpu().numpy() for t in (got.logprobs, got.entropy, got.top_ids, got.top_logprobs))
    assert np.array_equal(ids, want[2])
    for a, b in ((lp, want[0]), (entropy, want[1]), (top, want[3])):
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isinf(a), np.isinf(b))
        fine = np.isfinite(b)
        assert np.all(np.abs(a[fine] - b[fine]) <= 4e-6 + 2.0 ** -21 * np.abs(b[fine]))
    return got


def pick(T, V, seed, skip=0):
    tokens = torch.randint(V, (T,), generator=torch.Generator().manual_seed(seed))
    if skip:
        tokens[::skip] = -1
    return tokens.to(DEV)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 2, 0), (3, 7, 5), (5, 33, 32), (2, 1000, 8), (4, 4096, 20), (3, 4097, 32),
                                     (2, 50257, 5), (1, 151936, 20), (9, 32003, 1)])
def test_against_the_oracle(P, dtype, T, V, top):
    check(P, logits_of(T, V, dtype, V + top), pick(T, V, T), top)


@pytest.mark.parametrize("T,V", [(40, 5000), (300, 1500), (700, 260)])
def test_many_rows_some_skipped(P, T, V):
    temps = torch.rand(T, device=DEV) * 1.5 + 0.2
    check(P, logits_of(T, V, "bf16", T), pick(T, V, T, skip=7), 6, temps)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [64, 5000, 151936])
def test_ties_go_to_the_lowest_index(P, dtype, V):
    """All equal; two values; the largest only at the row's end; zeros of both signs."""
    x = torch.zeros(5, V, device=DEV, dtype=TYPES[dtype])
    x[1, ::3] = 1.0
    x[2, -20:] = 2.0
    x[3, 1::2] = -0.0
    x[4] = torch.arange(V, device=DEV).remainder(3).to(x.dtype)
    check(P, x, pick(5, V, 1), 32)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_infinities_and_nan(P, dtype):
    V = 3001
    x = logits_of(9, V, dtype, 2)
    inf, nan = float("inf"), float("nan")
    tokens = pick(9, V, 3)
    x[0, 5:] = -inf                     # a few tokens left
    x[1] = -inf                         # nothing left
    x[2, 17] = nan
    x[3, 2900] = inf
    x[4] = torch.finfo(x.dtype).min     # every logit the type's lowest
    x[5, 1:] = torch.finfo(x.dtype).min
    x[6, int(tokens[6])] = -inf         # the given token masked
    x[7] = nan
    x[8, 1:] = -inf                     # one token left
    tokens[8] = 0
    check(P, x, tokens, 8)


def test_a_token_past_the_vocabulary(P):
    x, tokens = logits_of(3, 500, "bf16", 4), torch.tensor([3, 500, 499], device=DEV)
    check(P, x, tokens, 3, error=8)
    P.reset_device_error(DEV)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 0), (3, 5), (8, 16)])
def test_strided_and_unaligned_rows(P, dtype, offset, pad):
    V = 2003
    wide = logits_of(6, offset + V + pad, dtype, 5)
    check(P, wide[:, offset:offset + V], pick(6, V, 6), 4)
    check(P, wide.t().contiguous().t()[:, :V], pick(6, V, 7), 4)          # columns apart: taken through a copy


def test_wide_range_and_temperatures(P):
    x = logits_of(8, 9000, "fp32", 8, scale=200.0)
    temps = torch.tensor([1e-3, 0.01, 0.5, 1.0, 2.0, 10.0, 1e3, 1e6], device=DEV)
    got = P.token_logprobs(x, pick(8, 9000, 9), 4, temps)
    want = O.token_logprobs(x.double().cpu().numpy(), pick(8, 9000, 9).cpu().numpy(), 4, temps.double().cpu().numpy())
    assert np.array_equal(got.top_ids.cpu().numpy(), want[2])
    # |log p| up to 1e6 here: the two roundings of d dominate
    assert np.allclose(got.logprobs.cpu().numpy(), want[0], rtol=2.0 ** -21, atol=4e-6)
    assert np.allclose(got.entropy.cpu().numpy(), want[1], rtol=2.0 ** -18, atol=4e-6)


def test_replays_in_a_graph(P):
    x, tokens = logits_of(10, 20000, "bf16", 10), pick(10, 20000, 11, skip=4)
    P.token_logprobs(x, tokens, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = P.token_logprobs(x, tokens, 5)
    for seed in range(3):
        x.copy_(logits_of(10, 20000, "bf16", 20 + seed))
        graph.replay()
        again = P.token_logprobs(x, tokens, 5)
        torch.cuda.synchronize()
        for a, b in zip((got.logprobs, got.entropy, got.top_ids, got.top_logprobs),
                        (again.logprobs, again.entropy, again.top_ids, again.top_logprobs)):
            assert torch.equal(a, b)


def test_no_rows_and_refusals(P):
    empty = P.token_logprobs(torch.empty(0, 50, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 3)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 3)
    x, tokens = logits_of(2, 40, "bf16", 12), pick(2, 40, 13)
    for bad in ((x.double(), tokens, 1, None), (x[0], tokens, 1, None), (x, tokens[:1], 1, None), (x, tokens.float(), 1, None),
                (x, tokens, 33, None), (x, tokens, -1, None), (x[:, :4], tokens, 5, None), (x, tokens.cpu(), 1, None),
                (x, tokens, 1, torch.ones(3, device=DEV))):
        with pytest.raises(ValueError):
            P.token_logprobs(*bad)


def test_a_workspace_first_used_in_a_capture(P):
    """A workspace that a captured call is the first to name is zero from then on, not from that graph's first replay: in
    memory of the graphs' pool that held other data, a second graph and an eager call give the same numbers before it."""
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(2, 150000, device=DEV, generator=g)
    tokens = torch.tensor([3, 5], device=DEV)
    want = P.token_logprobs(x, tokens, 4)
    pool = torch.cuda.graph_pool_handle()
    dirty = torch.cuda.CUDAGraph()
    with torch.cuda.graph(dirty, pool):
        junk = [torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device=DEV) for _ in range(8)]
    dirty.replay()
    torch.cuda.synchronize()
    del junk
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool):
            outs.append(P.token_logprobs(x, tokens, 4, workspace="logprobs_first_in_a_capture"))
        graphs.append(graph)
    eager = P.token_logprobs(x, tokens, 4, workspace="logprobs_first_in_a_capture")
    for n in (1, 0, 1):
        for t in (outs[n].logprobs, outs[n].entropy, outs[n].top_ids, outs[n].top_logprobs):
            t.fill_(7)
        graphs[n].replay()
        torch.cuda.synchronize()
        for got in (outs[n], eager):
            for a, b in ((got.logprobs, want.logprobs), (got.entropy, want.entropy), (got.top_ids, want.top_ids),
                         (got.top_logprobs, want.top_logprobs)):
                assert torch.equal(a, b)
