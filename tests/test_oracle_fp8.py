"""The 64-bit oracles of the 8-bit cache and of the log probabilities against torch on the CPU."""
import numpy as np
import pytest
import torch

from oracle import fp8_cache as O
from oracle import logprobs as OL


def test_round_e4m3_matches_torch():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.round_e4m3(every), every, equal_nan=True)
    finite = np.unique(every[np.isfinite(every)])
    middle = (finite[1:] + finite[:-1]) / 2                      # every tie
    x = np.concatenate([middle, np.nextafter(middle, 1e9), np.nextafter(middle, -1e9),
                        np.random.default_rng(0).normal(size=4000) * 100]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.round_e4m3(x), want)
    assert O.round_e4m3([1e9, -np.inf, 449.0]).tolist() == [448.0, -448.0, 448.0]


@pytest.mark.parametrize("amax,scale", [(0.0, 2.0 ** -100), (448.0, 1.0), (448.5, 2.0), (224.0, 0.5), (1e-38, 2.0 ** -100),
                                        (1.0, 2.0 ** -8), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7), (3.3895e38, 2.0 ** 120)])
def test_scale_is_the_smallest_power_of_two(amax, scale):
    assert O.scale_for(amax) == scale


def test_store_starts_and_grows_groups():
    codes, scales = np.zeros((1, 1, 32, 2)), np.ones((1, 1, 2))
    O.store(np.full((3, 1, 2), 100.0), codes, scales, [0, 1, 2], 16)
    assert scales[0, 0].tolist() == [0.25, 1.0] and codes[0, 0, :4, 0].tolist() == [384.0, 384.0, 384.0, 0.0]
    O.store(np.full((1, 1, 2), 1000.0), codes, scales, [3], 16)       # raised: 100 is 96 of 4 * 25 -> 24 * 4
    assert scales[0, 0, 0] == 4.0 and codes[0, 0, :4, 0].tolist() == [24.0, 24.0, 24.0, 256.0]
    O.store(np.full((1, 1, 2), 1.0), codes, scales, [2], 16)          # never falls
    assert scales[0, 0, 0] == 4.0 and codes[0, 0, 2, 0] == 0.25
    O.store(np.full((1, 1, 2), 1.0), codes, scales, [0], 16)          # started again: the others stand for nothing
    assert scales[0, 0, 0] == 2.0 ** -8 and codes[0, 0, 0, 0] == 256.0 and codes[0, 0, 3, 0] == 256.0


def test_attention_matches_torch():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(3, 2, 128, 16, generator=g).double(), torch.randn(3, 2, 128, 16, generator=g).double()
    ks, vs = torch.rand(3, 2, 8, generator=g).double(), torch.rand(3, 2, 8, generator=g).double()
    q = torch.randn(3, 4, 16, generator=g).double()
    o, spread = O.paged_attention(q.numpy(), k.numpy(), v.numpy(), ks.numpy(), vs.numpy(), np.array([[2, 0]]), [0], [3],
                                  [200], 0.25)
    full = [(x * s.repeat_interleave(16, 2)[..., None])[[2, 0]].transpose(0, 1).reshape(2, 256, 16)[:, :200]
            for x, s in ((k, ks), (v, vs))]
    mask = torch.arange(200)[None, :] <= 197 + torch.arange(3)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1), full[0].repeat_interleave(2, 0), full[1].repeat_interleave(2, 0), attn_mask=mask, scale=0.25)
    np.testing.assert_allclose(o, want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-12)
    assert (spread > 0).all()
    none, _ = O.paged_attention(q.numpy(), k.numpy(), v.numpy(), ks.numpy(), vs.numpy(), np.array([[2, 0]]), [0], [3], [1],
                                0.25)
    assert np.all(none[:2] == 0) and np.any(none[2] != 0)


def test_logprobs_match_torch():
    x = torch.randn(4, 50, generator=torch.Generator().manual_seed(1)).double()
    x[1, 3] = float("-inf")
    x[2, 7] = x[2, 30] = 9.0
    x[3, 5] = float("nan")
    lp, entropy, ids, top = OL.token_logprobs(x.numpy(), [3, 3, 30, 0], 5, [1.0, 2.0, 0.5, 1.0])
    want = torch.log_softmax(x / torch.tensor([1.0, 2.0, 0.5, 1.0]).double()[:, None], dim=-1)
    assert lp[1] == -np.inf and np.isnan(lp[3]) and np.isnan(entropy[3])
    np.testing.assert_allclose(lp[[0, 2]], want[[0, 2], [3, 30]].numpy(), rtol=1e-12)
    p = want.exp()
    plain = -(p * torch.where(p > 0, want, 0.0)).sum(-1)
    np.testing.assert_allclose(entropy[:3], plain[:3].numpy(), rtol=1e-12)
    assert ids[2, :2].tolist() == [7, 30] and ids[3, 0] == 5
    np.testing.assert_allclose(top[:3], want[:3].gather(1, torch.from_numpy(ids[:3])).numpy(), rtol=1e-12)
