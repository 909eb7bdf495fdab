"""Arguments that the 8-bit cache, the device metadata and the log probabilities refuse before anything is launched: on the
host, through the Python checks (with tensors that pass for CUDA ones) and through the C ABI (addresses never read)."""
import pytest
import torch

FAKE = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from nanovllm_b200 import _lib
    return _lib.load()


def store_args(**kw):
    a = dict(key=FAKE, ks=1024, value=FAKE, vs=1024, kc=FAKE, vc=FAKE, ksc=FAKE, vsc=FAKE, slots=FAKE, N=8, heads=8, dim=128,
             blocks=4, bs=256, group=16, err=FAKE, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,message", [
    (dict(dim=64), b"head_dim"), (dict(group=8), b"scale_group"), (dict(group=64), b"scale_group"),
    (dict(bs=24), b"multiple"), (dict(key=None), b"null"), (dict(slots=None), b"null"), (dict(ksc=None), b"null"),
    (dict(N=-1), b"sizes"), (dict(N=16385), b"at most 16384"), (dict(ks=1022), b"8-byte"), (dict(key=FAKE + 4), b"aligned"),
    (dict(kc=FAKE + 8), b"aligned"), (dict(blocks=1 << 24), b"32 bits"), (dict(heads=0), b"sizes")])
def test_store_refuses(lib, bad, message):
    assert lib.specdec_store_kvcache_fp8(*store_args(**bad)) == 1
    assert message in lib.specdec_last_error()


def test_store_of_nothing_launches_nothing(lib):
    assert lib.specdec_store_kvcache_fp8(*store_args(N=0, key=None, value=None, slots=None)) == 0


def attention_args(**kw):
    a = dict(q=FAKE, T=8, qs=4096, H=32, heads=8, dim=128, kc=FAKE, vc=FAKE, ksc=FAKE, vsc=FAKE, blocks=4, bs=256, group=16,
             cq=FAKE, ck=FAKE, ctx=None, qps=0, R=1, tables=FAKE, W=4, maxq=8, scale=0.1, causal=1, out=FAKE, os=4096, ws=FAKE,
             wsb=1 << 24, err=FAKE, flags=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("status,bad,message", [
    (1, dict(dim=64), b"head_dim"), (1, dict(H=30), b"multiple"), (3, dict(H=24, maxq=1), b"group 3"),
    (3, dict(maxq=9), b"packed columns"), (3, dict(maxq=2 ** 30), b"packed columns"), (1, dict(maxq=0), b"max_seqlen_q"),
    (1, dict(bs=64), b"multiple of 128"), (1, dict(bs=0), b"multiple of 128"), (1, dict(group=64), b"scale_group"),
    (1, dict(R=0), b"sizes"), (1, dict(R=65536), b"sizes"), (1, dict(cq=None), b"context_lens"),
    (1, dict(cq=None, ck=None, ctx=FAKE, qps=9, T=99), b"fit"), (1, dict(cq=None, ck=None, ctx=FAKE, qps=8, R=2), b"fit"),
    (1, dict(q=None), b"null"), (1, dict(out=None), b"null"), (1, dict(ksc=None), b"null"), (1, dict(flags=2), b"flags"),
    (1, dict(q=FAKE + 2), b"aligned"), (1, dict(qs=4100), b"aligned"), (1, dict(kc=FAKE + 8), b"aligned"),
    (1, dict(vsc=FAKE + 4), b"aligned"), (1, dict(W=1 << 24), b"2^31"), (1, dict(blocks=1 << 30), b"32 bits")])
def test_attention_refuses(lib, status, bad, message):
    assert lib.specdec_paged_attention_fp8(*attention_args(**bad)) == status
    assert message in lib.specdec_last_error()


def metadata_args(**kw):
    a = dict(lengths=FAKE, last=FAKE, drafts=FAKE, lens=FAKE, R=4, k=7, tables=FAKE, tw=8, nb=FAKE, free=FAKE, count=FAKE,
             cap=10, bs=256, rows=4, tokens=32, pad=9, width=8, b64=FAKE, b32=FAKE, ticket=FAKE, err=FAKE, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,message", [
    (dict(rows=3), b"rows"), (dict(rows=0, R=0), b"rows"), (dict(rows=65536), b"rows"), (dict(k=-1), b"drafts"),
    (dict(k=1024), b"drafts"), (dict(tokens=0), b"positive"), (dict(width=0), b"positive"), (dict(bs=0), b"positive"),
    (dict(tw=1 << 24), b"32 bits"), (dict(lengths=None), b"null"), (dict(nb=None), b"null"), (dict(count=None), b"together"),
    (dict(b32=None), b"null"), (dict(ticket=None), b"null")])
def test_metadata_refuses(lib, bad, message):
    assert lib.specdec_verify_metadata(*metadata_args(**bad)) == 1
    assert message in lib.specdec_last_error()


@pytest.mark.parametrize("blocks", [-1, 2 ** 31 // 256, 2 ** 40])
def test_metadata_refuses_a_cache_past_32_bits(lib, blocks):
    args = metadata_args()
    assert lib.specdec_verify_metadata_ex(*args[:-1], blocks, args[-1]) == 1
    assert b"32 bits" in lib.specdec_last_error()


def logprob_args(**kw):
    a = dict(x=FAKE, dtype=1, T=8, V=1000, stride=1000, tokens=FAKE, temps=None, top=5, lp=FAKE, ent=FAKE, ids=FAKE, tlp=FAKE,
             ws=FAKE, wsb=1 << 30, err=FAKE, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,message", [
    (dict(dtype=7), b"dtype"), (dict(stride=999), b"sizes"), (dict(T=65536), b"sizes"), (dict(T=-1), b"sizes"),
    (dict(V=0), b"sizes"), (dict(V=(1 << 24) + 1, stride=1 << 25), b"sizes"), (dict(top=33), b"num_top"),
    (dict(top=-1), b"num_top"), (dict(V=4, top=5), b"num_top"), (dict(x=None), b"null"), (dict(ids=None), b"null"),
    (dict(x=FAKE + 1), b"aligned"), (dict(ws=None), b"null"), (dict(ws=FAKE + 8), b"aligned")])
def test_logprobs_refuse(lib, bad, message):
    assert lib.specdec_token_logprobs(*logprob_args(**bad)) == 1
    assert message in lib.specdec_last_error()


def test_logprobs_of_no_rows_launch_nothing(lib):
    assert lib.specdec_token_logprobs(*logprob_args(T=0, x=None)) == 0


def test_cpu_tensors_are_refused():
    from nanovllm_b200.attention_fp8 import FP8Cache, store_kvcache_fp8
    from nanovllm_b200.logprobs import token_logprobs
    c = FP8Cache.allocate(2, 128, 2, torch.device("cpu"))
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        store_kvcache_fp8(x, x, c.k_cache, c.v_cache, c.k_scale, c.v_scale, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64))


def test_cache_geometry_is_checked():
    from nanovllm_b200.attention_fp8 import FP8Cache, _cache_geometry
    c = FP8Cache.allocate(3, 256, 2, torch.device("cpu"), group=32)
    assert _cache_geometry(c.k_cache, c.v_cache, c.k_scale, c.v_scale) == (3, 2, 256, 32)
    k, v = c.dequantised()
    assert k.shape == (3, 256, 2, 128) and v.dtype == torch.float32
    for bad in (dict(k=c.k_cache.view(torch.uint8)), dict(v=c.v_cache[:2]), dict(ks=c.k_scale.double()),
                dict(vs=c.v_scale[:, :, :4]), dict(ks=c.k_scale[:, :1], vs=c.v_scale[:, :1]),
                dict(k=c.k_cache.transpose(0, 1), v=c.v_cache.transpose(0, 1))):
        a = {**dict(k=c.k_cache, v=c.v_cache, ks=c.k_scale, vs=c.v_scale), **bad}
        with pytest.raises(ValueError):
            _cache_geometry(a["k"], a["v"], a["ks"], a["vs"])
    for group, size in ((8, 256), (32, 48), (64, 256)):
        with pytest.raises(ValueError, match="group"):
            FP8Cache.allocate(1, size, 2, torch.device("cpu"), group=group)
