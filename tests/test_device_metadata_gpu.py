"""verify_metadata on the GPU against the host's pack_verify_metadata, draft_placement and a stack of free blocks: equal."""
import math

import numpy as np
import pytest
import torch

from nanovllm_b200.batch_metadata import RowState, draft_placement, pack_verify_metadata, packed_sizes, packed_views

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def M():
    from nanovllm_b200 import device_metadata
    device_metadata.reset_device_error(DEV)
    return device_metadata


def case(R, k, block_size, low, high, num_rows, width, seed, full=False, fill=1.0):
    """Request state on the host: rows hold the blocks of the tokens already stored."""
    rng = np.random.default_rng(seed)
    lengths = rng.integers(low, high + 1, size=R)
    lens = np.full(R, k + 1) if full else rng.integers(1, k + 2, size=R)
    held = -(-(lengths - 1) // block_size)
    need = -(-(lengths - 1 + lens) // block_size)
    pool = int(np.maximum(held, need).sum()) + 5
    perm = rng.permutation(pool).astype(np.int32)
    tables = np.full((R, width + 2), -7, dtype=np.int32)
    used = 0
    for r in range(R):
        tables[r, :held[r]] = perm[used:used + held[r]]
        used += held[r]
    pads = (num_rows - R) * (k + 1)
    return dict(k=k, block_size=block_size, num_rows=num_rows, width=width, lengths=lengths, lens=lens, held=held, need=need,
                tables=tables, free=perm[used:], pad=pool, tokens=int(lens.sum()) + int(pads * fill),
                last=rng.integers(0, 150000, size=R), drafts=rng.integers(0, 150000, size=(R, k)))


def expected(s):
    """The packed arrays, the grown tables, the counts and the free count that the host code gives."""
    R = len(s["lengths"])
    tables, free = s["tables"].copy(), s["free"].tolist()
    rows = []
    for r in range(R):
        for j in range(int(s["held"][r]), int(s["need"][r])):
            tables[r, j] = free.pop()
        have = max(int(s["held"][r]), int(s["need"][r]))
        rows.append(RowState(int(s["lengths"][r]), int(s["last"][r]), tables[r, :have].tolist()))
    n64, n32 = packed_sizes(s["num_rows"], s["tokens"], s["width"])
    b64, b32 = np.zeros(n64, dtype=np.int64), np.zeros(n32, dtype=np.int32)
    pack_verify_metadata(rows, s["lens"].tolist(), s["k"], s["block_size"], s["num_rows"], s["tokens"], s["pad"], s["width"],
                         b64, b32)
    at, source = draft_placement(s["lens"], s["k"])
    b64[at] = s["drafts"].reshape(-1)[source]
    return b64, b32, tables, np.maximum(s["held"], s["need"]), len(free)


def on_device(s):
    n64, n32 = packed_sizes(s["num_rows"], s["tokens"], s["width"])
    t = lambda x, d: torch.tensor(np.ascontiguousarray(x), dtype=d, device=DEV)  # noqa: E731
    return dict(lengths=t(s["lengths"], torch.int64), last_tokens=t(s["last"], torch.int64), drafts=t(s["drafts"], torch.int64),
                verified_lens=t(s["lens"], torch.int64), block_tables=t(s["tables"], torch.int32),
                num_blocks=t(s["held"], torch.int32), free_blocks=t(s["free"], torch.int32),
                free_count=t([len(s["free"])], torch.int32), block_size=s["block_size"], num_rows=s["num_rows"],
                num_tokens=s["tokens"], pad_block_id=s["pad"], width=s["width"],
                buf64=torch.full((n64,), -9, dtype=torch.int64, device=DEV),
                buf32=torch.full((n32,), -9, dtype=torch.int32, device=DEV))


def check(d, want):
    b64, b32, tables, counts, left = want
    assert np.array_equal(d["buf64"].cpu().numpy(), b64) and np.array_equal(d["buf32"].cpu().numpy(), b32)
    assert np.array_equal(d["block_tables"].cpu().numpy(), tables)
    assert np.array_equal(d["num_blocks"].cpu().numpy(), counts) and d["free_count"].item() == left


@pytest.mark.parametrize("R,k,bs,low,high,num_rows,width", [
    (1, 7, 256, 1, 1, 1, 1), (1, 1, 128, 128, 128, 4, 9), (3, 7, 256, 250, 257, 8, 4), (8, 7, 256, 1, 600, 8, 3),
    (9, 15, 128, 1, 2000, 20, 17), (64, 7, 256, 900, 1100, 64, 17), (33, 0, 256, 1, 5000, 40, 24), (500, 7, 256, 1, 16000, 512, 64),
    (1000, 3, 16, 1, 300, 1003, 20), (5, 40, 8, 1, 20, 6, 8)])
@pytest.mark.parametrize("full", [False, True])
def test_equals_the_host_metadata(M, R, k, bs, low, high, num_rows, width, full):
    s = case(R, k, bs, low, high, num_rows, width, R + k, full)
    d = on_device(s)
    M.verify_metadata(**d)
    assert M.device_error(DEV) == 0
    check(d, expected(s))
    before = d["buf32"].clone()
    M.verify_metadata(**d)                 # the rows now hold their blocks: the same metadata, nothing taken
    check(d, expected(s))
    assert torch.equal(before, d["buf32"])


def test_fixed_lengths_without_a_stack(M):
    s = case(20, 7, 256, 100, 3000, 20, 13, 3, full=True)
    want = expected(s)
    d = on_device(s)
    M.verify_metadata(**d)
    again = on_device(s)
    again.update(verified_lens=None, free_blocks=None, free_count=None, block_tables=d["block_tables"],
                 num_blocks=d["num_blocks"])
    M.verify_metadata(**again)
    assert M.device_error(DEV) == 0
    assert np.array_equal(again["buf64"].cpu().numpy(), want[0]) and np.array_equal(again["buf32"].cpu().numpy(), want[1])


@pytest.mark.parametrize("fill", [0.0, 0.3, 0.77, 1.0])
def test_padding_rows(M, fill):
    s = case(5, 7, 256, 1, 700, 12, 5, 7, fill=fill)
    d = on_device(s)
    M.verify_metadata(**d)
    assert M.device_error(DEV) == 0
    check(d, expected(s))


def test_all_padding(M):
    s = case(0, 7, 256, 1, 2, 4, 3, 8)
    d = on_device(s)
    M.verify_metadata(**d)
    assert M.device_error(DEV) == 0
    check(d, expected(s))


@pytest.mark.parametrize("spoil,code", [
    (dict(verified_lens=0), 7), (dict(verified_lens=9), 7), (dict(lengths=0), 7), (dict(lengths=-5), 7),
    (dict(lengths=2 ** 40), 7), (dict(num_blocks=-1), 7), (dict(num_blocks=100), 7), (dict(free_count=0), 6),
    (dict(free_count=-3), 6)])
def test_bad_rows_and_a_dry_stack_assign_nothing(M, spoil, code):
    s = case(6, 7, 128, 120, 128, 7, 4, 9, full=True)
    d = on_device(s)
    (name, value), = spoil.items()
    d[name][d[name].numel() // 2] = value
    state = {n: d[n].clone() for n in ("block_tables", "num_blocks", "free_count")}
    M.verify_metadata(**d)
    assert M.device_error(DEV) == code
    M.reset_device_error(DEV)
    assert all(torch.equal(state[n], d[n]) for n in state)
    v = packed_views(d["buf64"], d["buf32"], s["num_rows"], s["tokens"], s["width"])
    assert (v["cu_seqlens_q"] == 0).all() and (v["cu_seqlens_k"] == 0).all() and (v["slot_mapping"] == -1).all()
    assert (v["block_tables"] == s["pad"]).all() and (v["input_ids"] == 0).all() and (v["positions"] == 0).all()
    good = on_device(s)                    # the next call is untouched by it
    M.verify_metadata(**good)
    assert M.device_error(DEV) == 0
    check(good, expected(s))


@pytest.mark.parametrize("length", [2 ** 63 - 1, 2 ** 63 - 7, 2 ** 63 - 8, 2 ** 62, 2 ** 31, -2 ** 63, 4 * 128 - 6, 4 * 128 - 7])
def test_lengths_up_to_the_type_s_end(M, length):
    """A length whose sum with the row's 8 tokens wraps in 64 bits is refused like any other past the table's 6 blocks of 128
    (of which width 4 are asked for); the longest that fits is served."""
    s = case(6, 7, 128, 120, 128, 7, 4, 14, full=True)
    d = on_device(s)
    d["lengths"][2] = length
    before = d["block_tables"].clone()
    M.verify_metadata(**d)
    v = packed_views(d["buf64"], d["buf32"], s["num_rows"], s["tokens"], s["width"])
    if length == 4 * 128 - 7:
        assert M.device_error(DEV) == 0
        assert v["positions"][16:24].tolist() == list(range(4 * 128 - 8, 4 * 128)) and d["num_blocks"][2].item() == 4
        return
    assert M.device_error(DEV) == 7
    M.reset_device_error(DEV)
    assert torch.equal(before, d["block_tables"]) and (v["cu_seqlens_k"] == 0).all() and (v["slot_mapping"] == -1).all()


@pytest.mark.parametrize("where", ["held", "stack"])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, 2 ** 27, "cache"])
def test_block_ids_outside_the_cache_assign_nothing(M, where, bad):
    """One id among 40 rows that is negative, whose slots pass 32 bits, or that the cache does not have: nothing is assigned
    and every row is empty, also with the ids of other rows good.  An id that no row needs does not matter."""
    s = case(40, 7, 16, 100, 700, 44, 45, 15, full=True, fill=0.5)
    blocks = s["pad"] if bad == "cache" else None
    d = on_device(s)
    d["cache_blocks"] = blocks
    grown = int((s["need"] - s["held"]).sum())
    assert 8 <= grown < len(s["free"])
    d["free_blocks"][len(s["free"]) - grown - 1] = -5          # below what this call takes
    d["block_tables"][3, int(s["held"][3]):] = -9              # past what row 3 holds
    M.verify_metadata(**{**d, **{n: d[n].clone() for n in ("block_tables", "num_blocks", "free_count", "buf64", "buf32")}})
    assert M.device_error(DEV) == 0
    value = s["pad"] if bad == "cache" else bad
    if where == "held":
        r = int(np.argmax(s["held"] > 1))
        d["block_tables"][r, 1] = value
    else:
        d["free_blocks"][len(s["free"]) - 7] = value
    state = {n: d[n].clone() for n in ("num_blocks", "free_count", "free_blocks")}
    held_blocks = lambda t: t[torch.arange(t.shape[1], device=DEV) < d["num_blocks"][:, None]]  # noqa: E731
    before = held_blocks(d["block_tables"])
    for _ in range(2):                                         # the ticket is left as it was found
        M.verify_metadata(**d)
        assert M.device_error(DEV) == 9
        M.reset_device_error(DEV)
        assert all(torch.equal(state[n], d[n]) for n in state)
        assert torch.equal(held_blocks(d["block_tables"]), before)
        v = packed_views(d["buf64"], d["buf32"], s["num_rows"], s["tokens"], s["width"])
        assert (v["cu_seqlens_q"] == 0).all() and (v["cu_seqlens_k"] == 0).all() and (v["slot_mapping"] == -1).all()
        assert (v["block_tables"] == s["pad"]).all() and (v["input_ids"] == 0).all() and (v["positions"] == 0).all()
    good = on_device(s)                    # the next call is untouched by it
    M.verify_metadata(**good, cache_blocks=s["pad"])
    assert M.device_error(DEV) == 0
    check(good, expected(s))
    with pytest.raises(ValueError, match="cache_blocks"):
        M.verify_metadata(**good, cache_blocks=0)


def test_tokens_that_do_not_fit(M):
    s = case(6, 7, 128, 1, 300, 7, 4, 10)
    for tokens in (int(s["lens"].sum()) - 1, int(s["lens"].sum()) + 9):
        M.verify_metadata(**on_device(dict(s, tokens=tokens)))
        assert M.device_error(DEV) == 7
        M.reset_device_error(DEV)


def test_replayed_graph_follows_the_requests(M):
    """Rounds on the device alone: a captured call, then lengths and last tokens advanced as an acceptance would."""
    s = case(12, 7, 128, 1, 400, 16, 8, 11, full=True)
    d = on_device(s)
    M.verify_metadata(**{**on_device(s)})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.verify_metadata(**d)
    rng = np.random.default_rng(12)
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        want = expected(s)
        check(d, want)
        took = len(s["free"]) - want[4]
        accepted = rng.integers(0, 8, size=12)
        s.update(tables=want[2], held=want[3], free=s["free"][:len(s["free"]) - took], lengths=s["lengths"] + accepted + 1,
                 last=rng.integers(0, 1000, size=12), drafts=rng.integers(0, 1000, size=(12, 7)))
        s["need"] = -(-(s["lengths"] - 1 + s["lens"]) // 128)
        if np.maximum(s["need"] - s["held"], 0).sum() > len(s["free"]):
            break
        d["lengths"].add_(torch.tensor(accepted + 1, device=DEV))
        d["last_tokens"].copy_(torch.tensor(s["last"]))
        d["drafts"].copy_(torch.tensor(s["drafts"]))
    assert M.device_error(DEV) == 0


def test_refusals(M):
    s = case(3, 7, 256, 1, 500, 4, 3, 13)
    d = on_device(s)
    for name, bad in (("lengths", d["lengths"].int()), ("lengths", d["lengths"][:2]), ("drafts", d["drafts"][:, ::2]),
                      ("block_tables", d["block_tables"].long()), ("num_blocks", d["num_blocks"][:1]),
                      ("free_blocks", None), ("buf64", d["buf64"][:-1]), ("buf32", d["buf32"].cpu()),
                      ("verified_lens", d["verified_lens"].int())):
        with pytest.raises(ValueError):
            M.verify_metadata(**{**d, name: bad})
