"""The 8-bit cache's kernels where rows and runs hold nothing or no numbers, and at the sizes by which their forms are chosen, against plain
64-bit arithmetic (plain_e4m3.py) with the tolerances that test_cache_e4m3_gpu.py derives."""
import math

import numpy as np
import pytest
import torch

import plain_e4m3 as P
from test_cache_e4m3_gpu import ACTS, DEV, adt, check_write, dev, filled, make_pages, make_runs, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def assert_codes(got, want):
    """Equal, but for a few rotated keys that lie next to a border between two codes: a 32-bit rounding, 2^-24 of a number, crosses the
    nearest of borders 2^-4 of it apart in one case of 2^19."""
    off = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert off.sum() <= 3 + 1e-5 * off.size and (np.abs(got - want)[off] <= 2.0 ** -3 * np.maximum(np.abs(got), np.abs(want))[off] + 2.0 ** -9).all(), off.sum()


# ------------------------------------------------------------------------------------------------ a row that is not a number
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("opts", [dict(), dict(window=20), dict(chunk=50), dict(softcap=5.0), dict(window=70, softcap=3.0)])
@pytest.mark.parametrize("row", [0, 40, 100])
def test_weights_of_a_prompt_with_a_query_that_is_not_a_number(ops, act, opts, row):
    """It gives NaN to the positions that it sees and changes no bit of any other's weight.  (101 tokens: the last group of 16 is
    filled up with the last one.)"""
    past, T, nh, G, D = 30, 101, 4, 2, 64
    first, _plain = filled(ops, [past + T], 2, G, D, weights=True)
    second = ops.E4m3Pages(first.k, first.v, first.k_scale, first.v_scale, first.table, first.weight.clone())
    q = torch.randn((T, nh * D), generator=torch.Generator().manual_seed(2)).to(adt(act)).to(DEV)
    bad = q.clone()
    bad[row, D + 3] = math.nan      # head 1, of kv head 0
    runs = make_runs([0], [past], [T])
    want = ops.attention_e4m3(q, first, 1, nh, opts.get("window"), 0.125, act, runs, softcap=opts.get("softcap"), chunk=opts.get("chunk"), add_weights=True)
    got = ops.attention_e4m3(bad, second, 1, nh, opts.get("window"), 0.125, act, runs, softcap=opts.get("softcap"), chunk=opts.get("chunk"), add_weights=True)
    i = past + row
    lo = max(0, i - opts.get("window", 10 ** 6) + 1, i // opts.get("chunk", 10 ** 6) * opts.get("chunk", 0))
    have, ought = (P.read_pages(p, D).weight[0, 1] for p in (second, first))
    assert np.isnan(have[0, lo:i + 1]).all() and not np.isnan(have[0, :lo]).any() and not np.isnan(have[0, i + 1:]).any()
    assert np.array_equal(have[0, :lo], ought[0, :lo]) and np.array_equal(have[0, i + 1:], ought[0, i + 1:])
    assert np.array_equal(have[1], ought[1])
    same = torch.ones((T, nh), dtype=torch.bool)
    same[row, 1] = False
    assert got.view(T, nh, D)[row, 1].isnan().all()
    assert torch.equal(got.view(T, nh, D)[same.to(DEV)], want.view(T, nh, D)[same.to(DEV)])


# ------------------------------------------------------------------------------------------------ runs without tokens
def padded(cu, slots, start, **kw):
    """Runs of a batch of single tokens, some of whose sequences bring none."""
    return {"cu_seqlens": dev(cu), "slots": dev(slots), "start": dev(start), "max_new": 1, "min_new": 0, "max_end": max(start) + 1, "decode": True, **kw}


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("cu", [[0, 1, 2, 2], [0, 1, 1, 2], [0, 0, 0, 1]])
@pytest.mark.parametrize("rotary", [64, 20])
def test_queries_of_rows_behind_the_last_sequence(ops, act, cu, rotary):
    """As many rows as sequences, of which some bring no token: every row has its queries, and only places of tokens are written."""
    nh, G, D = 5, 2, 64
    pages = make_pages(ops, 3, 64, 1, G, D, weights=True)
    pages.weight.fill_(7.0)
    x, at = torch.randn((3, (nh + 2 * G) * D), generator=torch.Generator().manual_seed(1)), [90, 5, 1234]
    inv = (1e4 ** (-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))).float()
    torch.full((3, nh * D), math.nan, dtype=adt(act), device=DEV)      # (what the result's memory may hold)
    q = ops.rope_kv_write_e4m3(x.to(DEV), dev(at), inv.to(DEV), 0, rotary, pages, 0, nh, act, padded(cu, [2, 0, 1], [5, 9, 0]))
    full = x.double().numpy().reshape(3, -1, D)
    turned = P.rotate(full[:, :nh + G], np.array(at), inv.double().numpy(), 0)
    err = np.abs(q.double().cpu().numpy().reshape(3, nh, D) - turned[:, :nh])
    assert (err <= 2.0 ** -21 * np.abs(full).max() + (np.abs(turned[:, :nh]) * 2.0 ** -8 if act == "bfloat16" else 0.0)).all()
    got, want = P.read_pages(pages, D), P.PlainPages(3, 1, G, D, 64)
    want.weight[:] = 7.0
    for b, (s, a) in enumerate(zip([2, 0, 1], [5, 9, 0])):
        if cu[b + 1] > cu[b]:
            want.write(s, 0, a, turned[cu[b]:cu[b] + 1, nh:], full[cu[b]:cu[b] + 1, nh + G:])
    for m in "kv":
        assert np.array_equal(got.scale[m], want.scale[m])
        assert_codes(got.code[m], want.code[m])
    assert np.array_equal(got.weight, want.weight)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("cu", [[0, 1, 2, 2], [0, 1, 1, 2], [0, 0, 0, 1]])
@pytest.mark.parametrize("lens", [[300, 70, 5], [1500, 70, 2100], [4200, 1100, 900]])
def test_single_tokens_beside_sequences_that_bring_none(ops, act, cu, lens):
    """Those change neither an output nor a weight."""
    first, _plain = filled(ops, lens, 2, 2, 64, weights=True)
    second = ops.E4m3Pages(first.k, first.v, first.k_scale, first.v_scale, first.table, first.weight.clone())
    q = torch.randn((3, 4 * 64), generator=torch.Generator().manual_seed(2)).to(adt(act)).to(DEV)
    got = ops.attention_e4m3(q, first, 1, 4, None, 0.125, act, padded(cu, [0, 1, 2], [n - 1 for n in lens]), add_weights=True)
    for b in range(3):
        if cu[b + 1] > cu[b]:
            want = ops.attention_e4m3(q[cu[b]:cu[b] + 1].contiguous(), second, 1, 4, None, 0.125, act, make_runs([b], [lens[b] - 1], [1]), add_weights=True)
            assert torch.equal(got[cu[b]], want[0])
    assert torch.equal(first.weight, second.weight)


# ------------------------------------------------------------------------------------------------ writes
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rotary,pairing", [(256, 0), (256, 1), (254, 0), (254, 1)])
def test_writes_at_the_most_shared_memory(ops, act, rotary, pairing):
    """The angles of 64 rows of heads of 256: 64 KiB, and what the kernel has beside them."""
    check_write(ops, act, 1, 1, 256, rotary, pairing, False, 64, [([0], [64]), ([0], [3]), ([0], [130])])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [1030, 2050, 4099])
def test_queries_of_several_tokens_to_a_workgroup(ops, act, T):
    """Two, four and eight of them; positions that follow one another, and some that do not."""
    nh, D, rotary = 3, 32, 24
    pages, rng = make_pages(ops, 1, T, 1, 1, D), np.random.RandomState(T)
    inv = (1e4 ** (-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))).float()
    at = 50_000 + np.arange(T) + np.cumsum(rng.rand(T) < 0.1) * 13
    x = torch.randn((T, nh * D), generator=torch.Generator().manual_seed(4))
    for pairing in (0, 1):
        q = ops.rope_kv_write_e4m3(x.to(DEV), dev(at.tolist()), inv.to(DEV), pairing, rotary, pages, 0, nh, act, make_runs([0], [0], [T]), write=False)
        want = P.rotate(x.double().numpy().reshape(T, nh, D), at, inv.double().numpy(), pairing)
        off = np.abs(q.double().cpu().numpy().reshape(T, nh, D) - want)
        assert (off <= 2.0 ** -21 * np.abs(x.numpy()).max() + (np.abs(want) * 2.0 ** -8 if act == "bfloat16" else 0.0)).all()


@pytest.mark.parametrize("step", [0, 1, 3, -2])
@pytest.mark.parametrize("start", [0, 37])
def test_codes_of_keys_whose_positions_do_not_follow_one_another(ops, step, start):
    """Whole tiles and parts of tiles: the codes of 64-bit angles, but for the few keys that lie next to a border between two."""
    T, D, rng = 300, 128, np.random.RandomState(abs(step))
    pages, freq = make_pages(ops, 1, start + T, 1, 2, D), torch.tensor(10000.0 ** (-np.arange(64) / 64), dtype=torch.float32)
    plain = P.PlainPages(1, 1, 2, D, pages.table.shape[1] * 64)
    at = 70_000 + step * np.arange(T) + np.cumsum(rng.rand(T) < 0.05) * 11
    x = torch.randn(T, 5 * D, generator=torch.Generator().manual_seed(1))
    full = x.double().numpy().reshape(T, 5, D)
    turned = P.rotate(full[:, 1:3], at, freq.double().numpy(), 0)
    if start:
        k, v = rng.randn(start, 2, D), rng.randn(start, 2, D)
        plain.write(0, 0, 0, k, v)
        P.fill_pages(pages, plain, D)
    ops.rope_kv_write_e4m3(x.to(DEV), dev(at.tolist()), freq.to(DEV), 0, D, pages, 0, 1, "float32", make_runs([0], [start], [T]))
    plain.write(0, 0, start, turned, full[:, 3:])
    got = P.read_pages(pages, D)
    assert np.array_equal(got.scale["k"], plain.scale["k"]) and np.array_equal(got.code["v"], plain.code["v"])
    assert_codes(got.code["k"], plain.code["k"])
