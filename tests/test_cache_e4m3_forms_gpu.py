"""The 8-bit cache's kernels where rows and runs hold nothing or no numbers, and at the sizes by which their forms are chosen, against plain
64-bit arithmetic (plain_e4m3.py) with the tolerances that test_cache_e4m3_gpu.py derives."""
import math

import numpy as np
import pytest
import torch

import plain_e4m3 as P
from test_cache_e4m3_gpu import ACTS, DEV, adt, check_attention, check_write, dev, filled, make_pages, make_runs, ops  # noqa: F401

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


# ------------------------------------------------------------------------------------------------ capped scores
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("cap", [1.5, 30.0, 1000.0])
@pytest.mark.parametrize("new", [1, 3])
def test_weights_of_capped_scores(ops, act, cap, new):
    """Scores that are eighths up to 1, without rounding.  In steps of 2^-24: the cap is off by 10 of a score (its argument, the argument's
    square, five terms and their product with the score, a rounding or two each), which counts twice, by itself and in its row's sum; that sum by 32 (200 numbers, some by lanes, and the
    exponential's 2); its logarithm, of 16 at most, and the difference from it by 8 each, rounded, and 16 more for the logarithm; the weight's own
    exponential by 2: 86, of a weight, whatever the cap."""
    n, D = 200, 16
    pages, plain = filled(ops, [n], 1, 1, D, weights=True)
    rng = np.random.RandomState(5)
    plain.code["k"][0, 0, 0] = rng.randint(-8, 9, plain.code["k"][0, 0, 0].shape) / 8
    plain.scale["k"][0, 0, 0], plain.weight[:] = 1.0, 0.0
    P.fill_pages(pages, plain, D)
    q = torch.zeros((new, 2 * D), dtype=adt(act))
    q[:, 0], q[:, D + 3] = 1.0, -1.0
    ops.attention_e4m3(q.to(DEV), pages, 0, 2, None, 1.0, act, make_runs([0], [n - new], [new]), softcap=cap, add_weights=True)
    want = sum(P.attend(q[:, h * D:(h + 1) * D].double().numpy(), plain.values("k", 0, 0, 0)[:n], plain.values("v", 0, 0, 0)[:n],
                        list(range(n - new, n)), 1.0, softcap=cap)[1] for h in range(2))
    off = np.abs(P.read_pages(pages, D).weight[0, 0, 0, :n] - want) / want
    assert off.max() <= 86 * 2.0 ** -24, off.max()


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


# ------------------------------------------------------------------------------------------------ prompts whose tiles go to two halves of a workgroup
HALVES = [
    (4, 2, 64, [577], [577], dict()),                              # ten tiles, no past
    (4, 4, 128, [513], [70], dict()),                              # nine tiles, the last of one position
    (2, 1, 80, [640, 50, 700], [200, 50, 1], dict()),              # heads narrower than their kernel's, a sequence without tiles for one half
    (3, 3, 48, [530], [129], dict()),
    (2, 2, 64, [900, 513], [300, 17], dict(window=448)),
    (2, 1, 64, [650], [650], dict(window=500, sink=True)),
    (4, 2, 80, [600], [90], dict(sink=True)),
    (4, 2, 64, [700], [257], dict(softcap=5.0)),
    (2, 1, 128, [580], [100], dict(bias=True, sink=True)),
    (2, 2, 64, [640], [200], dict(chunk=300)),
    (2, 1, 16, [1100], [64], dict(softcap=4.0, sink=True, window=600, bias=True, chunk=1000)),
]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("nh,G,D,lens,new,opts", HALVES)
def test_prompts_in_two_halves(ops, act, nh, G, D, lens, new, opts):
    """At most 512 workgroups and at least 512 positions in reach; one group of 16 tokens to a wave."""
    assert -(-max(new) // 64) * nh * len(new) <= 512 and -(-max(new) // 128) * nh * len(new) <= 256
    assert min(max(lens), opts.get("window", 10 ** 6) + 64) >= 512
    check_attention(ops, act, nh, G, D, lens, new, weights=True, **opts)


@pytest.mark.parametrize("nh,G,D,lens,new,opts", [(96, 1, 64, [640], [260], dict()), (130, 2, 128, [570], [135], dict(sink=True)),
                                                  (100, 1, 80, [515], [257], dict(softcap=5.0)), (90, 1, 48, [700], [257], dict(window=450, bias=True))])
def test_prompts_in_two_halves_with_two_groups(ops, nh, G, D, lens, new, opts):
    """The same with two groups of 16 tokens to a wave."""
    assert 256 < -(-max(new) // 128) * nh <= 512
    check_attention(ops, "bfloat16", nh, G, D, lens, new, weights=True, **opts)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("odd", [0, 1])
def test_halves_whose_scores_are_all_minus_infinity(ops, act, odd):
    """Every second tile's scores overflow to -inf, which leaves one half of the workgroup without weight; a row that sees no other tile is 0.
    A query that is not a number beside them.  (Scores of -512: their maxima and sums are rounded by 2^-15, and half as much again
    in the pass of the weights, which the exponential turns into 2^-13 of a weight.)"""
    n, D = 600, 16
    pages, plain = filled(ops, [n], 1, 1, D, weights=True)
    q = torch.zeros((n, 2 * D), dtype=adt(act))
    q[:, 0] = -2.0 ** 118
    q[17, D + 4] = math.nan
    lost = np.arange(plain.code["k"].shape[3]) // 64 % 2 == odd
    plain.code["k"][0, 0, 0] = 0.0
    plain.code["k"][0, 0, 0, :, 0] = np.where(lost, 1.0, 2.0 ** -9)
    plain.scale["k"][0, 0, 0] = np.where(lost[::16], 2.0 ** 11, 2.0 ** -100)
    P.fill_pages(pages, plain, D)
    before = plain.weight[0, 0, 0].copy()
    out = ops.attention_e4m3(q.to(DEV), pages, 0, 2, None, 1.0, act, make_runs([0], [0], [n]), add_weights=True).double().cpu().numpy().reshape(n, 2, D)
    assert np.isnan(out[17, 1]).all() and np.isfinite(out[:17]).all() and np.isfinite(out[18:]).all() and np.isfinite(out[17, 0]).all()
    keys, values = plain.values("k", 0, 0, 0)[:n], plain.values("v", 0, 0, 0)[:n]
    seeing = np.arange(0 if odd else 64, n)
    assert (out[:seeing[0], 0] == 0).all()
    o, w, spread, _reach = P.attend(q.double().numpy()[seeing, :D], keys, values, seeing.tolist(), 1.0)
    assert not w[lost[:n]].any()
    rounding = 2.0 ** -8 if act == "bfloat16" else 0.0
    assert (np.abs(out[seeing, 0] - o) <= ((rounding + 2.0 ** -13) * spread + rounding * np.abs(o)) * 1.01).all()
    rest = np.concatenate([np.arange(17), np.arange(18, n)])
    _o, w1, _s, _r = P.attend(np.zeros((n - 1, D)), keys, values, rest.tolist(), 1.0)
    gave = P.read_pages(pages, D).weight[0, 0, 0]
    assert np.isnan(gave[:18]).all() and (gave[n:] == before[n:]).all()
    total = (before[:n] + w + w1)[18:]
    assert (np.abs(gave[18:n] - total) <= (w + w1)[18:] * 2.0 ** -12 + total * 2.0 ** -22).all()


# ------------------------------------------------------------------------------------------------ single tokens whose waves go through several runs
def random_pages(ops, lens, G, D, seed=0):
    """Pages of codes drawn at random (no NaN), with scales of 2^-6 to 2^-3."""
    pages, g = make_pages(ops, len(lens), max(lens), 1, G, D, weights=True, seed=seed), torch.Generator().manual_seed(seed)
    for t in (pages.k, pages.v):
        code = torch.randint(0, 120, t.shape, generator=g, dtype=torch.uint8) + 128 * torch.randint(0, 2, t.shape, generator=g, dtype=torch.uint8)
        t.view(torch.uint8).copy_(code)
    for t in (pages.k_scale, pages.v_scale):
        t.copy_(torch.exp2(torch.randint(-6, -2, t.shape, generator=g).float()))
    pages.weight.copy_(torch.rand(pages.weight.shape, generator=g))
    return pages


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("nh,G,D,lens,opts", [(16, 16, 32, [4500, 3999, 2100, 1300, 4097, 70, 3500, 4200], dict()),
                                              (20, 20, 48, [4096, 3000, 1100, 4400, 3700, 2048], dict(window=3500)),
                                              (32, 16, 80, [3900, 4000, 3100, 1025, 2500, 3333, 4100], dict(softcap=5.0))])
def test_waves_that_go_through_several_runs(ops, act, nh, G, D, lens, opts):
    """Outputs and weights have the bits of each sequence alone, whose waves take a run each, and are right."""
    B = len(lens)
    assert 64 * G * B > 6144       # more runs, of 64 at most to a sequence, than waves
    pages = random_pages(ops, lens, G, D)
    plain = P.read_pages(pages, D)
    alone = ops.E4m3Pages(pages.k, pages.v, pages.k_scale, pages.v_scale, pages.table, pages.weight.clone())
    q = (torch.randn((B, nh * D), generator=torch.Generator().manual_seed(3)) * 0.05).to(adt(act))
    args = dict(softcap=opts.get("softcap"), add_weights=True)
    got = ops.attention_e4m3(q.to(DEV), pages, 0, nh, opts.get("window"), 0.125, act, make_runs(list(range(B)), [n - 1 for n in lens], [1] * B), **args)
    for b, n in enumerate(lens):
        one = ops.attention_e4m3(q[b:b + 1].to(DEV), alone, 0, nh, opts.get("window"), 0.125, act, make_runs([b], [n - 1], [1]), **args)
        assert torch.equal(one[0], got[b]), b
    assert torch.equal(pages.weight, alone.weight)
    after = P.read_pages(pages, D).weight
    for b in (0, B - 1):
        n, given, slack = lens[b], np.zeros((G, lens[b])), np.zeros((G, lens[b]))
        for h in range(nh):
            kvh = h // (nh // G)
            o, w, spread, reach = P.attend(q[b].double().numpy().reshape(nh, D)[h][None], plain.values("k", b, 0, kvh)[:n], plain.values("v", b, 0, kvh)[:n],
                                           [n - 1], 0.125, opts.get("window"), opts.get("softcap"))
            e = (D + 16) * 2.0 ** -24 * reach + 2.0 ** -20 * reach * ("softcap" in opts) + opts.get("softcap", 0.0) * 2e-7 + 2.0 ** -21
            rel = 2 * e + (2.0 ** -8 if act == "bfloat16" else 2.0 ** -22) + n * 2.0 ** -24
            off = np.abs(got[b].double().cpu().numpy().reshape(nh, D)[h] - o[0])
            assert (off <= rel * spread[0] * 1.01 + (np.abs(o[0]) * 2.0 ** -8 * 1.01 if act == "bfloat16" else 0.0)).all(), (b, h)
            given[kvh] += w
            slack[kvh] += w * (2 * e[0] + 2.0 ** -20)
        total = plain.weight[b, 0, :, :n] + given
        assert (np.abs(after[b, 0, :, :n] - total) <= slack + total * 2.0 ** -22 + 1e-12).all(), b


# ------------------------------------------------------------------------------------------------ writes
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rotary,pairing", [(256, 0), (256, 1), (254, 0), (254, 1)])
def test_writes_at_the_most_shared_memory(ops, act, rotary, pairing):
    """The angles of 64 rows of heads of 256: 64 KiB, and what the kernel has beside them."""
    check_write(ops, act, 1, 1, 256, rotary, pairing, False, 64, [([0], [64]), ([0], [3]), ([0], [130])])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("nh,G,D,rotary,pairing,bias,seqs,longest", [
    (2, 16, 16, 16, 0, True, 12, 900), (3, 5, 48, 0, 0, False, 20, 900), (1, 5, 32, 20, 1, True, 60, 900), (1, 16, 32, 12, 0, False, 12, 900),
    (1, 16, 144, 144, 0, True, 2, 2100)])
def test_writes_of_several_kv_heads_to_a_workgroup(ops, act, nh, G, D, rotary, pairing, bias, seqs, longest):
    """1,024 tiles times kv heads and more, most of which nothing falls into; first blocks that are there in part; rows of one head that
    are not finite, which leave its workgroup's other heads as they are."""
    assert ((longest + 62) // 64 + 1) * seqs * G >= 1024
    rng = np.random.RandomState(seqs)
    start, new = [(5 * i + 3) % 40 for i in range(seqs)], [1 + 7 * i % 40 for i in range(seqs)]
    new[seqs // 3], new[seqs - 1] = longest, 130
    slots, T = rng.permutation(seqs).tolist(), sum(new)
    pages, plain = make_pages(ops, seqs, longest + 40, 1, G, D, weights=True), P.PlainPages(seqs, 1, G, D, -(-(longest + 40) // 64) * 64)
    for s, n in zip(slots, start):
        if n:
            plain.write(s, 0, 0, rng.randn(n, G, D), rng.randn(n, G, D))
    plain.weight[:] = 7.0
    P.fill_pages(pages, plain, D)
    W = (nh + 2 * G) * D
    x, b = torch.randn((T, W), generator=torch.Generator().manual_seed(3)), (torch.randn((W,), generator=torch.Generator().manual_seed(4)) * 0.3).to(adt(act))
    for t, head, number in ((7, nh + 3, math.nan), (150, nh + 3, math.inf), (150, nh + G + 1, 2.0 ** 121), (151, nh + G + 2, -math.inf), (T - 1, nh, math.nan)):
        x[t, head * D + t % D] = number
    positions = np.concatenate([np.arange(a, a + n) for a, n in zip(start, new)])
    inv = (1e4 ** (-torch.arange(rotary // 2, dtype=torch.float64) / max(rotary // 2, 1))).float()
    ops.rope_kv_write_e4m3(x.to(DEV), dev(positions.tolist()), inv.to(DEV), pairing, rotary, pages, 0, nh, act, make_runs(slots, start, new),
                           bias=b.to(DEV) if bias else None)
    full, t = (x + b.float() if bias else x).double().numpy().reshape(T, nh + 2 * G, D), 0
    with np.errstate(invalid="ignore"):      # (infinities turn to NaN)
        turned = P.rotate(full[:, nh:nh + G], positions, inv.double().numpy(), pairing)
    for s, a, n in zip(slots, start, new):
        plain.write(s, 0, a, turned[t:t + n], full[t:t + n, nh + G:])
        t += n
    got = P.read_pages(pages, D)
    for m in "kv":
        assert np.array_equal(got.scale[m], plain.scale[m])
        assert_codes(got.code[m], plain.code[m]) if m == "k" and rotary else np.testing.assert_array_equal(got.code[m], plain.code[m])
    assert np.array_equal(got.weight, plain.weight)


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
