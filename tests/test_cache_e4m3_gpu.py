"""The 8-bit cache's kernels (csrc/cache_e4m3.hip, csrc/attention_e4m3.hip) against plain 64-bit arithmetic (plain_e4m3.py).

Tolerances.  Values are rounded to codes as they are given, so their codes and scales have to be equal; so have keys that are not
rotated.  A rotated key is a few 32-bit operations off (2^-21 of its pair's length is allowed), which may move it over the border
between two codes: it has to be within half a code's step and that of the 64-bit one.  Attention: a score's 32-bit sum of D
products is off by at most (D + 16) 2^-24 of sum |q k| scale, a probability by twice that and the exponential's 2^-21; the
bfloat16 library rounds probabilities before the product with the values, and its output: bfloat16 has 8 significant bits, so half a step
is 2^-8 of a number just above a power of two (1 + 2^-8 lies between 1 and 1 + 2^-7), twice; sums over L keys add L 2^-24."""
import math

import numpy as np
import pytest
import torch

import plain_e4m3 as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ACTS = ["bfloat16", "float32"]


@pytest.fixture(scope="module")
def ops():
    from turboquant_cpp_amd.csrc import ops as _ops
    for a in ACTS:
        _ops.library(a)
    return _ops


def adt(act):
    return torch.float32 if act == "float32" else torch.bfloat16


def dev(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make_runs(slots, start, new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return {"cu_seqlens": dev(cu), "slots": dev(slots), "start": dev(start), "max_new": max(new), "min_new": min(new),
            "max_end": max(a + n for a, n in zip(start, new)), "decode": max(new) == 1}


def make_pages(ops, slots, capacity, layers, G, D, page=64, weights=False, seed=0):
    per = -(-capacity // page)
    order = torch.randperm(slots * per, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return ops.E4m3Pages.empty(slots * per + 1, layers, G, D, page, (order.view(slots, per) + 1).to(DEV), weights)


def filled(ops, lens, layers, G, D, page=64, weights=False, seed=0, slots=None, loud=4.0):
    """Pages whose slot b holds lens[b] positions of random keys and values, and the same in plain form."""
    rng = np.random.RandomState(seed)
    pages = make_pages(ops, slots or len(lens), max(lens) + 1, layers, G, D, page, weights, seed)
    plain = P.PlainPages(slots or len(lens), layers, G, D, pages.table.shape[1] * page)
    for b, n in enumerate(lens):
        for layer in range(layers):
            k, v = (rng.randn(n, G, D) * np.exp2(rng.randn(n, 1, 1)) * np.where(rng.rand(D) < 0.05, loud, 1.0) for _ in range(2))
            plain.write(b, layer, 0, k, v)
    if weights:
        plain.weight[:] = np.float32(rng.rand(*plain.weight.shape))
    P.fill_pages(pages, plain, D)
    return pages, plain


# ------------------------------------------------------------------------------------------------ the write
def check_write(ops, act, nh, G, D, rotary, pairing, bias, page, steps, amplitude=1.0, ahead=0, seed=1, loud=None):
    """Steps of (slots, new tokens) one after the other: what the pages hold after each, and the queries."""
    g = torch.Generator().manual_seed(seed)
    n_slots = 1 + max(s for slots, _ in steps for s in slots)
    total = [sum(n for slots, new in steps for s, n in zip(slots, new) if s == i) for i in range(n_slots)]
    pages = make_pages(ops, n_slots, max(total), 3, G, D, page, True, seed)
    pages.weight.fill_(7.0)
    plain = P.PlainPages(n_slots, 3, G, D, pages.table.shape[1] * page)
    inv = (1e4 ** (-torch.arange(rotary // 2, dtype=torch.float64) / max(rotary // 2, 1))).float()
    length = [0] * n_slots
    W = (nh + 2 * G) * D
    for at, (slots, new) in enumerate(steps):
        T = sum(new)
        wide = torch.randn((T, W + 8), generator=g) * (1.0 if loud is None else loud[at])
        x = wide[:, :W]
        b = (torch.randn((W,), generator=g) * 0.3).to(torch.bfloat16 if act == "bfloat16" else torch.float32) if bias else None
        start = [length[s] for s in slots]
        positions = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)]) + ahead
        q = ops.rope_kv_write_e4m3(wide.to(DEV)[:, :W], positions.to(torch.int32).to(DEV), inv.to(DEV), pairing, rotary, pages, 1, nh, act,
                                   make_runs(slots, start, new), bias=None if b is None else b.to(DEV), amplitude=amplitude)
        full = (x if b is None else x + b.float()).double().numpy().reshape(T, nh + 2 * G, D)
        turned = P.rotate(full[:, :nh + G], positions.numpy(), inv.double().numpy(), pairing, amplitude)
        want_q, size = turned[:, :nh].reshape(T, -1), np.abs(full).max()
        err = np.abs(q.double().cpu().numpy() - want_q)
        # (a pair's numbers may be of unlike sizes: 2^-21 of the largest number there is)
        assert (err <= 2.0 ** -21 * amplitude * size + (np.abs(want_q) * 2.0 ** -8 if act == "bfloat16" else 0.0)).all(), err.max()
        got_before, t = P.read_pages(pages, D), 0
        for s, a, n in zip(slots, start, new):
            plain.write(s, 1, a, turned[t:t + n, nh:], full[t:t + n, nh + G:])
            t += n
            length[s] += n
            for h in range(G):
                blocks = -(-length[s] // 16)
                assert np.array_equal(got_before.scale["v"][s, 1, h, :blocks], plain.scale["v"][s, 1, h, :blocks]), (at, s, h)
                assert np.array_equal(got_before.code["v"][s, 1, h, :length[s]], plain.code["v"][s, 1, h, :length[s]]), (at, s, h)
                assert np.array_equal(got_before.scale["k"][s, 1, h, :blocks], plain.scale["k"][s, 1, h, :blocks]), (at, s, h)
                gk, pk = got_before.code["k"][s, 1, h, :length[s]], plain.code["k"][s, 1, h, :length[s]]
                if rotary == 0 and amplitude == 1.0:
                    assert np.array_equal(gk, pk)
                else:       # a neighbouring code where the rotated key lies at a border: few, and by one step
                    off = gk != pk
                    assert off.mean() <= 1e-3 and (np.abs(gk - pk)[off] <= 2.0 ** -3 * np.maximum(np.abs(gk), np.abs(pk))[off] + 2.0 ** -9).all()
                    # (the next write starts from what is there)
                    plain.code["k"][s, 1, h, :length[s]] = gk
                assert (got_before.weight[s, 1, h, :length[s]] == 0).all()
                assert (got_before.weight[s, 1, h, length[s]:] == 7).all()
        for layer in (0, 2):        # the other layers' part of every page is untouched
            assert not got_before.code["k"][:, layer].any() and not got_before.code["v"][:, layer].any()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("nh,G,D,rotary,pairing,bias,page", [
    (4, 4, 64, 64, 0, False, 64), (6, 2, 80, 32, 1, True, 128), (5, 1, 16, 0, 0, True, 64), (2, 2, 256, 256, 1, False, 64),
    (7, 1, 48, 20, 0, False, 192), (3, 3, 128, 128, 0, True, 64)])
def test_write(ops, act, nh, G, D, rotary, pairing, bias, page):
    check_write(ops, act, nh, G, D, rotary, pairing, bias, page,
                [([0, 2, 1], [1, 130, 17]), ([1, 0], [1, 1]), ([2, 0, 1], [3, 70, 47]), ([0, 1, 2], [1, 1, 1]), ([2], [65])])


def test_write_far_positions_and_amplitude(ops):
    check_write(ops, "float32", 4, 2, 32, 32, 0, False, 64, [([0], [40]), ([0], [1])], amplitude=1.2, ahead=1_000_000)
    check_write(ops, "bfloat16", 4, 2, 32, 32, 1, False, 64, [([0], [40]), ([0], [1])], amplitude=0.7, ahead=131_071)


@pytest.mark.parametrize("act", ACTS)
def test_write_blocks_that_grow(ops, act):
    """One token at a time, each larger or smaller than the last: blocks take larger scales and what they hold is rounded to them."""
    steps = [([0, 1], [1, 1])] * 40
    loud = [2.0 ** ((i * 7) % 23 - 11) for i in range(40)]
    check_write(ops, act, 2, 2, 32, 0, 0, False, 64, steps, loud=loud)
    check_write(ops, act, 2, 1, 48, 16, 0, True, 64, [([0], [5]), ([0], [3]), ([0], [20]), ([0], [2]), ([0], [2])], loud=[1e-6, 1.0, 1e4, 1e-3, 1e30])


def test_write_of_the_smallest_and_largest_numbers(ops):
    for value in (0.0, 2.0 ** -149, 1e-38, 2.0 ** -100 * 448, 448.0, 449.0, 1.75, 1.7500001, 2.0 ** 119, 1.3e36):
        pages = make_pages(ops, 1, 64, 1, 1, 16)
        plain = P.PlainPages(1, 1, 1, 16, 64)
        x = torch.zeros((3, 48))
        x[:, 16:32] = torch.linspace(-1, 1, 16) * value
        x[:, 32:] = torch.linspace(1, -0.5, 16) * value
        ops.rope_kv_write_e4m3(x.to(DEV), dev([0, 1, 2]), torch.zeros((0,), device=DEV), 0, 0, pages, 0, 1, "bfloat16", make_runs([0], [0], [3]))
        plain.write(0, 0, 0, x[:, None, 16:32].double().numpy(), x[:, None, 32:].double().numpy())
        got = P.read_pages(pages, 16)
        for m in "kv":
            assert np.array_equal(got.scale[m], plain.scale[m]), (value, m)
            assert np.array_equal(got.code[m], plain.code[m]), (value, m)


@pytest.mark.parametrize("act", ACTS)
def test_numbers_that_are_not_finite(ops, act):
    """A row with such a number in its key or value keeps NaN for its key and 0 for its value; its block's other rows are as without
    it; who sees it gets NaN, who does not is not touched."""
    nh, G, D = 2, 2, 32
    for bad in (math.nan, math.inf, -math.inf, 2.0 ** 120):
        pages = make_pages(ops, 1, 128, 1, G, D)
        g = torch.Generator().manual_seed(3)
        x = torch.randn((40, (nh + 2 * G) * D), generator=g)
        x[9, nh * D + 5] = bad                  # a key of head 0
        x[20, (nh + G + 1) * D + 7] = bad       # a value of head 1
        runs = make_runs([0], [0], [40])
        q = ops.rope_kv_write_e4m3(x.to(DEV), torch.arange(40, dtype=torch.int32, device=DEV), torch.zeros((0,), device=DEV), 0, 0, pages, 0, nh, act, runs)
        plain = P.PlainPages(1, 1, G, D, 128)
        full = x.double().numpy().reshape(40, nh + 2 * G, D)
        plain.write(0, 0, 0, full[:, nh:nh + G], full[:, nh + G:])
        got = P.read_pages(pages, D)
        for m in "kv":
            assert np.array_equal(got.scale[m], plain.scale[m])
            assert np.array_equal(got.code[m], plain.code[m], equal_nan=True)
        out = ops.attention_e4m3(q, pages, 0, nh, None, D ** -0.5, act, runs).float().cpu().view(40, nh, D)
        assert out[:9, 0].isfinite().all() and out[9:, 0].isnan().all()
        assert out[:20, 1].isfinite().all() and out[20:, 1].isnan().all()
        win = ops.attention_e4m3(q, pages, 0, nh, 4, D ** -0.5, act, runs).float().cpu().view(40, nh, D)
        assert win[:9, 0].isfinite().all() and win[9:13, 0].isnan().all() and win[13:, 0].isfinite().all()
        for t in (8, 12, 13, 39):      # single tokens
            one = make_runs([0], [t], [1])
            o = ops.attention_e4m3(q[t:t + 1].contiguous(), pages, 0, nh, 4, D ** -0.5, act, one).float().cpu().view(nh, D)
            assert bool(o[0].isnan().all()) == (9 <= t < 13) and bool(o[0].isfinite().all()) == (not 9 <= t < 13)


def test_write_of_queries_alone(ops):
    pages = make_pages(ops, 1, 64, 2, 1, 32)
    x = torch.randn((5, 3 * 32), generator=torch.Generator().manual_seed(1))
    inv = torch.ones(16)
    q = ops.rope_kv_write_e4m3(x.to(DEV), dev([0, 1, 2, 3, 4]), inv.to(DEV), 0, 32, pages, 1, 3, "float32", make_runs([0], [0], [5]), write=False)
    want = P.rotate(x.double().numpy().reshape(5, 3, 32), np.arange(5), np.ones(16), 0)
    assert np.abs(q.cpu().double().numpy().reshape(5, 3, 32) - want).max() < 1e-5
    assert not pages.k.float().any() and not pages.k_scale.any()


# ------------------------------------------------------------------------------------------------ attention
def check_attention(ops, act, nh, G, D, lens, new, page=64, window=None, softcap=None, bias=False, chunk=None, sink=None, weights=False,
                    seed=0, plain_pages=None):
    pages, plain = plain_pages or filled(ops, lens, 2, G, D, page, weights, seed)
    rng = np.random.RandomState(seed + 100)
    slots = list(rng.permutation(len(lens)))
    start = [lens[s] - new[s] for s in slots]
    count = [new[s] for s in slots]
    T, scale = sum(count), D ** -0.5
    q = torch.from_numpy(rng.randn(T, nh * D)).to(adt(act))
    r = [np.float32(np.abs(rng.randn(nh))) for _ in range(2)] if bias else None
    sk = np.float32(rng.randn(nh) * 2) if sink is True else sink
    before = plain.weight.copy()
    runs = make_runs(slots, start, count)
    out = ops.attention_e4m3(q.to(DEV), pages, 1, nh, window, scale, act, runs, softcap=softcap, chunk=chunk, add_weights=weights,
                             distance_bias=None if r is None else tuple(torch.from_numpy(x).to(DEV) for x in r),
                             sink=None if sk is None else torch.from_numpy(sk).to(DEV))
    got = out.double().cpu().numpy().reshape(T, nh, D)
    after = P.read_pages(pages, D).weight if weights else None
    t = 0
    for s, a, n in zip(slots, start, count):
        want_w, slack = np.zeros((G, lens[s])), np.zeros((G, lens[s]))
        for h in range(nh):
            kvh = h // (nh // G)
            k, v = plain.values("k", s, 1, kvh)[:lens[s]], plain.values("v", s, 1, kvh)[:lens[s]]
            o, w, spread, reach = P.attend(q[t:t + n].double().numpy().reshape(n, nh, D)[:, h], k, v, list(range(a, a + n)), scale, window,
                                           softcap, None if r is None else (float(r[0][h]), float(r[1][h])), chunk,
                                           None if sk is None else float(sk[h]))
            # (the cap's and the bias's own 32-bit functions: 2^-20 of what they are given, and 1e-6 of a cap)
            e = (D + 16) * 2.0 ** -24 * reach + 2.0 ** -20 * (reach + (10.0 if bias else 0.0)) * (softcap is not None or bias) + \
                (softcap or 0.0) * 2e-7 + 2.0 ** -21
            rel = 2 * e + (2.0 ** -8 if act == "bfloat16" else 2.0 ** -22) + lens[s] * 2.0 ** -24
            bound = rel[:, None] * spread * 1.01 + (np.abs(o) * 2.0 ** -8 * 1.01 if act == "bfloat16" else 0.0) + 1e-30
            off = np.abs(got[t:t + n, h] - o)
            assert (off <= bound).all(), (s, h, float((off / bound).max()))
            want_w[kvh] += w
            slack[kvh] += w * (2 * e.max() + n * 2.0 ** -24 + 2.0 ** -20)
        if weights:
            total = before[s, 1, :, :lens[s]] + want_w
            off = np.abs(after[s, 1, :, :lens[s]] - total)
            assert (off <= slack + total * nh // G * 2.0 ** -23 + total * 2.0 ** -22 + 1e-12).all(), (s, off.max())
            assert np.array_equal(after[s, 1, :, lens[s]:], before[s, 1, :, lens[s]:]) and np.array_equal(after[s, 0], before[s, 0])
        t += n
    return pages, q, out, runs


SHAPES = [(4, 4, 64), (6, 2, 80), (5, 1, 16), (34, 2, 128), (3, 3, 192), (7, 1, 256), (2, 2, 128), (8, 4, 48)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("nh,G,D", SHAPES)
def test_single_tokens(ops, act, nh, G, D):
    check_attention(ops, act, nh, G, D, [1, 63, 64, 65, 200, 129], [1] * 6, weights=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("nh,G,D", SHAPES)
def test_prompts(ops, act, nh, G, D):
    check_attention(ops, act, nh, G, D, [1, 70, 131, 64], [1, 70, 50, 3], weights=True, page=128)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("opts", [dict(window=1), dict(window=20), dict(window=64, sink=True), dict(softcap=5.0), dict(bias=True),
                                  dict(chunk=50), dict(sink=True, softcap=3.0, window=77, bias=True, chunk=90), dict(window=10_000)])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 150]])
def test_options(ops, act, opts, new):
    check_attention(ops, act, 4, 2, 64, [45, 130, 211], new, weights=True, **opts)


@pytest.mark.parametrize("act", ACTS)
def test_long_caches(ops, act):
    """Beyond position 4,096, where runs of single tokens grow longer, beside short sequences; one head, so that the plain side is quick."""
    check_attention(ops, act, 1, 1, 32, [4095, 4096, 4097, 9001, 5, 12_300], [1] * 6, weights=True)
    check_attention(ops, act, 1, 1, 32, [4300, 4097], [1] * 2, window=300, weights=True)


def test_prompts_of_two_groups_to_a_wave(ops):
    """Enough workgroups that a wave takes 32 tokens."""
    check_attention(ops, "bfloat16", 128, 2, 128, [600], [520], weights=True)
    check_attention(ops, "bfloat16", 128, 1, 64, [700], [513], window=100, sink=True)


@pytest.mark.parametrize("act", ACTS)
def test_every_code_comes_back(ops, act):
    """A cache of one position gives back its value: every code with several scales, to the bit."""
    D = 256
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0           # (no NaN among values)
    for e in (-100, -20, 0, 13, 110):
        pages = make_pages(ops, 1, 64, 1, 1, D)
        page = int(pages.table[0, 0])
        pages.v.view(torch.uint8)[page, 0, 0, torch.from_numpy(P.v_place(D, 0)).to(DEV)] = codes.to(DEV)
        pages.v_scale[page] = 2.0 ** e
        want = codes.view(torch.float8_e4m3fn).float() * 2.0 ** e
        for n_new in (1, 2):
            q = torch.zeros((n_new, D), dtype=adt(act), device=DEV)
            out = ops.attention_e4m3(q, pages, 0, 1, None, 1.0, act, make_runs([0], [0], [n_new]))
            assert torch.equal(out[0].float().cpu(), want), (act, e, n_new)


@pytest.mark.parametrize("act", ACTS)
def test_what_lies_behind_a_sequence_is_not_read(ops, act):
    """NaN keys and the largest values behind the end, in the tile's rest and in other slots' pages, change no bit."""
    for new in ([1, 1], [30, 77]):
        pages, plain = filled(ops, [45, 130], 2, 2, 64, weights=True)
        _, q, want, runs = check_attention(ops, act, 4, 2, 64, [45, 130], new, plain_pages=(pages, plain))
        for s, n in enumerate([45, 130]):
            plain.code["k"][s, :, :, n:] = np.nan
            plain.code["v"][s, :, :, n:] = 448.0
        P.fill_pages(pages, plain, 64)
        again = ops.attention_e4m3(q.to(DEV), pages, 1, 4, None, 64 ** -0.5, act, runs)
        assert torch.equal(again, want)


@pytest.mark.parametrize("act", ACTS)
def test_rows_without_weight(ops, act):
    """Scores that are all -inf: 0, with and without a sink of -inf; a sink alone decides."""
    pages, plain = filled(ops, [70], 2, 1, 16, weights=True)
    q = torch.zeros((70, 2 * 16), dtype=adt(act), device=DEV)
    q[:, 0] = -math.inf
    plain.code["k"][0, 1, 0, :, :] = 0.0
    plain.code["k"][0, 1, 0, :, 0] = 1.0
    P.fill_pages(pages, plain, 16)
    # head 0: every score is -inf; head 1: zeros
    for new, start in ((70, 0), (1, 69)):
        runs = make_runs([0], [start], [new])
        before = pages.weight.clone()
        for sink in (None, torch.tensor([-math.inf, -math.inf], device=DEV)):
            out = ops.attention_e4m3(q[start:start + new].contiguous(), pages, 1, 2, None, 1.0, act, runs, sink=sink, add_weights=True)
            assert (out.view(new, 2, 16)[:, 0] == 0).all() and out.isfinite().all()
        assert pages.weight.isfinite().all()
        given = (pages.weight - before)[pages.table[0].long(), 1].sum().item()
        assert abs(given - 2 * new) < 1e-2 * new      # head 1 alone gives weight, one a row and call
        pages.weight.copy_(before)


@pytest.mark.parametrize("act", ACTS)
def test_a_token_does_not_depend_on_the_others(ops, act):
    """The same bits alone, in a batch, and with other limits told (as a step that is replayed for longer sequences is)."""
    lens = [4100, 70, 260, 4500, 3]
    pages, _ = filled(ops, lens, 2, 2, 64)
    q = torch.randn((5, 4 * 64), generator=torch.Generator().manual_seed(2)).to(adt(act)).to(DEV)
    together = ops.attention_e4m3(q, pages, 1, 4, None, 0.125, act, make_runs([0, 1, 2, 3, 4], [n - 1 for n in lens], [1] * 5))
    for i, n in enumerate(lens):
        runs = make_runs([i], [n - 1], [1])
        assert torch.equal(ops.attention_e4m3(q[i:i + 1].contiguous(), pages, 1, 4, None, 0.125, act, runs)[0], together[i])
        runs["max_end"] = min(4544, n + 1000)
        assert torch.equal(ops.attention_e4m3(q[i:i + 1].contiguous(), pages, 1, 4, None, 0.125, act, runs)[0], together[i])


# ------------------------------------------------------------------------------------------------ eviction
def check_choice(ops, lens, keep, first, recent, layers=2, G=2, weight=None, page=64, seed=0):
    pages = make_pages(ops, len(lens) + 1, max(max(lens), 1), layers, G, 16, page, True, seed)
    rng = np.random.RandomState(seed)
    slots = [int(s) for s in rng.permutation(len(lens) + 1)[:len(lens)]]
    w = np.float32(rng.rand(layers, G, len(lens), pages.table.shape[1] * page)) if weight is None else weight
    table = pages.table.cpu().numpy()
    host = pages.weight.cpu().numpy()
    for b, s in enumerate(slots):
        for i, pg in enumerate(table[s]):
            host[pg] = w[:, :, b, i * page:(i + 1) * page]
    pages.weight.copy_(torch.from_numpy(host))
    got = ops.evict_choose(pages, dev(slots), dev(lens), max(lens), keep, first, recent).cpu().numpy()
    for b, n in enumerate(lens):
        for layer in range(layers):
            for h in range(G):
                assert got[b, layer, h].tolist() == P.choose(w[layer, h, b], n, keep, first, recent), (b, layer, h)


@pytest.mark.parametrize("lens,keep,first,recent", [
    ([1], 1, 0, 0), ([2], 1, 0, 0), ([100, 64, 65], 33, 4, 10), ([100, 300, 7], 64, 0, 64), ([500, 100], 64, 64, 0), ([300, 10, 0], 20, 3, 4),
    ([1025, 2048, 1024], 1000, 1, 999), ([777], 776, 0, 0)])
def test_choice(ops, lens, keep, first, recent):
    check_choice(ops, lens, keep, first, recent)


def test_choice_of_equal_weights_and_unusual_ones(ops):
    n, shape = 700, (2, 2, 1, 704)
    rng = np.random.RandomState(1)
    check_choice(ops, [n], 200, 5, 30, weight=np.zeros(shape, np.float32))
    check_choice(ops, [n], 200, 5, 30, weight=np.float32(rng.randint(0, 3, shape)))
    w = np.float32(rng.randint(-2, 3, shape))
    w[rng.rand(*shape) < 0.1] = np.nan
    w[rng.rand(*shape) < 0.1] = np.inf
    w[rng.rand(*shape) < 0.1] = -np.inf
    w[rng.rand(*shape) < 0.1] = -0.0
    for keep in (1, 50, 200, 650, 699):
        check_choice(ops, [n], keep, 0, 0, weight=w)
    check_choice(ops, [n], 300, 0, 0, weight=np.float32(1.0 + rng.randint(0, 5, shape) * 2.0 ** -23))      # the last bits decide


def test_choice_of_long_sequences(ops):
    """More weights than stay in LDS."""
    rng = np.random.RandomState(2)
    w = np.float32(rng.randint(0, 50, (1, 1, 2, 40_000)) / 7)
    check_choice(ops, [40_000, 16_500], 16_390, 4, 100, layers=1, G=1, weight=w, page=64)


@pytest.mark.parametrize("D,page,keep,lens", [(64, 64, 70, [200, 71]), (80, 128, 128, [300, 129]), (16, 64, 1, [5, 64]), (256, 64, 65, [190, 100]),
                                              (128, 192, 100, [400, 101])])
def test_move(ops, D, page, keep, lens):
    pages, plain = filled(ops, lens, 2, 2, D, page, True, slots=2 * len(lens), loud=2.0 ** 30)      # scales far apart: codes are rounded again
    src, dst = list(range(len(lens))), list(range(len(lens), 2 * len(lens)))
    kept = ops.evict_choose(pages, dev(src), dev(lens), max(lens), keep, min(2, keep), 0)
    raw = pages.k.view(torch.uint8).clone()
    ops.evict_move(pages, dev(src), dev(dst), kept)
    got = P.read_pages(pages, D)
    host = kept.cpu().numpy()
    for s, d in zip(src, dst):
        P.move(plain, s, d, host[s], page)
    for m in "kv":
        assert np.array_equal(got.code[m], plain.code[m]) and np.array_equal(got.scale[m], plain.scale[m]), m
    assert np.array_equal(got.weight, plain.weight)
    assert torch.equal(raw[pages.table[:len(lens)].long()], pages.k.view(torch.uint8)[pages.table[:len(lens)].long()])


def test_move_of_many_tiles(ops):
    """Enough workgroups (more than 2,048) that one tile of values at a time goes through shared memory."""
    lens, keep = [1300, 1217], 650
    pages, plain = filled(ops, lens, 8, 16, 32, 64, True, slots=4, loud=2.0 ** 30)
    kept = ops.evict_choose(pages, dev([0, 1]), dev(lens), max(lens), keep, 4, 100)
    assert -(-keep // 64) * 8 * 16 * 2 > 2048
    ops.evict_move(pages, dev([0, 1]), dev([2, 3]), kept)
    got, host = P.read_pages(pages, 32), kept.cpu().numpy()
    for s in (0, 1):
        P.move(plain, s, s + 2, host[s], 64)
    for m in "kv":
        assert np.array_equal(got.code[m], plain.code[m]) and np.array_equal(got.scale[m], plain.scale[m]), m
    assert np.array_equal(got.weight, plain.weight)


@pytest.mark.parametrize("step", [0, 1, 3, -2])
def test_positions_that_do_not_follow_one_another(ops, step):
    """What a run's tokens turn by is what `positions` says, one by one: steps of any size, and now and then another."""
    T, D, rng = 150, 128, np.random.RandomState(abs(step))
    pages, freq = make_pages(ops, 1, T, 1, 2, D), torch.tensor(10000.0 ** (-np.arange(64) / 64), dtype=torch.float32)
    at = 70_000 + step * np.arange(T) + np.cumsum(rng.rand(T) < 0.05) * 11
    x = torch.randn(T, 8 * D, generator=torch.Generator().manual_seed(1))
    q = ops.rope_kv_write_e4m3(x.to(DEV), dev(at.tolist()), freq.to(DEV), 0, D, pages, 0, 4, "float32", make_runs([0], [0], [T]))
    x = x.double().numpy().reshape(T, 8, D)
    want, length = P.rotate(x[:, :4], at, freq.double().numpy(), 0), np.hypot(x[:, :4, :64], x[:, :4, 64:])
    off = np.abs(q.cpu().double().numpy().reshape(T, 4, D) - want)
    assert (off <= 2.0 ** -21 * np.concatenate([length, length], -1)).all()
    k = P.rotate(x[:, 4:6], at, freq.double().numpy(), 0)
    got = P.read_pages(pages, D)
    for h in range(2):
        held, scale = got.values("k", 0, 0, h)[:T], got.scale["k"][0, 0, h].repeat(P.BLOCK)[:T, None]
        assert (np.abs(held - k[:, h]) <= (2.0 ** -4 + 2.0 ** -20) * np.abs(k[:, h]) + 2.0 ** -10 * scale + 2.0 ** -20 * np.abs(k[:, h]).max()).all()


def test_a_bias_from_any_place_on(ops):
    """Views of a bias that start between multiples of 16 bytes."""
    pages = make_pages(ops, 1, 20, 1, 2, 32)
    for dtype in (torch.bfloat16, torch.float32):
        bias = torch.randn(1 + 8 * 32, dtype=dtype, device=DEV)
        x, pos, freq = torch.randn(3, 8 * 32, device=DEV), dev([0, 1, 2]), torch.rand(16, device=DEV)
        q = [ops.rope_kv_write_e4m3(x, pos, freq, 0, 32, pages, 0, 4, "bfloat16", make_runs([0], [0], [3]), bias=b)
             for b in (bias[1:], bias[1:].clone())]
        assert torch.equal(*q)


def test_short_caches_at_the_most_shared_memory(ops):
    """14 tiles of 9 heads of 128 to a kv head: 64 bytes more than go through one launch."""
    check_attention(ops, "bfloat16", 9, 1, 128, [895], [1])
    check_attention(ops, "bfloat16", 9, 1, 128, [830], [1])


def test_move_of_few_positions_and_bad_places(ops):
    """Sequences of fewer positions than are asked for; positions and slots that lie outside are passed over."""
    pages, plain = filled(ops, [40, 150], 1, 1, 32, 64, True, slots=4)
    kept = torch.full((2, 1, 1, 130), -1, dtype=torch.int32)
    kept[0, 0, 0, :40] = torch.arange(40)
    kept[1, 0, 0, :3] = torch.tensor([0, 149, 100_000])
    ops.evict_move(pages, dev([0, 1]), dev([2, 3]), kept.to(DEV))
    kept[1, 0, 0, 2] = -1
    for s in (0, 1):
        P.move(plain, s, s + 2, kept[s].numpy(), 64)
    got = P.read_pages(pages, 32)
    for m in "kv":
        assert np.array_equal(got.code[m], plain.code[m]) and np.array_equal(got.scale[m], plain.scale[m])
    before = pages.k.view(torch.uint8).clone()
    ops.evict_move(pages, dev([0, 77]), dev([-1, 2]), kept.to(DEV))
    assert torch.equal(before, pages.k.view(torch.uint8))
    assert (ops.evict_choose(pages, dev([-5, 9]), dev([60, 60]), 60, 10) == -1).all()


def test_a_key_that_is_not_a_number_moves_along(ops):
    pages, plain = filled(ops, [100], 1, 1, 32, 64, True, slots=2)
    plain.code["k"][0, 0, 0, 50] = np.nan
    P.fill_pages(pages, plain, 32)
    kept = torch.arange(0, 100, 2, dtype=torch.int32).view(1, 1, 1, 50)
    ops.evict_move(pages, dev([0]), dev([1]), kept.to(DEV))
    got = P.read_pages(pages, 32)
    assert np.isnan(got.code["k"][1, 0, 0, 25]).all() and np.isnan(got.code["k"][1]).sum() == 32


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("act", ACTS)
def test_together(ops, act):
    """A conversation as the engine runs one: a prompt, single tokens with weights, eviction into other pages, and on from there with
    positions that run ahead of the places."""
    nh, G, D, page = 4, 2, 64, 64
    pages = make_pages(ops, 3, 400, 1, G, D, page, True, 5)
    plain = P.PlainPages(3, 1, G, D, 448)
    inv = (1e4 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().to(DEV)
    g = torch.Generator().manual_seed(9)

    def step(slot, start, n, ahead):
        x = torch.randn((n, (nh + 2 * G) * D), generator=g)
        positions = torch.arange(start + ahead, start + ahead + n, dtype=torch.int32)
        runs = make_runs([slot], [start], [n])
        q = ops.rope_kv_write_e4m3(x.to(DEV), positions.to(DEV), inv, 0, D, pages, 0, nh, act, runs)
        before = P.read_pages(pages, D)
        out = ops.attention_e4m3(q, pages, 0, nh, None, 0.125, act, runs, add_weights=True)
        after = P.read_pages(pages, D)
        full = x.double().numpy().reshape(n, nh + 2 * G, D)
        plain.write(slot, 0, start, P.rotate(full[:, nh:nh + G], positions.numpy(), inv.double().cpu().numpy(), 0), full[:, nh + G:])
        for h in range(nh):
            kvh = h // 2
            o, w, spread, reach = P.attend(q.double().cpu().numpy().reshape(n, nh, D)[:, h], before.values("k", slot, 0, kvh)[:start + n],
                                           before.values("v", slot, 0, kvh)[:start + n], list(range(start, start + n)), 0.125)
            bound = (2.0 ** -8 if act == "bfloat16" else 2.0 ** -15) * (spread + np.abs(o))
            assert (np.abs(out.double().cpu().numpy().reshape(n, nh, D)[:, h] - o) <= bound).all()
            plain.weight[slot, 0, kvh, :start + n] += w
        assert np.allclose(after.weight[slot, 0, :, :start + n], plain.weight[slot, 0, :, :start + n], rtol=1e-4, atol=1e-6)
        assert (after.code["k"][slot, 0, :, :start + n] != plain.code["k"][slot, 0, :, :start + n]).mean() < 1e-3
        assert np.array_equal(after.code["v"][slot, 0, :, :start + n], plain.code["v"][slot, 0, :, :start + n])

    step(0, 0, 150, 0)
    for i in range(3):
        step(0, 150 + i, 1, 0)
    kept = ops.evict_choose(pages, dev([0]), dev([153]), 153, 77, 4, 20)
    host = kept.cpu().numpy()
    held = P.read_pages(pages, D)
    for h in range(G):
        assert host[0, 0, h].tolist() == P.choose(np.float32(held.weight[0, 0, h]), 153, 77, 4, 20)
    ops.evict_move(pages, dev([0]), dev([2]), kept)
    P.move(held, 0, 2, host[0], page)
    for name in ("code", "scale"):
        for m in "kv":
            getattr(plain, name)[m][2] = getattr(held, name)[m][2]
    plain.weight[2] = held.weight[2]
    for i in range(2):
        step(2, 77 + i, 1, 76)
    step(2, 79, 33, 76)


@pytest.mark.parametrize("act", ACTS)
def test_captured_and_replayed(ops, act):
    """A step of single tokens as a graph, replayed between eager steps on the same pages: the bits of the eager step."""
    nh, G, D, lens = 4, 2, 64, [70, 300, 5]
    inv = torch.ones((D // 2,), device=DEV)
    x = torch.randn((3, (nh + 2 * G) * D), generator=torch.Generator().manual_seed(1)).to(DEV)

    def made():
        return filled(ops, lens, 2, G, D, weights=True)[0]

    def step(pages, runs, positions, qkv):
        q = ops.rope_kv_write_e4m3(qkv, positions, inv, 0, D, pages, 1, nh, act, runs)
        return ops.attention_e4m3(q, pages, 1, nh, None, 0.125, act, runs, add_weights=True)

    want_pages, pages = made(), made()
    runs = make_runs([2, 0, 1], [lens[s] - 1 for s in (2, 0, 1)], [1, 1, 1])
    runs["max_end"] = 320
    positions, qkv = dev([4, 69, 299]), x.clone()
    step(made(), runs, positions, qkv)          # kernels are loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pages, runs, positions, qkv)
    for i in range(4):
        qkv.copy_(x * (i + 1))
        graph.replay()
        got = out.clone()
        want = step(want_pages, runs, positions, x * (i + 1))
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        for a, b in ((pages.k, want_pages.k), (pages.v, want_pages.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(pages.weight, want_pages.weight) and torch.equal(pages.k_scale, want_pages.k_scale)


def test_on_another_stream(ops):
    pages, _ = filled(ops, [300, 70], 2, 2, 64, weights=True)
    q = torch.randn((2, 4 * 64), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    runs = make_runs([0, 1], [299, 69], [1, 1])
    want = ops.attention_e4m3(q, pages, 1, 4, None, 0.125, "bfloat16", runs)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.attention_e4m3(q, pages, 1, 4, None, 0.125, "bfloat16", runs)
    side.synchronize()
    assert torch.equal(got, want)
