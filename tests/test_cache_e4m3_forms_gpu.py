"""The 8-bit cache's kernels where rows and runs hold nothing or no numbers."""
import math

import numpy as np
import pytest
import torch

import plain_e4m3 as P
from test_cache_e4m3_gpu import ACTS, DEV, adt, filled, make_runs, ops  # noqa: F401

pytestmark = pytest.mark.gpu


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
