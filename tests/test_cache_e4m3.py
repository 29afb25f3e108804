"""A cache in 8 bits without a GPU: which layers keep one, the bookkeeping of positions that are let go, and what the entry points
refuse, which they must find out before they call into the library (here a stand-in that records calls)."""
import dataclasses
import types

import numpy as np
import pytest
import torch

from turboquant_cpp_amd.cache.paged import CacheError, CacheFull, PagedCache
from turboquant_cpp_amd.csrc import ops
from turboquant_cpp_amd.engine.batch import pack_step
from turboquant_cpp_amd.engine.generate import GenerationOptions, generate, kept_when_full
from turboquant_cpp_amd.parts.base import CacheNeed


def need(window=None, able=True, chunk=None, heads=2, dim=16):
    return CacheNeed(heads, dim, window, chunk=chunk, reads_e4m3=able)


def cache_of(*needs, tokens=64 * 8, **kw):
    kw = {"kv_cache": "e4m3", "track_weights": True, **kw}
    return PagedCache([n if isinstance(n, tuple) else (n, None, None) for n in needs], tokens, torch.bfloat16, None, **kw)


# ------------------------------------------------------------------------------------------------ which layers
def test_layers_that_can_read_8_bits_keep_them():
    c = cache_of(need(), need(able=False), need())
    assert [(g.key.e4m3, g.entries) for g in c.groups] == [(True, [0, 2]), (False, [1])]
    assert c.kv(2).layer == 1 and c.kv(0).layer == 0
    assert [g.host_table.shape[0] - c.max_slots for g in c.groups] == [1, 0]


def test_a_cache_that_another_layer_reads_has_to_suit_both():
    shared = cache_of(need(), (need(), None, 0), need())
    assert [(g.key.e4m3, g.entries) for g in shared.groups] == [(True, [0, 2])] and not shared.kv(1).owns and shared.kv(1).layer == 0
    other = cache_of(need(), (need(able=False), None, 0), need())
    assert [(g.key.e4m3, g.entries) for g in other.groups] == [(False, [0]), (True, [2])]


def test_a_cache_that_cannot_be_is_refused():
    with pytest.raises(CacheError, match="none of the model's layers"):
        cache_of(need(able=False))
    with pytest.raises(CacheError, match="multiple of 64"):
        cache_of(need(), page_size=32)
    with pytest.raises(CacheError, match="'same' or 'e4m3'"):
        cache_of(need(), kv_cache="int4")
    with pytest.raises(CacheError, match="8 bits alone"):
        cache_of(need(), kv_cache="same")
    with pytest.raises(CacheError, match="on a GPU"):
        PagedCache([(need(), None, None)], 64, torch.bfloat16, torch.device("cpu"), kv_cache="e4m3")
    same = cache_of(need(), kv_cache="same", track_weights=False)
    assert not same.groups[0].key.e4m3 and same.groups[0].host_table.shape[0] == same.max_slots


def test_the_mixers_that_can():
    from tiny_configs import TINY
    from turboquant_cpp_amd.engine.model import model_from_config
    able = {name: [n.reads_e4m3 for n, _s, _c in model_from_config(cfg, "float32").cache_needs()] for name, (cfg, _i) in TINY.items()}
    assert able["A"] == [True, True] and able["C"] == [True] * 3 and able["D"] == [True] * 4
    assert able["B"] == [False] * 3      # heads of 24 numbers


# ------------------------------------------------------------------------------------------------ positions that are let go
def grown(cache, n):
    slot = cache.open()
    cache.reserve(slot, n)
    cache.commit(slot)
    return slot


def test_letting_positions_go_moves_a_sequence_to_other_pages():
    c = cache_of(need(), need(dim=32), tokens=64 * 6, max_slots=2)
    slot = grown(c, 200)
    before = [g.host_table[slot, :4].tolist() for g in c.groups]
    c.begin_evict(slot, 70)
    assert all((g.host_table[g.spare, :2] >= 0).all() and g.pool.n_free == 0 for g in c.groups)
    c.end_evict(slot, 70)
    for g, old in zip(c.groups, before):
        assert not set(g.host_table[slot, :2].tolist()) & set(old) and (g.host_table[slot, 2:] < 0).all()
        assert (g.host_table[g.spare] < 0).all() and g.pool.n_free == 4
    assert c.length(slot) == 70 and c.slots[slot].dropped == 130 and c.positions_of([slot], [70]) == [200]
    assert c.reserve(slot, 1) == 70      # the next token's place
    c.commit(slot)
    c.begin_evict(slot, 64)
    c.end_evict(slot, 64)
    assert c.slots[slot].dropped == 137 and c.length(slot) == 64
    c.close(slot)
    assert all(g.pool.n_free == 6 for g in c.groups)
    assert c.slots[c.open()].dropped == 0


def test_letting_positions_go_that_was_broken_off_changes_nothing():
    c = cache_of(need(), tokens=64 * 6, max_slots=2)
    slot = grown(c, 200)
    g = c.groups[0]
    before = g.host_table[slot].tolist()
    c.begin_evict(slot, 70)
    c.end_evict(slot, 70, done=False)
    assert g.host_table[slot].tolist() == before and (g.host_table[g.spare] < 0).all() and g.pool.n_free == 2
    assert c.length(slot) == 200 and c.slots[slot].dropped == 0


def test_what_cannot_be_let_go():
    c = cache_of(need(), tokens=64 * 4, max_slots=2)
    slot = grown(c, 200)
    with pytest.raises(CacheFull, match="needs 2 pages"):      # 4 pages are held: none is free
        c.begin_evict(slot, 100)
    assert c.groups[0].pool.n_free == 0 and (c.groups[0].host_table[c.groups[0].spare] < 0).all()
    for keep in (0, 200, 300):
        with pytest.raises(CacheError, match="can stay"):
            c.begin_evict(slot, keep)
    with pytest.raises(CacheError, match="weights"):
        d = cache_of(need(), track_weights=False)
        d.begin_evict(grown(d, 100), 10)
    for other, why in ((need(able=False), "every layer"), (need(window=100), "window"), (need(chunk=64), "window or chunks")):
        d = cache_of(need(), other)
        with pytest.raises(CacheError, match=why):
            d.begin_evict(grown(d, 100), 10)
    d = cache_of(need(), tokens=64 * 6)
    slot = grown(d, 200)
    d.begin_evict(slot, 70)
    d.end_evict(slot, 70)
    with pytest.raises(CacheError, match="has let positions go"):
        d.truncate(slot, 10)
    d.reserve(slot, 1)
    with pytest.raises(CacheError, match="running step"):
        d.begin_evict(slot, 10)


def test_tokens_behind_positions_that_were_let_go():
    b = pack_step([3, 1], [10, 0], [[5, 6, 7], [8]], [[2], [0]], "cpu", ahead=[100, 0])
    assert b.positions.tolist() == [110, 111, 112, 0] and b.start_dev.tolist() == [10, 0] and b.start == [10, 0]
    b = pack_step([3, 1], [10, 0], [[5, 6, 7], [8]], [[2], [0]], "cpu")
    assert b.positions.tolist() == [10, 11, 12, 0]


def test_what_a_full_sequence_keeps():
    for n in range(1, 300):
        keep, first, recent = kept_when_full(n)
        assert 1 <= keep <= max(1, n // 2) and first >= 0 and recent >= 0 and first + recent <= keep and first <= 4
    assert kept_when_full(4096) == (2048, 4, 1022)


def test_generation_asks_for_what_the_engine_cannot():
    engine = types.SimpleNamespace(no_eviction=lambda: "because")
    with pytest.raises(ValueError, match="because"):
        generate(engine, [[1]], GenerationOptions(when_full="evict"))
    with pytest.raises(ValueError, match="when_full"):
        generate(engine, [[1]], GenerationOptions(when_full="shift"))


# ------------------------------------------------------------------------------------------------ refusals
class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 4 if name.endswith("scratch") else 0
        return call


@pytest.fixture
def pretend(monkeypatch):
    """CPU tensors taken for GPU 0's, and a library that only records that it was called."""
    lib = Library()
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: getattr(t, "pretended", 0))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "library", lambda act: lib)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    return lib


def aligned(t):
    """The same numbers from a multiple of 16 bytes on."""
    room = torch.empty(t.numel() + 16, dtype=t.dtype)
    skip = -room.data_ptr() % 16 // t.element_size()
    return room[skip:skip + t.numel()].view(t.shape).copy_(t)


def pools(pages=5, layers=2, G=2, D=32, page=64, slots=2, per=2, weights=True):
    code = lambda: aligned(torch.zeros(pages, layers, G, page * D, dtype=torch.uint8)).view(torch.float8_e4m3fn)
    return dict(k=code(), v=code(), k_scale=torch.zeros(pages, layers, G, page // 16), v_scale=torch.zeros(pages, layers, G, page // 16),
                table=torch.zeros(slots, per, dtype=torch.int32), weight=torch.zeros(pages, layers, G, page) if weights else None)


def elsewhere(t):
    t.pretended = 1
    return t


def test_pages_that_cannot_be(pretend):
    ops.E4m3Pages(**pools())
    for bad in (dict(D=24), dict(page=32), dict(page=96), dict(D=272), dict(pages=0)):
        with pytest.raises(ops.KernelError, match="E4m3Pages"):
            ops.E4m3Pages(**pools(**bad))
    good = pools()
    for name, t in (("k", good["k"].view(torch.uint8)), ("v", good["v"][:, :1]), ("v", aligned(torch.zeros(5, 2, 2, 4096, dtype=torch.uint8)).view(torch.float8_e4m3fn)),
                    ("k_scale", good["k_scale"].double()), ("v_scale", good["v_scale"][:-1]), ("table", good["table"].long()),
                    ("table", good["table"][0]), ("weight", torch.zeros(5, 2, 2, 32)), ("table", good["table"].t()),
                    ("v_scale", elsewhere(good["v_scale"].clone()))):
        with pytest.raises(ops.KernelError, match="E4m3Pages"):
            ops.E4m3Pages(**{**good, name: t})
    with pytest.raises(dataclasses.FrozenInstanceError):
        ops.E4m3Pages(**good).table = None


def runs_of(start=(0, 3), new=(5, 1), **kw):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    out = {"cu_seqlens": i32(np.cumsum([0, *new]).tolist()), "slots": i32(list(range(len(new)))), "start": i32(list(start)),
           "max_new": max(new), "min_new": min(new), "max_end": max(a + b for a, b in zip(start, new)), "decode": max(new) == 1}
    return {**out, **kw}


BAD_RUNS = [dict(max_end=0), dict(max_end=129), dict(max_new=0), dict(max_new=7), dict(decode=True),
            dict(slots=torch.zeros(3, dtype=torch.int32)), dict(slots=torch.zeros(2, dtype=torch.int64)),
            dict(start=torch.zeros(2, dtype=torch.int32)[:1]), dict(cu_seqlens=torch.zeros(2, dtype=torch.int32))]


def test_writes_that_are_refused(pretend):
    pages = ops.E4m3Pages(**pools())
    base = dict(qkv=aligned(torch.zeros(6, 8 * 32)), positions=torch.zeros(6, dtype=torch.int32), inv_freq=torch.zeros(16), pairing=0,
                rotary_dim=32, pages=pages, layer=1, num_heads=4, act="bfloat16", runs=runs_of())
    assert ops.rope_kv_write_e4m3(**base).shape == (6, 128) and pretend.calls == ["tq_e4m3_write"]
    wide = aligned(torch.zeros(6, 8 * 32 + 4))
    ops.rope_kv_write_e4m3(**{**base, "qkv": wide[:, :256], "bias": torch.zeros(256), "rotary_dim": 0, "inv_freq": torch.zeros(0)})
    ops.rope_kv_write_e4m3(**{**base, "qkv": base["qkv"][:, :128], "write": False})
    pretend.calls.clear()
    bad = [dict(runs=runs_of(**r)) for r in BAD_RUNS]
    bad += [dict(layer=2), dict(layer=-1), dict(num_heads=0), dict(num_heads=5), dict(rotary_dim=31), dict(rotary_dim=34), dict(rotary_dim=-2),
            dict(pairing=2), dict(inv_freq=torch.zeros(15)), dict(inv_freq=torch.zeros(16, dtype=torch.float64)), dict(qkv=base["qkv"].bfloat16()),
            dict(qkv=base["qkv"][:5]), dict(qkv=aligned(torch.zeros(6, 257))[:, :256]), dict(qkv=wide[:, 1:257]), dict(write=False),
            dict(qkv=aligned(torch.zeros(256, 6)).t()), dict(positions=torch.zeros(5, dtype=torch.int32)), dict(positions=torch.zeros(6)),
            dict(bias=torch.zeros(255)), dict(bias=torch.zeros(256, dtype=torch.float16)), dict(positions=elsewhere(torch.zeros(6, dtype=torch.int32))),
            dict(positions=torch.zeros(0, dtype=torch.int32)), dict(act="float16")]
    for b in bad:
        with pytest.raises((ops.KernelError, ValueError, KeyError)):
            ops.rope_kv_write_e4m3(**{**base, **b})
        assert not pretend.calls, b


def test_attention_that_is_refused(pretend):
    pages = ops.E4m3Pages(**pools())
    base = dict(q=aligned(torch.zeros(6, 128, dtype=torch.bfloat16)), pages=pages, layer=1, num_heads=4, window=None, scale=0.1, act="bfloat16",
                runs=runs_of())
    assert ops.attention_e4m3(**base).shape == (6, 128) and pretend.calls == ["tq_e4m3_attention"]
    pretend.calls.clear()
    bad = [dict(runs=runs_of(**r)) for r in BAD_RUNS]
    bad += [dict(layer=2), dict(num_heads=3), dict(num_heads=0), dict(window=0), dict(chunk=0), dict(softcap=0.0), dict(softcap=-1.0),
            dict(softcap=float("inf")), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=base["q"].float()), dict(q=base["q"][:, :64]),
            dict(q=base["q"][0]), dict(q=base["q"][:0]), dict(sink=torch.zeros(3)), dict(sink=torch.zeros(4, dtype=torch.bfloat16)),
            dict(distance_bias=(torch.zeros(4), torch.zeros(3))), dict(q=aligned(torch.zeros(6 * 128 + 1, dtype=torch.bfloat16))[1:].view(6, 128)),
            dict(pages=ops.E4m3Pages(**pools(weights=False)), add_weights=True), dict(sink=elsewhere(torch.zeros(4)))]
    for b in bad:
        with pytest.raises(ops.KernelError):
            ops.attention_e4m3(**{**base, **b})
        assert not pretend.calls, b


def test_choices_and_moves_that_are_refused(pretend):
    pages = ops.E4m3Pages(**pools())
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    choose = dict(pages=pages, slots=i32(0), lengths=i32(100), max_length=100, keep=10, first=4, recent=6)
    kept = ops.evict_choose(**choose)
    assert kept.shape == (1, 2, 2, 10) and kept.dtype == torch.int32
    move = dict(pages=pages, src_slots=i32(0), dst_slots=i32(1), kept=kept)
    ops.evict_move(**move)
    assert pretend.calls == ["tq_e4m3_choose", "tq_e4m3_move"]
    pretend.calls.clear()
    for b in (dict(keep=0), dict(first=5), dict(recent=-1), dict(first=-1), dict(max_length=129), dict(max_length=-1), dict(lengths=i32(1, 2)),
              dict(slots=torch.zeros(1)), dict(slots=i32(0)[0]), dict(pages=ops.E4m3Pages(**pools(weights=False))), dict(lengths=elsewhere(i32(3)))):
        with pytest.raises(ops.KernelError):
            ops.evict_choose(**{**choose, **b})
    for b in (dict(dst_slots=i32(0, 1)), dict(src_slots=i32(0).long()), dict(kept=kept[:, :1]), dict(kept=kept.long()), dict(kept=kept[0]),
              dict(kept=kept[..., :0]), dict(kept=kept[..., ::2]), dict(kept=torch.zeros(1, 2, 2, 129, dtype=torch.int32)), dict(dst_slots=elsewhere(i32(1)))):
        with pytest.raises(ops.KernelError):
            ops.evict_move(**{**move, **b})
    assert not pretend.calls


def test_pages_of_another_device_than_the_current_one(pretend, monkeypatch):
    pages = ops.E4m3Pages(**pools())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ops.KernelError, match="not the current device"):
        ops.evict_choose(pages, torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 10, 5)
    with pytest.raises(ops.KernelError, match="not the current device"):
        ops.attention_e4m3(torch.zeros(1, 128, dtype=torch.bfloat16), pages, 0, 4, None, 1.0, "bfloat16", runs_of((0,), (1,)))
    assert not pretend.calls


def test_a_sequence_that_has_let_positions_go_is_not_continued_by_its_history():
    """Its length is not the number of tokens that it has seen."""
    from turboquant_cpp_amd.engine.generate import continue_in_slot
    c = cache_of(need(), tokens=64 * 6, max_slots=2)
    slot = grown(c, 200)
    c.begin_evict(slot, 70)
    c.end_evict(slot, 70)
    engine = types.SimpleNamespace(cache=c, length=c.length)
    with pytest.raises(CacheError, match="let positions go"):
        continue_in_slot(engine, slot, list(range(100)) * 3)
