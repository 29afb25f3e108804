"""Models whose layers keep keys and values in 8 bits.

Against plain 64-bit arithmetic (``Stored``): whatever has been rounded on the way into the cache is read out of the cache's pages and
checked to be what was to be written, within the rounding (half a step: 2^-4 of the number or 2^-10 of its block's scale, once more
that where a block grew), and the plain model's attention then works on what the pages hold.  So neither a code that lies next to a
border nor a block that grew later blurs the comparison, and the bounds are those of the other engine tests: 1e-4 in 32 bits, 4 % of
the largest logit in bfloat16, 1.5 % at nine in ten.  The models have no experts, so no choice between such can turn.

Against the same engine with pages in the activations' type, for every design with layers that can: its attention finds the
numbers that the 8-bit pages hold in its own pages (``Twin``).  In 32 bits the two then agree to 1e-4 of the logits' root mean square;
in bfloat16 each may be off as those designs' own tests allow (median 3 %, nine in ten 6 %), so two differ by twice that."""
import importlib
import json

import numpy as np
import pytest
import torch

import plain_e4m3 as P
from plain_qwen2moe import PlainQwen2Moe, matvec_rows, rope_frequencies
from tiny_configs import TINY

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACTS = ["float32", "bfloat16"]
DENSE = {name: {**TINY[name][0], "mlp_only_layers": list(range(TINY[name][0]["num_hidden_layers"]))} for name in "ACD"}
MATS = "kv"


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from turboquant_cpp_amd.engine.model import write_random_model_dir
    made = {}

    def get(name, act):
        if (name, act) not in made:
            d = str(tmp_path_factory.mktemp(f"e4m3_{name}_{act}"))
            write_random_model_dir(d, DENSE[name], 3, 0.1, 0.02, act)
            made[name, act] = d, Stored(d)
        return made[name, act]
    return get


def engine_of(folder, act, max_tokens=2048, weights=False, **kw):
    from turboquant_cpp_amd.engine.model import load_model
    from turboquant_cpp_amd.engine.step import Engine
    return Engine(load_model(folder, act=act, device=DEV), max_tokens=max_tokens, kv_cache="e4m3", track_weights=weights, **kw)


class Stored(PlainQwen2Moe):
    """The plain model whose attention works on what a cache of 8 bits holds."""

    def step(self, tokens, place, position, held, act):
        """Logits of tokens at places ``place`` .. of the cache and positions ``position`` ..; ``held``: layer -> (keys and values
        {m: [G, places, hd]}, their scales).  Notes in ``received`` the weight that each place gets, layer by layer."""
        self.place, self.position, self.held, self.act, self.received = place, position, held, act, []
        return self.logits(tokens)

    def attention_layer(self, l, xb):
        p, t = f"model.layers.{l}.self_attn.", self.t
        T, g = xb.shape[0], self.nh // self.nkv
        x = {n: matvec_rows(t[p + n + "_proj.weight"], xb) + (t[p + n + "_proj.bias"] if self.has_bias else 0.0) for n in "qkv"}
        x = {n: a.view(T, -1, self.hd).numpy() for n, a in x.items()}
        freq = rope_frequencies(self.hd, self.theta)
        at = self.position + np.arange(T)
        q, k = P.rotate(x["q"], at, freq, 0), P.rotate(x["k"], at, freq, 0)
        held, scales = self.held[l]
        places = self.place + np.arange(T)
        for m, own in (("k", k), ("v", x["v"])):
            stored, scale = held[m][:, places].swapaxes(0, 1), scales[m][:, places].swapaxes(0, 1)[..., None]
            arithmetic = 1e-5 if self.act == "float32" else 0.04
            bound = 2.0 ** -4 * np.abs(own) + 2.0 ** -9 * scale + arithmetic * np.abs(own).max()
            assert (np.abs(stored - own) <= bound).all(), f"layer {l}: {m} differs by {(np.abs(stored - own) - bound).max():.2e} more than rounding"
        window = self.layer_window(l)
        out, received = np.zeros_like(q), np.zeros((self.nkv, held["k"].shape[1]))
        for h in range(self.nh):
            o, w, _s, _r = P.attend(q[:, h], held["k"][h // g], held["v"][h // g], places.tolist(), self.hd ** -0.5, window=window)
            out[:, h] = o
            received[h // g] += w
        self.received.append(received)
        return matvec_rows(t[p + "o_proj.weight"], torch.from_numpy(out.reshape(T, -1)))


def snapshot(engine, tables, slot):
    """layer -> (what the pages of ``slot`` hold, their scales), through the tables as they were during the step."""
    out = {}
    for g, table in zip(engine.cache.groups, tables):
        pages, D = g.pages8, g.key.head_dim
        row = [max(int(p), 0) for p in table[slot]]
        place = {m: np.stack([f(D, j) for j in range(pages.page_size)]) for m, f in (("k", P.k_place), ("v", P.v_place))}
        codes = {m: t[row].float().cpu().double().numpy() for m, t in (("k", pages.k), ("v", pages.v))}
        scale = {m: t[row].cpu().double().numpy() for m, t in (("k", pages.k_scale), ("v", pages.v_scale))}
        for i, e in enumerate(g.entries):
            by = {m: np.concatenate(list(scale[m][:, i]), axis=-1).repeat(P.BLOCK, axis=-1) for m in MATS}
            out[e] = {m: np.concatenate(list(codes[m][:, i][..., place[m]]), axis=-2) * by[m][..., None] for m in MATS}, by
    return out


class Watched:
    """An engine whose steps are checked against the plain model; ``weight`` is what each place should have received."""

    def __init__(self, engine, plain, act):
        self.engine, self.plain, self.act, self.weight = engine, plain, act, {}

    def step(self, slots, lists):
        cache = self.engine.cache
        starts = [cache.length(s) for s in slots]
        positions = cache.positions_of(slots, starts)
        during, kept_sync = [], cache.sync
        cache.sync = lambda: (during.append([g.host_table.copy() for g in cache.groups]), kept_sync())[1]
        try:
            logits = self.engine.step(slots, lists, [list(range(len(t))) for t in lists]).double().cpu()
        finally:
            cache.sync = kept_sync
        row, errs, top = 0, [], 0.0
        for slot, toks, start, pos in zip(slots, lists, starts, positions):
            want = self.plain.step(toks, start, pos, snapshot(self.engine, during[0], slot), self.act)
            errs += (logits[row:row + len(toks)] - want).abs().max(dim=-1).values.tolist()
            top = max(top, want.abs().max().item())
            row += len(toks)
            for l, received in enumerate(self.plain.received):
                have = self.weight.setdefault((slot, l), np.zeros_like(received))
                have[:, start:start + len(toks)] = 0.0
                have += received
        errs = np.array(errs)
        if self.act == "float32":
            assert errs.max() < 1e-4, f"logits differ by {errs.max():.2e} at row {errs.argmax()}"
        else:
            assert errs.max() < 0.04 * top and np.quantile(errs, 0.9) < 0.015 * top, (errs.max() / top, np.quantile(errs, 0.9) / top)
        return logits

    def check_weights(self, slot):
        n = self.engine.length(slot)
        for g in self.engine.cache.groups:
            row = g.host_table[slot]
            have = g.pages8.weight[[max(int(p), 0) for p in row]].cpu().double().numpy()
            for i, e in enumerate(g.entries):
                got = np.concatenate(list(have[:, i]), axis=-1)[:, :n]
                bound = 1e-3 if self.act == "float32" else 0.05
                assert np.abs(got - self.weight[slot, e][:, :n]).max() <= bound * max(1.0, self.weight[slot, e][:, :n].max()), f"layer {e}"


def tokens(V, n, seed):
    return torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("name", ["A", "C", "D"])
def test_steps_against_plain_arithmetic(folders, name, act):
    """Prompts of unequal lengths together, one that goes on in portions, single tokens beside each other, a slot used again."""
    folder, plain = folders(name, act)
    engine = engine_of(folder, act, use_graphs=False)
    assert all(g.key.e4m3 for g in engine.cache.groups) and engine.native is None
    w, V = Watched(engine, plain, act), engine.vocab_size
    a, b = engine.open(2)
    w.step([a, b], [tokens(V, 100, 1), tokens(V, 37, 2)])
    w.step([b, a], [tokens(V, 30, 3), tokens(V, 1, 4)])
    for i in range(4):
        w.step([a, b], [[5 + i], [9 + i]])
    engine.close([a])
    a = engine.open(1)[0]
    w.step([a], [[1]])
    w.step([a, b], [tokens(V, 17, 5), [3]])


@pytest.mark.parametrize("act", ACTS)
def test_letting_positions_go_against_plain_arithmetic(folders, act):
    """Weights that positions receive, which stay, the pages behind a move bit by bit, and the steps after it, twice."""
    folder, plain = folders("A", act)
    engine = engine_of(folder, act, weights=True, use_graphs=False)
    w, V = Watched(engine, plain, act), engine.vocab_size
    assert engine.no_eviction() is None
    a, b = engine.open(2)
    w.step([a, b], [tokens(V, 150, 1), tokens(V, 40, 2)])
    for i in range(3):
        w.step([a, b], [[5 + i], [9 + i]])
    for keep, first, recent in ((70, 4, 20), (33, 0, 0)):
        w.check_weights(a)
        w.check_weights(b)
        g, length = engine.cache.groups[0], engine.length(a)
        before = P.read_pages(g.pages8, g.key.head_dim)
        spare = g.spare
        kept = np.array([[P.choose(before.weight[a, l, h], length, keep, first, recent) for h in range(g.key.num_kv_heads)]
                         for l in range(len(g.entries))])
        P.move(before, a, spare, kept, 64)
        position = length + engine.cache.slots[a].dropped
        engine.evict([a, b], keep, first=first, recent=recent) if keep == 33 else engine.evict([a], keep, first=first, recent=recent)
        after = P.read_pages(g.pages8, g.key.head_dim)
        for m in MATS:
            assert np.array_equal(after.code[m][a][:, :, :keep], before.code[m][spare][:, :, :keep])
            assert np.array_equal(after.scale[m][a][..., :-(-keep // 16)], before.scale[m][spare][..., :-(-keep // 16)])
        assert np.array_equal(after.weight[a][..., :keep], before.weight[spare][..., :keep])
        assert engine.length(a) == keep and engine.cache.positions_of([a], [keep]) == [position]
        for l in range(len(g.entries)):
            w.weight[a, l] = after.weight[a, l].copy()
            w.weight[b, l] = after.weight[b, l].copy()
        for i in range(3):
            w.step([a, b], [[15 + i], [19 + i]])
        w.step([a], [tokens(V, 21, 7)])
    engine.close([a, b])
    assert all(g.pool.n_free == g.pool.n_pages for g in engine.cache.groups)


@pytest.mark.parametrize("act", ACTS)
def test_replayed_steps_have_the_bits_of_eager_ones(folders, act):
    """Decode steps as graphs, with positions let go between replays, other sequences in the slots and prompts in between."""
    folder, _plain = folders("A", act)
    runs = []
    for graphs in (False, True):
        engine = engine_of(folder, act, weights=True, use_graphs=graphs)
        V, out = engine.vocab_size, []
        a, b = engine.open(2)
        engine.step([a, b], [tokens(V, 150, 1), tokens(V, 63, 2)])
        for i in range(6):
            out.append(engine.step([a, b], [[5 + i], [9 + i]]))
        engine.evict([a, b], 64, recent=32)
        for i in range(4):
            out.append(engine.step([a, b], [[25 + i], [29 + i]]))
            out.append(engine.step_from_device([b, a], torch.tensor([7 + i, 8 + i], dtype=torch.int32, device=DEV)).clone())
        c = engine.open(1)[0]
        out.append(engine.step([c], [tokens(V, 30, 5)]))
        for i in range(3):
            out.append(engine.step([c, a], [[i], [i]]))
        assert graphs == bool(engine.graphs and engine.graphs.graphs)
        out += [g.pages8.weight.clone() for g in engine.cache.groups]
        runs.append(out)
    assert all(torch.equal(x, y) for x, y in zip(*runs, strict=True))


@pytest.mark.parametrize("act", ACTS)
def test_a_sequence_that_is_full_goes_on(folders, act):
    """Generation through the entry point far beyond the context, in a batch with one that ends before it: the tokens of the same
    steps made one by one."""
    from turboquant_cpp_amd import Model
    from turboquant_cpp_amd.engine.generate import kept_when_full
    folder, _plain = folders("A", act)
    V = DENSE["A"]["vocab_size"]
    prompts, n, ctx = [tokens(V, 60, 1), tokens(V, 9, 2)], 300, 128
    options = dict(temperature=0.0, rep_penalty=1.0, stop_tokens=[], max_batch=2, context_length=ctx, dtype=act, kv_cache="e4m3")
    with Model(folder, when_full="evict", max_tokens=n, **options) as model:
        got = model.generate_detailed(prompts, loop_detection=False)
        assert [r.finish_reason for r in got] == ["length"] * 2 and [len(r.tokens) for r in got] == [n] * 2
        assert all(r.cached_positions <= ctx for r in got) and model.generate_detailed([tokens(V, ctx + 1, 3)])[0].finish_reason == "context"
        ended = model.generate_detailed(prompts, loop_detection=False, when_full="end")
        assert [r.finish_reason for r in ended] == ["context"] * 2 and all(r.tokens == g.tokens[:len(r.tokens)] for r, g in zip(ended, got))
    engine = engine_of(folder, act, weights=True, use_graphs=False, max_positions=ctx, max_slots=2, max_tokens=2 * ctx + 64)
    slots = engine.open(2)
    out, logits = [[], []], engine.step(slots, prompts)
    for _ in range(n - 1):
        for o, t in zip(out, logits.argmax(-1).tolist()):
            o.append(t)
        engine.evict([s for s in slots if engine.length(s) == ctx], *kept_when_full(ctx))
        logits = engine.step(slots, [[o[-1]] for o in out])
    for o, t in zip(out, logits.argmax(-1).tolist()):
        o.append(t)
    assert out == [r.tokens for r in got]


@pytest.mark.parametrize("act", ACTS)
def test_a_conversation_saved_and_loaded(folders, act, tmp_path):
    from turboquant_cpp_amd import Model
    folder, _plain = folders("C", act)
    V, path = DENSE["C"]["vocab_size"], str(tmp_path / "kv.safetensors")
    options = dict(temperature=0.0, stop_tokens=[], max_tokens=12, context_length=512, dtype=act, max_batch=2)
    history = tokens(V, 130, 1)
    with Model(folder, kv_cache="e4m3", **options) as model:
        model.feed(history)
        model.save_context(path)
        want = model.chat(history + [5, 6])
    with Model(folder, kv_cache="e4m3", **options) as model:
        model.load_context(path)
        assert model.chat_tokens == history
        assert model.chat(history + [5, 6]) == want
    from turboquant_cpp_amd.engine.step import Engine
    with Model(folder, kv_cache="e4m3", **options) as model:      # what each position has received goes along, or starts at nothing
        weighing = Engine(model._model, 1024, kv_cache="e4m3", track_weights=True)
        slot = weighing.open(1)[0]
        weighing.step([slot], [history])
        saved = weighing.cache.export_slot(slot)
        again, bare = weighing.cache.import_slot(saved), model.engine.cache.import_slot(saved)
        for a, b in zip(weighing.cache.export_slot(again)["groups"], saved["groups"]):
            assert all(torch.equal(a[n], b[n]) for n in ("keys", "values", "key_scales", "value_scales", "weights"))
        for a, b in zip(model.engine.cache.export_slot(bare)["groups"], saved["groups"]):
            assert torch.equal(a["keys"], b["keys"]) and "weights" not in a
        for a in weighing.cache.export_slot(weighing.cache.import_slot(model.engine.cache.export_slot(bare)))["groups"]:
            assert not a["weights"].any()
    with Model(folder, **options) as model, pytest.raises(RuntimeError, match="another layout"):
        model.load_context(path)
    with Model(folder, **options) as model:
        model.feed(history)
        model.save_context(path)
    with Model(folder, kv_cache="e4m3", **options) as model, pytest.raises(RuntimeError, match="another layout"):
        model.load_context(path)


def test_what_a_model_refuses(folders):
    from turboquant_cpp_amd import Model
    from turboquant_cpp_amd.cache.paged import CacheError
    from turboquant_cpp_amd.engine.step import StepError
    folder, _plain = folders("C", "bfloat16")      # layers with a window
    with pytest.raises(ValueError, match="window"):
        Model(folder, kv_cache="e4m3", when_full="evict")
    with pytest.raises(CacheError, match="8 bits alone"):
        Model(folder, when_full="evict")
    with pytest.raises(CacheError, match="'same' or 'e4m3'"):
        Model(folder, kv_cache="int4")
    with pytest.raises(ValueError, match="when_full"):
        Model(folder, when_full="shift")
    engine = engine_of(folders("A", "bfloat16")[0], "bfloat16", weights=True)
    slot = engine.open(1)[0]
    engine.step([slot], [[1] * 50])
    for args in ((10, 5, 6), (0, 0, 0), (10, -1, 2)):
        with pytest.raises(StepError):
            engine.evict([slot], *args)
    with pytest.raises(StepError, match="twice"):
        engine.evict([slot, slot], 10)
    engine.evict([slot], 50)      # nothing to let go
    assert engine.length(slot) == 50


def test_the_command_line(folders, capsys):
    from turboquant_cpp_amd import cli
    folder, _plain = folders("A", "bfloat16")
    assert cli.main([folder, "-p", "1,2,3", "-n", "200", "-T", "0", "--ctx", "64", "--kv-cache", "e4m3", "--when-full", "evict", "-M", "--json",
                     "--max-batch", "1", "--rep-penalty", "1.5", "--stop-id", "-1"]) == 0
    out, err = capsys.readouterr()
    assert json.loads(out)[0]["finish_reason"] in ("length", "loop") and "kv=e4m3" in err and "KV type:              e4m3" in err
    # 2 layers x 4 kv heads x 16 numbers: bytes, and a quarter of one for the scale (and 4 for the weight) per kv head
    assert f"Per-token V (e4m3): {2 * 4 * (16 + 0.25) / 1024:.2f} KB" in err
    assert cli.main([folder, "-p", "1,2,3;4,5", "-n", "4", "-T", "0", "--ctx", "64", "--kv-cache", "e4m3", "--profile"]) == 0
    assert "attention_e4m3" in capsys.readouterr().err


# ------------------------------------------------------------------------------------------------ every design
def case_of(design, case, folder, act):
    c = importlib.import_module(f"{design}_cases")
    c.write_folder(folder, c.CASES[case], c.tensors(c.CASES[case], 0))
    return folder, c.CASES[case]["vocab"]


class Twin:
    """Runs an engine with pages of 8 bits, and one with pages of the activations' type whose attention finds in them what the
    former's hold."""

    def __init__(self, monkeypatch, folder, act):
        from turboquant_cpp_amd.csrc import ops
        from turboquant_cpp_amd.engine.model import load_model
        from turboquant_cpp_amd.engine.step import Engine
        monkeypatch.setenv("TQ_HOST", "python")
        model = load_model(folder, act=act, device=DEV)
        self.eight = Engine(model, max_tokens=1024, use_graphs=False, kv_cache="e4m3", track_weights=True)
        self.same = Engine(model, max_tokens=1024, use_graphs=False)
        self.act, self.seen, self.groups = act, [], {}
        for g in self.eight.cache.groups:
            if g.key.e4m3:
                for e in g.entries:
                    self.groups[e] = g
        self.attention, self.attention_e4m3 = ops.attention, ops.attention_e4m3
        monkeypatch.setattr(ops, "attention_e4m3", self.watch)
        monkeypatch.setattr(ops, "attention", self.put)

    def watch(self, q, pages, layer, *args, **kw):
        out = self.attention_e4m3(q, pages, layer, *args, **kw)
        self.seen.append((P.read_pages(pages, pages.head_dim), layer))
        return out

    def put(self, q, k_pages, v_pages, layer_offset, positions, slot_of_token, table, page_size, page_stride, nh, nkv, hd, *args, **kw):
        where = [(g, e) for g in self.same.cache.groups if k_pages.data_ptr() == g.k_pages.data_ptr()
                 for e in g.entries if g.offset_of(e) == layer_offset and e in self.groups]
        if where:
            (g, e), (held, layer) = where[0], self.seen.pop(0)
            assert self.groups[e].entries.index(e) == layer
            pools = {"k": k_pages.view(-1, page_stride)[:, layer_offset:].unflatten(1, (-1, hd))[:, :nkv * page_size].unflatten(1, (nkv, page_size)),
                     "v": v_pages.view(-1, page_stride)[:, layer_offset:].unflatten(1, (-1, page_size))[:, :nkv * hd].unflatten(1, (nkv, hd)).transpose(2, 3)}
            ends = {}
            for s, p in zip(slot_of_token.tolist(), positions.tolist()):
                ends[s] = max(ends.get(s, 0), p + 1)
            for s, end in ends.items():
                for i, pg in enumerate(table[s].tolist()):
                    n = min(page_size, end - i * page_size)
                    if pg < 0 or n <= 0:
                        continue
                    for m in MATS:
                        lo = i * page_size
                        new = np.stack([held.values(m, s, layer, h)[lo:lo + n] for h in range(nkv)])
                        scale = held.scale[m][s, layer].repeat(P.BLOCK, axis=-1)[:, lo:lo + n, None]
                        own = pools[m][pg, :, :n].double().cpu().numpy()
                        slack = 1e-5 if self.act == "float32" else 0.04
                        assert (np.abs(own - new) <= 2.0 ** -4 * np.abs(own) + 2.0 ** -9 * scale + slack * np.abs(own).max()).all(), (e, m, s, i)
                        pools[m][pg, :, :n] = torch.from_numpy(new).to(pools[m])
        return self.attention(q, k_pages, v_pages, layer_offset, positions, slot_of_token, table, page_size, page_stride, nh, nkv, hd, *args, **kw)

    def step(self, slots, lists):
        wants = [list(range(len(t))) for t in lists]
        got, want = (e.step(slots, lists, wants).double().cpu() for e in (self.eight, self.same))
        assert not self.seen
        d = got - want
        d = d - d.mean(dim=1, keepdim=True)
        scale = (want - want.mean(dim=1, keepdim=True)).square().mean().sqrt()
        return (d.square().mean(dim=1).sqrt() / scale).tolist()


@pytest.mark.parametrize("design,case,act", [
    ("felepel", "attention_only", "float32"), ("felepel", "attention_only", "bfloat16"), ("felepel", "experts", "float32"),
    ("felepel", "odd", "float32"), ("gokezen", "attention_only", "float32"), ("gokezen", "attention_only", "bfloat16"),
    ("gokezen", "loop_only", "float32"), ("gokezen", "odd", "float32"), ("gokezen", "wide", "float32"), ("taminex", "attention_only", "float32"),
    ("taminex", "attention_only", "bfloat16"), ("taminex", "odd", "float32"), ("taminex", "regular", "float32")])
def test_designs_against_their_pages_in_the_activations_type(monkeypatch, tmp_path, design, case, act):
    folder, V = case_of(design, case, str(tmp_path / "m"), act)
    twin = Twin(monkeypatch, folder, act)
    a, b = twin.eight.open(2)
    assert twin.same.open(2) == [a, b]
    errs = twin.step([a, b], [tokens(V, 100, 1), tokens(V, 37, 2)])
    errs += twin.step([b, a], [tokens(V, 30, 3), tokens(V, 1, 4)])
    for i in range(4):
        errs += twin.step([a, b], [[5 + i], [9 + i]])
    if act == "float32":
        assert max(errs) < 1e-4, f"row {int(np.argmax(errs))} of {len(errs)} differs by {max(errs):.2e}"
    else:
        assert np.median(errs) < 0.06 and np.quantile(errs, 0.9) < 0.12, (np.median(errs), np.quantile(errs, 0.9))


def test_a_conversation_that_has_let_positions_go(folders, tmp_path):
    """Its cache is not what it has seen: it starts over, cannot be continued in its slot, and is not saved."""
    from turboquant_cpp_amd import Model
    from turboquant_cpp_amd.cache.paged import CacheError
    from turboquant_cpp_amd.engine.generate import continue_in_slot
    folder, _plain = folders("A", "bfloat16")
    V = DENSE["A"]["vocab_size"]
    history, path = tokens(V, 100, 1), str(tmp_path / "kv.safetensors")
    with Model(folder, kv_cache="e4m3", when_full="evict", temperature=0.0, stop_tokens=[], max_tokens=6, context_length=256, max_batch=2) as model:
        want = model.chat(history + [5, 6])
        for again in (history + [5, 6], history + [5, 6] + want):
            model.reset_chat()
            model.feed(history)
            model.engine.evict([model._chat_slot], 50)
            with pytest.raises(RuntimeError, match="let positions go"):
                model.save_context(path)
            with pytest.raises(CacheError, match="let positions go"):
                continue_in_slot(model.engine, model._chat_slot, again)
            fed = model.feed(again)
            assert fed == len(again) and model.engine.cache.slots[model._chat_slot].dropped == 0
            model.reset_chat()
            model.feed(history)
            model.engine.evict([model._chat_slot], 50)
            assert model.chat(history + [5, 6]) == want


def test_whose_turn_it_is_to_end_where_nothing_is_free(folders):
    """Two sequences need pages at once, one to let positions go and the other to grow: the longer one ends, its pages let the other go on."""
    from turboquant_cpp_amd.engine.generate import GenerationOptions, generate
    folder, _plain = folders("A", "bfloat16")
    engine = engine_of(folder, "bfloat16", max_tokens=192, weights=True, max_slots=2, max_positions=100)
    V = engine.vocab_size
    options = GenerationOptions(max_tokens=20, temperature=0.0, rep_penalty=1.0, loop_detection=False, max_batch=2, when_full="evict")
    got = generate(engine, [tokens(V, 99, 1), tokens(V, 63, 2)], options)
    assert [r.finish_reason for r in got] == ["context", "length"] and [len(r.tokens) for r in got] == [2, 20]
    got = generate(engine, [tokens(V, 63, 2), tokens(V, 99, 1)], options)
    assert [r.finish_reason for r in got] == ["length", "context"]
