"""Calls of the operators of the 8-bit cache, as a user of this library makes them: the write that rotates queries and keys and
fills the pages, attention over the pages (prompts and single tokens, with and without the sums of the weights that each position
receives), and eviction by those sums.

A page holds keys and values as e4m3 codes (``torch.float8_e4m3fn``) with one scale, a power of two, for each block of 16
positions of a layer's kv head:

* pools ``k``, ``v`` [pages, layers, kv heads, page_size * head_dim]; ``k_scale``, ``v_scale`` float32 [pages, layers, kv heads,
  page_size / 16]; ``weight`` float32 [pages, layers, kv heads, page_size]; ``table`` int32 [slots, logical pages];
* within a tile of 64 positions keys lie [head_dim / 16][64 positions][16 numbers] and values [head_dim][4][4][4], where position
  16 j + 4 c + i of the tile stands at [c][j][i].

A block's scale is the smallest power of two, 2^-100 at least, whose 448 fold is no smaller than the block's largest magnitude; a
block that grows by a larger number takes the larger scale, and the codes it holds are rounded to it.

Weights of attention start from zero in every pass (a request's cache does), so that a pass can be repeated on the same state.
"""
from __future__ import annotations

import math
import zlib

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = 16
LEAST = -100


# ------------------------------------------------------------------------------------------------------------------ cases

def listed():
    """Head layouts are those of the Qwen1.5-MoE-A2.7B (16 heads, 16 kv heads, 128) and Qwen2-57B-A14B (28, 4, 128) sizes that the
    library is measured at, and of smaller models."""
    write = dict(op="write", act="bfloat16", rotary=128, pairing=0, bias=False, page=64)
    attend = dict(op="attend", act="bfloat16", window=0, softcap=0.0, sink=False, weights=False, page=64)
    return [
        # eight running conversations write one decoded token each, most of them inside a block
        dict(write, name="write_tokens_8", seqs=8, shortest=1, longest=1, past=4001, heads=16, kv_heads=16, dim=128),
        # a long prompt of one request
        dict(write, name="write_prompt_4096", seqs=1, shortest=4096, longest=4096, past=0, heads=16, kv_heads=16, dim=128),
        # ragged follow-ups behind what the conversations hold, with the product's bias added here
        dict(write, name="write_ragged_12", seqs=12, shortest=3, longest=900, past=1205, heads=28, kv_heads=4, dim=128, bias=True),
        # the 32-bit path, neighbouring pairs, part of a head rotated
        dict(write, name="write_f32_partial", act="float32", seqs=5, shortest=1, longest=333, past=77, heads=6, kv_heads=2, dim=80,
             rotary=32, pairing=1, bias=False, page=128),
        # the reply of one short conversation: latency
        dict(attend, name="token_1_short", kind="token", seqs=1, shortest=500, longest=500, heads=16, kv_heads=16, dim=128),
        # eight conversations at the context that the library's headline is measured at
        dict(attend, name="token_8_at_8192", kind="token", seqs=8, shortest=8192, longest=8192, heads=16, kv_heads=16, dim=128),
        # a full batch of unequal conversations whose caches will be evicted: weights are kept
        dict(attend, name="token_64_weights", kind="token", seqs=64, shortest=300, longest=4100, heads=28, kv_heads=4, dim=128,
             weights=True),
        # one prompt
        dict(attend, name="prompt_2048", kind="prompt", seqs=1, shortest=2048, longest=2048, past=0, heads=16, kv_heads=16, dim=128),
        # ragged turns behind long conversations, with weights kept and capped scores
        dict(attend, name="prompt_ragged_weights", kind="prompt", seqs=3, shortest=130, longest=2311, past=3907, heads=28, kv_heads=4,
             dim=128, softcap=50.0, weights=True),
        # the 32-bit path behind a window, with a sink
        dict(attend, name="prompt_f32_window", kind="prompt", act="float32", seqs=2, shortest=300, longest=1100, past=450, heads=8,
             kv_heads=2, dim=64, window=256, sink=True),
        # a conversation of a small model goes back to half its context
        dict(op="evict", name="evict_one", seqs=1, shortest=1500, longest=1500, keep=750, first=4, recent=128, layers=2, kv_heads=4,
             dim=64, page=64),
        # a batch at its context's end, several layers at once
        dict(op="evict", name="evict_batch", seqs=8, shortest=7900, longest=8192, keep=4096, first=4, recent=1024, layers=6,
             kv_heads=16, dim=128, page=64),
    ]


def draw(rng):
    """One more call: sizes spread over their logarithm, odd ones among them."""
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads = rng.choice([(16, 16), (28, 4), (8, 2), (6, 3), (12, 1), (20, 5)])
    dim = rng.choice([32, 48, 64, 80, 96, 128, 128, 128, 192, 256])
    act = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    page = rng.choice([64, 64, 128])
    op = rng.choice(["write", "token", "token", "prompt", "prompt", "evict"])
    if op == "write":
        seqs, longest = size(1, 24), size(1, 2000)
        while seqs * longest > 8000:
            seqs = max(1, seqs // 2)
        return dict(op="write", act=act, seqs=seqs, shortest=rng.randint(1, longest), longest=longest, past=rng.choice([0, size(1, 3000)]),
                    heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([0, dim // 4 * 2, dim]), pairing=rng.randint(0, 1),
                    bias=rng.random() < 0.5, page=page)
    more = dict(window=rng.choice([0, 0, size(20, 2000)]), softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.3,
                weights=rng.random() < 0.4, page=page)
    if op == "token":
        seqs, longest = size(1, 48), size(1, 12000)
        while seqs * longest * kv_heads * dim > 8 * 8192 * 16 * 128:
            seqs, longest = max(1, seqs // 2), max(1, longest * 3 // 4)
        return dict(op="attend", kind="token", act=act, seqs=seqs, shortest=rng.randint(1, longest), longest=longest, heads=heads,
                    kv_heads=kv_heads, dim=dim, **more)
    if op == "prompt":
        seqs, longest, past = size(1, 5), size(2, 2200), rng.choice([0, 0, size(1, 2500)])
        while seqs * longest * (longest + past) * heads * dim > 3 * 2311 * 6218 * 16 * 128 // 2:
            seqs, longest = max(1, seqs - 1), max(2, longest * 3 // 4)
        return dict(op="attend", kind="prompt", act=act, seqs=seqs, shortest=rng.randint(1, longest), longest=longest, past=past,
                    heads=heads, kv_heads=kv_heads, dim=dim, **more)
    seqs, longest, layers = size(1, 12), size(40, 8000), rng.randint(1, 6)
    while seqs * longest * layers * kv_heads * dim > 8 * 8192 * 6 * 16 * 128:
        seqs = max(1, seqs // 2)
    shortest = rng.randint(max(1, longest // 2), longest)
    keep = rng.randint(max(1, shortest // 3), shortest)
    first = rng.choice([0, min(4, keep)])
    return dict(op="evict", seqs=seqs, shortest=shortest, longest=longest, keep=keep, first=first, recent=rng.randint(0, keep - first),
                layers=layers, kv_heads=kv_heads, dim=dim, page=page)


def _lengths(case, name="longest"):
    """Unequal sizes from the shortest to the longest, in a mixed order."""
    n = case["seqs"]
    sizes = np.round(np.linspace(case["longest"], case["shortest"], n)).astype(np.int64)
    return [int(v) for v in np.random.RandomState(7).permutation(sizes)]


def _past(case):
    """What the sequences hold before the call: as long as ``past`` at the most, no two alike."""
    top = case.get("past", 0)
    return [max(0, top - 37 * i - (top // 9) * i) if top else 0 for i in range(case["seqs"])]


# ------------------------------------------------------------------------------------------------------------------ inputs

def _places(case, capacity, seed, slots):
    """A page table whose pages lie in a mixed order, and the number of pages (one more than the table names)."""
    per = -(-capacity // case["page"])
    order = np.random.RandomState(seed % (1 << 31)).permutation(slots * per) + 1
    return torch.from_numpy(order.reshape(slots, per).astype(np.int32)).to(DEVICE), slots * per + 1


def _quantise(x):
    """[..., rows, dim] -> (codes, scales): blocks of 16 rows."""
    y = x.unflatten(-2, (-1, BLOCK))
    scale = _scale_of(y.abs().amax((-1, -2)))
    return (y / scale[..., None, None]).flatten(-3, -2).to(torch.float8_e4m3fn), scale


def _scale_of(top):
    """The smallest power of two, 2^LEAST at least, with top <= 448 of it."""
    part, power = torch.frexp(top)                  # top = part 2^power, part in [0.5, 1); 448 = 0.875 2^9
    power = torch.where(part > 0.875, power - 8, power - 9).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, power, torch.full_like(power, LEAST)))


def _random_rows(g, *shape):
    """Keys or values as models have them: numbers around zero, a few dimensions of a head much larger than the others."""
    x = torch.randn(shape, generator=g, device=DEVICE)
    loud = torch.rand(shape[-1], generator=g, device=DEVICE) < 0.04
    return x * torch.where(loud, 6.0, 1.0) * torch.exp2(torch.randn(shape[:-1], generator=g, device=DEVICE) * 0.4)[..., None]


def _bytes(t):
    return t.view(torch.uint8)


def _k_layout(rows, page):
    """[..., page, dim] codes -> [..., page * dim] as keys lie in a page."""
    x = _bytes(rows).unflatten(-1, (-1, 16)).unflatten(-3, (page // 64, 64)).transpose(-2, -3)
    return x.flatten(-4).contiguous().view(torch.float8_e4m3fn)


def _v_layout(rows, page):
    x = _bytes(rows).unflatten(-2, (page // 64, 4, 4, 4))           # [tile, j, c, i, dim]
    x = x.permute(*range(x.dim() - 5), -5, -1, -3, -4, -2)           # [tile, dim, c, j, i]
    return x.flatten(-5).contiguous().view(torch.float8_e4m3fn)


def _k_rows(pages, dim):
    """[..., page * dim] as keys lie -> [..., page, dim]"""
    x = _bytes(pages).unflatten(-1, (-1, dim // 16, 64, 16)).transpose(-2, -3)
    return x.flatten(-2).flatten(-3, -2).contiguous().view(torch.float8_e4m3fn)


def _v_rows(pages, dim):
    x = _bytes(pages).unflatten(-1, (-1, dim, 4, 4, 4))              # [tile, dim, c, j, i]
    x = x.permute(*range(x.dim() - 5), -5, -2, -3, -1, -4)           # [tile, j, c, i, dim]
    return x.flatten(-5, -2).contiguous().view(torch.float8_e4m3fn)


def _pools(case, layers, n_pages, g, filled):
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    out = {}
    for name, layout in (("k", _k_layout), ("v", _v_layout)):
        if filled:
            codes, scale = _quantise(_random_rows(g, n_pages, layers, G, page, D))
            out[name], out[name + "_scale"] = layout(codes, page), scale
        else:
            out[name] = torch.zeros((n_pages, layers, G, page * D), dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn)
            out[name + "_scale"] = torch.zeros((n_pages, layers, G, page // BLOCK), device=DEVICE)
    return out


def _runs(slots, start, new):
    """A step's tokens as runs of consecutive positions, one per sequence, as the step function describes them."""
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    cu = np.concatenate([[0], np.cumsum(new)])
    return {"cu_seqlens": dev(cu.tolist()), "slots": dev(slots), "start": dev(start), "max_new": max(new), "min_new": min(new),
            "max_end": max(a + n for a, n in zip(start, new)), "decode": max(new) == 1}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed((seed * 1000003 + zlib.crc32(case["op"].encode())) % (1 << 62))
    new, B = _lengths(case), case["seqs"]
    G, D = case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["op"] == "evict":
        slots = [int(v) for v in np.random.RandomState(3).permutation(2 * B)]       # half of them have the kept positions behind it
        table, n_pages = _places(case, max(new), seed, 2 * B)
        state |= _pools(case, case["layers"], n_pages, g, filled=True)
        # a few positions get most of the weight, as trained heads have it; whole runs of positions get none at all
        w = torch.exp2(torch.randn((n_pages, case["layers"], G, case["page"]), generator=g, device=DEVICE) * 4)
        state["weight"] = torch.where(torch.rand(w.shape, generator=g, device=DEVICE) < 0.1, torch.zeros_like(w), w)
        state |= {"table": table, "src": torch.tensor(slots[:B], dtype=torch.int32, device=DEVICE),
                  "dst": torch.tensor(slots[B:], dtype=torch.int32, device=DEVICE),
                  "lengths": torch.tensor(new, dtype=torch.int32, device=DEVICE), "max_length": max(new)}
        return state
    past = [n - 1 for n in new] if case.get("kind") == "token" else _past(case)
    if case.get("kind") == "token":
        new = [1] * B
    slots = [int(v) for v in np.random.RandomState(5).permutation(B + 1)[:B]]
    runs = _runs(slots, past, new)
    table, n_pages = _places(case, runs["max_end"], seed, B + 1)
    T, H = sum(new), case["heads"]
    state |= {"runs": runs, "table": table, "sizes": new, "start": past}
    state["seq"] = torch.repeat_interleave(torch.arange(B), torch.tensor(new)).to(DEVICE)
    state["row"] = torch.cat([torch.arange(a, a + n) for a, n in zip(past, new)]).to(DEVICE)
    state |= _pools(case, 2, n_pages, g, filled=case["op"] == "attend" or max(past) > 0)
    state["layer"] = 1
    if case["op"] == "write":
        state["qkv"] = torch.cat([_random_rows(g, T, H + 2 * G, D).flatten(1)])
        state["bias"] = torch.randn((H + 2 * G) * D, generator=g, device=DEVICE) * 0.5 if case["bias"] else None
        # positions run ahead of the places where a sequence has let positions go
        state["positions"] = (state["row"] + 1000 * (state["seq"] % 2)).to(torch.int32)
        n = case["rotary"] // 2
        state["freq"] = (1e6 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().to(DEVICE)
    else:
        state["q"] = (torch.randn((T, H * D), generator=g, device=DEVICE) * 0.6).to(DTYPES[case["act"]])
        state["sink"] = torch.randn(H, generator=g, device=DEVICE) + 1.0 if case["sink"] else None
        state["weight"] = torch.zeros((n_pages, 2, G, case["page"]), device=DEVICE) if case["weights"] else None
    return state


# ------------------------------------------------------------------------------------------------------------------ passes

def run(s):
    c = s["case"]
    if own:
        return _OWN[c["op"]](s, c)
    return _PLAIN[c["op"]](s, c)


def _own_pages(s):
    from turboquant_cpp_amd.csrc import ops
    return ops, ops.E4m3Pages(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s.get("weight"))


def _own_write(s, c):
    ops, pages = _own_pages(s)
    q = ops.rope_kv_write_e4m3(s["qkv"], s["positions"], s["freq"], c["pairing"], c["rotary"], pages, s["layer"], c["heads"], c["act"],
                               s["runs"], bias=s["bias"])
    return [q, s["k"], s["v"], s["k_scale"], s["v_scale"]]


def _own_attend(s, c):
    ops, pages = _own_pages(s)
    if c["weights"]:
        s["weight"].zero_()
    out = ops.attention_e4m3(s["q"], pages, s["layer"], c["heads"], c["window"] or None, c["dim"] ** -0.5, c["act"], s["runs"],
                             softcap=c["softcap"] or None, sink=s["sink"], add_weights=c["weights"])
    return [out, s["weight"]] if c["weights"] else [out]


def _own_evict(s, c):
    ops, pages = _own_pages(s)
    kept = ops.evict_choose(pages, s["src"], s["lengths"], s["max_length"], c["keep"], first=c["first"], recent=c["recent"])
    ops.evict_move(pages, s["src"], s["dst"], kept)
    return [kept, s["k"], s["v"], s["k_scale"], s["v_scale"], s["weight"]]


_OWN = {"write": _own_write, "attend": _own_attend, "evict": _own_evict}


def _plain_write(s, c):
    T, H, G, D, page, layer = s["qkv"].shape[0], c["heads"], c["kv_heads"], c["dim"], c["page"], s["layer"]
    x = (s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]).view(T, H + 2 * G, D)
    qk, n = x[:, :H + G], c["rotary"] // 2
    if n:
        angle = s["positions"].double()[:, None] * s["freq"].double()
        cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
        a, b = (qk[..., :n], qk[..., n:2 * n]) if c["pairing"] == 0 else (qk[..., 0:2 * n:2], qk[..., 1:2 * n:2])
        turned = (a * cos - b * sin, a * sin + b * cos)
        turned = torch.cat(turned, -1) if c["pairing"] == 0 else torch.stack(turned, -1).flatten(-2)
        qk = torch.cat([turned, qk[..., 2 * n:]], -1)
    q = qk[:, :H].reshape(T, H * D).to(DTYPES[c["act"]])
    # the pages that the step's tokens fall into, each brought to rows, changed and laid out again
    slot = s["runs"]["slots"].long()[s["seq"]]
    place = s["table"][slot, s["row"] // page].long()
    touched, at = torch.unique(place, return_inverse=True)
    at_row = at * page + s["row"] % page
    block = at_row // BLOCK
    n_blocks = touched.numel() * page // BLOCK
    is_new = torch.zeros(touched.numel() * page, dtype=torch.bool, device=DEVICE).index_fill_(0, at_row, True)
    # rows of a block that the sequence held before: those before the step's first token, where that lies inside the block
    first = s["runs"]["start"].long()[s["seq"]]
    held = torch.zeros(n_blocks, dtype=torch.long, device=DEVICE)
    held[block] = torch.where(s["row"] // BLOCK == first // BLOCK, first % BLOCK, torch.zeros_like(first))
    is_old = (torch.arange(BLOCK, device=DEVICE) < held[:, None]) & ~is_new.view(-1, BLOCK)
    for name, vals, to_rows, to_pages in (("k", qk[:, H:], _k_rows, _k_layout), ("v", x[:, H + G:], _v_rows, _v_layout)):
        pool, scale = _bytes(s[name])[:, layer], s[name + "_scale"][:, layer]
        codes = to_rows(pool[touched].view(torch.float8_e4m3fn), D).transpose(1, 2).reshape(-1, G, D)      # [rows, G, D]
        was = scale[touched].transpose(1, 2).reshape(n_blocks, G)
        top = torch.zeros((n_blocks, G), device=DEVICE).index_reduce_(0, block, vals.abs().amax(-1), "amax")
        now = torch.maximum(_scale_of(top), torch.where(held[:, None] > 0, was, torch.zeros_like(was)))
        changed = torch.zeros(n_blocks, dtype=torch.bool, device=DEVICE).index_fill_(0, block, True)
        now = torch.where(changed[:, None], now, was)
        old = (codes.float().view(n_blocks, BLOCK, G, D) * (was / now)[:, None, :, None]).to(torch.float8_e4m3fn)
        codes = torch.where(is_old.view(-1, 1, 1), _bytes(old.view(-1, G, D)), _bytes(codes))
        codes[at_row] = _bytes((vals / now[block][..., None]).to(torch.float8_e4m3fn))
        pool[touched] = _bytes(to_pages(codes.view(torch.float8_e4m3fn).view(-1, page, G, D).transpose(1, 2), page))
        scale[touched] = now.view(-1, page // BLOCK, G).transpose(1, 2)
    return [q, s["k"], s["v"], s["k_scale"], s["v_scale"]]


def _held_values(s, c):
    """Keys and values of the step's sequences in 32 bits, [B, G, positions, dim]."""
    D, layer = c["dim"], s["layer"]
    pages = s["table"][s["runs"]["slots"].long()].long()
    out = []
    for name, to_rows in (("k", _k_rows), ("v", _v_rows)):
        codes = to_rows(_bytes(s[name])[pages, layer].view(torch.float8_e4m3fn), D)      # [B, pages, G, page, D]
        scale = s[name + "_scale"][pages, layer].repeat_interleave(BLOCK, -1)
        out.append((codes.float() * scale[..., None]).transpose(1, 2).flatten(2, 3))
    return out


def _plain_attend(s, c):
    B, H, G, D, T = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["q"].shape[0]
    N, g = max(s["sizes"]), c["heads"] // c["kv_heads"]
    k, v = _held_values(s, c)
    L = k.shape[2]
    place = torch.arange(T, device=DEVICE) - s["runs"]["cu_seqlens"].long()[s["seq"]]
    q = torch.zeros((B, N, H, D), device=DEVICE)
    q[s["seq"], place] = s["q"].float().view(T, H, D)
    q = q.view(B, N, G, g, D).permute(0, 2, 3, 1, 4).reshape(B, G, g * N, D)
    score = (q @ k.transpose(2, 3) * D ** -0.5).view(B, G, g, N, L)
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    at = torch.full((B, N), -1, dtype=torch.long, device=DEVICE)
    at[s["seq"], place] = s["row"]
    j = torch.arange(L, device=DEVICE)
    sees = j <= at[..., None]
    if c["window"]:
        sees &= j > at[..., None] - c["window"]
    score = torch.where(sees[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    if c["sink"]:
        top = torch.maximum(top, s["sink"].view(1, G, g, 1, 1))
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + torch.exp(s["sink"].view(1, G, g, 1, 1) - top)
    p = torch.where(sees[:, None, None], p / total, 0.0)
    o = (p.view(B, G, g * N, L) @ v).view(B, H, N, D)
    out = o[s["seq"], :, place].reshape(T, H * D).to(DTYPES[c["act"]])
    if not c["weights"]:
        return [out]
    s["weight"].zero_()
    pages = s["table"][s["runs"]["slots"].long()].long()
    s["weight"][pages, s["layer"]] = p.sum((2, 3)).view(B, G, -1, c["page"]).transpose(1, 2)
    return [out, s["weight"]]


def _plain_evict(s, c):
    G, D, page, keep = c["kv_heads"], c["dim"], c["page"], c["keep"]
    src, dst = s["table"][s["src"].long()].long(), s["table"][s["dst"].long()].long()
    w = s["weight"][src].permute(0, 2, 3, 1, 4).flatten(3)                       # [B, layers, G, positions]
    j, n = torch.arange(w.shape[-1], device=DEVICE), s["lengths"].long().view(-1, 1, 1, 1)
    always = (j < c["first"]) | ((j >= n - c["recent"]) & (j < n))
    rank = torch.where(j < n, torch.where(always, math.inf, w.double()), -math.inf)
    kept = torch.sort(torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep], dim=-1).values
    n_pages = -(-keep // page)
    fill = n_pages * page - keep
    index = torch.cat([kept, kept[..., :1].expand(*kept.shape[:3], fill)], -1) if fill else kept
    is_row = torch.arange(n_pages * page, device=DEVICE) < keep
    for name, to_rows, to_pages in (("k", _k_rows, _k_layout), ("v", _v_rows, _v_layout)):
        rows = _bytes(to_rows(_bytes(s[name])[src].view(torch.float8_e4m3fn), D)).permute(0, 2, 3, 1, 4, 5).flatten(3, 4)
        scale = s[name + "_scale"][src].permute(0, 2, 3, 1, 4).flatten(3)
        mine = torch.gather(scale, 3, index // BLOCK) * is_row                    # each kept row's scale
        block = mine.unflatten(-1, (-1, BLOCK)).amax(-1)                           # [B, layers, G, blocks]
        took = torch.gather(rows, 3, index[..., None].expand(*index.shape, D))
        ratio = torch.where(block > 0, 1 / block, 0.0).repeat_interleave(BLOCK, -1) * mine
        codes = (took.view(torch.float8_e4m3fn).float() * ratio[..., None]).to(torch.float8_e4m3fn)
        codes = codes.unflatten(3, (n_pages, page)).permute(0, 3, 1, 2, 4, 5)
        _bytes(s[name])[dst[:, :n_pages]] = _bytes(to_pages(codes, page))
        blocks = block.unflatten(3, (n_pages, page // BLOCK)).permute(0, 3, 1, 2, 4)
        s[name + "_scale"][dst[:, :n_pages]] = blocks
    took = (torch.gather(w, 3, index) * is_row).unflatten(3, (n_pages, page)).permute(0, 3, 1, 2, 4)
    s["weight"][dst[:, :n_pages]] = took
    return [kept.to(torch.int32), s["k"], s["v"], s["k_scale"], s["v_scale"], s["weight"]]


_PLAIN = {"write": _plain_write, "attend": _plain_attend, "evict": _plain_evict}


# ------------------------------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    G, D, B = case["kv_heads"], case["dim"], case["seqs"]
    size = 2 if case.get("act") == "bfloat16" else 4
    new = _lengths(case)
    if case["op"] == "evict":
        rows = B * case["layers"] * G
        return {"bytes": sum(new) * case["layers"] * G * 4 + rows * case["keep"] * (2 * 2 * D + 4 + 4), "flops": sum(new) * case["layers"] * G}
    H = case["heads"]
    if case["op"] == "write":
        T = sum(new)
        return {"bytes": T * ((H + 2 * G) * D * 4 + H * D * size + 2 * G * D), "flops": T * (H + G) * case["rotary"] * 3}
    token = case["kind"] == "token"
    start = [n - 1 for n in new] if token else _past(case)
    new = [1] * B if token else new
    window = case["window"] or 1 << 60
    pairs = sum(sum(min(a + i + 1, window) for i in range(n)) for a, n in zip(start, new))
    held = sum(min(a + n, window + n - 1) for a, n in zip(start, new))
    flops = pairs * H * D * 4 + (pairs * H * D * 2 if case["weights"] and not token else 0)
    return {"bytes": held * G * D * 2 + sum(new) * H * D * 2 * size + (held * G * 8 if case["weights"] else 0), "flops": flops}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits

def _round_e4m3(y):
    """The nearest number with four significant bits, steps of 2^-9 at the least, ties to the even one; in 64 bits."""
    _, power = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(power - 4, min=-9))
    return torch.round(y / step) * step


def _as_codes(v):
    """Codes' numbers as they are compared: in 64 bits."""
    return v.to(torch.float32).double()


def exact(case, seed):
    s, c = prepare(case, seed), case
    return {"write": _exact_write, "attend": _exact_attend, "evict": _exact_evict}[c["op"]](s, c)


def _row_of(name, page, D, j):
    """Where position j's numbers lie in a page of ``page`` positions (numpy, [D])."""
    d, t, r = np.arange(D), j // 64, j % 64
    if name == "k":
        return t * 64 * D + (d // 16) * 1024 + r * 16 + d % 16
    return t * 64 * D + d * 64 + (r % 16) // 4 * 16 + r // 16 * 4 + r % 4


def _rows_of(name, page, D):
    return torch.from_numpy(np.stack([_row_of(name, page, D, j) for j in range(page)])).to(DEVICE)      # [page, D]


def _exact_write(s, c):
    H, G, D, page, layer, n = c["heads"], c["kv_heads"], c["dim"], c["page"], s["layer"], c["rotary"] // 2
    if len(s["sizes"]) * max(s["sizes"]) > 20000:
        return None
    x = s["qkv"].double().view(-1, H + 2 * G, D)
    if s["bias"] is not None:       # the sum is the operator's input in 32 bits
        x = (s["qkv"] + s["bias"]).double().view(-1, H + 2 * G, D)
    qk = x[:, :H + G].clone()
    for i in range(n):
        lo, hi = (i, i + n) if c["pairing"] == 0 else (2 * i, 2 * i + 1)
        turn = s["positions"].double() * s["freq"][i].double()
        a, b = x[:, :H + G, lo], x[:, :H + G, hi]
        qk[..., lo] = a * torch.cos(turn)[:, None] - b * torch.sin(turn)[:, None]
        qk[..., hi] = a * torch.sin(turn)[:, None] + b * torch.cos(turn)[:, None]
    pools = {m: (_as_codes(s[m]), s[m + "_scale"].double().clone()) for m in ("k", "v")}
    table, t0 = s["table"].cpu().numpy(), 0
    slots = s["runs"]["slots"].tolist()
    for b, (start, count) in enumerate(zip(s["start"], s["sizes"])):
        for block in range(start // BLOCK, (start + count - 1) // BLOCK + 1):
            lo, hi = max(start, block * BLOCK), min(start + count, (block + 1) * BLOCK)
            pg = int(table[slots[b], block * BLOCK // page])
            inside = block * BLOCK % page
            for m, vals in (("k", qk[:, H:]), ("v", x[:, H + G:])):
                codes, scales = pools[m]
                new = vals[t0 + lo - start:t0 + hi - start]                              # [rows, G, D]
                top = new.abs().amax((0, 2))
                e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -140) / 448))
                e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
                e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp(min=LEAST)
                scale = torch.exp2(e)
                old = list(range(block * BLOCK, lo))
                was = scales[pg, layer, :, inside // BLOCK].clone()
                if old:
                    scale = torch.maximum(scale, was)
                where = lambda r: torch.from_numpy(np.stack([_row_of(m, page, D, q % page) for q in r])).to(DEVICE)  # noqa: E731
                if old:
                    at = where(old)
                    codes[pg, layer][:, at] = _round_e4m3(codes[pg, layer][:, at] * (was / scale)[:, None, None])
                codes[pg, layer][:, where(range(lo, hi))] = _round_e4m3(new.transpose(0, 1) / scale[:, None, None])
                scales[pg, layer, :, inside // BLOCK] = scale
        t0 += count
    return [qk[:, :H].reshape(-1, H * D), pools["k"][0], pools["v"][0], pools["k"][1], pools["v"][1]]


def _exact_attend(s, c):
    H, G, D, page, layer = c["heads"], c["kv_heads"], c["dim"], c["page"], s["layer"]
    g = H // G
    where = {m: _rows_of(m, page, D) for m in ("k", "v")}
    out = torch.zeros((s["q"].shape[0], H, D), dtype=torch.float64, device=DEVICE)
    weight = None if s["weight"] is None else torch.zeros(s["weight"].shape, dtype=torch.float64, device=DEVICE)
    t0, slots = 0, s["runs"]["slots"].tolist()
    for b, (start, count) in enumerate(zip(s["start"], s["sizes"])):
        end = start + count
        pages = s["table"][slots[b], :-(-end // page)].long()
        held = {}
        for m in ("k", "v"):
            v = _as_codes(_bytes(s[m])[pages, layer].view(torch.float8_e4m3fn))           # [pages, G, page * D]
            v = v[..., where[m]] * s[m + "_scale"][pages, layer].double().repeat_interleave(BLOCK, -1)[..., None]
            held[m] = v.transpose(0, 1).reshape(G, -1, D)[:, :end]
        i, j = torch.arange(start, end, device=DEVICE)[:, None], torch.arange(end, device=DEVICE)[None]
        sees = (j <= i) & ((j > i - c["window"]) if c["window"] else (j >= 0))
        for h in range(H):
            q = s["q"][t0:t0 + count, h * D:(h + 1) * D].double()
            score = q @ held["k"][h // g].T / math.sqrt(D)
            if c["softcap"]:
                score = c["softcap"] * torch.tanh(score / c["softcap"])
            score = score.masked_fill(~sees, -math.inf)
            if c["sink"]:
                score = torch.cat([score, s["sink"][h].double().expand(count, 1)], 1)
            p = torch.softmax(score, 1)[:, :end]
            out[t0:t0 + count, h] = p @ held["v"][h // g]
            if weight is not None:
                total = torch.nn.functional.pad(p.sum(0), (0, pages.numel() * page - end))
                weight[pages, layer, h // g] += total.view(-1, page)
        t0 += count
    return [out.flatten(1)] + ([] if weight is None else [weight])


def _exact_evict(s, c):
    G, D, page, keep, L = c["kv_heads"], c["dim"], c["page"], c["keep"], c["layers"]
    if c["seqs"] * L * G > 800:
        return None
    where = {m: _rows_of(m, page, D) for m in ("k", "v")}
    pools = {m: (_as_codes(s[m]), s[m + "_scale"].double().clone()) for m in ("k", "v")}
    weight = s["weight"].double().clone()
    n_pages = -(-keep // page)
    host = s["weight"].cpu().numpy()
    kept = np.zeros((c["seqs"], L, G, keep), dtype=np.int32)
    for b in range(c["seqs"]):
        src = s["table"][int(s["src"][b])].long()
        dst = s["table"][int(s["dst"][b]), :n_pages].long()
        n, at = int(s["lengths"][b]), src.cpu().numpy()
        for layer in range(L):
            for h in range(G):
                w = host[at, layer, h].reshape(-1)[:n]
                always = [j for j in range(n) if j < c["first"] or j >= n - c["recent"]]
                rest = np.setdiff1d(np.arange(n), always)
                rest = rest[np.lexsort((rest, -w[rest].astype(np.float64)))][:keep - len(always)]
                mine = np.sort(np.concatenate([np.array(always, dtype=np.int64), rest]))
                kept[b, layer, h] = mine
                mine = torch.from_numpy(mine).to(DEVICE)
                for m in ("k", "v"):
                    codes, scales = pools[m]
                    v = codes[src, layer, h][:, where[m]].reshape(-1, D)[mine]
                    v = v * scales[src, layer, h].repeat_interleave(BLOCK, -1).reshape(-1)[mine][:, None]
                    own_scale = scales[src, layer, h].repeat_interleave(BLOCK, -1).reshape(-1)[mine]
                    pad = n_pages * page - keep
                    v, own_scale = torch.nn.functional.pad(v, (0, 0, 0, pad)), torch.nn.functional.pad(own_scale, (0, pad))
                    top = own_scale.view(-1, BLOCK).amax(1)
                    v = torch.where(top.repeat_interleave(BLOCK)[:, None] > 0, v / top.repeat_interleave(BLOCK)[:, None], 0.0)
                    flat = torch.zeros((n_pages, page * D), dtype=torch.float64, device=DEVICE)
                    flat[:, where[m]] = _round_e4m3(v).view(n_pages, page, D)
                    codes[dst, layer, h] = flat
                    scales[dst, layer, h] = top.view(n_pages, -1)
                weight[dst, layer, h] = torch.nn.functional.pad(s["weight"][src, layer, h].double().reshape(-1)[mine],
                                                                (0, n_pages * page - keep)).view(n_pages, page)
    return [torch.from_numpy(kept).to(DEVICE), pools["k"][0], pools["v"][0], pools["k"][1], pools["v"][1], weight]
