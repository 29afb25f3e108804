"""The 8-bit cache in plain 64-bit arithmetic: rounding to e4m3 with a scale for each block of 16 positions, the write that appends
to blocks, attention over what the blocks stand for, the choice of positions by weight and their move.  Written from the
formulas, on the CPU, one block and one row at a time."""
from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = 16


def round_e4m3(y: np.ndarray) -> np.ndarray:
    """The nearest number with four significant bits, in steps of 2^-9 at the least; ties to the even one."""
    y = np.asarray(y, dtype=np.float64)
    _, power = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(power - 4, -9))
    return np.round(y / step) * step


def scale_of(top: float) -> float:
    """The smallest power of two, 2^-100 at least, with top <= 448 of it."""
    e = -100
    while top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def usable(x) -> np.ndarray:
    return np.abs(x) < 2.0 ** 120      # (false for NaN)


class PlainPages:
    """Codes [slots, layers, kv heads, positions, dim] and scales of a cache, without pages."""

    def __init__(self, slots, layers, G, D, positions):
        positions = -(-positions // BLOCK) * BLOCK
        self.code = {m: np.zeros((slots, layers, G, positions, D)) for m in "kv"}
        self.scale = {m: np.zeros((slots, layers, G, positions // BLOCK)) for m in "kv"}
        self.weight = np.zeros((slots, layers, G, positions))

    def values(self, m, slot, layer, h):
        return self.code[m][slot, layer, h] * np.repeat(self.scale[m][slot, layer, h], BLOCK)[:, None]

    def write(self, slot, layer, start, k, v):
        """k, v [n, G, D] to positions start, start + 1, .."""
        n = k.shape[0]
        for h in range(k.shape[1]):
            good = usable(k[:, h]).all(-1) & usable(v[:, h]).all(-1)
            for block in range(start // BLOCK, (start + n - 1) // BLOCK + 1):
                lo, hi = max(start, block * BLOCK), min(start + n, (block + 1) * BLOCK)
                mine = slice(lo - start, hi - start)
                for m, x in (("k", k), ("v", v)):
                    code, scale = self.code[m][slot, layer, h], self.scale[m][slot, layer, h]
                    rows, ok = x[mine, h], good[mine]
                    s = scale_of(float(np.abs(rows[ok]).max()) if ok.any() else 0.0)
                    if lo > block * BLOCK and scale[block] > s:
                        s = scale[block]
                    if lo > block * BLOCK and scale[block] != s:
                        code[block * BLOCK:lo] = round_e4m3(code[block * BLOCK:lo] * (scale[block] / s))
                    scale[block] = s
                    code[lo:hi] = np.where(ok[:, None], round_e4m3(np.where(ok[:, None], rows, 0.0) / s), np.nan if m == "k" else 0.0)
            self.weight[slot, layer, h, start:start + n] = 0.0


def rotate(x, positions, inv_freq, pairing, amplitude=1.0):
    """x [T, heads, D] turned by positions [T]; the first 2 n numbers of a head are n pairs."""
    x, n = np.array(x, dtype=np.float64), len(inv_freq)
    for i in range(n):
        lo, hi = (i, i + n) if pairing == 0 else (2 * i, 2 * i + 1)
        turn = np.asarray(positions, dtype=np.float64) * float(inv_freq[i])
        c, s = amplitude * np.cos(turn)[:, None], amplitude * np.sin(turn)[:, None]
        a, b = x[..., lo].copy(), x[..., hi].copy()
        x[..., lo], x[..., hi] = a * c - b * s, a * s + b * c
    return x


def attend(q, k, v, places, scale, window=None, softcap=None, bias=None, chunk=None, sink=None):
    """One head: q [n, D] of tokens at ``places``, k, v [L, D] -> outputs [n, D], weights [L], and per row two measures of how far a
    32-bit computation may be off: sum_j p_j |v_j| and the largest sum_d |q_d k_jd| scale."""
    L = k.shape[0]
    out, weight = np.zeros((len(places), v.shape[1])), np.zeros(L)
    spread, reach = np.zeros((len(places), v.shape[1])), np.zeros(len(places))
    for r, i in enumerate(places):
        lo = max(0, i - window + 1) if window else 0
        if chunk:
            lo = max(lo, i // chunk * chunk)
        j = np.arange(lo, i + 1)
        s = (k[j] @ q[r]) * scale
        if softcap:
            s = softcap * np.tanh(s / softcap)
        if bias is not None:
            s = s - bias[0] * np.log1p(bias[1] * (i - j))
        top = max(s.max(), sink if sink is not None else -math.inf)
        if top == -math.inf:
            continue
        e = np.exp(s - top)
        p = e / (e.sum() + (math.exp(sink - top) if sink is not None else 0.0))
        out[r], spread[r] = p @ v[j], p @ np.abs(v[j])
        weight[j] += p
        reach[r] = (np.abs(k[j]) @ np.abs(q[r])).max() * abs(scale)
    return out, weight, spread, reach


def choose(weight, n, keep, first, recent):
    """The positions that stay of n with these weights, ascending; -1 behind them where there are fewer."""
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    always = [j for j in range(n) if j < first or j >= n - recent]
    rest = [j for j in range(n) if first <= j < n - recent]
    rank = [math.inf if w != w else w for w in weight[:n].tolist()]
    # (NaN is above +inf)
    rest.sort(key=lambda j: (not math.isnan(weight[j]), -rank[j], j))
    return sorted(always + rest[:keep - len(always)])


def move(plain: PlainPages, src, dst, kept, page):
    """kept [layers, G, keep] of slot src to slot dst."""
    L, G, keep = kept.shape
    end = -(-keep // page) * page
    for layer in range(L):
        for h in range(G):
            for m in "kv":
                code = np.zeros((end, plain.code[m].shape[-1]))
                own = np.zeros(end)
                for i, j in enumerate(kept[layer, h]):
                    if j >= 0:
                        code[i], own[i] = plain.code[m][src, layer, h, j], plain.scale[m][src, layer, h, j // BLOCK]
                top = own.reshape(-1, BLOCK).max(1)
                ratio = np.divide(own, np.repeat(top, BLOCK), out=np.zeros_like(own), where=np.repeat(top, BLOCK) > 0)
                plain.code[m][dst, layer, h, :end] = round_e4m3(code * ratio[:, None])
                plain.scale[m][dst, layer, h, :end // BLOCK] = top
            w = np.zeros(end)
            for i, j in enumerate(kept[layer, h]):
                if j >= 0:
                    w[i] = plain.weight[src, layer, h, j]
            plain.weight[dst, layer, h, :end] = w


# ------------------------------------------------------------------------------------------------ pages in the library's layout
def k_place(D, j):
    """Where position j of a page holds its numbers 0 .. D - 1 (keys)."""
    d = np.arange(D)
    return j // 64 * 64 * D + d // 16 * 1024 + j % 64 * 16 + d % 16


def v_place(D, j):
    return j // 64 * 64 * D + np.arange(D) * 64 + j % 16 // 4 * 16 + j % 64 // 16 * 4 + j % 4


def read_pages(pages, D) -> PlainPages:
    """What the library's pages hold, slot by slot (positions without a page: zeros)."""
    n_pages, L, G, ps = (*pages.k.shape[:3], pages.page_size)
    table = pages.table.cpu().numpy()
    out = PlainPages(table.shape[0], L, G, D, table.shape[1] * ps)
    raw = {m: t.float().cpu().double().numpy() for m, t in (("k", pages.k), ("v", pages.v))}
    scale = {m: t.cpu().double().numpy() for m, t in (("k", pages.k_scale), ("v", pages.v_scale))}
    place = {m: np.stack([f(D, j) for j in range(ps)]) for m, f in (("k", k_place), ("v", v_place))}
    for slot in range(table.shape[0]):
        for i, pg in enumerate(table[slot]):
            if pg < 0:
                continue
            for m in "kv":
                out.code[m][slot, :, :, i * ps:(i + 1) * ps] = raw[m][pg][..., place[m]]
                out.scale[m][slot, :, :, i * ps // BLOCK:(i + 1) * ps // BLOCK] = scale[m][pg]
            if pages.weight is not None:
                out.weight[slot, :, :, i * ps:(i + 1) * ps] = pages.weight[pg].cpu().double().numpy()
    return out


def fill_pages(pages, plain: PlainPages, D) -> None:
    """Puts what ``plain`` holds into the library's pages."""
    ps, table = pages.page_size, pages.table.cpu().numpy()
    place = {m: np.stack([f(D, j) for j in range(ps)]) for m, f in (("k", k_place), ("v", v_place))}
    raw = {m: t.float().cpu().numpy() for m, t in (("k", pages.k), ("v", pages.v))}
    scale = {m: t.cpu().numpy() for m, t in (("k", pages.k_scale), ("v", pages.v_scale))}
    weight = None if pages.weight is None else pages.weight.cpu().numpy()
    for slot in range(table.shape[0]):
        for i, pg in enumerate(table[slot]):
            if pg < 0:
                continue
            for m in "kv":
                raw[m][pg][..., place[m]] = plain.code[m][slot, :, :, i * ps:(i + 1) * ps]
                scale[m][pg] = plain.scale[m][slot, :, :, i * ps // BLOCK:(i + 1) * ps // BLOCK]
            if weight is not None:
                weight[pg] = plain.weight[slot, :, :, i * ps:(i + 1) * ps]
    for m, t, s in (("k", pages.k, pages.k_scale), ("v", pages.v, pages.v_scale)):
        t.copy_(torch.from_numpy(raw[m]).to(torch.float8_e4m3fn))
        s.copy_(torch.from_numpy(scale[m]))
    if weight is not None:
        pages.weight.copy_(torch.from_numpy(weight))
