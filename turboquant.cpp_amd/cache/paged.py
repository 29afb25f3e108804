"""The cache: a slot for each live sequence, keys and values of every layer in pages, and state of
fixed size per sequence.

The reference keeps one run state per sequence with flat ``[layers][max_seq][kv_dim]`` arrays
(/root/reference/src/engine/tq_transformer.c:208-281) and, beside them, recurrent state of fixed size
(``delta_state``, ``conv_state``, tq_transformer.c:290-313); its block cache in ``src/cache`` hands out
blocks on demand with create / append / seq_len / free calls and status checks
(/root/reference/src/cache/tq_paged_cache.c:35-243).  This cache serves many sequences at once:

* A *slot* stands for one live sequence: its length, its pages, its row of every state tensor.
  Slots are opened when a batch starts, closed when its sequence ends, and handed out again.
* Keys and values live in *pages* of ``page_size`` positions.  Layers whose needs agree (kv heads,
  width of a key row, width of a value row, window) form a *group* with storage of its own: one pool of
  pages (a group that keeps a window has a pool for its windows only: what every sequence's window, and the
  ``window_step`` positions that one step may add to it, can hold), each page holding the rows of all the group's layers for ``page_size`` positions of one sequence:
  keys laid out ``[layer][kv head][row][head_dim]``, values transposed, ``[layer][kv head][value_dim][row]``
  (both as the attention kernels' operands want them).  Keys and values have pools of their own, so their
  rows may differ in width, and a group whose layers keep one row per position only (``value_dim`` 0) has no
  value pool at all.  A group that keeps a window gives back the pages that have fallen out of every later
  token's window, so its sequences hold pages for the window only; a group whose tokens see their own chunk of
  positions only gives back the pages that lie wholly before the chunk of the sequence's next token.
* The page table of a group, ``[slot][logical page] -> page`` (-1: none), lives on the device and is
  updated only when pages change hands; kernels find a token's rows through its slot.
* A schedule entry that reads another entry's cache gets a view of that entry's storage and none
  of its own.
* With ``kv_cache="e4m3"`` the groups whose mixers (and all that read their cache) can work on pages of 8 bits keep such
  (``ops.E4m3Pages``); the others stay as they are.  If every group does, without windows and chunks, and keeps the attention
  weight that each position receives (``track_weights``), positions can be let go: they are copied to other pages, and the sequence's
  length is what is left, while its tokens' positions go on counting (``Slot.dropped`` is the difference).

All bookkeeping is on the host and independent of the device, so it is tested without one.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch


# what a group's pools hold (CacheGroup.pools), in the order in which a saved sequence lists them
POOLS = ("keys", "values", "key_scales", "value_scales", "weights")


class CacheError(RuntimeError):
    pass


class CacheFull(CacheError):
    """No page or slot is free for what was asked."""


class PagePool:
    """Free list of the pages of one group."""

    def __init__(self, n_pages: int):
        self.n_pages = n_pages
        self._free = list(range(n_pages - 1, -1, -1))   # pop() hands out low numbers first
        self._held = bytearray(n_pages)

    @property
    def n_free(self) -> int:
        return len(self._free)

    def take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise CacheFull(f"cache needs {n} more pages, {len(self._free)} of {self.n_pages} are free")
        pages = [self._free.pop() for _ in range(n)]
        for p in pages:
            self._held[p] = 1
        return pages

    def give_back(self, pages) -> None:
        for p in pages:
            if not 0 <= p < self.n_pages or not self._held[p]:
                raise CacheError(f"page {p} is given back but is not held")
            self._held[p] = 0
            self._free.append(p)


@dataclass(frozen=True)
class GroupKey:
    num_kv_heads: int
    head_dim: int
    value_dim: int
    window: int | None
    chunk: int | None = None
    keep_first: int = 0
    e4m3: bool = False


@dataclass
class KVView:
    """What a mixer needs to reach its keys and values."""
    k_pages: torch.Tensor | None      # flat pool of the group's keys
    v_pages: torch.Tensor | None      # flat pool of the group's values (None: the group keeps keys only)
    table: torch.Tensor | None        # int32 [slots, logical pages]
    layer_offset: int                 # offset of the layer's key rows inside a key page, in elements
    page_size: int
    page_stride: int                  # elements per key page
    window: int | None
    owns: bool                        # False: this run reads another run's keys and values and writes none
    v_layer_offset: int = 0           # the same for values; equal to the keys' when both rows are as wide
    v_page_stride: int = 0
    value_dim: int = 0
    pages8: "object | None" = None    # ops.E4m3Pages: the group keeps 8 bits, and k_pages and v_pages are None
    layer: int = 0                    # the entry's layer in them


class CacheGroup:
    def __init__(self, key: GroupKey, entries: list[int], n_pages: int, page_size: int, max_slots: int,
                 max_pages_per_seq: int, dtype: torch.dtype, device, track_weights: bool = False):
        self.key = key
        self.entries = entries
        self.page_size = page_size
        self.layer_elems = key.num_kv_heads * page_size * key.head_dim
        self.v_layer_elems = key.num_kv_heads * page_size * key.value_dim
        self.page_stride = len(entries) * self.layer_elems
        self.v_page_stride = len(entries) * self.v_layer_elems
        self.pool = PagePool(n_pages)
        self.max_pages_per_seq = max_pages_per_seq
        # (one row more where positions can be let go: the pages that they are copied to, before they become the sequence's)
        self.spare = max_slots if key.e4m3 else None
        rows = max_slots + (1 if key.e4m3 else 0)
        self.host_table = np.full((rows, max_pages_per_seq), -1, dtype=np.int32)
        self.dirty: set[int] = set()
        self.device = device
        self._staging = None
        self.k_pages = self.v_pages = self.table = self.pages8 = None     # without a device: bookkeeping only
        if device is not None and key.e4m3:
            if torch.device(device).type != "cuda":
                raise CacheError("a cache of 8 bits lies on a GPU")
            from ..csrc import ops
            self.table = torch.full((rows, max_pages_per_seq), -1, dtype=torch.int32, device=device)
            self.pages8 = ops.E4m3Pages.empty(n_pages, len(entries), key.num_kv_heads, key.head_dim, page_size, self.table, track_weights)
        elif device is not None:
            # zeroed once: rows beyond a sequence's length are read by tiled kernels (and masked), so they
            # must always hold finite numbers; pages that come back from a sequence do
            self.k_pages = torch.zeros(n_pages * self.page_stride, dtype=dtype, device=device)
            if self.v_page_stride:
                self.v_pages = torch.zeros(n_pages * self.v_page_stride, dtype=dtype, device=device)
            self.table = torch.full((rows, max_pages_per_seq), -1, dtype=torch.int32, device=device)

    def pools(self) -> dict[str, torch.Tensor]:
        """The pools of the group's pages, [pages, numbers of a page] each, by what they hold."""
        p = self.pages8
        if p is not None:
            held = (p.k.view(torch.uint8), p.v.view(torch.uint8), p.k_scale, p.v_scale, p.weight)
            return {n: t.view(t.shape[0], -1) for n, t in zip(POOLS, held) if t is not None}
        out = {"keys": self.k_pages.view(-1, self.page_stride)}
        if self.v_pages is not None:
            out["values"] = self.v_pages.view(-1, self.v_page_stride)
        return out

    def position_bytes(self) -> tuple[float, float]:
        """What a position costs in all the group's layers: keys (with the weight it has received, where that is kept), values.
        A scale is shared by 16 positions, so the numbers need not be whole."""
        rows = len(self.entries) * self.key.num_kv_heads
        if self.pages8 is not None:
            return rows * (self.key.head_dim + 4 / 16 + (4 if self.pages8.weight is not None else 0)), rows * (self.key.value_dim + 4 / 16)
        return rows * self.key.head_dim * self.k_pages.element_size(), rows * self.key.value_dim * self.k_pages.element_size()

    def offset_of(self, entry: int) -> int:
        return self.entries.index(entry) * self.layer_elems

    def v_offset_of(self, entry: int) -> int:
        return self.entries.index(entry) * self.v_layer_elems

    def first_needed_page(self, length: int) -> int:
        """Lowest logical page that a token at position >= length can still attend to."""
        first = 0
        if self.key.window is not None:
            first = max(0, length - self.key.window + 1)
        if self.key.chunk is not None:      # the token at position `length` and all later ones see its chunk's start at the earliest
            first = max(first, length // self.key.chunk * self.key.chunk)
        return first // self.page_size

    @property
    def kept_pages(self) -> int:
        """Logical pages from the start that hold positions every later token sees: they are never given back."""
        return -(-self.key.keep_first // self.page_size)

    def needed_pages(self, length: int) -> list[int]:
        """The logical pages that a sequence of ``length`` positions holds after a commit, in ascending order."""
        last = (length - 1) // self.page_size if length else -1
        first = self.first_needed_page(length)
        return [p for p in range(last + 1) if p >= first or p < self.kept_pages]

    def sync(self) -> None:
        """Sends the rows of the page table that changed to the device.  On a GPU they go through pinned memory
        with copies that the host does not wait for (a copy from ordinary memory returns only when everything
        issued before it has run, a decode step that was issued ahead included); the pinned rows are written again
        only after an event behind the last copies has passed."""
        if not self.dirty or self.table is None:
            self.dirty.clear()
            return
        rows = sorted(self.dirty)
        self.dirty.clear()
        n = len(rows)
        if torch.device(self.device).type != "cuda":
            self.table[torch.tensor(rows, dtype=torch.int64)] = torch.from_numpy(self.host_table[rows])
            return
        st = self._staging
        if st is None or st["rows"].shape[0] < n:
            cap = max(n, 8)
            st = self._staging = {"rows": torch.empty((cap, self.max_pages_per_seq), dtype=torch.int32).pin_memory(),
                                  "idx": torch.empty((cap,), dtype=torch.int64).pin_memory(),
                                  "copied": torch.cuda.Event()}
        else:
            st["copied"].synchronize()
        st["rows"].numpy()[:n] = self.host_table[rows]
        st["idx"].numpy()[:n] = rows
        dev_rows = st["rows"][:n].to(self.device, non_blocking=True)
        dev_idx = st["idx"][:n].to(self.device, non_blocking=True)
        st["copied"].record()
        self.table.index_copy_(0, dev_idx, dev_rows)


@dataclass
class Slot:
    index: int
    length: int = 0
    live: bool = False
    reserved: int = 0                 # positions reserved beyond length by the running step
    dropped: int = 0                  # positions that were let go: the next token's position is length + dropped


class PagedCache:
    """Slots, page groups and per-sequence state for one model.

    ``needs``: for every schedule entry ``(cache_need or None, state_need or None, cache_of or None)``.
    ``max_tokens``: the most positions live sequences hold at once, each rounded up to whole pages.
    """

    def __init__(self, needs, max_tokens: int, dtype: torch.dtype, device, page_size: int = 64,
                 max_slots: int | None = None, max_positions: int | None = None, window_step: int = 2048,
                 kv_cache: str = "same", track_weights: bool = False):
        """``kv_cache``: "same" (pages in the activations' type) or "e4m3" (pages of 8 bits where the mixers can read them).
        ``track_weights``: those pages also keep the attention weight that each position receives.
        ``window_step``: the most positions that one step adds to a sequence where a group keeps a window; such a
        group's pool is sized for ``max_slots`` windows of that reach, and whoever runs longer steps cuts them
        (``step_limit`` says so: None where no pool is smaller for it)."""
        if page_size < 1 or max_tokens < 1 or window_step < 1:
            raise CacheError("page_size, max_tokens and window_step must be positive")
        if kv_cache not in ("same", "e4m3"):
            raise CacheError(f"kv_cache is 'same' or 'e4m3', got {kv_cache!r}")
        if kv_cache == "e4m3" and page_size % 64:
            raise CacheError(f"pages of 8 bits hold a multiple of 64 positions, not {page_size}")
        if track_weights and kv_cache != "e4m3":
            raise CacheError("pages of 8 bits alone keep the weights that positions receive")
        self.kv_cache, self.track_weights = kv_cache, track_weights
        self.page_size = page_size
        self.n_pages = -(-max_tokens // page_size)
        self.max_slots = min(self.n_pages, 4096) if max_slots is None else max_slots
        per_seq = self.n_pages if max_positions is None else min(self.n_pages, -(-max_positions // page_size))
        self.max_positions = per_seq * page_size if max_positions is None else min(per_seq * page_size, max_positions)
        self.dtype, self.device = dtype, device
        self.slots = [Slot(i) for i in range(self.max_slots)]
        self._free_slots = list(range(self.max_slots - 1, -1, -1))

        by_key: dict[GroupKey, list[int]] = {}
        self._entry_group: dict[int, tuple[CacheGroup, int, bool]] = {}
        self._needs = list(needs)
        # an entry's pages are of 8 bits if its own mixer and every one that reads its cache can work on such
        e4m3 = {e: kv_cache == "e4m3" and n.reads_e4m3 for e, (n, _s, of) in enumerate(self._needs) if n is not None and of is None}
        for n, _state, of in self._needs:
            if n is not None and of in e4m3:
                e4m3[of] = e4m3[of] and n.reads_e4m3
        if kv_cache == "e4m3" and not any(e4m3.values()):
            raise CacheError("none of the model's layers can read pages of 8 bits")
        for e, (cache_need, _state, cache_of) in enumerate(self._needs):
            if cache_need is not None and cache_of is None:
                by_key.setdefault(GroupKey(cache_need.num_kv_heads, cache_need.head_dim, cache_need.value_width,
                                           cache_need.window, cache_need.chunk,
                                           cache_need.keep_first if cache_need.window is not None else 0, e4m3[e]), []).append(e)
        # A sequence holds, of a group with a window, the pages that its last `window` positions touch, and during a
        # step those of the step's new positions too, until the step is committed: window + window_step positions
        # lie in at most that many pages plus two.
        self.step_limit: int | None = None
        self.groups: list[CacheGroup] = []
        for key, entries in by_key.items():
            pages = self.n_pages
            if key.window is not None:
                for_windows = self.max_slots * (-(-(key.window + window_step) // page_size) + 2 + -(-key.keep_first // page_size))
                if for_windows < pages:
                    pages, self.step_limit = for_windows, window_step
            self.groups.append(CacheGroup(key, entries, pages, page_size, self.max_slots, per_seq, dtype, device, track_weights))
        self._v_offset: dict[int, int] = {}
        for g in self.groups:
            for e in g.entries:
                self._entry_group[e] = (g, g.offset_of(e), True)
                self._v_offset[e] = g.v_offset_of(e)
        for e, (cache_need, _state, cache_of) in enumerate(self._needs):
            if cache_need is not None and cache_of is not None:
                if cache_of not in self._entry_group or not self._entry_group[cache_of][2]:
                    raise CacheError(f"schedule entry {e} reads the cache of entry {cache_of}, which keeps none of its own")
                g, off, _ = self._entry_group[cache_of]
                src = self._needs[cache_of][0]
                if (src.num_kv_heads, src.head_dim, src.value_width) != \
                        (cache_need.num_kv_heads, cache_need.head_dim, cache_need.value_width):
                    raise CacheError(f"schedule entry {e} reads the cache of entry {cache_of} but their head counts or sizes differ")
                if src.window is not None and (cache_need.window is None or cache_need.window > src.window):
                    raise CacheError(f"schedule entry {e} looks further back than entry {cache_of}, whose cache it reads, keeps")
                if src.window is not None and cache_need.keep_first > src.keep_first:
                    raise CacheError(f"schedule entry {e} keeps more first positions in sight than entry {cache_of}, whose cache it reads, keeps")
                if src.chunk is not None and cache_need.chunk != src.chunk:
                    raise CacheError(f"schedule entry {e} reads the cache of entry {cache_of}, which keeps chunks of {src.chunk} positions only")
                self._entry_group[e] = (g, off, False)
                self._v_offset[e] = self._v_offset[cache_of]

        self.states: dict[int, torch.Tensor] = {}
        for e, (_cache, state_need, _of) in enumerate(self._needs):
            if state_need is not None and device is not None:
                self.states[e] = torch.zeros((self.max_slots, *state_need.shape), dtype=state_need.dtype, device=device)

    # ------------------------------------------------------------ slots
    @property
    def n_live(self) -> int:
        return self.max_slots - len(self._free_slots)

    def open(self) -> int:
        """A slot for a new sequence of length 0 with zeroed state."""
        if not self._free_slots:
            raise CacheFull(f"all {self.max_slots} slots hold live sequences")
        i = self._free_slots.pop()
        s = self.slots[i]
        s.length, s.live, s.reserved, s.dropped = 0, True, 0, 0
        for st in self.states.values():
            st[i].zero_()
        return i

    def close(self, slot: int) -> None:
        """Ends a sequence: its pages and its slot go back."""
        s = self._live(slot)
        for g in self.groups:
            row = g.host_table[slot]
            held = row[row >= 0]
            if held.size:
                g.pool.give_back(held.tolist())
                row[:] = -1
                g.dirty.add(slot)
        s.live, s.length, s.reserved, s.dropped = False, 0, 0, 0
        self._free_slots.append(slot)

    def length(self, slot: int) -> int:
        return self._live(slot).length

    def _live(self, slot: int) -> Slot:
        if not 0 <= slot < self.max_slots or not self.slots[slot].live:
            raise CacheError(f"slot {slot} holds no live sequence")
        return self.slots[slot]

    # ------------------------------------------------------------ a step's positions
    def reserve(self, slot: int, n_new: int) -> int:
        """Makes room for positions length .. length+n_new-1 in every group; returns the first of them."""
        s = self._live(slot)
        if s.reserved:
            raise CacheError(f"slot {slot} already has positions reserved for a running step")
        end = s.length + n_new
        if end > self.max_positions:
            raise CacheFull(f"sequence in slot {slot} would reach {end} positions, the cache holds {self.max_positions} per sequence")
        first_page, last_page = s.length // self.page_size, (end - 1) // self.page_size
        for g in self.groups:
            row = g.host_table[slot]
            missing = [p for p in range(first_page, last_page + 1) if row[p] < 0]
            if missing:
                try:
                    pages = g.pool.take(len(missing))
                except CacheFull:
                    self._undo_reserve(slot, g)
                    raise
                row[missing] = pages
                g.dirty.add(slot)
        s.reserved = n_new
        return s.length

    def room_for(self, slots, counts) -> None:
        """Raises CacheFull if the groups that keep every position (and each sequence's own bound) have no room for
        ``counts[i]`` more positions in ``slots[i]``, all together; takes nothing.  For a step that is run in cuts:
        the groups with a window have room for every cut by the size of their pools."""
        need = 0
        for slot, n in zip(slots, counts):
            s = self._live(slot)
            if s.length + n > self.max_positions:
                raise CacheFull(f"sequence in slot {slot} would reach {s.length + n} positions, the cache holds {self.max_positions} per sequence")
            held = (s.length + self.page_size - 1) // self.page_size
            need += (s.length + n + self.page_size - 1) // self.page_size - held
        for g in self.groups:
            if g.key.window is None and need > g.pool.n_free:
                raise CacheFull(f"cache needs {need} more pages, {g.pool.n_free} of {g.pool.n_pages} are free")

    def needs_page(self, slot: int, n_new: int = 1) -> bool:
        """Whether ``n_new`` more positions would take a page that the sequence does not hold yet."""
        s = self._live(slot)
        first_page, last_page = s.length // self.page_size, (s.length + n_new - 1) // self.page_size
        if last_page >= self.groups[0].max_pages_per_seq if self.groups else False:
            return True
        return any((g.host_table[slot][first_page:last_page + 1] < 0).any() for g in self.groups)

    @property
    def n_free_slots(self) -> int:
        return len(self._free_slots)

    def _undo_reserve(self, slot: int, failed: CacheGroup | None) -> None:
        """Gives back the pages beyond the sequence's length, in the groups before ``failed`` (None: in all)."""
        s = self.slots[slot]
        keep_upto = (s.length - 1) // self.page_size if s.length else -1
        for g in self.groups:
            if g is failed:
                break
            row = g.host_table[slot]
            extra = [p for p in range(keep_upto + 1, g.max_pages_per_seq) if row[p] >= 0]
            if extra:
                g.pool.give_back(row[extra].tolist())
                row[extra] = -1
                g.dirty.add(slot)

    def cancel(self, slot: int) -> None:
        """The step that reserved positions did not run: they do not count, and pages taken for them go back."""
        s = self._live(slot)
        s.reserved = 0
        self._undo_reserve(slot, None)

    def commit(self, slot: int) -> None:
        """The step that reserved positions has run: they now count, and pages that no later token's
        window reaches go back to their pool."""
        s = self._live(slot)
        s.length += s.reserved
        s.reserved = 0
        for g in self.groups:
            first = g.first_needed_page(s.length)
            if first > 0:
                row = g.host_table[slot]
                old = [p for p in range(g.kept_pages, first) if row[p] >= 0]
                if old:
                    g.pool.give_back(row[old].tolist())
                    row[old] = -1
                    g.dirty.add(slot)

    # ------------------------------------------------------------ a sequence that outlives its request
    def truncate(self, slot: int, length: int) -> None:
        """Forgets the positions from ``length`` on, so that the sequence can go on from there with other tokens.
        Refused (CacheError) where that cannot be done: a group with a window has given back pages that a token at
        ``length`` would look at, or the model keeps fixed-size state per sequence, which has no earlier value."""
        s = self._live(slot)
        if s.reserved:
            raise CacheError(f"slot {slot} has positions reserved for a running step")
        if not 0 <= length <= s.length:
            raise CacheError(f"slot {slot} holds {s.length} positions, not {length}")
        if length == s.length:
            return
        if s.dropped:
            raise CacheError(f"slot {slot} has let positions go: what is left are not the first ones of what it has seen")
        if any(state is not None for _c, state, _o in self._needs):
            raise CacheError("a model with fixed-size state per sequence cannot go back to an earlier position")
        for g in self.groups:
            row = g.host_table[slot]
            if any(row[p] < 0 for p in g.needed_pages(length)):
                raise CacheError(f"the window of a group has given back pages that position {length} would look at")
        for g in self.groups:
            row = g.host_table[slot]
            needed = set(g.needed_pages(length))
            gone = [p for p in range(g.max_pages_per_seq) if row[p] >= 0 and p not in needed]
            if gone:
                g.pool.give_back(row[gone].tolist())
                row[gone] = -1
                g.dirty.add(slot)
        s.length = length

    # ------------------------------------------------------------ positions that are let go
    def no_eviction(self) -> str | None:
        """Why positions cannot be let go, or None."""
        if not self.groups or not all(g.key.e4m3 for g in self.groups):
            return "every layer that keeps a cache has to keep one of 8 bits"
        if not self.track_weights:
            return "the cache does not keep the weights that positions receive (track_weights)"
        if any(g.key.window is not None or g.key.chunk is not None for g in self.groups):
            return "layers with a window or chunks count on the places of all positions"
        return None

    def dropped(self, slot: int) -> int:
        """How many positions of its sequence have been let go."""
        return self._live(slot).dropped

    def positions_of(self, slots, places) -> list[int]:
        """The positions of tokens at these places of the slots' sequences."""
        return [p + self.slots[s].dropped for s, p in zip(slots, places)]

    def begin_evict(self, slot: int, keep: int) -> None:
        """Pages for ``keep`` positions of a sequence that holds more, in the spare row of every group's table."""
        s, why = self._live(slot), self.no_eviction()
        if why is not None:
            raise CacheError(f"positions cannot be let go: {why}")
        if s.reserved:
            raise CacheError(f"slot {slot} has positions reserved for a running step")
        if not 1 <= keep < s.length:
            raise CacheError(f"slot {slot} holds {s.length} positions: fewer than these and at least one can stay, not {keep}")
        n = -(-keep // self.page_size)
        short = [g for g in self.groups if g.pool.n_free < n]
        if short:
            raise CacheFull(f"letting positions go needs {n} pages to copy the others to, {short[0].pool.n_free} of {short[0].pool.n_pages} are free")
        for g in self.groups:
            g.host_table[g.spare, :n] = g.pool.take(n)
            g.dirty.add(g.spare)

    def end_evict(self, slot: int, keep: int, done: bool = True) -> None:
        """The spare row's pages become the sequence's (or, not ``done``, go back), and the others go back."""
        s = self._live(slot)
        for g in self.groups:
            row, spare = g.host_table[slot], g.host_table[g.spare]
            gone = row if done else spare
            g.pool.give_back(gone[gone >= 0].tolist())
            if done:
                row[:] = spare
                g.dirty.add(slot)
            spare[:] = -1
            g.dirty.add(g.spare)
        if done:
            s.dropped += s.length - keep
            s.length = keep

    def export_slot(self, slot: int) -> dict:
        """What the cache holds of one sequence, on the host: its length, per group the logical pages it holds
        (first page, keys [pages, page elements], values) and per entry its row of fixed-size state."""
        s = self._live(slot)
        if s.reserved:
            raise CacheError(f"slot {slot} has positions reserved for a running step")
        out = {"length": s.length, "page_size": self.page_size, "dropped": s.dropped, "groups": [], "states": {}}
        for g in self.groups:
            first = g.first_needed_page(s.length)
            row = g.host_table[slot]
            pages = [int(row[p]) for p in g.needed_pages(s.length)]
            if any(p < 0 for p in pages):
                raise CacheError(f"slot {slot} does not hold all pages of its {s.length} positions")
            idx = torch.tensor(pages, dtype=torch.int64, device=self.device)
            entry = {"first_page": first, "entries": list(g.entries), "key": (g.key.num_kv_heads, g.key.head_dim, g.key.value_dim, g.key.window, g.key.chunk, g.key.keep_first),
                     "keys": None, "values": None}
            if g.key.e4m3:
                entry["key"] += (True,)
            entry.update({name: pool[idx].cpu() for name, pool in g.pools().items()})
            out["groups"].append(entry)
        for e, st in self.states.items():
            out["states"][e] = st[slot].cpu()
        return out

    def import_slot(self, data: dict) -> int:
        """A new slot that holds what ``export_slot`` gave (of a cache of the same model, page size and type)."""
        if data["page_size"] != self.page_size or len(data["groups"]) != len(self.groups):
            raise CacheError("the saved sequence comes from a cache of another layout")
        for g, d in zip(self.groups, data["groups"]):
            saved = tuple(d["key"])
            saved += (None,) * (5 - len(saved))
            saved += (0,) * (6 - len(saved))
            saved += (False,) * (7 - len(saved))
            pools = g.pools()
            # (weights alone may be missing or left over: a cache that does not keep them has no use for them, one that does starts them at 0)
            if saved != (g.key.num_kv_heads, g.key.head_dim, g.key.value_dim, g.key.window, g.key.chunk, g.key.keep_first, g.key.e4m3) or \
                    list(d["entries"]) != list(g.entries) or \
                    any(d.get(n) is None or d[n].dtype != t.dtype or d[n].shape[1] != t.shape[1] for n, t in pools.items() if n != "weights" or d.get(n) is not None) or \
                    (d["values"] is None) != ("values" not in pools):
                raise CacheError("the saved sequence comes from a cache of another layout")
        if int(data.get("dropped", 0)) and self.no_eviction() is not None:
            raise CacheError("the saved sequence has let positions go, which this cache cannot do")
        slot = self.open()
        try:
            length = int(data["length"])
            if length:
                self.reserve(slot, length)
                self.commit(slot)
            for g, d in zip(self.groups, data["groups"]):
                first = g.first_needed_page(length)
                needed = g.needed_pages(length)
                if d["first_page"] != first or d["keys"].shape[0] != len(needed):
                    raise CacheError("the saved pages do not cover the saved length")
                row = g.host_table[slot]
                idx = torch.tensor([int(row[p]) for p in needed], dtype=torch.int64, device=self.device)
                if idx.numel():
                    for name, pool in g.pools().items():
                        pool[idx] = d[name].to(self.device) if d.get(name) is not None else torch.zeros((), dtype=pool.dtype, device=self.device)
            self.slots[slot].dropped = int(data.get("dropped", 0))
            for e, st in data["states"].items():
                self.states[int(e)][slot].copy_(st.to(self.device))
        except BaseException:
            self.slots[slot].reserved = 0
            self.close(slot)
            raise
        return slot

    def sync(self) -> None:
        for g in self.groups:
            g.sync()

    # ------------------------------------------------------------ views
    def kv(self, entry: int) -> KVView:
        if entry not in self._entry_group:
            raise CacheError(f"schedule entry {entry} keeps no keys and values")
        g, off, owns = self._entry_group[entry]
        return KVView(g.k_pages, g.v_pages, g.table, off, g.page_size, g.page_stride, self._needs[entry][0].window, owns,
                      self._v_offset[entry], g.v_page_stride, g.key.value_dim, g.pages8,
                      g.entries.index(entry if owns else self._needs[entry][2]))

    def state(self, entry: int) -> torch.Tensor:
        if entry not in self.states:
            raise CacheError(f"schedule entry {entry} keeps no per-sequence state")
        return self.states[entry]

    def pages_held(self) -> dict[int, int]:
        """Pages in use per group index."""
        return {i: g.pool.n_pages - g.pool.n_free for i, g in enumerate(self.groups)}

    def bytes(self) -> int:
        n = 0
        for g in self.groups:
            if g.table is not None:
                n += sum(t.numel() * t.element_size() for t in g.pools().values())
        return n
