"""The cache of a batch: a slot per sequence, keys and values per layer, fixed-size state beside them.

What the reference keeps per conversation (src/model.rs:686-728, src/cuda.rs:9826-9870) is kept
here per slot.  Layers with different needs are grouped: every mixer states what it wants
(`CacheRequest`: all keys, or a window of them; row geometry), equal requests share a group, and
each group has its own pages, page tables and storage.  This mirrors the reference sizing
its caches by attention layers only and its state buffers by the other layers
(src/model.rs:240-253, src/model.rs:738-741).  Fixed-size per-sequence state (the reference's
`conv_state`/`ssm_state`, zeroed on reset, src/model.rs:692-695, src/model.rs:772-777) lives in a
`[slot, ...]` tensor per schedule entry that asks for one (with one more row at the end, where the padding
rows of fixed-size launches land); the Llama decoder asks for none.

Storage of a group: K and V, each `[entry, page, kv_head, PAGE_TOKENS, head_dim]` (V with `v_head_dim` in
place of `head_dim` where a mixer's values are not as wide as its keys).  One page of one kv head is a
contiguous block, which is what the decode kernel streams.

Several slots may continue the same sequence (`fork`, `reorder`): they hold its pages together, and a slot gets a page of its
own, with a copy of what is filled of it, when it is about to write to one that others hold (`reserve`).

Kinds of request: "full" keeps every position; "window" only the last `window` positions; "chunk" only the
positions of the chunk of `window` positions (counted from position 0) that the sequence's newest token lies in.
The last two give pages back as the sequence moves on.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .pages import PAGE_TOKENS, CacheFullError, PagePool, SlotAllocator, pages_for


@dataclass(frozen=True)
class CacheRequest:
    """What a mixer wants kept per token.  kind "full": every position stays visible;
    kind "window": only the last `window` positions are ever read again; kind "chunk": only positions p with
    floor(p / window) equal to that of the reader's own position.  `v_head_dim`: the values' width when it is not
    the keys' `head_dim`.  `values_in_keys`: nothing is stored for the values; a position's value is the leading
    `v_head_dim` numbers of its key row (a latent that serves as both), and `LayerMemory.v` is None.  `keep_first`: a
    window cache also keeps the sequence's first so many positions for good."""
    kind: str
    num_kv_heads: int
    head_dim: int
    window: Optional[int] = None
    v_head_dim: Optional[int] = None
    values_in_keys: bool = False
    keep_first: int = 0

    def __post_init__(self):
        if self.kind not in ("full", "window", "chunk"):
            raise ValueError(f"unknown cache kind {self.kind!r}")
        if self.kind in ("window", "chunk") and (self.window is None or self.window < 1):
            raise ValueError(f"a {self.kind} cache needs a positive size")
        if self.v_head_dim is not None and self.v_head_dim < 1:
            raise ValueError("the values' width must be positive")
        if self.keep_first < 0 or (self.keep_first and self.kind != "window"):
            raise ValueError("only a window cache keeps first positions, and not a negative number of them")
        if self.values_in_keys and self.value_dim > self.head_dim:
            raise ValueError("values that live in the key rows cannot be wider than the keys")

    @property
    def value_dim(self) -> int:
        return self.head_dim if self.v_head_dim is None else self.v_head_dim


@dataclass(frozen=True)
class StateRequest:
    """Fixed-size memory per sequence, zero when the sequence starts."""
    shape: Tuple[int, ...]
    dtype: torch.dtype = torch.float32


@dataclass
class LayerMemory:
    """What one schedule entry sees of the cache during a step."""
    k: Optional[torch.Tensor]             # [page, kv_head, PAGE_TOKENS, head_dim] of this entry, or None
    v: Optional[torch.Tensor]
    block_table: Optional[torch.Tensor]   # device int32 [max_slots, max_pages_per_seq] of the entry's group
    window: Optional[int]
    writes: bool                          # False when the entry reads another entry's memory
    state: Optional[torch.Tensor]         # [max_slots + 1, *shape] or None; the last row (slot -1) is for padding rows
    chunk: Optional[int] = None           # size of the chunks of a "chunk" group
    block_state: Optional[torch.Tensor] = None   # the same kind of memory for the layer's arrangement itself (always the entry's own)


class _Group:
    def __init__(self, request: CacheRequest, n_pages: int, max_slots: int, max_pages_per_seq: int,
                 dtype: torch.dtype, device: torch.device):
        self.request = request
        self.entries: List[int] = []
        self.pool = PagePool(n_pages)
        self.pages: Dict[int, List[int]] = {}          # slot -> page numbers by page index (0 = released)
        self.first_live: Dict[int, int] = {}           # slot -> first page index still held
        self.table_host = np.zeros((max_slots, max_pages_per_seq), dtype=np.int32)
        self.table_dev: Optional[torch.Tensor] = None
        self.dirty: Dict[int, Tuple[int, int]] = {}    # slot -> [first, end) page indices not yet on the device
        self.k: Optional[torch.Tensor] = None
        self.v: Optional[torch.Tensor] = None
        self.dtype = dtype
        self.device = device
        self.n_pages = n_pages

    def allocate(self) -> None:
        r = self.request
        shape = (len(self.entries), self.n_pages + 1, r.num_kv_heads, PAGE_TOKENS, r.head_dim)
        # zero-filled once: rows past a sequence's length are never read, but the padding rows of
        # fixed-size launches read the trash page, which must hold finite numbers
        self.k = torch.zeros(shape, dtype=self.dtype, device=self.device)
        self.v = None if r.values_in_keys else torch.zeros(shape[:-1] + (r.value_dim,), dtype=self.dtype, device=self.device)
        self.table_dev = torch.zeros(self.table_host.shape, dtype=torch.int32, device=self.device)


class SequenceCache:
    def __init__(self, requests: Sequence[Tuple[int, Optional[CacheRequest], Optional[StateRequest], Optional[int]]],
                 *, max_tokens: int, max_slots: int, max_seq_len: int, dtype: torch.dtype,
                 device: torch.device | str = "cpu"):
        """`requests`: one tuple per schedule entry: (entry index, cache request or None,
        state request or None, memory_of or None[, state request of the layer's arrangement or None])."""
        if max_tokens < 1:
            raise ValueError("max_tokens must be positive")
        self.device = torch.device(device)
        self.dtype = dtype
        self.max_tokens = int(max_tokens)
        self.n_pages = pages_for(max_tokens)
        # a sequence whose every position stays cached cannot be longer than the pool; one that only keeps windows can
        keeps_all = any(r[1] is not None and r[1].kind == "full" and r[3] is None for r in requests)
        self.max_seq_len = int(min(max_seq_len, self.n_pages * PAGE_TOKENS)) if keeps_all else int(max_seq_len)
        self.max_pages_per_seq = pages_for(self.max_seq_len)
        self.slots = SlotAllocator(max_slots)
        self.max_slots = max_slots
        self.lengths = [0] * max_slots
        self.turns = [0] * max_slots                   # counts up whenever what a slot holds, or where its next tokens go, may change
        self._groups: List[_Group] = []
        self._group_of_entry: Dict[int, Tuple[_Group, int]] = {}
        self._reads_from: Dict[int, int] = {}
        self._state: Dict[int, torch.Tensor] = {}
        self._block_state: Dict[int, torch.Tensor] = {}
        by_request: Dict[CacheRequest, _Group] = {}
        requests = [tuple(r) + (None,) * (5 - len(r)) for r in requests]
        for entry, creq, sreq, memory_of, breq in requests:
            if breq is not None:      # an arrangement's own state is never borrowed: an entry that reads another's cache keeps its own
                self._block_state[entry] = torch.zeros((max_slots + 1,) + tuple(breq.shape), dtype=breq.dtype, device=self.device)
            if memory_of is not None:
                self._reads_from[entry] = memory_of
                continue
            if creq is not None:
                g = by_request.get(creq)
                if g is None:
                    g = _Group(creq, self.n_pages, max_slots, self.max_pages_per_seq, dtype, self.device)
                    by_request[creq] = g
                    self._groups.append(g)
                self._group_of_entry[entry] = (g, len(g.entries))
                g.entries.append(entry)
            if sreq is not None:
                # one row more than there are slots: padding rows of a fixed-size launch carry slot -1, which
                # indexes this last row, as they write keys and values to the trash page
                self._state[entry] = torch.zeros((max_slots + 1,) + tuple(sreq.shape), dtype=sreq.dtype, device=self.device)
        for g in self._groups:
            g.allocate()

    # ---- sizes ------------------------------------------------------------------------------
    def bytes_per_token(self) -> int:
        total = 0
        esz = torch.empty((), dtype=self.dtype).element_size()
        for g in self._groups:
            stored = g.request.head_dim + (0 if g.request.values_in_keys else g.request.value_dim)
            total += len(g.entries) * g.request.num_kv_heads * stored * esz
        return total

    def state_bytes_per_sequence(self) -> int:
        return sum(t[0].numel() * t.element_size() for d in (self._state, self._block_state) for t in d.values())

    @property
    def free_pages(self) -> int:
        return min((g.pool.free_pages for g in self._groups), default=self.n_pages)

    @property
    def groups(self) -> List[_Group]:
        return self._groups

    # ---- slots ------------------------------------------------------------------------------
    def open_slot(self) -> int:
        s = self.slots.take()
        self.lengths[s] = 0
        self.turns[s] += 1
        for g in self._groups:
            g.pages[s] = []
            g.first_live[s] = 0
        for d in (self._state, self._block_state):
            for t in d.values():
                t[s].zero_()
        return s

    def close_slot(self, slot: int) -> None:
        if not self.slots.live(slot):
            raise RuntimeError(f"slot {slot} is closed but not open")
        for g in self._groups:
            held = [p for p in g.pages.pop(slot) if p != PagePool.TRASH_PAGE]
            g.pool.give_back(held)
            g.first_live.pop(slot, None)
            g.table_host[slot, :] = 0
            g.dirty.pop(slot, None)      # a closed slot's row is never read; it is rewritten when pages come
        self.lengths[slot] = 0
        self.slots.give_back(slot)

    def length(self, slot: int) -> int:
        return self.lengths[slot]

    def reserve(self, wanted: Sequence[Tuple[int, int]]) -> None:
        """Pages for every (slot, new length) pair, in every group; all or nothing.  What will be written, from a slot's
        length on, lies in pages that the slot holds alone afterwards: the one its last tokens share with others is copied."""
        for slot, new_len in wanted:
            if not self.slots.live(slot):
                raise RuntimeError(f"slot {slot} is not open")
            if new_len > self.max_seq_len:
                raise CacheFullError(f"context full ({self.max_seq_len} tokens): slot {slot} would hold {new_len}")
        for g in self._groups:
            need = sum(max(0, pages_for(n) - len(g.pages[s])) for s, n in wanted)
            shared: Dict[int, int] = {}                     # page held by others too -> how many of `wanted` want it for themselves
            for s, n in wanted if g.pool.shared else ():
                for page in self._written(g, s, n):
                    if g.pool.holders(page) > 1:
                        shared[page] = shared.get(page, 0) + 1
            need += sum(min(w, g.pool.holders(page) - 1) for page, w in shared.items())
            if need > g.pool.free_pages:
                raise CacheFullError(
                    f"the cache is full: {need} more pages of {PAGE_TOKENS} tokens wanted, {g.pool.free_pages} of {g.pool.n_pages} free")
        for s, _ in wanted:
            self.turns[s] += 1
        for g in self._groups:
            for s, n in wanted:
                have = len(g.pages[s])
                more = pages_for(n) - have
                if more > 0:
                    new = g.pool.take(more)
                    g.pages[s].extend(new)
                    g.table_host[s, have:have + more] = new
                    self._mark(g, s, have, have + more)
            copies: List[Tuple[int, int, int]] = []
            for s, n in wanted if g.pool.shared else ():
                first = self.lengths[s] // PAGE_TOKENS
                for i, page in enumerate(self._written(g, s, n), start=first):
                    if g.pool.holders(page) < 2:
                        continue
                    own = g.pool.take(1)[0]
                    filled = self.lengths[s] - i * PAGE_TOKENS
                    if filled > 0:
                        copies.append((page, own, filled))
                    g.pool.give_back([page])
                    g.pages[s][i] = own
                    g.table_host[s, i] = own
                    self._mark(g, s, i, i + 1)
            if copies:
                self._copy_rows(g, copies)

    def _written(self, g: _Group, slot: int, new_len: int) -> List[int]:
        """The slot's pages, among those it has, that tokens from its length up to `new_len` go to."""
        if new_len <= self.lengths[slot]:
            return []
        return g.pages[slot][self.lengths[slot] // PAGE_TOKENS:pages_for(new_len)]

    @staticmethod
    def _mark(g: _Group, slot: int, lo: int, hi: int) -> None:
        was = g.dirty.get(slot, (lo, hi))
        g.dirty[slot] = (min(was[0], lo), max(was[1], hi))

    def _to_device(self, values) -> torch.Tensor:
        t = torch.tensor(values, dtype=torch.int32, pin_memory=self.device.type == "cuda")
        return t.to(self.device, non_blocking=True)

    def _copy_rows(self, g: _Group, copies: Sequence[Tuple[int, int, int]]) -> None:
        """(page, page to copy to, filled rows), keys and values of all the group's entries, on the current stream."""
        storage = [t for t in (g.k, g.v) if t is not None]
        if self.device.type != "cuda":
            for src, dst, rows in copies:
                for t in storage:
                    t[:, dst, :, :rows] = t[:, src, :, :rows]
            return
        from ..kernels import ops
        src, dst, rows = self._to_device([list(x) for x in zip(*copies)]).unbind(0)
        ops.copy_pages(storage, src, dst, rows)

    # ---- several continuations of one sequence ---------------------------------------------------
    def fork(self, slot: int) -> int:
        """Another slot that holds what `slot` holds: the same pages, a copy of its fixed-size state."""
        if not self.slots.live(slot):
            raise RuntimeError(f"slot {slot} is not open")
        new = self.open_slot()
        for g in self._groups:
            g.pages[new] = list(g.pages[slot])
            g.first_live[new] = g.first_live[slot]
            g.pool.share([p for p in g.pages[new] if p != PagePool.TRASH_PAGE])
            n = len(g.pages[new])
            g.table_host[new, :n] = g.pages[new]
            self._mark(g, new, 0, n)
        for d in (self._state, self._block_state):
            for t in d.values():
                t[new].copy_(t[slot])
        self.lengths[new] = self.lengths[slot]
        return new

    def reorder(self, slots: Sequence[Sequence[int]], parents: Sequence[Sequence[int]]) -> None:
        """Every sequence's slots take over from others of them: slot slots[s][j] holds afterwards what slots[s][parents[s][j]]
        held before.  Pages are shared, fixed-size states move on the device.  Every sequence has equally many slots."""
        flat = [s for row in slots for s in row]
        if len(set(flat)) != len(flat):
            raise ValueError("a slot is named twice")
        for row, up in zip(slots, parents):
            if len(row) != len(slots[0]) or len(up) != len(row) or any(not 0 <= p < len(row) for p in up):
                raise ValueError("every sequence wants equally many slots, and a parent among them for each")
        if len(slots) != len(parents):
            raise ValueError(f"{len(slots)} sequences, parents of {len(parents)}")
        for s in flat:
            if not self.slots.live(s):
                raise RuntimeError(f"slot {s} is not open")
        moves = [(row[j], row[p]) for row, up in zip(slots, parents) for j, p in enumerate(up) if p != j]
        if not moves:
            return
        was = {s: self.lengths[s] for s in flat}
        for g in self._groups:
            old = {s: (g.pages[s], g.first_live[s]) for s in flat}
            for to, src in moves:
                g.pool.share([p for p in old[src][0] if p != PagePool.TRASH_PAGE])
            for to, src in moves:
                pages = list(old[src][0])
                g.pool.give_back([p for p in old[to][0] if p != PagePool.TRASH_PAGE])
                g.pages[to], g.first_live[to] = pages, old[src][1]
                before, n = old[to][0], len(pages)
                same = next((i for i, (a, b) in enumerate(zip(before, pages)) if a != b), min(len(before), n))
                g.table_host[to, n:len(before)] = 0
                g.table_host[to, same:n] = pages[same:]
                if same < n:
                    self._mark(g, to, same, n)
        for to, src in moves:
            self.lengths[to] = was[src]
            self.turns[to] += 1
        states = [t for d in (self._state, self._block_state) for t in d.values()]
        if not states:
            return
        if self.device.type != "cuda":
            to, src = torch.tensor([m[0] for m in moves]), torch.tensor([m[1] for m in moves])
            for t in states:
                t[to] = t[src]
            return
        from ..kernels import ops
        ops.reorder_states(states, self._to_device([list(r) for r in slots]), self._to_device([list(r) for r in parents]))

    def commit(self, slot: int, new_len: int) -> None:
        """The slot now holds `new_len` tokens.  Window and chunk groups give back pages no later query can see."""
        self.lengths[slot] = new_len
        for g in self._groups:
            if g.request.kind == "window":
                # a query at position p >= new_len reads keys > p - window >= new_len - window
                dead_before = max(0, new_len - g.request.window + 1) // PAGE_TOKENS
            elif g.request.kind == "chunk":
                # a query at position p >= new_len reads keys from the start of its own chunk, at or after the start
                # of the chunk that position new_len lies in
                dead_before = ((new_len // g.request.window) * g.request.window) // PAGE_TOKENS
            else:
                continue
            # a window that keeps first positions never gives back the pages they lie in
            first = max(g.first_live[slot], pages_for(g.request.keep_first)) if g.request.kind == "window" else g.first_live[slot]
            if dead_before > first:
                pages = g.pages[slot]
                g.pool.give_back([pages[i] for i in range(first, dead_before)])
                for i in range(first, dead_before):
                    pages[i] = PagePool.TRASH_PAGE
                g.table_host[slot, first:dead_before] = 0    # never read again: the device copy may keep them
                g.first_live[slot] = dead_before

    def reset(self, slot: int) -> None:
        """The slot starts over: no tokens, pages given back, fixed-size state zero (src/model.rs:772-777)."""
        if not self.slots.live(slot):
            raise RuntimeError(f"slot {slot} is not open")
        for g in self._groups:
            held = [p for p in g.pages[slot] if p != PagePool.TRASH_PAGE]
            g.pool.give_back(held)
            g.pages[slot] = []
            g.first_live[slot] = 0
            g.table_host[slot, :] = 0
            g.dirty.pop(slot, None)
        for d in (self._state, self._block_state):
            for t in d.values():
                t[slot].zero_()
        self.lengths[slot] = 0
        self.turns[slot] += 1

    def truncate(self, slot: int, pos: int) -> int:
        """Rewinds a slot to `pos` tokens (src/model.rs:799-821: lowering the position is enough for
        attention caches).  Returns the length actually reached: fixed-size state and released window
        pages cannot be rewound, so with those the slot stays where it is.  Pages past that length go back."""
        cur = self.lengths[slot]
        if pos < cur and not (self._state or self._block_state or any(g.request.kind in ("window", "chunk") and g.first_live[slot] * PAGE_TOKENS > 0 for g in self._groups)):
            cur = self.lengths[slot] = pos
        self.turns[slot] += 1
        keep = pages_for(cur)
        for g in self._groups:
            pages = g.pages[slot]
            if len(pages) > keep:
                g.pool.give_back(pages[keep:])
                g.table_host[slot, keep:len(pages)] = 0
                del pages[keep:]
        return cur

    # ---- device side ------------------------------------------------------------------------
    def sync_tables(self) -> None:
        """Copies the changed stretches of the page tables to the device, on the stream of the kernels
        that read them.  Only rows that gained pages since the last call are touched.

        The host does not wait: the stretches are first copied into page-locked staging memory of this call's own
        (a copy from ordinary memory would hold the host until everything queued on the stream has run, one whole step
        in a decode loop that otherwise runs ahead of the device), and go to the device from there in stream order.
        The staging memory is handed back to torch's allocator, which reuses it only after those copies ran; the
        host's own table may change again at once (a slot closed, a page taken) without touching what is under way."""
        on_gpu = self.device.type == "cuda"
        for g in self._groups:
            if not g.dirty:
                continue
            if not on_gpu:
                for slot, (lo, hi) in g.dirty.items():
                    g.table_dev[slot, lo:hi].copy_(torch.from_numpy(g.table_host[slot, lo:hi]))
                g.dirty.clear()
                continue
            stretches = [(slot, lo, hi) for slot, (lo, hi) in g.dirty.items() if hi > lo]
            total = sum(hi - lo for _, lo, hi in stretches)
            if total:
                stage = torch.empty((total,), dtype=torch.int32, pin_memory=True)
                view = stage.numpy()
                at = 0
                for slot, lo, hi in stretches:
                    view[at:at + hi - lo] = g.table_host[slot, lo:hi]
                    g.table_dev[slot, lo:hi].copy_(stage[at:at + hi - lo], non_blocking=True)
                    at += hi - lo
            g.dirty.clear()

    def memory(self, entry: int) -> LayerMemory:
        src = self._reads_from.get(entry, entry)
        writes = entry not in self._reads_from
        gi = self._group_of_entry.get(src)
        state = self._state.get(src)
        block_state = self._block_state.get(entry)
        if gi is None:
            return LayerMemory(None, None, None, None, writes, state, None, block_state)
        g, idx = gi
        return LayerMemory(g.k[idx], g.v[idx] if g.v is not None else None, g.table_dev, g.request.window if g.request.kind == "window" else None,
                           writes, state, g.request.window if g.request.kind == "chunk" else None, block_state)
