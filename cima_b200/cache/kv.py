"""The cache: a slot for each live sequence, keys and values for each layer in pages, and
fixed-size state for each slot beside them.

Layout.  Layers whose mixers ask for the same storage (KV heads, head size, window, planes) form a
*group*.  A group owns ``[layers, pages, planes (k|v, or one shared), kv_heads, page_size, head_dim]`` and one block
table ``[slots, width]`` of page ids that all its layers share.  A group that keeps every key
gives a sequence one page per ``page_size`` positions; a group with a window of ``w`` keys gives
it a ring of ``ceil(w / page_size) + 1`` pages, position ``p`` living in ring entry
``(p / page_size) % ring``; those are the pages that can still hold a key within the window of
the newest position.  A slot's pages go back to their pools when the slot is closed and are
handed to later sequences with their old contents, which nothing reads: every kernel is given
the sequence's length.

Sequences may share pages.  ``fork`` opens slots that hold what another holds: the same pages, which count their
holders, and copies of its state (of a window's ring too, whose pages are written over).  A slot that is about to write into a page that
others hold gets a copy of what it keeps of it first (``reserve``; the copies run together in ``flush``), so a sequence never sees
another's tokens, and a page goes back to its pool with its last holder.  ``compact`` moves the held pages to the lowest ids.
``shared_groups`` tells an attention which sequences of a step have pages in common.

The reference keeps one sequence: per layer K and V of ``[kv_heads, max_seq, head_dim]`` and one
cursor (src/models/transformer.rs:764, :916-917; src/kernels.cu:440-454), its fixed-size state
(position counter, penalty ring, next token) in separate device buffers (:716-729).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .pages import CacheFull, FreeList


@dataclass(frozen=True)
class KVRequest:
    """What a mixer needs per position: keys and values of ``n_kv_heads`` heads of ``head_dim``;
    ``window`` 0 = all positions are kept, w > 0 = only the last w need to be.  ``planes`` 2 = keys and values
    are kept apart; 1 = one vector per position and head serves as both (a latent that the mixer projects
    keys and values from)."""
    n_kv_heads: int
    head_dim: int
    window: int = 0
    planes: int = 2


@dataclass(frozen=True)
class StateRequest:
    """Fixed-size state per sequence: a tensor ``[slots, *shape]``, zeroed when a slot is opened."""
    name: str
    shape: Tuple[int, ...]
    dtype: torch.dtype = torch.float32


class CapacityError(RuntimeError):
    """A sequence would grow beyond the positions the model or the cache allows."""


@dataclass
class LayerKV:
    """What an attention kernel needs to find a layer's keys and values."""
    storage: torch.Tensor        # [pages, planes (k|v, or 1), kv_heads, page_size, head_dim] of this layer
    block_table: torch.Tensor    # [slots, width] int32, shared by the group
    page_size: int
    ring_pages: int              # 0 = one table entry per page of positions; R = ring of R entries
    window: int
    group: int
    planes: int = 2


@dataclass
class SharedPrefixes:
    """Which sequences of a step hold the same pages for a prefix, as an attention kernel wants it (int32 on the device; ``KVCache.shared_groups``
    finds them).  The pages of a group are the first ones of all its sequences' tables and lie below their newest positions."""
    order: torch.Tensor          # [seqs] the step's sequences, group by group, those of no group at any place
    own_page: torch.Tensor       # [seqs] pages that sequence i has in common with its group (0: it is in none); its own begin there
    groups: torch.Tensor         # [groups, 3] place of the group's first sequence in ``order``, sequences, pages
    most: int                    # sequences of the largest group
    pages: int = 0               # a bound on the pages of a group (0: not known), for the choice of splits only
    alone: Optional[bool] = None # whether some sequence is in no group (None: where there are more than the groups could hold), for splits and order only

    @staticmethod
    def pack(groups: Sequence[Tuple[Sequence[int], int]], n_seqs: int, places: int = 0) -> np.ndarray:
        """``KVCache.shared_groups``' answer for a step of ``n_seqs`` sequences as the three arrays one behind the other, with at least ``places`` groups (the
        further ones have no sequences)."""
        order = [i for members, _ in groups for i in members]
        out = np.zeros(2 * n_seqs + 3 * max(len(groups), places), dtype=np.int32)
        out[:n_seqs] = order + sorted(set(range(n_seqs)) - set(order))
        at = 0
        for k, (members, pages) in enumerate(groups):
            out[n_seqs + np.asarray(members)] = pages
            out[2 * n_seqs + 3 * k:2 * n_seqs + 3 * k + 3] = at, len(members), pages
            at += len(members)
        return out

    @classmethod
    def over(cls, packed: torch.Tensor, n_seqs: int, most: int, pages: int = 0, alone: Optional[bool] = None) -> "SharedPrefixes":
        """The arrays of ``packed`` (on the device) as views."""
        return cls(packed[:n_seqs], packed[n_seqs:2 * n_seqs], packed[2 * n_seqs:].view(-1, 3), most, pages, alone)


class KVGroup:
    def __init__(self, index: int, request: KVRequest, layers: List[int], n_pages: int, n_slots: int,
                 page_size: int, max_pages_per_seq: int, dtype: torch.dtype, device):
        self.index = index
        self.request = request
        self.layers = layers
        self.page_size = page_size
        ring = -(-request.window // page_size) + 1 if request.window > 0 else 0
        self.ring_pages = ring if 0 < ring < max_pages_per_seq else 0
        self.width = self.ring_pages or max_pages_per_seq
        self.pool = FreeList(n_pages, f"page of group {index}")
        self.pages_of: List[List[int]] = [[] for _ in range(n_slots)]
        self.holders = np.zeros(n_pages, dtype=np.int32)          # slots that hold a page
        self.shared = 0                                           # pages that more than one slot holds
        self.copies: List[Tuple[int, int, int]] = []              # (from, to, positions) that the next flush copies
        self.table_host = np.zeros((n_slots, self.width), dtype=np.int32)
        self.block_table = torch.zeros((n_slots, self.width), dtype=torch.int32, device=device)
        if request.planes not in (1, 2):
            raise ValueError(f"a cache request has {request.planes} planes; 2 (keys | values) or 1 (shared) are possible")
        self.storage = torch.zeros((len(layers), n_pages, request.planes, request.n_kv_heads, page_size, request.head_dim),
                                   dtype=dtype, device=device)
        self.dirty: set = set()

    def pages_needed(self, length: int) -> int:
        n = -(-length // self.page_size)
        return min(n, self.ring_pages) if self.ring_pages else n

    def written(self, slot: int, start: int, length: int) -> List[int]:
        """Places among the slot's pages that positions start .. length - 1 lie in (none where there are none) and that other slots hold too."""
        if not self.shared or start >= length:
            return []
        held = self.pages_of[slot]
        return [i for i in range(start // self.page_size, min(len(held), -(-length // self.page_size))) if self.holders[held[i]] > 1]

    def grow(self, slot: int, start: int, length: int) -> None:
        """Take the pages that ``length`` positions need beyond those held, and pages of its own in place of shared ones that positions
        from ``start`` on are about to be written to; what the slot keeps of those is copied by the next ``flush``.  All or nothing."""
        held = self.pages_of[slot]
        own = self.written(slot, start, length)
        more = max(0, self.pages_needed(length) - len(held))
        if not own and not more:
            return
        new = self.pool.take(len(own) + more)
        for p in new:
            self.holders[p] = 1
        for i, p in zip(own, new):
            old = held[i]
            keep = min(self.page_size, start - i * self.page_size)
            if keep > 0:
                self.copies.append((old, p, keep))
            self.drop(old)
            held[i] = p
            self.table_host[slot, i] = p
        for p in new[len(own):]:
            self.table_host[slot, len(held)] = p
            held.append(p)
        self.dirty.add(slot)

    def hold(self, page: int) -> None:
        """One more holder of a held page."""
        self.holders[page] += 1
        if self.holders[page] == 2:
            self.shared += 1

    def drop(self, page: int) -> bool:
        """One holder fewer; whether it was the last (the caller gives the page back)."""
        self.holders[page] -= 1
        if self.holders[page] == 1:
            self.shared -= 1
        return self.holders[page] == 0

    def share(self, src: int, dst: int, length: int) -> None:
        """The pages of ``src``'s first ``length`` positions are ``dst``'s (which holds none) as well."""
        pages = self.pages_of[src][:self.pages_needed(length)]
        for p in pages:
            self.hold(p)
        self.pages_of[dst] = pages
        self.table_host[dst, :len(pages)] = pages
        self.dirty.add(dst)

    def duplicate(self, src: int, dst: int, length: int) -> None:
        """``dst`` (which holds none) gets pages of its own with the contents of those of ``src``'s first ``length`` positions."""
        n = self.pages_needed(length)
        new = self.pool.take(n)
        for i, (a, b) in enumerate(zip(self.pages_of[src], new)):
            self.holders[b] = 1
            self.copies.append((a, b, self.page_size if self.ring_pages else min(self.page_size, length - i * self.page_size)))
        self.pages_of[dst] = new
        self.table_host[dst, :n] = new
        self.dirty.add(dst)

    def release(self, slot: int) -> None:
        self.pool.give([p for p in self.pages_of[slot] if self.drop(p)])
        self.pages_of[slot] = []

    def trim(self, slot: int, length: int) -> int:
        keep = self.pages_needed(length)
        back = self.pages_of[slot][keep:]
        self.pool.give([p for p in back if self.drop(p)])
        del self.pages_of[slot][keep:]
        return len(back)

    def compact(self) -> int:
        """Held pages beyond as many as are held move to free ones below; how many moved."""
        n = self.pool.held
        high = [p for p in range(n, self.pool.n) if self.holders[p]]
        moves = dict(zip(high, (p for p in range(n) if not self.holders[p])))
        if not moves:
            return 0
        self.pool.move(moves.items())
        for old, new in moves.items():
            self.holders[new], self.holders[old] = self.holders[old], 0
            self.copies.append((old, new, self.page_size))
        for slot, pages in enumerate(self.pages_of):
            if any(p in moves for p in pages):
                self.pages_of[slot] = pages = [moves.get(p, p) for p in pages]
                self.table_host[slot, :len(pages)] = pages
                self.dirty.add(slot)
        return len(moves)

    def plans(self) -> List[np.ndarray]:
        """The pending copies as plans without an order of their own: one, or several to be run one after another where a page is both
        written and read or written again (a page that was copied from, given back and taken anew)."""
        out: List[list] = []
        read, wrote = set(), set()
        for a, b, n in self.copies:
            if not out or a in wrote or b in read or b in wrote:
                out.append([])
                read, wrote = set(), set()
            out[-1].append((a, b, n))
            read.add(a)
            wrote.add(b)
        self.copies = []
        return [np.array(p, dtype=np.int32) for p in out]

    def flush(self) -> None:
        if not self.dirty:
            return
        rows = sorted(self.dirty)
        idx = torch.as_tensor(rows, dtype=torch.long, device=self.block_table.device)
        self.block_table.index_copy_(0, idx, torch.from_numpy(self.table_host[rows]).to(self.block_table.device))
        self.dirty.clear()

    def nbytes(self) -> int:
        return self.storage.numel() * self.storage.element_size()


class KVCache:
    """Slots, pages and per-sequence state of one model.

    ``requests[i]`` is what the mixer at site ``i`` (the i-th entry of the model's schedule; "layer"
    below) asks for: a list of ``KVRequest`` / ``StateRequest`` (possibly empty).  ``shares[i] = j``
    lets site ``i`` read site ``j``'s keys and values instead of holding its own.  ``max_tokens`` is the most positions that live
    sequences hold at any time, each sequence's count rounded up to ``page_size``.
    """

    def __init__(self, requests: Sequence[Sequence[object]], max_tokens: int, max_position: int,
                 dtype: torch.dtype, device, page_size: int = 64, max_seqs: Optional[int] = None,
                 shares: Optional[Dict[int, int]] = None, extra_state: Sequence[StateRequest] = (), kernels=None):
        """``kernels``: the kernel library, which copies pages and state on a GPU (``fork``, ``compact``)."""
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size {page_size} must be a positive multiple of 16")
        if max_tokens <= 0:
            raise ValueError(f"max_tokens {max_tokens} must be positive")
        self.page_size = page_size
        self.n_pages = -(-max_tokens // page_size)
        self.max_tokens = self.n_pages * page_size
        self.max_position = max_position
        self.n_slots = max(1, min(self.n_pages, max_seqs if max_seqs else 4096))
        self.max_pages_per_seq = -(-min(self.max_tokens, max_position) // page_size)
        self.dtype = dtype
        self.device = device
        self.kernels = kernels
        self.slots = FreeList(self.n_slots, "slot")
        self.lengths = np.zeros(self.n_slots, dtype=np.int64)
        self.groups: List[KVGroup] = []
        self._layer_group: Dict[int, Tuple[int, int]] = {}
        self.state: Dict[str, torch.Tensor] = {}
        self.has_mixer_state = False      # a mixer keeps state of fixed size per sequence (it cannot be rewound)
        shares = dict(shares or {})
        by_key: Dict[KVRequest, List[int]] = {}
        for layer, reqs in enumerate(requests):
            for r in reqs:
                if isinstance(r, KVRequest):
                    if layer in shares:
                        raise ValueError(f"layer {layer} both asks for keys/values and reads layer {shares[layer]}'s")
                    by_key.setdefault(r, []).append(layer)
                elif isinstance(r, StateRequest):
                    self._add_state(r)
                    self.has_mixer_state = True
                else:
                    raise TypeError(f"layer {layer}: unknown cache request {r!r}")
        for r in extra_state:
            self._add_state(r)
        for gi, (req, layers) in enumerate(by_key.items()):
            g = KVGroup(gi, req, layers, self.n_pages, self.n_slots, page_size, self.max_pages_per_seq, dtype, device)
            self.groups.append(g)
            for li, layer in enumerate(layers):
                if layer in self._layer_group:
                    raise ValueError(f"layer {layer} asks for keys and values twice")
                self._layer_group[layer] = (gi, li)
        for layer, src in shares.items():
            if src not in self._layer_group:
                raise ValueError(f"layer {layer} reads the cache of layer {src}, which holds none")
            self._layer_group[layer] = self._layer_group[src]

    # ------------------------------------------------------------------ state
    def _add_state(self, r: StateRequest) -> None:
        if r.name in self.state:
            raise ValueError(f"per-sequence state '{r.name}' is asked for twice")
        self.state[r.name] = torch.zeros((self.n_slots, *r.shape), dtype=r.dtype, device=self.device)

    # ------------------------------------------------------------------ views
    def layer_kv(self, layer: int) -> LayerKV:
        gi, li = self._layer_group[layer]
        g = self.groups[gi]
        return LayerKV(storage=g.storage[li], block_table=g.block_table, page_size=self.page_size,
                       ring_pages=g.ring_pages, window=g.request.window, group=gi, planes=g.request.planes)

    def most_tokens_going_on(self) -> Optional[int]:
        """The most tokens that a sequence which already holds positions may add in one step whose rows read the
        cache, or None for no limit.  A window group keeps a ring of ceil(w / page) + 1 pages: the step's keys are
        all appended before any row reads, so a row's oldest key survives only while the step adds at most a page."""
        return self.page_size if any(g.ring_pages for g in self.groups) else None

    def has_kv(self, layer: int) -> bool:
        return layer in self._layer_group

    def nbytes(self) -> int:
        return (sum(g.nbytes() for g in self.groups)
                + sum(t.numel() * t.element_size() for t in self.state.values()))

    # ------------------------------------------------------------------ slots
    def open(self, count: int) -> List[int]:
        """Slots for ``count`` new sequences, empty, their state zeroed."""
        got = self.slots.take(count)
        for s in got:
            assert self.lengths[s] == 0 and all(not g.pages_of[s] for g in self.groups), \
                f"slot {s} was handed out with contents"
        if got and self.state:
            idx = torch.as_tensor(got, dtype=torch.long, device=self.device)
            for t in self.state.values():
                t.index_fill_(0, idx, 0)
        return got

    def reserve(self, slot: int, length: int) -> None:
        """Make room for ``slot`` to hold ``length`` positions; all or nothing."""
        if not self.slots.is_held(slot):
            raise ValueError(f"slot {slot} is not open")
        if length > self.max_position:
            raise CapacityError(f"slot {slot}: {length} positions exceed the model's max_position {self.max_position}")
        if length < self.lengths[slot]:
            raise ValueError(f"slot {slot}: a sequence of {self.lengths[slot]} positions cannot shrink to {length}")
        start = int(self.lengths[slot])
        for g in self.groups:                         # room in every group before any takes a page
            need = max(0, g.pages_needed(length) - len(g.pages_of[slot])) + len(g.written(slot, start, length))
            if need > g.pool.free:
                raise CacheFull(f"slot {slot} cannot grow to {length} positions: {need} {g.pool.what}(s) wanted, {g.pool.free} of {g.pool.n} free "
                                f"(the cache holds {self.max_tokens} positions in pages of {self.page_size})")
        for g in self.groups:
            g.grow(slot, start, length)

    def must_fit(self, wanted: Sequence[Tuple[int, int]]) -> None:
        """Raise (``CapacityError`` / ``CacheFull``) unless every (slot, length) of ``wanted`` can be reserved
        together; takes nothing.  A step asks this before it reserves anything, so one that does not fit leaves
        no sequence with pages it did not commit."""
        for slot, length in wanted:
            if length > self.max_position:
                raise CapacityError(f"slot {slot}: {length} positions exceed the model's max_position {self.max_position}")
        for g in self.groups:
            need = sum(max(0, g.pages_needed(length) - len(g.pages_of[slot])) for slot, length in wanted)
            if g.shared:                              # the last holder of a page writes into the page itself
                writers: Dict[int, int] = {}
                for slot, length in wanted:
                    for i in g.written(slot, int(self.lengths[slot]), length):
                        p = g.pages_of[slot][i]
                        writers[p] = writers.get(p, 0) + 1
                need += sum(min(n, int(g.holders[p]) - 1) for p, n in writers.items())
            if need > g.pool.free:
                raise CacheFull(f"the step needs {need} more pages of group {g.index}, {g.pool.free} are free "
                                f"(the cache holds {self.max_tokens} positions in pages of {self.page_size})")

    def commit(self, slot: int, length: int) -> None:
        """Record that ``slot`` now holds ``length`` positions (after the step that wrote them)."""
        for g in self.groups:
            if len(g.pages_of[slot]) < g.pages_needed(length):
                raise ValueError(f"slot {slot}: {length} positions committed but not reserved")
        self.lengths[slot] = length

    def length(self, slot: int) -> int:
        return int(self.lengths[slot])

    def can_rewind(self, slot: int, length: int) -> bool:
        """Whether ``slot`` may go back to its first ``length`` positions and go on from there.  Always to where it
        is; further back only if every group keeps all keys (a ring has overwritten old ones) and no mixer keeps
        state of its own (which belongs to the sequence's end)."""
        held = int(self.lengths[slot])
        if length == held:
            return True
        return 0 <= length < held and not self.has_mixer_state and not any(g.ring_pages for g in self.groups)

    def rewind(self, slot: int, length: int) -> None:
        """Forget the positions from ``length`` on (their pages stay with the slot and are written again)."""
        if not self.slots.is_held(slot):
            raise ValueError(f"slot {slot} is not open")
        if not self.can_rewind(slot, length):
            raise ValueError(f"slot {slot} holds {int(self.lengths[slot])} positions and cannot go back to {length}")
        self.lengths[slot] = length

    # ------------------------------------------------------------------ sequences that share pages
    def fork(self, slot: int, count: int = 1, share: bool = True) -> List[int]:
        """``count`` new slots that hold what ``slot`` holds, its state included, and go on from there each for itself.  Their pages are
        ``slot``'s own until one of them writes into one (``share`` False, and a window's ring: copies from the start).  All or nothing."""
        if not self.slots.is_held(slot):
            raise ValueError(f"slot {slot} is not open")
        if count < 0:
            raise ValueError(f"a sequence cannot be forked {count} times")
        length = int(self.lengths[slot])
        for g in self.groups:
            need = count * g.pages_needed(length) if g.ring_pages or not share else 0
            if need > g.pool.free:
                raise CacheFull(f"slot {slot} cannot be forked {count} times: {need} {g.pool.what}(s) wanted, {g.pool.free} of {g.pool.n} free "
                                f"(the cache holds {self.max_tokens} positions in pages of {self.page_size})")
        new = self.slots.take(count)
        for s in new:
            for g in self.groups:
                (g.share if share and not g.ring_pages else g.duplicate)(slot, s, length)
            self.lengths[s] = length
        self.run_copies()                             # (in the stream's order: behind what wrote them, before what goes on)
        if new:
            plan = np.array([(slot, s, 1) for s in new], dtype=np.int32)
            for t in (t for t in self.state.values() if t.numel()):
                self._copy(t.view(1, self.n_slots, 1, 1, 1, -1), plan)
        return new

    def compact(self) -> int:
        """Move the held pages of every group to its lowest ids (what lies above is one free stretch then); how many pages moved.  What
        sequences hold stays what it was."""
        self.run_copies()
        moved = sum(g.compact() for g in self.groups)
        self.flush()
        return moved

    def run_copies(self) -> None:
        """Run the copies of pages that are pending, on the current stream."""
        for g in self.groups:
            if g.copies:
                for plan in g.plans():
                    self._copy(g.storage, plan)

    def _copy(self, storage: torch.Tensor, plan: np.ndarray) -> None:
        plan = torch.from_numpy(plan)
        if storage.is_cuda:
            if self.kernels is None:
                raise RuntimeError("the cache was made without the kernel library, which copies pages on a GPU")
            with torch.cuda.device(storage.device):
                self.kernels.copy_pages(storage, plan)
            return
        for a, b, n in plan.tolist():                 # host memory (bookkeeping without a GPU)
            storage[:, b, :, :, :n] = storage[:, a, :, :, :n]

    def shared_groups(self, slots: Sequence[int]) -> List[Tuple[List[int], int]]:
        """Groups of sequences of a step that hold the same pages for a prefix, as (places in ``slots``, pages): of the nested prefixes that
        a page's holders may have in common, those that spare the most pages.  Whole pages below each sequence's next position only;
        a sequence is in one group at most.  Empty where nothing is shared."""
        g = next((g for g in self.groups if not g.ring_pages), None)          # (what is shared is shared alike in every group that keeps all keys)
        if g is None or not g.shared or len(slots) < 2:
            return []
        slots = list(slots)
        full = [int(self.lengths[s]) // self.page_size for s in slots]
        rows = g.table_host[slots]

        # the tree of the prefixes, a node after the one that it is under (not by recursion: a sequence forked from the one before makes it as deep as
        # there are sequences): members, pages common to them, nodes below
        nodes: List[Tuple[List[int], int, List[int]]] = []
        todo = [(list(range(len(slots))), 0, -1)]
        while todo:
            members, depth, above = todo.pop()
            most = min(full[i] for i in members)
            same = (rows[members, depth:most] == rows[members[0], depth:most]).all(0)
            common = depth + (int(same.argmin()) if not same.all() else most - depth)
            if above >= 0:
                nodes[above][2].append(len(nodes))
            nodes.append((members, common, []))
            children: Dict[int, List[int]] = {}
            for i in members:
                if full[i] > common:
                    children.setdefault(int(rows[i, common]), []).append(i)
            todo += [(c, common, len(nodes) - 1) for c in reversed(list(children.values())) if len(c) > 1]
        # from below: a node's own prefix, or the best of those under it, whichever spares more
        spared = [0] * len(nodes)
        whole = [False] * len(nodes)
        for k in range(len(nodes) - 1, -1, -1):
            members, common, below = nodes[k]
            under = sum(spared[j] for j in below)
            whole[k] = (len(members) - 1) * common >= under
            spared[k] = max((len(members) - 1) * common, under)
        out, look = [], [0]
        while look:
            k = look.pop()
            members, common, below = nodes[k]
            if not whole[k]:
                look += reversed(below)
            elif common:
                out.append((members, common))
        return out

    def trim(self, slot: int) -> int:
        """Give back the slot's pages behind those that its positions lie in (taken ahead, or left by a rewind); how many."""
        if not self.slots.is_held(slot):
            raise ValueError(f"slot {slot} is not open")
        return sum(g.trim(slot, int(self.lengths[slot])) for g in self.groups)

    def free_tokens(self) -> int:
        """Positions that the free pages could still hold (the scarcest group decides)."""
        return min((g.pool.free for g in self.groups), default=self.n_pages) * self.page_size

    def held_tokens(self, slot: int) -> int:
        """Positions that the pages of ``slot`` hold room for (the group with the fewest pages decides)."""
        return min((len(g.pages_of[slot]) for g in self.groups), default=0) * self.page_size

    def shared_tokens(self, slot: int, start: int, length: int) -> int:
        """Positions of pages that ``slot`` shares and will need in its own right to be written from ``start`` to ``length``."""
        return max((len(g.written(slot, start, length)) for g in self.groups), default=0) * self.page_size

    def close(self, slots: Sequence[int]) -> None:
        """Give the slots and their pages back; later sequences use them again."""
        slots = list(slots)
        for s in slots:
            if not self.slots.is_held(s):
                raise ValueError(f"slot {s} is closed but is not open")
        self.slots.give(slots)
        for s in slots:
            for g in self.groups:
                g.release(s)
            self.lengths[s] = 0

    def flush(self) -> None:
        """Run what copies of pages are pending, and bring the device's block tables up to date with the host's."""
        self.run_copies()
        for g in self.groups:
            g.flush()

    def check(self) -> None:
        """Invariants of the bookkeeping (tests call this after every operation)."""
        self.slots.check()
        for g in self.groups:
            g.pool.check()
            seen: Dict[int, int] = {}
            for s in range(self.n_slots):
                pages = g.pages_of[s]
                if not self.slots.is_held(s):
                    assert not pages, f"closed slot {s} holds pages in group {g.index}"
                assert len(set(pages)) == len(pages), f"slot {s} holds a page of group {g.index} twice"
                for p in pages:
                    assert g.pool.is_held(p), f"page {p} of group {g.index} is in a table but free"
                    seen[p] = seen.get(p, 0) + 1
                assert g.table_host[s, :len(pages)].tolist() == pages, f"slot {s}: the table and its pages differ"
                assert len(pages) >= g.pages_needed(int(self.lengths[s])), f"slot {s} holds too few pages"
            for p in range(g.pool.n):
                assert g.holders[p] == seen.get(p, 0), f"page {p} of group {g.index} is held {seen.get(p, 0)} times, counted {g.holders[p]}"
            assert g.shared == sum(1 for n in seen.values() if n > 1), f"group {g.index}: shared pages are miscounted"
            assert len(seen) == g.pool.held, f"group {g.index}: {g.pool.held - len(seen)} page(s) held by no slot"
            keeping = [k for k in self.groups if not k.ring_pages]
            if g in keeping:                          # sequences share the same places in every group that keeps all keys
                for s in range(self.n_slots):
                    assert [g.holders[p] for p in g.pages_of[s]] == [keeping[0].holders[p] for p in keeping[0].pages_of[s]], f"slot {s} shares differently in group {g.index}"
