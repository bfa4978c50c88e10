"""The cache of a model: a slot per live sequence, paged keys and values per layer,
and per-sequence state of fixed size.

The reference keeps one tensor [layers, kv_heads, max_seq_len, head_dim] for one
sequence (src/model/kv_cache.rs:23-53) and a position counter that the caller
advances (src/model/mod.rs:93).  Here many sequences live at once:

* a *slot* stands for one sequence; it records the sequence's length and is given
  back when the sequence ends, then used again;
* layers whose mixers ask for the same thing form a *group* with storage of its own.
  A paged group holds keys and values in pages of `PAGE` positions, per layer all key
  pages [pages, kv_heads, PAGE * head_dim] and then all value pages (keys as
  [PAGE, head_dim], values transposed as [value_dim, PAGE]), and a table from (slot,
  position // PAGE) to a page.  A group with a window gives pages back as soon as every
  position in them has left the window of the sequence's next position; the pages of
  the first `keep_first` positions are never given back while the sequence lives;
* a state group holds [layers, slots, *shape], zeroed when a slot is taken.

A sequence may go on from where another one stands (`fork`): it then holds the same pages, each of which knows how many
sequences hold it, and a copy of the state.  A page that several hold is never written: the step that would write to it
gives its sequence a page of its own with the positions so far (`prepare`).

All decisions are taken on the host; the device only sees the page tables.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Union

import numpy as np
import torch

from ..csrc.build import PAGE_TOKENS
from .pages import CacheCapacityError, CacheRollbackError, CacheStateError, FreeList
from .requests import PagedKVRequest, PagedLatentRequest, StateRequest

PAGE = PAGE_TOKENS   # tokens per cache page: the number the kernels were compiled with


def pages_for(n_tokens: int) -> int:
    return (n_tokens + PAGE - 1) // PAGE


@dataclass
class PagedView:
    """What an attention mixer gets for its layer."""
    k_pages: torch.Tensor       # [pages, kv_heads, PAGE, head_dim]
    v_pages: torch.Tensor       # [pages, kv_heads, value_dim, PAGE]: values lie transposed
    page_table: torch.Tensor    # [slots, pages per sequence] int32, on the device
    window: Optional[int]
    group: "PagedGroup"
    keep_first: int = 0


@dataclass
class LatentView:
    """What a latent-attention mixer gets for its layer."""
    pages: torch.Tensor         # [pages, PAGE, width]
    page_table: torch.Tensor    # [slots, pages per sequence] int32, on the device
    window: Optional[int]
    group: "PagedGroup"


class PagedGroup:
    """Pages of one kind of content (keys and values per head, or one latent vector per
    position) with their pool and page table; what a page holds does not matter to the
    bookkeeping."""

    def __init__(self, request: Union[PagedKVRequest, PagedLatentRequest], layers: Sequence[int],
                 n_pages: int, max_slots: int, table_width: int, dtype: torch.dtype,
                 device: torch.device):
        self.request = request
        self.layers = list(layers)
        self.n_pages = n_pages
        self.pool = FreeList(n_pages, "cache page")
        self.holders = np.zeros(n_pages, dtype=np.int32)   # sequences that hold a page
        self.forked = False                 # several may hold one page: a fork has been made since the pool was last empty
        if isinstance(request, PagedLatentRequest):
            shape = (len(self.layers), n_pages, PAGE * request.width)
        else:
            self._k_elems = n_pages * request.num_kv_heads * PAGE * request.head_dim
            shape = (len(self.layers),
                     self._k_elems + n_pages * request.num_kv_heads * PAGE * request.value_dim)
        self.storage = torch.zeros(shape, dtype=dtype, device=device)
        # columns of the table that hold the first `keep_first` positions: a window never returns them
        self.kept_cols = pages_for(getattr(request, "keep_first", 0)) if request.window else 0
        self.table_host = np.full((max_slots, table_width), -1, dtype=np.int32)
        self.table_dev = torch.full((max_slots, table_width), -1, dtype=torch.int32, device=device)
        self.first_live = [0] * max_slots   # first table column that still holds a page
        self.n_cols = [0] * max_slots       # table columns filled so far
        self._dirty: set = set()
        self.bytes_copied = 0   # host-to-device bytes of page-table rows so far
        # rows on their way to the device are snapshots in pinned memory (several in rotation):
        # the host may change the table again before an earlier copy has run
        self._staging = None
        self._staging_events = []
        self._turn = 0

    def pages_needed(self, slot: int, new_len: int) -> int:
        return max(0, pages_for(new_len) - self.n_cols[slot])

    def grow(self, slot: int, new_len: int) -> None:
        need = self.pages_needed(slot, new_len)
        if need == 0:
            return
        if pages_for(new_len) > self.table_host.shape[1]:
            raise CacheCapacityError(
                f"a sequence of {new_len} tokens is longer than the cache was sized for "
                f"({self.table_host.shape[1] * PAGE})")
        got = self.pool.take(need)
        c = self.n_cols[slot]
        self.holders[got] = 1
        self.table_host[slot, c:c + need] = got
        self.n_cols[slot] = c + need
        self._dirty.add(slot)

    def _drop(self, pages) -> None:
        """One sequence less holds each of these pages (-1: none); those that none holds any more go back."""
        pages = [int(p) for p in pages if p >= 0]
        self.holders[pages] -= 1
        self.pool.give_back(p for p in pages if self.holders[p] == 0)
        self.forked = self.forked and self.pool.held_count > 0

    def fork(self, src: Sequence[int], dst: Sequence[int], lengths: Sequence[int]) -> None:
        """Each slot dst[i] lets go of what it holds and holds the pages of the first lengths[i] positions of src[i] from now on.  (A
        step that was prepared and did not run to its end has left src[i] further pages, which it will write to: those stay its own.)"""
        cols = max(self.n_cols[s] for s in dst)
        gone = self.table_host[dst, :cols].ravel()
        gone = gone[gone >= 0]
        np.subtract.at(self.holders, gone, 1)
        keep = [min(self.n_cols[a], pages_for(n)) for a, n in zip(src, lengths)]
        rows = self.table_host[src]
        held = rows[:, :max(self.n_cols[a] for a in src)]
        held[np.arange(held.shape[1]) >= np.asarray(keep)[:, None]] = -1
        self.table_host[dst] = rows
        np.add.at(self.holders, held[held >= 0], 1)
        self.pool.give_back(np.unique(gone[self.holders[gone] == 0]).tolist())
        self.forked = True
        for a, b, c in zip(src, dst, keep):
            self.first_live[b], self.n_cols[b] = self.first_live[a], c
        self._dirty.update(dst)

    def writes_into_shared(self, slots: Sequence[int], lengths: Sequence[int]) -> List[int]:
        """Which of `slots` (indices into the list) need a page of their own before they write position lengths[i]: their last page is
        begun and several hold it.  Of sequences that hold one page together, the last need not copy it if no other holds it."""
        out, left = [], {}
        for i, (s, n) in enumerate(zip(slots, lengths)):
            if n % PAGE == 0:
                continue
            page = int(self.table_host[s, n // PAGE])
            holders = left.get(page, int(self.holders[page]))
            if holders > 1:
                out.append(i)
                left[page] = holders - 1
        return out

    def begun_copies(self, slots: Sequence[int], lengths: Sequence[int]) -> List[int]:
        """A new page for each of `slots` with what its page of position lengths[i] holds before that; no table names it yet."""
        if not slots:
            return []
        new = self.pool.take(len(slots))
        try:
            self.copy_pages([int(self.table_host[s, n // PAGE]) for s, n in zip(slots, lengths)], new, [n % PAGE for n in lengths])
        except Exception:
            self.pool.give_back(new)
            raise
        return new

    def unshare(self, slots: Sequence[int], lengths: Sequence[int], pages: Sequence[int]) -> None:
        """Puts the pages of `begun_copies` in the place of the pages of position lengths[i]."""
        for s, n, new in zip(slots, lengths, pages):
            self.holders[self.table_host[s, n // PAGE]] -= 1
            self.holders[new] = 1
            self.table_host[s, n // PAGE] = new
            self._dirty.add(s)

    def copy_pages(self, src: Sequence[int], dst: Sequence[int], counts: Sequence[int]) -> None:
        """The first counts[i] positions of page src[i] into page dst[i], in all layers."""
        r = self.request
        latent = isinstance(r, PagedLatentRequest)
        heads, dim, vdim = (1, r.width, 0) if latent else (r.num_kv_heads, r.head_dim, r.value_dim)
        if self.storage.is_cuda:
            from ..csrc import ops
            ops.core_ops(self.storage.dtype).copy_pages(self.storage.view(len(self.layers), -1), self.n_pages, heads, dim, vdim, src, dst, counts)
            return
        for layer in self.layers:              # (bookkeeping without a device)
            view = self.view(layer)
            for a, b, c in zip(src, dst, counts):
                if latent:
                    view.pages[b, :c] = view.pages[a, :c]
                else:
                    view.k_pages[b, :, :c] = view.k_pages[a, :, :c]
                    view.v_pages[b, :, :, :c] = view.v_pages[a, :, :, :c]

    def common_columns(self, groups: Sequence[Sequence[int]]) -> np.ndarray:
        """Per group of slots (all of one size) the leading columns in which their tables agree."""
        slots = np.asarray(groups)
        cols = np.asarray([max(self.n_cols[s] for s in g) for g in groups])
        width = int(cols.max())
        rows = self.table_host[slots, :width]                     # [groups, slots, columns]
        differ = np.ones((len(groups), width + 1), dtype=bool)    # (the column behind the last one ends what they have in common)
        differ[:, :width] = (rows != rows[:, :1]).any(axis=1)
        return np.minimum(differ.argmax(axis=1), cols)

    def trim(self, slot: int, next_pos: int) -> None:
        """Gives back the pages that no position >= next_pos can see any more."""
        w = self.request.window
        if not w:
            return
        first_needed_key = max(0, next_pos - w + 1)
        keep_from = min(first_needed_key // PAGE, self.n_cols[slot])
        f = self.first_live[slot]
        if keep_from > f:
            lo = max(f, self.kept_cols)      # columns below hold the kept first positions
            if keep_from > lo:
                self._drop(self.table_host[slot, lo:keep_from])
                self.table_host[slot, lo:keep_from] = -1
                self._dirty.add(slot)
            self.first_live[slot] = keep_from

    def can_truncate(self, slot: int, new_len: int) -> bool:
        """Whether the keys that position `new_len` will see are still held."""
        w = self.request.window
        if not w or new_len == 0:
            return True
        return max(0, new_len - w + 1) // PAGE >= self.first_live[slot]

    def truncate(self, slot: int, new_len: int) -> None:
        """Gives back the whole pages beyond `new_len` positions.  What lies beyond `new_len`
        in the last kept page stays there; kernels that read whole pages give it no weight, and
        the next tokens overwrite it."""
        keep = pages_for(new_len)
        f, c = self.first_live[slot], self.n_cols[slot]
        if keep >= c:
            return
        self._drop(self.table_host[slot, keep:c])
        self.table_host[slot, keep:c] = -1
        self.n_cols[slot] = keep
        self.first_live[slot] = min(f, keep)
        self._dirty.add(slot)

    def release(self, slot: int) -> None:
        c = self.n_cols[slot]
        self._drop(self.table_host[slot, :c])
        self.table_host[slot, :c] = -1
        self.first_live[slot] = 0
        self.n_cols[slot] = 0
        self._dirty.add(slot)

    def upload(self) -> None:
        if not self._dirty:
            return
        rows = sorted(self._dirty)
        self._dirty.clear()
        if not self.table_dev.is_cuda:
            idx = torch.as_tensor(rows, dtype=torch.long)
            self.table_dev.index_copy_(0, idx, torch.from_numpy(self.table_host[rows]))
            return
        chunk = 32   # rows per snapshot buffer
        width = self.table_host.shape[1]
        if self._staging is None:
            self._staging = torch.empty((4, chunk, width), dtype=torch.int32, pin_memory=True)
            self._staging_events = [None] * 4
        # One copy for dirty rows that lie close together, with those between (a reorder changes many rows, and a copy costs more than
        # 8 KB of it): [first, last] pairs, at most `chunk` rows long.
        spans: List[List[int]] = []
        for r in rows:
            if spans and r - spans[-1][0] < chunk and (r == spans[-1][1] + 1 or (len(rows) > 2 and (r - spans[-1][1] - 1) * width <= 2048)):
                spans[-1][1] = r
            else:
                spans.append([r, r])
        i = 0
        while i < len(spans):
            self._turn = (self._turn + 1) % 4
            if self._staging_events[self._turn] is not None:
                self._staging_events[self._turn].synchronize()
            stage = self._staging[self._turn]
            stage_np = stage.numpy()
            at = 0
            while i < len(spans) and at + spans[i][1] - spans[i][0] < chunk:
                first, end = spans[i][0], spans[i][1] + 1
                n = end - first
                stage_np[at:at + n] = self.table_host[first:end]
                self.table_dev[first:end].copy_(stage[at:at + n], non_blocking=True)
                self.bytes_copied += 4 * width * n
                at += n
                i += 1
            ev = self._staging_events[self._turn] or torch.cuda.Event()
            ev.record()
            self._staging_events[self._turn] = ev

    def view(self, layer: int):
        i = self.layers.index(layer)
        r = self.request
        if isinstance(r, PagedLatentRequest):
            return LatentView(self.storage[i].view(self.n_pages, PAGE, r.width), self.table_dev,
                              r.window, self)
        k = self.storage[i, :self._k_elems].view(self.n_pages, r.num_kv_heads, PAGE, r.head_dim)
        v = self.storage[i, self._k_elems:].view(self.n_pages, r.num_kv_heads, r.value_dim, PAGE)
        return PagedView(k, v, self.table_dev, r.window, self, r.keep_first if r.window else 0)


class StateGroup:
    def __init__(self, request: StateRequest, layers: Sequence[int], max_slots: int,
                 device: torch.device):
        self.request = request
        self.layers = list(layers)
        self.storage = torch.zeros((len(self.layers), max_slots, *request.shape),
                                   dtype=request.dtype, device=device)

    def reset(self, slot: int) -> None:
        self.storage[:, slot].zero_()

    def fork(self, src: Sequence[int], dst: Sequence[int], act_dtype: torch.dtype) -> None:
        """The state of each slot dst[i] becomes that of src[i], in all layers.  `act_dtype`: whose library is loaded already (bytes
        are copied, the state's type does not matter)."""
        if self.storage.is_cuda:
            from ..csrc import ops
            ops.core_ops(act_dtype).copy_slots(self.storage, src, dst)
        else:
            self.storage[:, list(dst)] = self.storage[:, list(src)]

    def view(self, layer: int) -> torch.Tensor:
        """[slots, *shape] of one layer."""
        return self.storage[self.layers.index(layer)]


class Cache:
    """`requests[k]` is what the mixer of the k-th entry of the layer order asks for
    (None: nothing, or it reads another entry's cache); "layer" below means such an entry.  `max_tokens` is the most tokens that live sequences hold
    at any time, each sequence's count rounded up to a multiple of PAGE."""

    def __init__(self, requests: Sequence[Union[PagedKVRequest, PagedLatentRequest, StateRequest, tuple, None]],
                 max_tokens: int, max_slots: Optional[int] = None,
                 max_seq_len: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda"):
        self.device = torch.device(device)
        self.dtype = dtype
        n_pages = max(1, pages_for(max_tokens))
        self.max_tokens = n_pages * PAGE
        self.max_slots = max_slots if max_slots else min(n_pages, 256)
        self.max_seq_len = min(max_seq_len, self.max_tokens) if max_seq_len else self.max_tokens
        table_width = pages_for(self.max_seq_len)
        self.slots = FreeList(self.max_slots, "sequence slot")
        self.lengths = [0] * self.max_slots
        self.paged: List[PagedGroup] = []
        self.states: List[StateGroup] = []
        self._of_layer: Dict[int, Union[PagedGroup, StateGroup]] = {}
        # A mixer made of several (branches side by side) asks for several things at once: a tuple
        # of requests, each of which joins the group of its kind under the key (entry, place).
        # A branch may itself ask for several things (a tuple inside the tuple): keys grow a place per level,
        # and `view` hands back tuples of the same shape.
        self._composite: Dict[int, object] = {}
        by_request: Dict[object, List[object]] = {}

        def walk(req, key):
            """Files every request of a (nested) tuple under its key; returns the keys in the tuple's shape."""
            if isinstance(req, (tuple, list)):
                return tuple(walk(sub, key + (j,)) for j, sub in enumerate(req))
            if req is None:
                return None
            by_request.setdefault(req, []).append(key)
            return key

        for layer, req in enumerate(requests):
            if isinstance(req, (tuple, list)):
                self._composite[layer] = walk(req, (layer,))
            elif req is not None:
                by_request.setdefault(req, []).append(layer)
        for req, layers in by_request.items():
            if isinstance(req, (PagedKVRequest, PagedLatentRequest)):
                g = PagedGroup(req, layers, n_pages, self.max_slots, table_width, dtype, self.device)
                self.paged.append(g)
            elif isinstance(req, StateRequest):
                g = StateGroup(req, layers, self.max_slots, self.device)
                self.states.append(g)
            else:
                raise TypeError(f"unknown cache request {req!r}")
            for layer in layers:
                self._of_layer[layer] = g

    # ---- slots -----------------------------------------------------------------
    def acquire(self, count: int = 1) -> List[int]:
        got = self.slots.take(count)
        for s in got:
            self.lengths[s] = 0
            for g in self.states:
                g.reset(s)
        return got

    def release(self, slots) -> None:
        slots = list(slots)
        for s in slots:
            if not self.slots.is_held(s):
                raise CacheStateError(f"sequence slot {s} is released but is not held")
        for s in slots:
            for g in self.paged:
                g.release(s)
            self.lengths[s] = 0
        self.slots.give_back(slots)

    def length(self, slot: int) -> int:
        return self.lengths[slot]

    def truncate(self, slot: int, length: int) -> None:
        """Shortens the sequence of `slot` to its first `length` tokens, so that its next step
        goes on from there.  The reference rolls its one sequence back by lowering the position
        counter (src/main.rs:1722-1726, the chat's /retry; src/model/mod.rs:234-237 for the
        return to zero); here whole pages beyond `length` also go back to the pool.

        Raises `CacheRollbackError`, and changes nothing, if a window has already given back
        keys that position `length` would see, or if `length` > 0 and a mixer keeps state of
        fixed size.  `length` = 0 is always possible: pages are given back and state is zeroed."""
        if not self.slots.is_held(slot):
            raise CacheStateError(f"sequence slot {slot} is shortened but is not held")
        cur = self.lengths[slot]
        if not 0 <= length <= cur:
            raise ValueError(f"a sequence of {cur} tokens cannot be shortened to {length}")
        if length == cur:
            return
        if length > 0:
            if self.states:
                raise CacheRollbackError(
                    "a mixer of this model keeps per-sequence state of fixed size, which cannot be "
                    "rolled back; only reset (length 0) is possible")
            for g in self.paged:
                if not g.can_truncate(slot, length):
                    w = g.request.window
                    raise CacheRollbackError(
                        f"slot {slot} cannot be shortened from {cur} to {length} tokens: position "
                        f"{length} sees keys from {max(0, length - w + 1)} on, but the window of {w} "
                        f"has already given back everything before {g.first_live[slot] * PAGE}")
        for g in self.paged:
            g.truncate(slot, length)
            g.upload()
        if length == 0:
            for g in self.states:
                g.reset(slot)
        self.lengths[slot] = length

    def reset(self, slot: int) -> None:
        """The sequence of `slot` starts again at its first token; the slot stays held."""
        self.truncate(slot, 0)

    # ---- one sequence going on from another one's cache ----------------------------
    def fork(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """The sequence of each held slot dst[i] ends and goes on as a copy of the sequence of src[i] (which may be a
        source several times, and is no destination).  Pages are held together from then on, state is copied."""
        src, dst = list(src), list(dst)
        if len(src) != len(dst):
            raise CacheStateError(f"{len(src)} sequences to copy and {len(dst)} slots for them")
        for s in src + dst:
            if not self.slots.is_held(s):
                raise CacheStateError(f"sequence slot {s} is copied but is not held")
        if len(set(dst)) != len(dst) or not set(dst).isdisjoint(src):
            raise CacheStateError("a sequence slot is written twice, or both copied from and written")
        if not src:
            return
        for g in self.states:            # (before the tables: a copy may be refused, where another device is the current one)
            g.fork(src, dst, self.dtype)
        for g in self.paged:
            g.fork(src, dst, [self.lengths[a] for a in src])
            g.upload()
        for a, b in zip(src, dst):
            self.lengths[b] = self.lengths[a]

    def reorder(self, slots: Sequence[int], parents: Sequence[int]) -> List[int]:
        """What a beam search does between two steps: place j goes on from the sequence at place parents[j].  Returns the slots in
        the new order.  A sequence that goes on keeps its slot in the first place that names it; the further
        places get copies in the slots of sequences that nobody names, so the fewest copies are made."""
        slots, parents = list(slots), list(parents)
        if len(parents) != len(slots) or (parents and not 0 <= min(parents) <= max(parents) < len(slots)):
            raise CacheStateError(f"{len(slots)} parents in [0, {len(slots)}) are needed, got {parents}")
        if len(set(slots)) != len(slots):
            raise CacheStateError("a sequence slot appears twice")
        named = set(parents)
        free = [s for j, s in enumerate(slots) if j not in named][::-1]
        out, src, dst, seen = [], [], [], set()
        for p in parents:
            if p in seen:
                src.append(slots[p])
                dst.append(free.pop())
                out.append(dst[-1])
            else:
                seen.add(p)
                out.append(slots[p])
        self.fork(src, dst)
        return out

    def common_columns(self, groups: Sequence[Sequence[int]]) -> List[int]:
        """Per group of slots (all of one size) the leading pages that their sequences hold together, in all layers."""
        if not self.paged or not groups:
            return [0] * len(groups)
        return np.minimum.reduce([g.common_columns(groups) for g in self.paged]).tolist()

    # ---- one step ----------------------------------------------------------------
    def prepare(self, slots: Sequence[int], new_lens: Sequence[int]) -> None:
        """Makes room for each sequence to reach its new length, gives a sequence that would write to a page
        which others hold too a page of its own, and brings the device's page tables up to date.  Nothing
        changes if there is no room or a copy is refused."""
        for s in slots:
            if not self.slots.is_held(s):
                raise CacheStateError(f"sequence slot {s} is used but is not held")
        if len(set(slots)) != len(slots):
            raise CacheStateError("a sequence slot appears twice in one step")
        for s, n in zip(slots, new_lens):
            if n > self.max_seq_len:
                raise CacheCapacityError(
                    f"a sequence of {n} tokens is longer than the cache was sized for "
                    f"({self.max_seq_len})")
        past = [self.lengths[s] for s in slots]
        copies = [g.writes_into_shared(slots, past) if g.forked else [] for g in self.paged]
        for g, shared in zip(self.paged, copies):
            need = sum(g.pages_needed(s, n) for s, n in zip(slots, new_lens)) + len(shared)
            if need > g.pool.free_count:
                raise CacheCapacityError(
                    f"the cache is full: this step needs {need} more pages of {PAGE} tokens, "
                    f"{g.pool.free_count} of {g.n_pages} are free")
        # The copies come before the tables change: they may be refused (where another device is the current one).
        copies = [([slots[i] for i in shared], [past[i] for i in shared]) if shared else ((), ()) for shared in copies]
        pages: List[List[int]] = []
        try:
            for g, (of, lens) in zip(self.paged, copies):
                pages.append(g.begun_copies(of, lens))
        except Exception:
            for g, got in zip(self.paged, pages):
                g.pool.give_back(got)
            raise
        for g, (of, lens), got in zip(self.paged, copies, pages):
            g.unshare(of, lens, got)
            for s, n in zip(slots, new_lens):
                g.grow(s, n)
            g.upload()

    def commit(self, slots: Sequence[int], new_lens: Sequence[int]) -> None:
        """Records the new lengths after a step and lets windows give pages back."""
        for s, n in zip(slots, new_lens):
            self.lengths[s] = n
            for g in self.paged:
                g.trim(s, n)
        for g in self.paged:
            g.upload()

    # ---- views ---------------------------------------------------------------------
    def view(self, layer: int):
        if layer in self._composite:
            def views(keys):
                if keys is None:
                    return None
                if keys and isinstance(keys[0], int):          # a key: (entry, place, ...)
                    return self._of_layer[keys].view(keys)
                return tuple(views(k) for k in keys)
            return views(self._composite[layer])
        g = self._of_layer.get(layer)
        return None if g is None else g.view(layer)

    def check(self) -> None:
        """Host-side consistency: nothing lost, nothing held twice."""
        self.slots.check()
        for g in self.paged:
            g.pool.check()
            seen: Dict[int, int] = {}
            for s in range(self.max_slots):
                pages = [int(p) for p in g.table_host[s] if p >= 0]
                if pages and not self.slots.is_held(s):
                    raise CacheStateError(f"free slot {s} still holds pages")
                if len(set(pages)) != len(pages):
                    raise CacheStateError(f"slot {s} holds a page twice")
                if any(p >= 0 and g.holders[p] > 1 for p in g.table_host[s, pages_for(self.lengths[s]):]):
                    raise CacheStateError(f"slot {s} holds a page beyond its length that others hold too")
                for p in pages:
                    if not g.pool.is_held(p):
                        raise CacheStateError(f"page {p} is in a table but free")
                    seen[p] = seen.get(p, 0) + 1
            for p, n in seen.items():
                if n != g.holders[p]:
                    raise CacheStateError(f"page {p} is in {n} places, held by {g.holders[p]}")
            if len(seen) != g.pool.held_count:
                raise CacheStateError("a held page is in no table")

    def bytes_held(self) -> int:
        return sum(g.storage.numel() * g.storage.element_size() for g in self.paged + self.states)
