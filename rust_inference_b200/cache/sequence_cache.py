"""The device cache: keys and values for every cache layer, one slot per sequence, and a
fixed-size per-sequence state area beside them.

Layers ask for what they need (`KVRequest`, `StateRequest`); layers with the same needs
form a *group* with storage of its own:

  kv group     K, V: [layers in group, pages, kv heads, page_size, head_dim], in the run
               dtype (V with a head size of its own when the request gives one).  A (page,
               kv head) is a dense [page_size, head_dim] tile.  Groups are keyed by (kv
               heads, head_dim, window, value head size), so layers that keep all keys and
               layers that look at a window do not share storage.  A request may say that its
               values are the leading channels of its keys (one row per position that serves as
               both, as attention over a shared latent keeps it): then there is no V, and the
               layer's `v` is its `k`.
               With `kv_dtype` int8 a group holds 8-bit codes and their scales instead (`kernels.quantized_cache`): K, V as above
               but int8, and per page and kv head one float32 scale for every 16 positions of each.  Layers whose request
               does not say that it can be held so are refused.
  state group  [layers in group, slots, *shape]: state of fixed size per sequence, zeroed
               when the slot is handed out (a recurrent mixer's matrix state, for one).

A mixer made of several mixers asks for several things at once: a tuple of requests, answered
by a `CompositeLayer` whose `parts` are the answers in the same order, each in its own group.  A member
may itself ask for several things (a recurrent mixer that keeps a matrix state and the last inputs of a
short convolution): tuples nest, and so do the answers.

All kv groups share one paging (`SlotPager`): position p of a slot lies in page
`page_table[slot, p // page_size]` at offset `p % page_size`, in every layer.  The
reference's per-layer `[max_seq_len, kv_dim]` pair with one length counter
(kv_cache.rs:25-50) is the one-slot, one-page-per-sequence case of this.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from .pager import SlotPager, CacheError, CacheFull  # noqa: F401

PAGE_SIZE = 64


@dataclass(frozen=True)
class KVRequest:
    n_kv_heads: int
    head_dim: int
    window: int | None = None      # None: the layer reads all keys
    v_head_dim: int | None = None  # None: values have the keys' head size
    values_in_keys: bool = False   # the values are the first v_head_dim channels of the keys: no storage of their own
    quantizable: bool = field(default=False, compare=False)    # the layer writes and reads a cache in 8 bits if it is given one


@dataclass(frozen=True)
class StateRequest:
    shape: tuple
    dtype: torch.dtype = torch.float32


@dataclass
class KVLayer:
    k: torch.Tensor                # [pages, kv heads, page_size, head_dim]
    v: torch.Tensor
    request: KVRequest


@dataclass
class StateLayer:
    state: torch.Tensor            # [slots, *shape]
    request: StateRequest


@dataclass
class CompositeLayer:
    parts: tuple                   # KVLayer / StateLayer, in the order of the request's members
    request: tuple


class SequenceCache:
    def __init__(self, requests: list, *, max_tokens: int, max_seq_len: int, dtype: torch.dtype,
                 device, n_slots: int | None = None, page_size: int = PAGE_SIZE, kv_dtype: torch.dtype | None = None):
        """requests[i] is what cache layer i needs (KVRequest, StateRequest or None).  `kv_dtype`: None, keys and values in the run
        dtype, or torch.int8.
        `max_tokens` is the number of positions all live sequences may hold together, each
        sequence's count rounded up to a whole page."""
        if kv_dtype not in (None, torch.int8):
            raise ValueError(f"cache: keys and values are kept in the run dtype or as int8, not {kv_dtype}")
        self.kv_dtype = kv_dtype
        self.device = torch.device(device)
        self.dtype = dtype
        self.page_size = page_size
        n_pages = max(1, -(-max_tokens // page_size))
        max_seq_len = min(max_seq_len, n_pages * page_size)
        if n_slots is None:
            n_slots = min(n_pages, 1024)
        self.pager = SlotPager(n_slots, n_pages, page_size, max_seq_len)
        self.max_seq_len = max_seq_len
        self.n_slots = n_slots
        self.n_pages = n_pages

        self.page_table_host = np.zeros((n_slots, self.pager.max_pages_per_slot), dtype=np.int32)
        self.page_table = torch.zeros((n_slots, self.pager.max_pages_per_slot), dtype=torch.int32,
                                      device=self.device)

        self._stage_bufs = [None] * 4
        self._stage_events = [None] * 4
        self._stage_turn = 0
        self.h2d_bytes = 0             # bytes of page-table entries copied to the device so far

        # group layers by their needs
        self.groups: dict = {}
        self._layers: list = [None] * len(requests)
        members: dict = {}                      # request -> [path]: the cache layer, then the places inside composites

        def enlist(req, path):
            """A composite's members are answered each in the group of its kind; a member may be a composite itself."""
            if isinstance(req, tuple):
                for m, sub in enumerate(req):
                    enlist(sub, path + (m,))
            elif req is not None:
                if kv_dtype is not None and isinstance(req, KVRequest) and not req.quantizable:
                    raise CacheError(f"cache layer {path[0]}: keys and values of this kind are not kept in 8 bits ({req})")
                members.setdefault(req, []).append(path)

        def composites(req, path):
            layer = CompositeLayer([None] * len(req), req)
            for m, sub in enumerate(req):
                if isinstance(sub, tuple):
                    layer.parts[m] = composites(sub, path + (m,))
            return layer

        for i, req in enumerate(requests):
            enlist(req, (i,))
            if isinstance(req, tuple):
                self._layers[i] = composites(req, (i,))

        def place(path, layer):
            if len(path) == 1:
                self._layers[path[0]] = layer
                return
            at = self._layers[path[0]]
            for m in path[1:-1]:
                at = at.parts[m]
            at.parts[path[-1]] = layer

        for req, users in members.items():
            if isinstance(req, KVRequest):
                shape = (len(users), n_pages, req.n_kv_heads, page_size, req.head_dim)
                if kv_dtype is not None:
                    from ..kernels import quantized_cache
                    if page_size != quantized_cache.PAGE_SIZE:
                        raise ValueError(f"cache: pages of {page_size} positions are not kept in 8 bits")
                    v_shape = shape[:-1] + (req.v_head_dim or req.head_dim,)
                    s_shape = shape[:3] + (page_size // quantized_cache.BLOCK,)
                    k, v = (torch.zeros(sh, dtype=kv_dtype, device=self.device) for sh in (shape, v_shape))
                    ks, vs = (torch.zeros(s_shape, dtype=torch.float32, device=self.device) for _ in range(2))
                    self.groups[req] = (k, v, ks, vs)
                    for j, path in enumerate(users):
                        place(path, quantized_cache.QuantizedPages(k[j], v[j], ks[j], vs[j], req))
                    continue
                k = torch.zeros(shape, dtype=dtype, device=self.device)
                if req.values_in_keys:
                    if (req.v_head_dim or req.head_dim) > req.head_dim:
                        raise ValueError(f"cache: values of {req.v_head_dim} channels do not fit inside keys of {req.head_dim}")
                    v = k
                    self.groups[req] = (k,)
                else:
                    v = torch.zeros(shape[:-1] + (req.v_head_dim or req.head_dim,), dtype=dtype, device=self.device)
                    self.groups[req] = (k, v)
                for j, path in enumerate(users):
                    place(path, KVLayer(k[j], v[j], req))
            elif isinstance(req, StateRequest):
                s = torch.zeros((len(users), n_slots) + tuple(req.shape), dtype=req.dtype,
                                device=self.device)
                self.groups[req] = (s,)
                for j, path in enumerate(users):
                    place(path, StateLayer(s[j], req))
            else:
                raise TypeError(f"cache layers {[path[0] for path in users]}: unknown request {req!r}")

        def freeze(layer):
            if isinstance(layer, CompositeLayer):
                layer.parts = tuple(freeze(part) for part in layer.parts)
            return layer

        for layer in self._layers:
            freeze(layer)

    # ---- what the model reads --------------------------------------------
    def layer(self, index: int):
        return self._layers[index]

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for g in self.groups.values() for t in g)

    # ---- slots -------------------------------------------------------------
    def alloc_slot(self) -> int:
        slot = self.pager.alloc_slot()
        for req, tensors in self.groups.items():
            if isinstance(req, StateRequest):
                tensors[0][:, slot].zero_()
        return slot

    def free_slot(self, slot: int) -> None:
        self.pager.free_slot(slot)

    def length(self, slot: int) -> int:
        return self.pager.length(slot)

    def _staging(self, n: int) -> torch.Tensor:
        """A pinned int32 buffer of n entries whose earlier use has been copied out: page-table
        updates go through these, so that publishing them never blocks the host on the stream."""
        i = self._stage_turn
        self._stage_turn = (i + 1) % len(self._stage_bufs)
        if self._stage_events[i] is not None:
            self._stage_events[i].synchronize()
        buf = self._stage_bufs[i]
        if buf is None or buf.numel() < n:
            buf = torch.empty(max(256, 2 * n), dtype=torch.int32).pin_memory()
            self._stage_bufs[i] = buf
        return buf

    def reserve(self, wants: list[tuple]) -> None:
        """Make room for (slot, new_length) pairs, all or nothing, and publish the page table
        entries that were added to the device (asynchronously, in stream order)."""
        added = {slot: pages for slot, pages in self.pager.reserve_many(wants).items() if pages}
        if not added:
            return
        total = sum(len(p) for p in added.values())
        self.h2d_bytes += 4 * total
        if self.device.type != "cuda":
            for slot, pages in added.items():
                have = self.pager.page_count(slot)
                self.page_table_host[slot, have - len(pages):have] = pages
                self.page_table[slot, have - len(pages):have] = torch.tensor(pages, dtype=torch.int32)
            return
        buf = self._staging(total)
        off = 0
        for slot, pages in added.items():
            have = self.pager.page_count(slot)
            self.page_table_host[slot, have - len(pages):have] = pages
            buf[off:off + len(pages)] = torch.tensor(pages, dtype=torch.int32)
            self.page_table[slot, have - len(pages):have].copy_(buf[off:off + len(pages)], non_blocking=True)
            off += len(pages)
        ev = torch.cuda.Event()
        ev.record()
        self._stage_events[(self._stage_turn - 1) % len(self._stage_bufs)] = ev

    def commit(self, slot: int, new_length: int) -> None:
        self.pager.set_length(slot, new_length)

    def lengths(self, slots: list) -> list:
        return self.pager.lengths(slots)

    def advance(self, slots: list, counts: list) -> None:
        """The end of a step: every slot's length moves on by the tokens it was given."""
        self.pager.advance(slots, counts)
