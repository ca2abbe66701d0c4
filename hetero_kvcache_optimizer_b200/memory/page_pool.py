"""Who owns the pages of a paged ``Int4KVStore``, kept on the device.

A page table alone says where a sequence's tokens lie; ``PagePool`` adds how many
table entries name each page (``refs``), so that sequences can share pages (the
samples of one prompt, the beams of a search), get new ones as they grow and
give them back. No call but ``free_pages`` reads anything back or waits for the
device (lists from the host travel in a launch's parameters), so all of them can
be captured in a CUDA graph beside the decode step; the same state always gives
the same page ids (the lowest free ones, in table order).

The reference keeps one cache per sequence and drops whole entries
(src/memory/dram_storage.py:20-255, src/memory/manager.py:1231-1299); it has no
sharing of pages to replace.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

from .. import _lib as L
from .. import kvstore as kv


class PagePool:
    """``store``: paged (its ``page_table`` and ``lengths`` are rewritten here).
    ``refs``: int32 [num_pages] counts to take over, e.g. of a pool that other
    stores hold pages of as well (default: counted from the table). Calls on one
    pool must not overlap (they share its workspace and its state)."""

    def __init__(self, store: kv.Int4KVStore, refs: Optional[torch.Tensor] = None):
        if not store.paged:
            raise ValueError("PagePool needs a paged store (Int4KVStore(num_pages=...))")
        self.store = store
        if refs is None:
            t = store.page_table.reshape(-1).long()
            held = (t >= 0) & (t < store.num_pages)
            refs = torch.zeros(store.num_pages, dtype=torch.int32, device=store.device)
            refs.index_add_(0, t[held], torch.ones_like(t[held], dtype=torch.int32))
        elif (refs.dtype != torch.int32 or refs.shape != (store.num_pages,) or not refs.is_contiguous()
              or refs.device != store.pool.device):
            raise ValueError(f"refs must be a contiguous int32 [{store.num_pages}] tensor on the store's device")
        self.refs = refs
        kv._require_cuda(store.pool, refs)
        self._struct = store.struct()  # addresses and geometry, which stay for the store's life
        self._ref = ctypes.byref(self._struct)
        nbytes = L.load().hkv_pages_workspace_bytes(self._ref, store.batch, store.kv_heads)
        if nbytes == 0:
            raise ValueError("unsupported store geometry")
        self._ws = torch.empty(nbytes, dtype=torch.uint8, device=store.pool.device)

    def _call(self, name: str, *args) -> None:
        st = self.store
        L.check(getattr(L.load(), name)(self._ref, st.batch, st.kv_heads, *args, self._ws.data_ptr(), self._ws.numel(),
                                        kv.raw_stream(self.refs.device)), name)

    def _per_sequence(self, x: Union[torch.Tensor, Sequence[int]], name: str) -> torch.Tensor:
        B = self.store.batch
        if isinstance(x, torch.Tensor):
            if x.shape != (B,) or x.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"{name} must be {B} integers, one per sequence")
            if x.is_cuda:
                if x.dtype == torch.int64:  # out of range stays out of range
                    x = x.clamp(-2**31, 2**31 - 1)
                return x.to(device=self.refs.device, dtype=torch.int32).contiguous()
        values = [int(v) for v in (x.tolist() if isinstance(x, torch.Tensor) else x)]
        if len(values) != B or any(not -2**31 <= v < 2**31 for v in values):
            raise ValueError(f"{name} must be {B} integers, one per sequence")
        with kv.launch_on(self.refs.device):
            out = torch.empty(B, dtype=torch.int32, device=self.refs.device)
            L.check(L.load().hkv_put_i32((ctypes.c_int32 * B)(*values), B, out.data_ptr(), kv.raw_stream(out.device)), "hkv_put_i32")
        return out

    def fork(self, parents: Union[torch.Tensor, Sequence[int]], stream=None) -> None:
        """Sequence b becomes what sequence ``parents[b]`` was, for all b at once
        (sampling several continuations, reordering the beams of a search); -1
        empties it. Full pages are shared; a partly filled last page goes to the
        lowest b with that parent and is copied for the others. An int32 tensor
        on the device is used as it is (a captured fork reads it at each replay;
        a list is kept as it was). Afterwards only tokens behind the lengths
        may be written: a sequence that is to be cut back into shared pages or
        filled anew is emptied (-1, ``free``) first."""
        with kv.launch_on(self.refs.device, stream):
            par = self._per_sequence(parents, "parents")
            self._call("hkv_pages_fork", self.refs.data_ptr(), par.data_ptr())

    def reserve(self, tokens: int = 1, tokens_of: Optional[torch.Tensor] = None, stream=None) -> None:
        """Room for ``tokens`` more tokens behind every sequence's length
        (``tokens_of`` int32 [B] lowers that per sequence): the pages it lacks
        are taken from the free ones. To be called before an append or a
        quantise-pack that may start a page."""
        with kv.launch_on(self.refs.device, stream):
            of = self._per_sequence(tokens_of, "tokens_of") if tokens_of is not None else None
            self._call("hkv_pages_reserve", self.refs.data_ptr(), int(tokens),
                       of.data_ptr() if of is not None else None)

    def free(self, sequences: Sequence[int], stream=None) -> None:
        """Empties the given sequences: their pages are free once no other
        sequence shares them."""
        gone = set(int(b) for b in sequences)
        if any(not 0 <= b < self.store.batch for b in gone):
            raise ValueError(f"sequences must lie in [0, {self.store.batch})")
        self.fork([-1 if b in gone else b for b in range(self.store.batch)], stream=stream)

    def compact(self, into: "PagePool", stream=None) -> None:
        """Copies every page in use (within the length of any sequence that names
        it) into another pool (same format, page size, batch and heads), in the
        order of the table: a sequence's pages become consecutive, so that a move
        to the host is a few long copies, and a smaller pool can take a
        thinned-out one. ``into`` is rewritten whole (table, lengths, counts);
        shared pages stay shared; this pool is left as it is."""
        a, b = self.store, into.store
        if (a.batch, a.kv_heads, a.fmt, a.group, a.page_tokens) != (b.batch, b.kv_heads, b.fmt, b.group, b.page_tokens):
            raise ValueError("compact needs a pool of the same batch, heads, format and page size")
        if a.pool.device != b.pool.device:
            raise ValueError("both pools must be on one device")
        with kv.launch_on(self.refs.device, stream):
            self._call("hkv_pages_compact", into._ref, into.refs.data_ptr())
        b.len_hint = a.len_hint

    def free_pages(self) -> int:
        """Pages that nobody names (waits for the device)."""
        return int((self.refs == 0).sum().item())
