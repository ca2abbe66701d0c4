"""Multi-layer tiered INT4 KV cache for decoding, built on libhetero_kv.

Per layer it keeps the three zones of HeteroKVManager (src/memory/manager.py:
sink + recent tail in fp16/bf16 HBM, the evicted body as packed INT4 pages)
and runs one decode step as ONE launch (``fused_append``, the default for the
fp16min format):

    decode_append  (new token -> recent ring; oldest ring row -> INT4 body;
                    split-KV GQA attention over body + sink/recent, LSE merge)

or, with ``fused_append=False`` (the default for the ref format), as the two
launches it fuses (append_kv, then decode). In the ref format the fused launch's
append job shares a warp with the metadata expansion of the CTA's first tiles
and holds the CTA back: 107.4 us per layer against 95.4 us for the two launches
(config 1); in fp16min the append has a warp of its own and the fused step is
the faster one (2.485 against 2.569 ms per 32-layer step). All state (lengths, ring heads) lives on the device, so a whole
multi-layer step can be captured once into a CUDA graph and replayed every token.

Several sequences from one prompt: ``attach_prefix`` puts a shared INT4 prefix in
front of every layer's cache (read once for all of its sequences), ``num_pages``
keeps the bodies in page pools, ``fork`` continues sequences from others (samples,
beams), and ``set_rotary`` lets a step take the queries and keys as the layer's
projections give them (normed and rotated in one launch before the append).
"""
from __future__ import annotations

import bisect
from typing import List, Optional, Sequence, Union

import torch

from . import _lib as L
from . import kvstore as kv
from .memory.page_pool import PagePool


class TieredKVDecoder:
    def __init__(self, num_layers: int, batch: int, q_heads: int, kv_heads: int, *,
                 sink: int = 64, recent: int = 1024, body_capacity: int = 32768,
                 fmt: str = "fp16min", group: int = 32, page_tokens: int = 256,
                 kv_dtype: torch.dtype = torch.float16, out_dtype: torch.dtype = torch.float32,
                 device="cuda", ctas: int = 0, fused_append: Optional[bool] = None,
                 early: Optional[bool] = None, num_pages: Optional[int] = None):
        # the fused launch takes at most 8 query heads per KV head; more run as
        # the two launches (the attention split in groups of at most 8)
        fused_ok = q_heads // kv_heads <= 8
        self.fused_append = (fmt != "ref" and fused_ok) if fused_append is None else fused_append
        if self.fused_append and not fused_ok:
            raise ValueError("fused_append needs at most 8 query heads per KV head")
        self.early = early
        self.num_layers, self.batch = num_layers, batch
        self.q_heads, self.kv_heads = q_heads, kv_heads
        self.sink, self.recent = sink, recent
        self.fmt, self.group = fmt, group
        self.kv_dtype, self.out_dtype = kv_dtype, out_dtype
        self.device = torch.device(device)
        self.ctas = ctas
        self.stores: List[kv.Int4KVStore] = []
        self.dense: List[kv.DenseKV] = []
        for _ in range(num_layers):
            self.stores.append(kv.Int4KVStore(batch, kv_heads, body_capacity, fmt=fmt, group=group,
                                              page_tokens=page_tokens, num_pages=num_pages, device=self.device))
            self.dense.append(kv.DenseKV(batch, kv_heads, sink + recent, dtype=kv_dtype,
                                         device=self.device))
        # with num_pages (pages per layer), the bodies' pages are owned by pools
        self.pools: List[PagePool] = [PagePool(st) for st in self.stores] if num_pages is not None else []
        self.prefixes: Optional[List[kv.SharedPrefix]] = None
        self._groups: List[tuple] = []  # per sequence, the group of its slot in each layer's prefix
        self._behind: List[tuple] = []  # ... and the one that its own tokens were computed behind
        self._mixed: List[int] = []     # sequences for which they differ
        self._nobody: Optional[torch.Tensor] = None
        self._rotary = None
        self.positions: Optional[torch.Tensor] = None
        self.body_len = 0
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.host_graph: Optional[torch.cuda.CUDAGraph] = None
        self._static = None
        self._host = None

    # ------------------------------------------------------------------ prefill
    def prefill_layer(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v [B, Hkv, S, 128]: the first ``sink`` tokens and the last
        ``recent`` stay dense, the rest is quantised into the INT4 body."""
        S = k.shape[2]
        d, st = self.dense[layer], self.stores[layer]
        ns = min(self.sink, S)
        nr = min(self.recent, S - ns)
        d.k[:, :, :ns] = k[:, :, :ns]
        d.v[:, :, :ns] = v[:, :, :ns]
        if nr:
            d.k[:, :, self.sink:self.sink + nr] = k[:, :, S - nr:]
            d.v[:, :, self.sink:self.sink + nr] = v[:, :, S - nr:]
        nb = S - ns - nr
        self._set_behind(self._groups)
        if self.pools:  # pages that others share as well must not be written
            self._empty_pool(layer)
            self.pools[layer].reserve(nb)
        if nb:
            kv.prefill(st, k[:, :, ns:ns + nb], v[:, :, ns:ns + nb])
        else:
            st.set_lengths(0)
        d.set_lengths(ns + nr if ns == self.sink else ns)
        d.ring_head.zero_()
        self.body_len = nb

    def set_state(self, body_len: int) -> None:
        """Declare that every layer holds ``body_len`` INT4 tokens and a full sink + ring
        (with ``num_pages``, on pages of each sequence's own)."""
        self._set_behind(self._groups)
        for l, (st, d) in enumerate(zip(self.stores, self.dense)):
            if self.pools:
                self._empty_pool(l)
                self.pools[l].reserve(body_len)
            st.set_lengths(body_len)
            d.set_lengths(self.sink + self.recent)
            d.ring_head.zero_()
        self.body_len = body_len

    # ------------------------------------------------------------------ several sequences from one prompt
    def _empty_pool(self, layer: int) -> None:
        if self._nobody is None:
            self._nobody = torch.full((self.batch,), -1, dtype=torch.int32, device=self.device)
        self.pools[layer].fork(self._nobody)

    def attach_prefix(self, prefixes: Optional[Sequence[kv.SharedPrefix]]) -> None:
        """One shared prefix per layer (None: none), in front of what the layer's
        cache holds; it stays attached until replaced. Steps then append and run
        ``kvstore.decode_shared`` (large groups: fastest with ``out_dtype`` bfloat16).
        A sequence's group is that of its slot in the
        batch: what the caches hold now is taken to belong behind it. A captured
        step is dropped: ``capture`` again."""
        if prefixes is not None:
            prefixes = list(prefixes)
            if len(prefixes) != self.num_layers:
                raise ValueError(f"attach_prefix needs {self.num_layers} prefixes, one per layer")
            for p in prefixes:
                if p.store.kv_heads != self.kv_heads or p.group_start[-1] > self.batch:
                    raise ValueError("a prefix with other KV heads or more sequences than the batch")
        self.prefixes = prefixes
        self._groups = ([tuple(bisect.bisect_right(p.group_start, b) if b < p.group_start[-1] else 0 for p in prefixes)
                         for b in range(self.batch)] if prefixes is not None else [])
        self._set_behind(self._groups)
        self.graph = self.host_graph = self._host = None

    def _set_behind(self, groups: List[tuple]) -> None:
        self._behind = list(groups)
        self._mixed = [b for b, (x, y) in enumerate(zip(self._behind, self._groups)) if x != y]

    def _check_context(self) -> None:
        """A fork moves a sequence's own tokens, not its slot's prefix: attention over
        both would be over a context that no prompt had."""
        if self._mixed:
            raise RuntimeError(f"sequences {self._mixed} were forked from another prefix group: their tokens do not follow their "
                               "slot's prefix (fork within groups, fill them anew, or attach_prefix with other groups)")

    def reserve(self, tokens: int) -> None:
        """Pages for ``tokens`` more body tokens in every layer (``num_pages`` only)."""
        if not self.pools:
            raise RuntimeError("reserve needs a decoder with num_pages")
        for pool in self.pools:
            pool.reserve(tokens)

    def fork(self, parents: Union[torch.Tensor, Sequence[int]]) -> None:
        """Sequence b continues from what sequence ``parents[b]`` was, in every layer
        and for all b at once (``num_pages`` only): body pages are shared or copied
        (``PagePool.fork``), the sink and recent rows and their state are copied, and
        ``positions`` of a captured step; -1 empties a sequence (its position is 0).
        ``reserve`` before the next steps.

        With a prefix attached, a parent lies in the sequence's own group (the prefix
        is the slot's): parents given on the host from another group leave sequences
        that the next step refuses, until they are filled anew, forked back or given
        another prefix; parents on the device are not known here and are the caller's
        to keep within the groups."""
        if not self.pools:
            raise RuntimeError("fork needs a decoder with num_pages")
        par = self.pools[0]._per_sequence(parents, "parents")
        if not isinstance(parents, torch.Tensor) and any(not -1 <= int(b) < self.batch for b in parents):
            raise ValueError(f"parents must be -1 or lie in [0, {self.batch})")
        if self._groups and not (isinstance(parents, torch.Tensor) and parents.is_cuda):
            old = self._behind
            self._set_behind([old[a] if 0 <= a < self.batch else self._groups[b] for b, a in enumerate(int(x) for x in parents)])
        at = par.long().clamp(0, self.batch - 1)  # values on the device are not known here
        gone = par != at
        if self.positions is not None:  # of the captured step's next tokens
            self.positions.copy_(self.positions.index_select(0, at).masked_fill_(gone, 0))
        for pool, d in zip(self.pools, self.dense):
            for t in (d.k, d.v, d.lengths, d.ring_head):
                t.copy_(t.index_select(0, at))
            d.lengths.masked_fill_(gone, 0)
            d.ring_head.masked_fill_(gone, 0)
            pool.fork(par)

    def set_rotary(self, table: torch.Tensor, q_weights: Optional[Sequence[torch.Tensor]] = None,
                   k_weights: Optional[Sequence[torch.Tensor]] = None, eps: float = 1e-6,
                   adjacent: bool = False) -> None:
        """Steps that are given positions take queries and keys before their norm
        and rotation: ``kvstore.norm_rope`` with ``table`` and the layers' head-norm
        weights (None: no norm) runs ahead of each layer's append. A step captured
        with positions holds the addresses of the table and weights before and is
        dropped: ``capture`` again."""
        for w in (q_weights, k_weights):
            if w is not None and len(w) != self.num_layers:
                raise ValueError(f"set_rotary needs {self.num_layers} weights, one per layer")
        self._rotary = (table, q_weights, k_weights, eps, adjacent)
        if self.positions is not None:
            self.graph = None

    def _ready(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, positions: Optional[torch.Tensor]):
        if positions is None:
            return q, k_new
        if self._rotary is None:
            raise RuntimeError("positions without set_rotary")
        table, qw, kw, eps, adjacent = self._rotary
        return kv.norm_rope(q, k_new, positions, table, qw[layer] if qw is not None else None,
                            kw[layer] if kw is not None else None, eps=eps, adjacent=adjacent)

    # ------------------------------------------------------------------ decode
    def step_layer(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                   out: Optional[torch.Tensor] = None, len_hint: Optional[int] = None,
                   early: bool = False) -> torch.Tensor:
        """One layer's decode step. ``early``: the launch just before this one on
        the stream does not write this layer's cache (another layer's step), so
        the fused launch may stream the cache while that one finishes."""
        st, d = self.stores[layer], self.dense[layer]
        hint = len_hint if len_hint is not None else self.body_len + 1
        if self.prefixes is not None:
            self._check_context()
            kv.append_kv(k_new, v_new, d, self.sink, st)
            return kv.decode_shared(q, self.prefixes[layer], st, d, out_dtype=self.out_dtype, out=out, ctas=self.ctas,
                                    body_len=hint, dense_len=self.sink + self.recent)
        if self.fused_append:
            return kv.decode_append(q, k_new, v_new, d, self.sink, st, out_dtype=self.out_dtype, out=out,
                                    ctas=self.ctas, body_len=hint, dense_len=self.sink + self.recent,
                                    early=early)
        kv.append_kv(k_new, v_new, d, self.sink, st)
        return kv.decode(q, st, d, out_dtype=self.out_dtype, out=out, ctas=self.ctas,
                         body_len=hint, dense_len=self.sink + self.recent)

    @property
    def launches_per_layer(self) -> int:
        """Kernel launches of one layer's decode step, with at most 8 query heads per
        KV head; ``norm_rope``'s (steps with positions) comes on top."""
        return 4 if self.prefixes is not None else 1 if self.fused_append else 2

    @property
    def _early(self) -> bool:
        # a step runs the layers in order, so with two or more layers the launch
        # before a layer's is always another layer's (which never writes its cache)
        return self.num_layers >= 2 if self.early is None else (self.early and self.num_layers >= 2)

    def _early_layer(self, layer: int) -> bool:
        # a call on layer 0's pool may be the launch just before a step
        return self._early and not (layer == 0 and self.pools)

    def step(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
             out: Optional[torch.Tensor] = None, len_hint: Optional[int] = None,
             positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q [L, B, Hq, 128], k_new/v_new [L, B, Hkv, 128] -> out [L, B, Hq, 128].
        ``positions`` (int32 or int64 [B], after ``set_rotary``): q and k_new are
        still to be normed and rotated."""
        if out is None:
            out = torch.empty(self.num_layers, self.batch, self.q_heads, 128, dtype=self.out_dtype,
                              device=self.device)
        for l in range(self.num_layers):
            ql, kl = self._ready(l, q[l], k_new[l], positions)
            self.step_layer(l, ql, kl, v_new[l], out=out[l], len_hint=len_hint, early=self._early_layer(l))
        self.body_len += 1
        return out

    def decode_only(self, q: torch.Tensor, out: torch.Tensor, len_hint: Optional[int] = None) -> None:
        """Attention of every layer without appending (cache unchanged)."""
        hint = len_hint if len_hint is not None else self.body_len
        self._check_context()
        for l in range(self.num_layers):
            if self.prefixes is not None:
                kv.decode_shared(q[l], self.prefixes[l], self.stores[l], self.dense[l], out_dtype=self.out_dtype, out=out[l],
                                 ctas=self.ctas, body_len=hint, dense_len=self.sink + self.recent)
                continue
            kv.decode(q[l], self.stores[l], self.dense[l], out_dtype=self.out_dtype, out=out[l],
                      ctas=self.ctas, body_len=hint, dense_len=self.sink + self.recent)

    # ------------------------------------------------------------------ CUDA graph
    def capture(self, max_steps: int, positions: Optional[torch.Tensor] = None) -> None:
        """Capture one decode step over static input/output buffers. The split
        grid is sized for a body of ``body_len + max_steps`` tokens; device-side
        lengths keep replays exact as the body grows. Steps captured before
        (``capture_host``'s too) are dropped. ``positions`` (after
        ``set_rotary``): the positions of the first step's tokens; the captured
        step norms and rotates its queries and keys and moves ``self.positions``
        on by one (negative ones, sequences that pad the batch, stay)."""
        self.graph = self.host_graph = self._host = None  # they hold the buffers that are replaced here
        Lyr, B = self.num_layers, self.batch
        q = torch.zeros(Lyr, B, self.q_heads, 128, dtype=torch.bfloat16, device=self.device)
        kn = torch.zeros(Lyr, B, self.kv_heads, 128, dtype=self.kv_dtype, device=self.device)
        vn = torch.zeros_like(kn)
        out = torch.empty(Lyr, B, self.q_heads, 128, dtype=self.out_dtype, device=self.device)
        hint = self.body_len + max_steps
        self._hint = hint
        self.positions = None if positions is None else positions.to(device=self.device, dtype=torch.int32).clone()

        def run():
            for l in range(Lyr):
                ql, kl = self._ready(l, q[l], kn[l], self.positions)
                self.step_layer(l, ql, kl, vn[l], out=out[l], len_hint=hint, early=self._early_layer(l))
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        g = torch.cuda.CUDAGraph()
        # warm the library (function attributes, workspace) outside capture, on a
        # throwaway copy of the state, then restore it
        snap = self._snapshot()
        with torch.cuda.stream(s):
            run()
        s.synchronize()
        self._restore(snap)
        with torch.cuda.graph(g, stream=s):
            run()
            if self.positions is not None:
                self.positions += self.positions >= 0  # a sequence that pads the batch stays one
        torch.cuda.current_stream(self.device).wait_stream(s)
        self.graph = g
        self._static = (q, kn, vn, out)

    def capture_host(self) -> None:
        """Capture the end-to-end step over engine-owned pinned host buffers
        (``host_buffers``: q, new K, new V in; out back), after ``capture``.
        Inputs go in on a side stream as three copies, each gating the first
        layer that reads it: layer 0's, layers 1-3's (small, lands while layer 0
        computes) and the rest (lands while layers 0-3 compute; the host link
        moves ~26 GB/s, so one copy of all later layers would hold layer 1 up).
        Outputs go back on another side stream
        as two copies: layers [0, L-2) once layer L-3 is done, and the last two
        layers at the end. Every dependency of a kernel on a copy, and every
        copy, costs microseconds of the step even when the data is ready, hence
        as few of them as the overlap allows (measured on the 32-layer config-1
        step: per-layer copies +138 us over the device-only step, this ~+55 us)."""
        assert self._static is not None, "capture() first"
        if self.positions is not None:
            raise RuntimeError("capture_host takes queries and keys that are rotated already: capture() without positions")
        q, kn, vn, out = self._static
        hq = torch.empty(q.shape, dtype=q.dtype, pin_memory=True)
        hk = torch.empty(kn.shape, dtype=kn.dtype, pin_memory=True)
        hv = torch.empty(vn.shape, dtype=vn.dtype, pin_memory=True)
        ho = torch.empty(out.shape, dtype=out.dtype, pin_memory=True)
        hint = self._hint
        Lyr = self.num_layers
        cuts = sorted({c for c in (Lyr - 2,) if 0 < c < Lyr}) + [Lyr]
        chunks = list(zip([0] + cuts[:-1], cuts))
        s = torch.cuda.Stream(device=self.device)
        s_in = torch.cuda.Stream(device=self.device)
        s_out = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        bounds = sorted({b for b in (1, 4) if b < Lyr}) + [Lyr]
        in_chunks = list(zip([0] + bounds[:-1], bounds))  # [0,1), [1,4), [4,L)
        ev_in = [torch.cuda.Event() for _ in in_chunks]
        ev_out = [torch.cuda.Event() for _ in chunks]
        # warm the capture stream's decode workspace outside capture (state restored)
        snap = self._snapshot()
        with torch.cuda.stream(s):
            for l in range(Lyr):
                self.step_layer(l, q[l], kn[l], vn[l], out=out[l], len_hint=hint, early=self._early_layer(l))
        s.synchronize()
        self._restore(snap)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            s_in.wait_stream(s)
            s_out.wait_stream(s)
            with torch.cuda.stream(s_in):
                for i, (a, b) in enumerate(in_chunks):
                    q[a:b].copy_(hq[a:b], non_blocking=True)
                    kn[a:b].copy_(hk[a:b], non_blocking=True)
                    vn[a:b].copy_(hv[a:b], non_blocking=True)
                    ev_in[i].record(s_in)
            ci = 0
            for l in range(Lyr):
                for i, (a, _) in enumerate(in_chunks):
                    if l == a:  # the first layer that reads input copy i
                        s.wait_event(ev_in[i])
                self.step_layer(l, q[l], kn[l], vn[l], out=out[l], len_hint=hint, early=self._early_layer(l))
                a, b = chunks[ci]
                if l == b - 1:
                    ev_out[ci].record(s)
                    with torch.cuda.stream(s_out):
                        s_out.wait_event(ev_out[ci])
                        ho[a:b].copy_(out[a:b], non_blocking=True)
                    ci += 1
            s.wait_stream(s_in)
            s.wait_stream(s_out)
        torch.cuda.current_stream(self.device).wait_stream(s)
        self.host_graph = g
        self._host = (hq, hk, hv, ho)

    @property
    def host_buffers(self):
        """Pinned host (q, new K, new V, out) of the pipelined end-to-end step.
        The step's copies read and write them asynchronously: write the next
        step's inputs, and read ``out``, only after the step has finished on
        the device (e.g. after a stream or event synchronisation)."""
        return self._host

    def _snapshot(self):
        return [(st.lengths.clone(), d.lengths.clone(), d.ring_head.clone(),
                 d.k.clone(), d.v.clone()) for st, d in zip(self.stores, self.dense)]

    def _restore(self, snap) -> None:
        for (bl, dl, rh, k, v), st, d in zip(snap, self.stores, self.dense):
            st.lengths.copy_(bl)
            d.lengths.copy_(dl)
            d.ring_head.copy_(rh)
            d.k.copy_(k)
            d.v.copy_(v)

    @property
    def static_buffers(self):
        return self._static

    def replay(self) -> None:
        if self.graph is None:
            raise RuntimeError("replay needs a captured step (capture; attach_prefix and set_rotary drop it)")
        self._check_context()
        self.graph.replay()
        self.body_len += 1

    def step_host(self, q_host: torch.Tensor, k_host: torch.Tensor, v_host: torch.Tensor,
                  out_host: torch.Tensor) -> None:
        """End-to-end step from (pinned) host buffers: H2D of the step's queries
        and new K/V, the captured step, D2H of the attention outputs. Given the
        engine's own ``host_buffers`` (after ``capture_host``) it replays the
        pipelined graph (per-layer copies overlapping the kernels); otherwise it
        copies everything in, replays the step and copies everything out."""
        if self._host is not None and all(a.data_ptr() == b.data_ptr() for a, b in
                                          zip((q_host, k_host, v_host, out_host), self._host)):
            self._check_context()
            self.host_graph.replay()
            self.body_len += 1
            return
        q, kn, vn, out = self._static
        q.copy_(q_host, non_blocking=True)
        kn.copy_(k_host, non_blocking=True)
        vn.copy_(v_host, non_blocking=True)
        self.replay()
        out_host.copy_(out, non_blocking=True)

    # ------------------------------------------------------------------ accounting
    def step_bytes(self, body_len: Optional[int] = None) -> int:
        """Algorithmic HBM bytes of one decode step (all layers): each INT4 code,
        meta, dense K/V byte, query and output read or written once, plus the
        append (new token in, evicted row in, packed row out, ring row out)."""
        nb = self.body_len if body_len is None else body_len
        return self.num_layers * (self.layer_attn_bytes(nb + 1) + self.layer_append_bytes())

    def layer_attn_bytes(self, body_tokens: int) -> int:
        """Without a shared prefix's bytes (its lengths are on the device)."""
        ng = 128 // self.group
        meta = 4 * ng + (ng if self.fmt == "ref" else 0)
        per_tok_body = 2 * (64 + meta)
        esz = torch.tensor([], dtype=self.kv_dtype).element_size()
        per_tok_dense = 2 * 128 * esz
        units = self.batch * self.kv_heads
        qo = self.batch * self.q_heads * 128 * (2 + torch.tensor([], dtype=self.out_dtype).element_size())
        return units * (body_tokens * per_tok_body + (self.sink + self.recent) * per_tok_dense) + qo

    def layer_append_bytes(self) -> int:
        ng = 128 // self.group
        meta = 4 * ng + (ng if self.fmt == "ref" else 0)
        esz = torch.tensor([], dtype=self.kv_dtype).element_size()
        units = self.batch * self.kv_heads
        return units * 2 * (128 * esz * 3 + 64 + meta)
