"""Fixed-active-set decode of sequences that go on behind shared prefixes.

The lifecycle is :class:`~moba_hip.PreparedDecode`'s (an exclusive lease,
persistent buffers overwritten by the next call, ``step`` / ``capture`` /
``close``).  A step takes one token per leased row before its rotation, turns
its key and query by prefix length plus own position, appends it and attends
the row's prefix and its own tokens: the page delta and positions, the rotary
append, the mean of a chunk that it closes, and the two of shared-prefix attention,
five launches whose arguments never change, so that one hipGraph replays them.  A
lease makes the plan of its batch and holds the partials of its step; a model's
layers have one each.
"""
from __future__ import annotations

import numpy as np
import torch

from . import decode_contract as contract
from .baseline_adapter import _require
from .cache_layout import IncrementalLayout, positive_int
from .ops import _lib
from .ops import decode as kernels
from .prepared_decode import PreparedDecode
from .shared_prefix import SharedPrefixPlan


class PreparedSharedDecode(PreparedDecode):
    def __init__(self, cache, sequence_ids, prefix_ids, num_q_heads, *, rotary=None, max_length=None,
                 check_finite=True):
        """``prefix_ids``: the prefix slot of each leased sequence, -1 for none.
        ``rotary``: the table by which keys and queries turn; without it they
        are expected turned.  ``max_length``: what a leased sequence may grow
        to (default: what its slot holds); the work of a step is cut for it."""
        self._handle = None
        with cache._lock, torch.cuda.device(cache.device):
            cache._guard()
            self.num_q_heads = positive_int(num_q_heads, "num_q_heads")
            capacity = cache._layout.max_seq_len
            self.max_length = capacity if max_length is None else positive_int(max_length, "max_length")
            _require([
                (lambda: self.num_q_heads % cache.num_kv_heads == 0, "Hq must be a multiple of Hkv"),
                (lambda: self.max_length <= capacity, "max_length exceeds max_seq_len"),
                (lambda: isinstance(check_finite, bool), "check_finite must be bool"),
            ])
            self.check_finite, self.cache, self.dense = check_finite, cache, True
            self._dev = cache.device.index
            self._lease = IncrementalLayout(cache._layout,
                                            contract.int_vector(sequence_ids, "sequence_ids"))
            self.ids = self._lease.ids
            self.prefix_ids, self.prefix_lengths = cache._prefixes(self.ids, prefix_ids)
            self.rotary = rotary
            if rotary is not None:
                cache._check_rotary(rotary, max(self.prefix_lengths))
                self._angles = rotary.cos_sin   # what the launches hold the address of
            self._plan = SharedPrefixPlan(self.prefix_ids, self.prefix_lengths, self.ids,
                                          self.num_q_heads, cache.num_kv_heads, cache.head_dim,
                                          max_suffix=self.max_length, device=cache.device)
            self._shared_buffers(len(self.ids))
            self._calls = self._launches(len(self.ids))
            self._uploaded = False    # the device delta holds a grant not yet committed
            self._delta_uploads = 0
            self._graph = None
            self.closed = self.failed = False
            cache._lessee = self   # the lease starts once everything above succeeded

    def _shared_buffers(self, rows):
        c, hq, d = self.cache, self.num_q_heads, self.cache.head_dim
        dev, dt = c.device, c.dtype
        self.q = torch.zeros((rows, hq, d), device=dev, dtype=dt)
        self.k = torch.zeros((rows, c.num_kv_heads, d), device=dev, dtype=dt)
        self.v = torch.zeros_like(self.k)
        self._turned = self.q if self.rotary is None else torch.empty_like(self.q)
        self.output = torch.empty_like(self.q)
        self.lse = torch.empty((rows, hq), device=dev, dtype=torch.float32)
        self.gpu_ids = torch.tensor(self.ids, device=dev, dtype=torch.int32)
        self.positions = torch.zeros(rows, device=dev, dtype=torch.int32)
        self.delta = torch.full((2, rows), -1, device=dev, dtype=torch.int32)
        by_slot = np.zeros(c._layout.batch_size, np.int32)
        by_slot[list(self.ids)] = self.prefix_lengths
        self._offsets = torch.from_numpy(by_slot).to(dev)
        self._work = torch.empty(self._plan.parts * hq * (d + 2), device=dev, dtype=torch.float32)

    def _launches(self, rows):
        """(entry, arguments without the stream) of a step, in order."""
        c, plan, ptr = self.cache, self._plan, _lib.ptr
        code, hq, hkv, d = kernels.DTYPE_CODE[c.dtype], self.num_q_heads, c.num_kv_heads, c.head_dim
        pages, page, width = c.k_cache.shape[0], c._layout.page_size, c._table.shape[1]
        kc, vc, table = ptr(c.k_cache), ptr(c.v_cache), ptr(c._table)
        ids, pos = ptr(self.gpu_ids), ptr(self.positions)
        calls = [("moba_hip_decode_metadata", (table, width, ptr(c._lengths), ids, pos,
                                               ptr(self.delta), rows, 1))]
        if self.rotary is None:
            calls.append(("moba_hip_paged_append", (ptr(self.k), ptr(self.v), code, rows, hkv, d, kc,
                                                    vc, page, table, width, ids, pos)))
        else:
            r = self.rotary
            calls.append(("moba_hip_append_rotary", (
                ptr(self.q), hq * d, d, ptr(self.k), hkv * d, d, ptr(self.v), hkv * d, d, code, rows,
                hq, hkv, d, ptr(self._angles), r.max_positions, r.rotary_dim, int(r.interleaved), kc, vc,
                pages, page, table, c._table.shape[0], width, ids, pos, ptr(self._offsets),
                ptr(self._turned), None)))
        calls.append(("moba_hip_block_means", (kc, code, hkv, d, page, table, width, ids, pos, rows, 1,
                                               c.chunk_size, ptr(c._means), c._means.shape[1])))
        meta, work = ptr(plan.meta), ptr(self._work)
        # a row's own tokens: its position and what lies before it
        calls.append(("moba_hip_shared_attention", (
            ptr(self._turned), code, rows, hq, hkv, d, d ** -0.5, kc, vc, pages, page, table, width,
            pos, 1, self.max_length, meta, plan.n_items, meta + plan._rows_at, meta + plan._parts_at,
            plan.max_parts, plan.uneven, work, work + 4 * plan.parts * hq * d, ptr(self.output),
            ptr(self.lse))))
        return calls

    @property
    def delta_uploads(self):
        return self._delta_uploads

    # parts of a step, as PreparedDecode has them for whole-model steps
    def _plan_step(self, stream):
        """Plans one token per row and uploads its page grants; changes nothing
        of the cache when it refuses (ValueError)."""
        step = self._lease.plan()
        if max(step.positions) >= self.max_length:
            raise ValueError("append exceeds max_length")
        if self.rotary is not None and self._angles.shape[0] <= max(
                p + n for p, n in zip(step.positions, self.prefix_lengths)):
            raise ValueError("positions exceed the rotary table")
        if step.updates or self._uploaded:
            try:   # from pinned memory, which torch keeps until the copy is done
                self.delta.copy_(torch.from_numpy(step.delta).pin_memory(), non_blocking=True)
            except BaseException:
                self.failed = True
                raise
            self._uploaded = bool(step.updates)
            self._delta_uploads += 1
        self._step = step
        return step.positions

    def _launch_step(self, stream):
        for name, args in self._calls:
            _lib.call(name, *args, stream)

    def _commit_step(self):
        self._lease.commit(self._step)
        self._uploaded = False

    def step(self, q, k, v, *, use_graph=False):
        """One token per leased row; argument and capacity errors change nothing."""
        with self.cache._lock, torch.cuda.device(self.cache.device):
            stream = self._usable()
            copies = self._bind_all(((q, self.q, "q"), (k, self.k, "k"), (v, self.v, "v")))
            if use_graph and self._graph is None:
                raise ValueError("capture('step') first")
            positions = self._plan_step(stream)
            try:
                with torch.no_grad():
                    for given, buffer in copies:
                        buffer.copy_(given)
                if use_graph:
                    self._graph.replay()
                else:
                    self._launch_step(stream)
                self._commit_step()
            except BaseException:   # the device may be a token ahead of the host, or on its way
                self.failed = True
                raise
            return self._result(positions)

    def attend(self, q, *, use_graph=False):
        raise ValueError("a shared decode has no attend; PagedKVCache.attend_shared serves one")

    def capture(self, kind="step"):
        """Records the device work of one step into a hipGraph.  Nothing runs
        and no cache state changes."""
        _require([(lambda: kind == "step", "kind must be step")])
        with self.cache._lock, torch.cuda.device(self.cache.device):
            self._usable()
            if self._graph is not None:
                raise ValueError("graph already captured")
            side = torch.cuda.Stream(device=self.cache.device)
            side.wait_stream(torch.cuda.current_stream(self.cache.device))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                self._launch_step(side.cuda_stream)
            self._graph = graph
            return self

    def close(self):
        super().close()
        self._graph = None
