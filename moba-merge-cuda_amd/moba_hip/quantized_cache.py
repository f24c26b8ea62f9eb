"""Paged KV cache in 8 bits: :class:`~moba_hip.PagedKVCache` whose pages hold codes and
scales (:mod:`moba_hip.quantized`), at half the bytes of a 16-bit cache.

Constructor, operations, errors and lifecycle are the 16-bit cache's, with
``format="int8"`` or ``"fp8"``; ``dtype`` is the type of its inputs and outputs.  Keys
and values are quantised as they are appended; chunk means, routing and attention are
those of the stored values.  At most 64 query heads of a kv head and 8192 chunks are
routed; what is refused for that is refused before anything is stored.  Sequences behind
shared prefixes are the 16-bit cache's alone.

:class:`PreparedQuantizedDecode` is its prepared decode: the page delta and positions, the
quantising append (with a ``rotary`` table the keys and queries turn inside it), the mean
of a chunk that it closes, the route, and the attention, five to seven launches whose
arguments never change, so that one hipGraph replays them.
"""
from __future__ import annotations

import numpy as np
import torch

from . import decode_contract as contract
from .baseline_adapter import _require
from .cache_layout import IncrementalLayout, positive_int
from .kv_cache import DecodeResult, PagedKVCache
from .ops import _lib
from .ops import decode as kernels
from .prepared_shared import PreparedSharedDecode
from .quantized import (_FORMATS, QuantizedPages, _attention_work, _check_format, _check_head_dim,
                        _pool_args, quantized_append, quantized_attention, quantized_read)

_ROUTE_WIDTH = 8192   # chunks that moba_hip_decode_route scores
_ROUTE_GROUP = 64     # query heads of a kv head


def _route_rules(nq, hq, hkv, width):
    return [(lambda: hq // hkv <= _ROUTE_GROUP, "at most 64 query heads per kv head are routed"),
            (lambda: width <= _ROUTE_WIDTH, "at most 8192 chunks are routed"),
            (lambda: nq * hkv * -(-(hq // hkv) // 16) < 2 ** 23,   # 2^32 threads
             "at most 2^23 blocks of 16 query heads are routed")]


class QuantizedKVCache(PagedKVCache):
    def __init__(self, batch_size, max_seq_len, num_kv_heads, head_dim, *, format="int8", **kwargs):
        _check_format(format)
        _check_head_dim(positive_int(head_dim, "head_dim"))
        self.format = format
        super().__init__(batch_size, max_seq_len, num_kv_heads, head_dim, **kwargs)

    def _allocate(self, pages, page):
        self.pages = QuantizedPages.empty(pages, page, self.num_kv_heads, self.head_dim,
                                          format=self.format, device=self.device)

    def _pool_tensors(self):
        return self.pages[:4]

    def _write(self, k, v, seq, pos):
        quantized_append(k, v, self.pages, self._table, seq, pos)

    def _write_rotary(self, k, v, seq, pos, rotary, q, offsets):
        return quantized_append(k, v, self.pages, self._table, seq, pos, rotary=rotary, q=q,
                                offsets=offsets)

    def _means_args(self):
        """Arguments of moba_hip_quantized_means before and after its items."""
        (k, _, ks, _, n, page), table = _pool_args(self.pages, self._table)
        return ((_FORMATS[self.pages.k.dtype], k, ks, n, page, self.num_kv_heads, self.head_dim, *table),
                (self.chunk_size, kernels.DTYPE_CODE[self.dtype], self._means.data_ptr(),
                 self._means.shape[1]))

    def _close_chunks(self, seq, chunks):
        n = seq.numel()
        if n:
            before, after = self._means_args()
            _lib.call("moba_hip_quantized_means", *before, seq.data_ptr(), chunks.data_ptr(), n, 0, *after,
                      _lib.stream_of(self.device))

    def _read(self, slot, n):
        if not n:
            return tuple(torch.empty((0, self.num_kv_heads, self.head_dim), dtype=self.dtype,
                                     device=self.device) for _ in range(2))
        pos = torch.arange(n, device=self.device, dtype=torch.int32)
        return quantized_read(self.pages, self._table, torch.full_like(pos, slot), pos, dtype=self.dtype)

    def _route_size(self, nq, hq, last, lengths, topk):
        """(remote chunks of a head, chunks to score) of nq routed queries, the farthest at
        position ``last`` of a cache of ``lengths``; raises what the route does not take."""
        remote = min(int(topk) - 1, self._candidates(lengths))
        width = max(remote, last // self.chunk_size) if remote else 0
        _require([(lambda: width * hq * nq < 2 ** 31, "route score grid exceeds int32 capacity"),
                  *_route_rules(nq, hq, self.num_kv_heads, width)])
        return remote, width

    def _check_decode(self, q, ids, counts, topk, dense):
        nq, hq, d = q.shape
        lengths = np.array(self.lengths)
        lengths[list(ids)] += counts
        limit = int(lengths[list(ids)].max())
        slots = 0 if dense else self._route_size(nq, hq, limit - 1, lengths, topk)[0] + 1
        _attention_work(nq, hq, self.num_kv_heads, d, slots, min(self.chunk_size, limit), limit)

    def _decode(self, q, ids, pos, dev_ids, dev_pos, topk, dense):
        q = q.contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
        nq, hq, d = q.shape
        selected = None
        if not dense:
            remote, width = self._route_size(nq, hq, max(pos), None, topk)
            selected = torch.empty((nq, hq, remote + 1), dtype=torch.int32, device=self.device)
            scores = (torch.empty((nq, hq, width), dtype=torch.float32, device=self.device)
                      if remote else None)
            _lib.call("moba_hip_decode_route", q.data_ptr(), kernels.DTYPE_CODE[self.dtype], nq, hq,
                      self.num_kv_heads, d, self._means.data_ptr(), self._means.shape[1],
                      dev_ids.data_ptr(), dev_pos.data_ptr(), self.chunk_size, width, remote,
                      _lib.ptr(scores), selected.data_ptr(), None, None, _lib.stream_of(self.device))
        out, lse = quantized_attention(q, self.pages, self._table, dev_ids, dev_pos + 1, selected=selected,
                                       chunk_size=None if dense else self.chunk_size,
                                       max_length=max(pos) + 1)
        return DecodeResult(out, lse, selected, ids, pos)

    def prepare_decode(self, sequence_ids, num_q_heads, *, topk=4, mode="moba", check_finite=True,
                       stable_routes=False, rotary=None):
        return PreparedQuantizedDecode(self, sequence_ids, num_q_heads, topk=topk, mode=mode,
                                       check_finite=check_finite, stable_routes=stable_routes,
                                       rotary=rotary)

    def attend_shared(self, *args, **kwargs):
        raise ValueError("shared prefixes need a 16-bit cache (PagedKVCache)")

    def prepare_shared_decode(self, *args, **kwargs):
        raise ValueError("shared prefixes need a 16-bit cache (PagedKVCache)")


class PreparedQuantizedDecode(PreparedSharedDecode):
    def __init__(self, cache, sequence_ids, num_q_heads, *, topk=4, mode="moba", check_finite=True,
                 stable_routes=False, rotary=None):
        """``rotary``: the table by which keys and queries turn; without it they are
        expected turned.  The others are :class:`~moba_hip.PreparedDecode`'s."""
        self._handle = None
        with cache._lock, torch.cuda.device(cache.device):
            cache._guard()
            self.num_q_heads = positive_int(num_q_heads, "num_q_heads")
            _require([
                (lambda: isinstance(cache, QuantizedKVCache), "QuantizedKVCache required"),
                (lambda: self.num_q_heads % cache.num_kv_heads == 0, "Hq must be a multiple of Hkv"),
                (lambda: isinstance(check_finite, bool), "check_finite must be bool"),
                (lambda: isinstance(stable_routes, bool), "stable_routes must be bool"),
            ])
            self.dense = contract.decode_mode(mode, topk)
            self.check_finite, self.stable_routes, self.cache = check_finite, stable_routes, cache
            self._dev = cache.device.index
            self._lease = IncrementalLayout(cache._layout,
                                            contract.int_vector(sequence_ids, "sequence_ids"))
            self.ids = self._lease.ids
            self.max_length = cache._layout.max_seq_len
            rows, hq = len(self.ids), self.num_q_heads
            width = max(1, (self.max_length - 1) // cache.chunk_size)   # closed chunks of a full row
            self.remote = 0 if self.dense else min(topk - 1, width)
            if not self.dense:
                _require([(lambda: rows * hq * width < 2 ** 31, "route score grid exceeds int32 capacity"),
                          *_route_rules(rows, hq, cache.num_kv_heads, width)])
            self.prefix_lengths = (0,) * rows
            self.rotary = rotary
            if rotary is not None:
                cache._check_rotary(rotary, 0)
                self._angles = rotary.cos_sin   # what the launches hold the address of
            self._quantized_buffers(rows, width)
            self._calls = self._launches(rows, width)
            self._uploaded = False    # the device delta holds a grant not yet committed
            self._delta_uploads = 0
            self._graph = self._attend_graph = None
            self.closed = self.failed = False
            cache._lessee = self   # the lease starts once everything above succeeded

    def _quantized_buffers(self, rows, width):
        c, hq, d = self.cache, self.num_q_heads, self.cache.head_dim
        dev, dt = c.device, c.dtype
        self.q = torch.zeros((rows, hq, d), device=dev, dtype=dt)
        self.k = torch.zeros((rows, c.num_kv_heads, d), device=dev, dtype=dt)
        self.v = torch.zeros_like(self.k)
        self._turned = self.q if self.rotary is None else torch.zeros_like(self.q)
        self.output = torch.empty_like(self.q)
        self.lse = torch.empty((rows, hq), device=dev, dtype=torch.float32)
        self.gpu_ids = torch.tensor(self.ids, device=dev, dtype=torch.int32)
        self.positions = torch.zeros(rows, device=dev, dtype=torch.int32)
        self.delta = torch.full((2, rows), -1, device=dev, dtype=torch.int32)
        self.selected = self.scores = None
        if not self.dense:
            self.selected = torch.full((rows, hq, self.remote + 1), -1, device=dev, dtype=torch.int32)
            self.scores = torch.empty((rows, hq, width), device=dev, dtype=torch.float32)
        slots, chunk = (0, 0) if self.dense else (self.remote + 1, min(c.chunk_size, self.max_length))
        self._work = torch.empty(
            _attention_work(rows, hq, c.num_kv_heads, d, slots, chunk, self.max_length), device=dev,
            dtype=torch.uint8)

    def _launches(self, rows, width):
        """(entry, arguments without the stream) of a step, in order: the first, those that
        an attend leaves out, and the rest."""
        c, ptr = self.cache, _lib.ptr
        code, hq, hkv, d = kernels.DTYPE_CODE[c.dtype], self.num_q_heads, c.num_kv_heads, c.head_dim
        pool, table = _pool_args(c.pages, c._table)
        form = _FORMATS[c.pages.k.dtype]
        ids, pos = ptr(self.gpu_ids), ptr(self.positions)

        def places(append):
            return ("moba_hip_decode_metadata", (ptr(c._table), c._table.shape[1], ptr(c._lengths), ids, pos,
                                                 ptr(self.delta), rows, append))
        r = self.rotary
        turn = (None, 0, 0, 0) if r is None else (ptr(self._angles), self._angles.shape[0], r.rotary_dim,
                                                  int(r.interleaved))
        q_in, q_heads, q_out = (None, 0, None) if r is None else (ptr(self.q), hq, ptr(self._turned))
        append = ("moba_hip_quantized_append", (
            q_in, hq * d, d, ptr(self.k), hkv * d, d, ptr(self.v), hkv * d, d, code, rows, q_heads, hkv, d,
            *turn, form, *pool, *table, ids, pos, None, q_out, None))
        before, after = c._means_args()
        means = ("moba_hip_quantized_means", (*before, ids, pos, rows, 1, *after))
        read = []
        if not self.dense:
            read.append(("moba_hip_decode_route", (
                ptr(self._turned), code, rows, hq, hkv, d, ptr(c._means), c._means.shape[1], ids, pos,
                c.chunk_size, width, self.remote, ptr(self.scores), ptr(self.selected), None, None)))
        slots = 0 if self.dense else self.remote + 1
        # a row's tokens: its position and what lies before it
        read.append(("moba_hip_quantized_attention", (
            ptr(self._turned), code, rows, hq, hkv, d, d ** -0.5, form, *pool, *table, ids, pos, 1,
            self.max_length, ptr(self.selected), slots, c.chunk_size if slots else 0, ptr(self._work),
            ptr(self.output), ptr(self.lse))))
        self._attend_calls = [places(0), *read]
        return [places(1), append, means, *read]

    def attend(self, q, *, use_graph=False):
        """The attention of a step at each row's last token, without appending."""
        with self.cache._lock, torch.cuda.device(self.cache.device):
            stream = self._usable()
            if self.rotary is not None:
                raise ValueError("a decode that turns its queries has no attend")
            copies = self._bind_all(((q, self.q, "q"),))
            if use_graph and self._attend_graph is None:
                raise ValueError("capture('attend') first")
            positions = tuple(n - 1 for n in self._lease.positions().tolist())
            if min(positions) < 0:
                raise ValueError("attend requires nonempty cached sequences")
            try:
                with torch.no_grad():
                    for given, buffer in copies:
                        buffer.copy_(given)
                if use_graph:
                    self._attend_graph.replay()
                else:
                    self._launch(self._attend_calls, stream)
            except BaseException:
                self.failed = True
                raise
            return self._result(positions)

    @staticmethod
    def _launch(calls, stream):
        for name, args in calls:
            _lib.call(name, *args, stream)

    def capture(self, kind="step"):
        """Records the device work of one step / attend into a hipGraph.  Nothing runs
        and no cache state changes."""
        _require([(lambda: kind in ("step", "attend"), "kind must be step or attend")])
        with self.cache._lock, torch.cuda.device(self.cache.device):
            self._usable()
            if (self._graph if kind == "step" else self._attend_graph) is not None:
                raise ValueError("graph already captured")
            if kind == "attend":
                if self.rotary is not None:
                    raise ValueError("a decode that turns its queries has no attend")
                if int(np.min(self._lease.positions())) == 0:
                    raise ValueError("attend capture requires nonempty cached sequences")
            side = torch.cuda.Stream(device=self.cache.device)
            side.wait_stream(torch.cuda.current_stream(self.cache.device))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                self._launch(self._calls if kind == "step" else self._attend_calls, side.cuda_stream)
            if kind == "step":
                self._graph = graph
            else:
                self._attend_graph = graph
            return self

    def close(self):
        super().close()
        self._attend_graph = None
