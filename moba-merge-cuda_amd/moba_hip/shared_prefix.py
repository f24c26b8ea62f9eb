"""Attention for a batch whose sequences share long prefixes.

A prefix (a system prompt, a document, a prompt that is sampled several times)
is stored once, in a slot of its own, and read once for all the query rows
behind it; each row then attends the tokens of its own slot.  The plan of a
batch holds which rows share what; their own lengths are read on the device, so
one plan serves every call on that batch, of whichever layer and step, that its
maker passes it to.  (The cache's ``attend_shared`` and its prepared steps make
plans of their own, one per cache and so one per layer.)
"""
from __future__ import annotations

import math
import struct

import numpy as np
import torch

from .cache_layout import positive_int
from .ops import _lib
from .rotary import _DTYPES, _check_index, _check_pool, _meet, _on_device, _span

# (row, q head of a kv head) pairs of a work item: its four waves have 32 each,
# or the same 32 and a quarter of the keys each (solo: a wave has an item's 32
# pairs and all of its keys alone)
_WIDE, _NARROW = 128, 32
# What the length of the ranges is chosen by: workgroups that a CU holds (up to
# 128 dims, above); an item's time beside its keys, us, the last one's and one of
# many; a key's, per dim, times what the items of one CU make of each other
# (alone, and per item; wide items, narrow ones); the rates at which partials are
# written and read, and K/V, bytes per us; the merge's time per range of a row, us.
# These ten, and three that stand in the formulas below (an item is long from 0.83 of
# the longest, half of a late one counts, a norm of order 7), are fitted to 140
# batches, each timed cut in 6 to 30 ways (prefixes to 128K tokens, 1 to 400 rows, 40
# to 256 dims): what is taken is 2% behind the best of them on average.
_CUS, _HELD = 256, (3, 2)
_ITEM, _OF_MANY, _KEY = 6.4, 5.0, 2.2e-4
_ON_A_CU = (0.8, 0.27), (0.65, 0.5)
_PARTIALS, _CACHE, _RANGE = 3.5e6, 4.5e6, 7.5e-3
_XCDS = 8   # workgroup L runs on XCD L % 8


def _slots(values, name, n=None):
    out = np.asarray(values.cpu() if isinstance(values, torch.Tensor) else values)
    if out.ndim != 1 or out.dtype.kind not in "iu" or (n is not None and len(out) != n):
        raise ValueError(f"{name} must be one integer per query row")
    if len(out) and (out.min() < -1 or out.max() >= 2 ** 31):
        raise ValueError(f"{name} entries must be -1 or more")
    return out.astype(np.int64)


class SharedPrefixPlan:
    """Which query rows share which prefix, cut into work items.

    ``prefix_ids``, ``prefix_lengths``, ``suffix_ids``: one entry per query
    row.  The row attends tokens [0, prefix_length) of page-table row
    ``prefix_id`` (-1: no prefix, with length 0) and then its own length of
    tokens of page-table row ``suffix_id`` (-1: none).  Rows of one
    (prefix_id, prefix_length) are served together, and so are rows of one
    suffix_id (several query tokens of a sequence, each with its own length).
    ``max_suffix`` bounds the own lengths (longer ones are cut to it).  A plan
    used on a stream other than the one it was made on is kept until that
    stream's work is done; a captured graph needs it as long as it is replayed.
    """

    def __init__(self, prefix_ids, prefix_lengths, suffix_ids, num_q_heads, num_kv_heads, head_dim,
                 *, max_suffix, device="cuda"):
        hq, hkv = positive_int(num_q_heads, "num_q_heads"), positive_int(num_kv_heads, "num_kv_heads")
        d = positive_int(head_dim, "head_dim")
        if hq % hkv:
            raise ValueError("Hq must be a multiple of Hkv")
        if d % 8 or d > 256:
            raise ValueError("head_dim must be a multiple of 8 in [8,256]")
        if isinstance(max_suffix, bool) or not isinstance(max_suffix, int) or \
                not 0 <= max_suffix <= 2 ** 30:
            raise ValueError("max_suffix must be a length, at most 2^30")
        prefix = _slots(prefix_ids, "prefix_ids")
        n = len(prefix)
        if n < 1:
            raise ValueError("one query row at least")
        length = _slots(prefix_lengths, "prefix_lengths", n)
        suffix = _slots(suffix_ids, "suffix_ids", n)
        if length.min() < 0 or (length[prefix < 0] != 0).any():
            raise ValueError("prefix_lengths must be 0 or more, and 0 without a prefix")
        if length.max() > 2 ** 30:
            raise ValueError("prefix_lengths must be at most 2^30")
        if n * hq >= 2 ** 31:
            raise ValueError("query grid exceeds int32 capacity")
        self.rows, self.num_q_heads, self.num_kv_heads, self.head_dim = n, hq, hkv, d
        self._q_shape = (n, hq, d)
        self.max_suffix = max_suffix
        self.max_prefix = int(length.max())
        self.max_slot = int(max(prefix[length > 0].max(initial=-1), suffix.max()))
        flat = self._build(prefix, length, suffix)
        self.meta = torch.from_numpy(flat).to(device)
        # what a call needs of the plan, for the native host path
        self._packed = struct.pack("13q", n, hq, hkv, d, self.max_slot, self.max_prefix, max_suffix,
                                   self.n_items, self._rows_at, self._parts_at, self.parts,
                                   self.max_parts, self.uneven)

    @property
    def device(self):
        return self.meta.device

    def _check(self):
        """Raises where ``meta``, which a caller may replace, is not what the
        kernels index."""
        m = self.meta
        if not isinstance(m, torch.Tensor) or m.dtype != torch.int32 or m.layout != torch.strided or \
                m.dim() != 1 or not m.is_contiguous() or \
                m.numel() != self._parts_at // 4 + 3 * self.rows or m.data_ptr() & 15:
            raise ValueError("plan.meta must be the plan's int32 records, contiguous and 16-byte aligned")

    def _build(self, prefix, length, suffix):
        """The device arrays: work items, segments' rows, rows' partials."""
        n, hkv, group = self.rows, self.num_kv_heads, self.num_q_heads // self.num_kv_heads
        # segments: the rows of one (prefix, length), then those of one own slot
        shared = np.nonzero(length > 0)[0]
        alone = np.nonzero((suffix >= 0) & (self.max_suffix > 0))[0]
        pairs, of_shared, n_shared = np.unique(prefix[shared] << 32 | length[shared],
                                               return_inverse=True, return_counts=True)
        slots, of_alone, n_alone = np.unique(suffix[alone], return_inverse=True, return_counts=True)
        row_list = np.concatenate((shared[np.argsort(of_shared, kind="stable")],
                                   alone[np.argsort(of_alone, kind="stable")]))
        slot = np.concatenate((pairs >> 32, slots))
        own = np.arange(len(slot)) >= len(pairs)
        tokens = np.where(own, -1, np.concatenate((pairs & (2 ** 32 - 1), slots)))
        bound = np.where(own, self.max_suffix, tokens)
        n_rows = np.concatenate((n_shared, n_alone))
        row_at = np.cumsum(n_rows) - n_rows
        # 33 to 128 pairs: one wide block of which a part is idle reads its keys
        # once (16 rows of 4 heads behind 32K tokens: 41 us; two narrow ones 43)
        size = np.where(n_rows * group > _NARROW, _WIDE, _NARROW)
        blocks = -(-n_rows * group // size)
        splits, solo = self._ranges(blocks * hkv, bound, own, size == _NARROW, n_rows)
        n_prefix, n_suffix = np.zeros(n, np.int64), np.zeros(n, np.int64)
        of_row = np.repeat(splits, n_rows)
        n_prefix[row_list[:len(shared)]] = of_row[:len(shared)]
        n_suffix[row_list[len(shared):]] = of_row[len(shared):]

        # one item per (segment, range, kv head, block); those of one (segment,
        # range, kv head) read the same keys
        count = splits * hkv * blocks
        seg = np.repeat(np.arange(len(slot)), count)
        local = np.arange(len(seg)) - np.repeat(np.cumsum(count) - count, count)
        block, part = local % blocks[seg], local // blocks[seg]
        m0 = block * size[seg]
        n_m = np.minimum(size[seg], n_rows[seg] * group - m0)
        first, last = m0 // group, (m0 + n_m - 1) // group
        only = np.where(first == last, row_list[row_at[seg] + first], -1)
        items = np.stack((row_at[seg], m0, n_m, slot[seg], part % hkv,
                          part // hkv | splits[seg] << 16, tokens[seg], only), axis=1)
        keys = np.cumsum(block == 0)
        # four waves' items of one workgroup: the kv heads of a row next to each
        # other, whose keys lie together and are as many
        single = (own & (size == _NARROW) & solo)[seg]
        singles, items, keys = items[single], items[~single], keys[~single]
        singles = np.concatenate((singles, np.zeros((-len(singles) % 4, 8), np.int64)))
        carriers = np.zeros((len(singles) // 4, 8), np.int64)
        carriers[:, 0], carriers[:, 2], carriers[:, 6] = 4 * np.arange(len(carriers)), -1, -1
        items = np.concatenate((items, carriers))
        keys = np.concatenate((keys, len(seg) + 1 + np.arange(len(carriers))))
        # Longest first; but a few items of own tokens behind a card full of
        # prefix ranges would start when those end, all alone
        n_own = int((items[:, 6] < 0).sum())
        card = _CUS * _HELD[self.head_dim > 128]
        if n_own <= card // 2 and len(items) > card:
            order = np.argsort(items[:, 6] >= 0, kind="stable")
            items, keys = items[order], keys[order]
        items = self._dealt(items, keys)
        self.n_items = len(items)
        items[items[:, 2] < 0, 0] += len(items)

        part_at = np.cumsum(n_prefix + n_suffix) - (n_prefix + n_suffix)
        self.parts = int((n_prefix + n_suffix).sum())
        self.uneven = int(n_alone.max(initial=0) > 1)  # rows of one own slot, of any lengths
        self.max_parts = int((n_prefix + n_suffix).max())
        arrays = [items.ravel(), singles.ravel(), row_list, part_at, part_at + n_prefix,
                  n_prefix + n_suffix]
        self._rows_at = 4 * (arrays[0].size + arrays[1].size)
        self._parts_at = self._rows_at + 4 * len(row_list)
        return np.concatenate(arrays).astype(np.int32)

    def _ranges(self, blocks, bounds, own, narrow, rows):
        """How the segments are cut: (ranges of each, whether narrow items of
        own tokens go to single waves).  A segment has ``blocks`` items per
        range, up to ``bounds`` keys (own lengths lie anywhere below their bound:
        half of it on average) and ``rows`` query rows.  Taken are ranges of about
        one length, the one that gives the shortest time by the figures above:
        as many heavy items as the CUs hold alike (256 rows behind 32K tokens, 8
        kv heads: 512 items, two a CU, 192 us; 640 204; 768 220)."""
        if not len(blocks):
            return np.zeros(0, np.int64), False
        alike, index, times = np.unique(np.stack((blocks, bounds, own, narrow, rows), axis=1), axis=0,
                                        return_inverse=True, return_counts=True)
        blocks, bounds, own, narrow, rows = alike.T
        hq, hkv, d = self.num_q_heads, self.num_kv_heads, self.head_dim
        held, share, narrow = _HELD[d > 128], np.where(own, 0.5, 1.0), narrow.astype(bool)
        alone, each = np.where(narrow[:, None], *_ON_A_CU[::-1]).T
        single = own.astype(bool) & narrow
        read = (bounds * share * times).sum() * hkv * d * 4 / _CACHE
        # ranges of the longest segment: a row of the arrays each
        top = int(bounds.argmax())
        most, row = max(1.0, int(bounds[top]) / 128), int(blocks[top] * hkv * times[top])
        tried = np.unique(np.concatenate((
            np.geomspace(1, most, 1 + math.ceil(8 * math.log2(most))).round(),
            np.clip(np.arange(1, held + 1) * _CUS // row, 1, most))))
        splits = np.minimum(np.ceil(bounds / np.ceil(bounds[top] / tried)[:, None]), 2 ** 15 - 1)
        joins = splits @ (rows * times) * hq * d * 8 / _PARTIALS + _RANGE * splits.max(axis=1)
        count, keys = blocks * splits * times, _KEY * d * np.ceil(bounds / splits)
        ways = []
        for solo in (False, True) if single.any() else (False,):
            waves = np.where(single & solo, 4, 1)   # items of a workgroup
            items, time = count / waves, keys * waves * share
            # the longest ones: rounds that fill the CUs, then each CU has the rest
            likely = _ITEM + time
            heavy = likely > 0.83 * likely.max(axis=1, keepdims=True)
            many = np.where(heavy, items, 0.0).sum(axis=1)
            rounds = np.ceil(many / (held * _CUS)) - 1
            rest = np.ceil(many / _CUS) - rounds * held
            full, last = [np.where(heavy, _ITEM + time * np.maximum(alone, each * n), 0.0).max(axis=1)
                          for n in (held, rest[:, None])]
            # the others, beside the last round; what it leaves no room for starts
            # when that ends, some of it earlier
            work = items * (_OF_MANY + time * each * held) / (held * _CUS)
            room = last * (rounds + 1 - many / (held * _CUS))
            late = np.where(heavy, 0.0, _ITEM + time * alone).max(axis=1)
            late = np.where(np.where(heavy, 0.0, work).sum(axis=1) > room, late, 0.0)
            longest = np.maximum(rounds * full + last + 0.5 * late,
                                 (_ITEM + keys * waves * alone).max(axis=1))
            work = work.sum(axis=1)   # of the whole card
            # what is far the longest hides the others
            ways.append(joins + (longest ** 7 + work ** 7 + read ** 7) ** (1 / 7))
        best, solo = np.unravel_index(np.argmin(np.stack(ways, axis=1)), (len(tried), len(ways)))
        return splits[best].astype(np.int64)[index.ravel()], bool(solo)

    @staticmethod
    def _dealt(items, keys):
        """The items as workgroups take them: those of the same ``keys`` go to
        one XCD, one after another, the XCDs in turn; an item of no pairs pads
        a short one."""
        if not len(items):
            return items
        turn = (np.cumsum(np.concatenate(([True], keys[1:] != keys[:-1]))) - 1) % _XCDS
        order = np.argsort(turn, kind="stable")
        held = np.bincount(turn, minlength=_XCDS)
        rank = np.arange(len(items)) - np.repeat(np.cumsum(held) - held, held)
        dealt = np.zeros((int(held.max()) * _XCDS, items.shape[1]), np.int64)
        dealt[rank * _XCDS + turn[order]] = items[order]
        return dealt


def _check_attention(q, k_cache, v_cache, page_table, suffix_lengths, plan):
    """Raises what is wrong with the arguments of a call."""
    _check_pool(k_cache, v_cache, page_table)
    _, page, hkv, d = k_cache.shape
    dev = k_cache.device
    if not isinstance(plan, SharedPrefixPlan):
        raise ValueError("plan must be a SharedPrefixPlan")
    plan._check()
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype != k_cache.dtype or \
            q.device != dev or plan.device != dev:
        raise ValueError("q must be [Nq,Hq,D] of the pool's device and dtype, and the plan on it")
    if q.requires_grad:
        raise ValueError("KV cache/decode is inference-only; detach Q/K/V")
    if tuple(q.shape) != plan._q_shape or (hkv, d) != (plan.num_kv_heads, plan.head_dim):
        raise ValueError("q and the pool must have the plan's rows, heads and head_dim")
    slots, width = page_table.shape
    if plan.max_slot >= slots or plan.max_prefix > width * page:
        raise ValueError("the plan's slots and prefix lengths must fit page_table")
    _check_index(suffix_lengths, "suffix_lengths", 1, dev, plan.rows)


def _scale(scale):
    """A scale that fp32 holds: one that it flushed to 0 would make NaN of masked
    scores, -inf times 0."""
    scale = float(scale)
    if not 2.0 ** -126 <= scale <= 1e30:
        raise ValueError("scale must be positive and finite, in [2^-126, 1e30]")
    return scale


def _check_output(t, name, shape, like, dtype):
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.dtype != dtype or \
            t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {list(shape)} {dtype} on the pool's device")


def shared_prefix_attention(q, k_cache, v_cache, page_table, suffix_lengths, plan, *, scale=None,
                            out=None, lse=None):
    """Softmax attention of q [Nq,Hq,D] over each row's shared prefix and its
    own tokens in a page pool; returns (out [Nq,Hq,D], lse [Nq,Hq] fp32, natural
    log).

    k_cache, v_cache [pages,page_size,Hkv,D] and page_table [slots,width] int32
    as in :func:`moba_hip.append_rotary`; ``suffix_lengths`` [Nq] int32: how many
    tokens of its own slot each row attends (read on the device, cut to
    [0, plan.max_suffix]).  ``scale`` (in [2^-126, 1e30]) defaults to D ** -0.5.
    q, the pool and ``out`` must be 16-byte aligned.  A row with nothing to
    attend gives zeros and an lse of -inf; a token in an unmapped page is not
    attended.  Nothing is read back, so a call can be captured into a graph
    (``out`` and ``lse``, contiguous, then keep their addresses)."""
    done = _lib.calls().shared_attention(q, k_cache, v_cache, page_table, suffix_lengths, plan, scale,
                                         out, lse)
    if done is not NotImplemented:
        return done
    _check_attention(q, k_cache, v_cache, page_table, suffix_lengths, plan)
    pages, page, hkv, d = k_cache.shape
    width = page_table.shape[1]
    n, hq = plan.rows, plan.num_q_heads
    scale = d ** -0.5 if scale is None else _scale(scale)
    q = q.contiguous()
    qp, kp, vp = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if (qp | kp | vp) & 15:
        raise ValueError("q and the pool must be 16-byte aligned")
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_output(out, "out", plan._q_shape, q, q.dtype)
        if out.data_ptr() & 15:
            raise ValueError("out must be 16-byte aligned")
        if _meet(_span(out), _span(k_cache)) or _meet(_span(out), _span(v_cache)):
            raise ValueError("out must not overlap the pool")
    if lse is None:
        lse = torch.empty((n, hq), dtype=torch.float32, device=q.device)
    else:
        _check_output(lse, "lse", (n, hq), q, torch.float32)
        if any(_meet(_span(lse), _span(t)) for t in (out, k_cache, v_cache)):
            raise ValueError("lse must not overlap out or the pool")
    parts = plan.parts * hq
    # partial sums [parts, D], then (max, sum) pairs
    work = torch.empty(parts * (d + 2), dtype=torch.float32, device=q.device)
    wp, meta = work.data_ptr(), plan.meta.data_ptr()
    _on_device(k_cache.get_device(), "moba_hip_shared_attention", qp, _DTYPES[q.dtype], n, hq, hkv,
               d, scale, kp, vp, pages, page, page_table.data_ptr(), width,
               suffix_lengths.data_ptr(), 0, min(plan.max_suffix, width * page), meta, plan.n_items,
               meta + plan._rows_at, meta + plan._parts_at, plan.max_parts, plan.uneven, wp,
               wp + 4 * parts * d, out.data_ptr(), lse.data_ptr())
    return out, lse
