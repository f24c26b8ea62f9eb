"""8-bit paged KV cache: a page pool that holds codes and scales, the append that
quantises tokens on their way into it (their keys turned by their positions first),
the read that gives them back in 16 bits, and the attention of new tokens over it.

:class:`QuantizedPages` is the pool.  The functions serve callers that own one and its
table on the device (nothing is read back, so a call can be captured into a graph);
:class:`moba_hip.QuantizedKVCache` plans the pages itself.

A row of D values (one head of one token) stands as codes c and a scale s, x ~ c s::

    a = max(max |x|, 2^-100),  s = a / top,  c = x top / a to the nearest code,
                                             ties to the even one

with top 127 (``"int8"``) or 448 (``"fp8"``, the 8-bit float e4m3).  int8 is off by at
most a / 254; fp8 by 2^-4 of each value (a / 458752, half the smallest step, where that is
more), so it keeps small values next to large ones.  A row that holds an infinity or a NaN has codes 0
and scale NaN: it reads back as NaN.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .cache_layout import positive_int
from .ops import _lib
from .rotary import (_DTYPES, RotaryTable, _check_index, _check_token_tensor, _meet, _on_device,
                     _raise_bad, _span)
from .shared_prefix import _check_output, _scale

_CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
_MAX_SLOTS = 16


def _code_width(head_dim):
    """Bytes of a row of codes: whole 16-byte pieces."""
    return -(-head_dim // 16) * 16


class QuantizedPages(NamedTuple):
    """A pool of 8-bit pages: codes ``k``, ``v`` [pages,Hkv,page_size,Dp] (int8 or
    float8_e4m3fn; Dp: head_dim rounded up to 16) and scales ``k_scale``, ``v_scale``
    [pages,Hkv,page_size] fp32; contiguous, the codes 16-byte aligned.  head_dim is a
    multiple of 8, at most 256.  A cell that is attended holds what an append wrote there:
    finite codes, those behind head_dim 0."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    head_dim: int

    @classmethod
    def empty(cls, num_pages, page_size, num_kv_heads, head_dim, *, format="int8", device="cuda"):
        """A pool whose cells are not yet written."""
        _check_format(format)
        n, p = positive_int(num_pages, "num_pages"), positive_int(page_size, "page_size")
        h, d = positive_int(num_kv_heads, "num_kv_heads"), positive_int(head_dim, "head_dim")
        _check_head_dim(d)
        _check_size(n, p, h, d)
        codes = [torch.empty((n, h, p, _code_width(d)), dtype=_CODES[format], device=device)
                 for _ in range(2)]
        scales = [torch.empty((n, h, p), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales, d)

    @property
    def format(self):
        return "int8" if self.k.dtype == torch.int8 else "fp8"


def _check_format(format):
    if format not in ("int8", "fp8"):
        raise ValueError("format must be int8 or fp8")


def _check_head_dim(d):
    if not 8 <= d <= 256 or d % 8:
        raise ValueError("8-bit head_dim must be a multiple of 8 in [8,256]")


def _check_size(pages, page, heads, d):
    if pages * page >= 2 ** 31:
        raise ValueError("page pool exceeds int32 token capacity")
    if pages * page * heads > 0xfffffff0 // (_code_width(d) // 16):
        raise ValueError("page pool exceeds 64 GiB of codes")


# The checks below name what is wrong with a call.  They are not on the path of
# one that holds: the native host path (csrc/python/calls.cpp) tests the same
# conditions, allocates and launches.

def _check_pages(pages, page_table):
    """Raises what is wrong with a pool and its table; returns their sizes."""
    if not isinstance(pages, QuantizedPages):
        raise ValueError("pages must be QuantizedPages")
    k = pages.k
    if not isinstance(k, torch.Tensor) or k.dim() != 4 or not k.numel():
        raise ValueError("pages.k must be nonempty [pages,Hkv,page_size,Dp]")
    if k.dtype not in _FORMATS:
        raise ValueError("pages.k must be int8 or float8_e4m3fn")
    if not k.is_cuda:
        raise ValueError("cache device must be CUDA")
    n, h, p, width = k.shape
    d = pages.head_dim
    if isinstance(d, bool) or not isinstance(d, int):
        raise ValueError("pages.head_dim must be an integer")
    _check_head_dim(d)
    if width != _code_width(d):
        raise ValueError("pages.k must have head_dim rounded up to 16 codes a row")
    for name, t, shape, dtype in (("v", pages.v, k.shape, k.dtype),
                                  ("k_scale", pages.k_scale, k.shape[:3], torch.float32),
                                  ("v_scale", pages.v_scale, k.shape[:3], torch.float32)):
        if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != dtype or t.device != k.device:
            raise ValueError(f"pages.{name} must be {list(shape)} {dtype} on the device of pages.k")
    if not all(t.is_contiguous() for t in pages[:4]):
        raise ValueError("pages must be contiguous")
    if (k.data_ptr() | pages.v.data_ptr()) & 15:
        raise ValueError("pages must be 16-byte aligned")
    spans = [_span(t) for t in pages[:4]]
    if any(_meet(a, b) for i, a in enumerate(spans) for b in spans[:i]):
        raise ValueError("the tensors of pages must not overlap")
    _check_size(n, p, h, d)
    _check_index(page_table, "page_table", 2, k.device)
    if not page_table.numel():
        raise ValueError("page_table must be nonempty")
    if page_table.shape[1] * p >= 2 ** 31:
        raise ValueError("page pool exceeds int32 token capacity")
    return n, h, p, d


def _check_tokens(t, name, n, heads, d, device, like=None):
    if isinstance(t, torch.Tensor) and (t.dtype not in _DTYPES or t.device != device):
        raise ValueError(f"{name} must be BF16 or FP16 on the pool's device")
    _check_token_tensor(t, name, n, heads, d, t if like is None else like)


def _pool_args(pages, page_table):
    """The pool as the entries take it, from the codes on, and its table."""
    n, _, p, _ = pages.k.shape
    return ((pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(), n, p),
            (page_table.data_ptr(), page_table.shape[0], page_table.shape[1]))


def quantized_append(k, v, pages, page_table, token_seq, token_pos, *, rotary=None, q=None, q_out=None,
                     offsets=None, check=False):
    """Writes N new tokens into an 8-bit page pool.  With ``rotary`` (a
    :class:`moba_hip.RotaryTable`) their keys turn first, quantised from the fp32
    result, and so do the queries ``q`` of the same tokens, which are returned in
    their own type (None without ``q``).

    k, v [N,Hkv,D] and q [N,Hq,D] (bf16 or fp16, alike) may be views with a contiguous
    last dimension.  page_table, token_seq, token_pos, offsets, q_out and check, and
    what becomes of tokens without a cell or an angle: as in
    :func:`moba_hip.append_rotary`."""
    if not check:
        done = _lib.calls().quantized_append(k, v, pages, page_table, token_seq, token_pos, rotary, q, q_out,
                                             offsets)
        if done is not NotImplemented:
            return done
    n_pages, hkv, page, d = _check_pages(pages, page_table)
    dev = pages.k.device
    n = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else 0
    _check_tokens(k, "k", n, hkv, d, dev)
    _check_tokens(v, "v", n, hkv, d, dev, k)
    if n < 1:
        raise ValueError("k has an invalid shape")
    _check_index(token_seq, "token_seq", 1, dev, n)
    _check_index(token_pos, "token_pos", 1, dev, n)
    if rotary is None:
        for name, t in (("q", q), ("q_out", q_out), ("offsets", offsets)):
            if t is not None:
                raise ValueError(f"{name} without rotary")
    else:
        if not isinstance(rotary, RotaryTable):
            raise ValueError("rotary must be a RotaryTable")
        rotary._check(d, dev)
        if offsets is not None:
            _check_index(offsets, "offsets", 1, dev, page_table.shape[0])
    hq = 0
    if q is not None:
        _check_tokens(q, "q", n, None, d, dev, k)
        hq = q.shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    if n * (hq + 2 * hkv) * _code_width(d) >= 2 ** 33:
        raise ValueError("append exceeds 2^33 elements")
    pools = [_span(t) for t in pages[:4]]
    for t in (k, v, q):
        if t is not None and any(_meet(_span(t), at) for at in pools):
            raise ValueError("append inputs must not alias KV cache storage; clone first")
    if q is not None:
        if q_out is None:
            q_out = torch.empty((n, hq, d), dtype=q.dtype, device=q.device)
        else:
            _check_tokens(q_out, "q_out", n, hq, d, dev, k)
            if not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous")
            at = _span(q_out)
            if any(_meet(at, o) for o in (*pools, _span(q), _span(k), _span(v))):
                raise ValueError("q_out must not overlap the inputs or the pool")
    status = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    qa = (None, 0, 0) if q is None else (q.data_ptr(), q.stride(0), q.stride(1))
    turn = ((None, 0, 0, 0) if rotary is None else
            (rotary.cos_sin.data_ptr(), rotary.max_positions, rotary.rotary_dim, rotary.interleaved))
    pool, table = _pool_args(pages, page_table)
    _on_device(pages.k.get_device(), "moba_hip_quantized_append", *qa, k.data_ptr(), k.stride(0),
               k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _DTYPES[k.dtype], n, hq, hkv, d, *turn,
               _FORMATS[pages.k.dtype], *pool, *table, token_seq.data_ptr(), token_pos.data_ptr(),
               _lib.ptr(offsets), _lib.ptr(q_out), _lib.ptr(status))
    if check:
        _raise_bad(status, token_seq, token_pos, page_table.shape[1] * page)
    return q_out


def quantized_read(pages, page_table, token_seq, token_pos, *, dtype=torch.bfloat16, check=False):
    """The values of N stored tokens, code times scale rounded once to ``dtype`` (bf16
    or fp16): (k, v), each [N,Hkv,D].  token_seq and token_pos [N] int32 as in
    :func:`quantized_append`; a cell may be named more than once.  A token of slot -1 is
    padding and reads as zeros; so does one outside the table or in an unmapped page,
    which ``check`` makes a RuntimeError after the launch."""
    if not check and dtype in _DTYPES:
        done = _lib.calls().quantized_read(pages, page_table, token_seq, token_pos, _DTYPES[dtype])
        if done is not NotImplemented:
            return done
    n_pages, hkv, page, d = _check_pages(pages, page_table)
    dev = pages.k.device
    if dtype not in _DTYPES:
        raise ValueError("dtype must be BF16 or FP16")
    _check_index(token_seq, "token_seq", 1, dev)
    n = token_seq.shape[0]
    if n < 1:
        raise ValueError("token_seq must be nonempty")
    _check_index(token_pos, "token_pos", 1, dev, n)
    if n * hkv * (d // 8) >= 2 ** 31:
        raise ValueError("read exceeds 2^31 pieces of 8 elements")
    k, v = (torch.empty((n, hkv, d), dtype=dtype, device=dev) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    pool, table = _pool_args(pages, page_table)
    _on_device(pages.k.get_device(), "moba_hip_quantized_read", _FORMATS[pages.k.dtype], *pool, hkv, d, *table,
               token_seq.data_ptr(), token_pos.data_ptr(), n, _DTYPES[dtype], k.data_ptr(), v.data_ptr(),
               _lib.ptr(status))
    if check:
        bad = int(status)
        if bad & 1:
            raise RuntimeError("token_seq entries must be slots of page_table, or -1")
        if bad & 2:
            raise RuntimeError("a token's position has no page")
    return k, v


def _attention_work(n, hq, hkv, d, slots, chunk, limit):
    """Bytes of the workspace of an attention; raises for one that passes its counters."""
    size = -1 if n * hq >= 2 ** 31 else _lib.load().moba_hip_quantized_attention_work(
        n, hq, hkv, d, slots, chunk, limit)
    if size < 0:
        raise ValueError("attention exceeds 2^31 units of 128 tokens or 2^23 blocks of 16 heads")
    return size


def quantized_attention(q, pages, page_table, q_seq, lengths, *, selected=None, chunk_size=None,
                        max_length=None, scale=None, out=None, lse=None):
    """Softmax attention of q [Nq,Hq,D] (bf16 or fp16) over an 8-bit pool: row r attends
    the first ``lengths[r]`` tokens of slot ``q_seq[r]``; returns (out [Nq,Hq,D], lse
    [Nq,Hq] fp32, natural log).

    q_seq, lengths [Nq] int32, read on the device; lengths are cut to [0, max_length]
    (default: what page_table can map).  The fewer tokens a small call may have, the
    fewer workgroups a tight ``max_length`` lets it start.  With ``selected``
    [Nq,Hq,slots] int32 (1 to 16 slots) a head attends, of those tokens, the ones in the
    chunks of ``chunk_size`` that it names (-1: none, any order, a chunk named twice
    counts once): MoBA's decode with :attr:`DecodeResult.selected_blocks`.  A slot
    outside the table (-1: padding) and a row or head with nothing to attend give
    zeros and an lse of -inf; a token in an unmapped page is not attended.  A head whose
    query holds an infinity or a NaN gets NaN.  ``scale`` (in [2^-126, 1e30]) defaults to
    D ** -0.5.  q and ``out`` are contiguous and 16-byte aligned.  Scores, and before their
    scales the products of q with the codes (up to 127 or 448), must be finite in fp32.
    Weights are summed before they are divided, up to 2^6 for a token, so that values must
    stay below 2^122 / length in size.  A call takes less than 2^31 units
    of 128 tokens and 2^23 blocks of up to 16 query heads of a row and kv head.  Nothing is
    read back, so a call can be captured into a graph; what becomes of its tensors on other
    streams and in a graph: as in :func:`moba_hip.append_rotary`."""
    if out is None and lse is None:
        done = _lib.calls().quantized_attention(q, pages, page_table, q_seq, lengths, selected, chunk_size,
                                                max_length, scale)
        if done is not NotImplemented:
            return done
    n_pages, hkv, page, d = _check_pages(pages, page_table)
    dev = pages.k.device
    n = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    _check_tokens(q, "q", n, None, d, dev)
    hq = q.shape[1]
    if n < 1 or hq % hkv:
        raise ValueError("q must be nonempty, Hq a multiple of Hkv")
    if not q.is_contiguous() or q.data_ptr() & 15:
        raise ValueError("q must be contiguous and 16-byte aligned")
    _check_index(q_seq, "q_seq", 1, dev, n)
    _check_index(lengths, "lengths", 1, dev, n)
    span = page_table.shape[1] * page
    limit = span if max_length is None else min(span, positive_int(max_length, "max_length"))
    scale = d ** -0.5 if scale is None else _scale(scale)
    slots = chunk = 0
    if selected is not None:
        _check_index(selected, "selected", 3, dev, n)
        slots = selected.shape[2]
        if selected.shape[1] != hq or not 1 <= slots <= _MAX_SLOTS:
            raise ValueError("selected must be [Nq,Hq,slots] with 1 to 16 slots")
        if chunk_size is None:
            raise ValueError("selected needs chunk_size")
        chunk = min(positive_int(chunk_size, "chunk_size"), limit)
    elif chunk_size is not None:
        raise ValueError("chunk_size without selected")
    size = _attention_work(n, hq, hkv, d, slots, chunk, limit)
    pools = [_span(t) for t in pages[:4]]
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_output(out, "out", tuple(q.shape), q, q.dtype)
        if out.data_ptr() & 15:
            raise ValueError("out must be 16-byte aligned")
    if lse is None:
        lse = torch.empty((n, hq), dtype=torch.float32, device=dev)
    else:
        _check_output(lse, "lse", (n, hq), q, torch.float32)
    read = pools + [_span(t) for t in (q, page_table, q_seq, lengths, selected) if t is not None]
    if any(_meet(_span(out), at) for at in read) or any(_meet(_span(lse), at) for at in [*read, _span(out)]):
        raise ValueError("out and lse must not overlap each other, the inputs or the pool")
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    pool, table = _pool_args(pages, page_table)
    _on_device(pages.k.get_device(), "moba_hip_quantized_attention", q.data_ptr(), _DTYPES[q.dtype], n, hq,
               hkv, d, scale, _FORMATS[pages.k.dtype], *pool, *table, q_seq.data_ptr(), lengths.data_ptr(), 0,
               limit, _lib.ptr(selected), slots, chunk, work.data_ptr(), out.data_ptr(), lse.data_ptr())
    return out, lse
