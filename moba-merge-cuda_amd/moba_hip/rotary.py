"""Rotary append: keys rotated by their positions on the way into a paged KV
cache, with the queries of the same tokens, in one launch.

:class:`RotaryTable` holds the cosines and sines of a model's rotation;
:func:`append_rotary` serves callers that own a page pool and its table on the
device (nothing is read back, so a call can be captured into a graph);
:meth:`moba_hip.PagedKVCache.append_rotary` plans the pages itself.
"""
from __future__ import annotations

import torch

from .cache_layout import positive_int
from .ops import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


class RotaryTable:
    """cos and sin of ``position * inv_freq[i]`` for every position below
    ``max_positions``, as one fp32 tensor ``cos_sin [max_positions,
    rotary_dim / 2, 2]``.  Angles are formed in 64 bits and rounded once (a
    32-bit angle of position 10^5 is off by up to 4e-3).

    ``rotary_dim`` is the number of leading dims of a head that turn (even);
    ``interleaved`` pairs dims (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
    ``inv_freq`` replaces ``base ** (-2i / rotary_dim)``; ``scaling``
    multiplies cos and sin."""

    def __init__(self, rotary_dim, max_positions, *, base=10000.0, inv_freq=None, scaling=1.0,
                 interleaved=False, device="cuda"):
        self._shape(positive_int(rotary_dim, "rotary_dim"), interleaved)
        n = positive_int(max_positions, "max_positions")
        if n >= 2 ** 31:
            raise ValueError("max_positions exceeds int32 capacity")
        half = self.rotary_dim // 2
        if inv_freq is None:
            inv = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
        else:
            inv = torch.as_tensor(inv_freq).to(device, torch.float64)
            if inv.shape != (half,):
                raise ValueError("inv_freq must be [rotary_dim / 2]")
        angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inv
        self._store(angle.cos() * scaling, angle.sin() * scaling)

    @classmethod
    def from_cos_sin(cls, cos, sin, *, interleaved=False):
        """The table of a model's own ``cos`` and ``sin`` [positions,
        rotary_dim / 2]."""
        ok = all(isinstance(t, torch.Tensor) and t.dim() == 2 and t.is_floating_point()
                 for t in (cos, sin))
        if not ok or cos.shape != sin.shape or cos.device != sin.device or not cos.numel() or \
                cos.shape[0] >= 2 ** 31:
            raise ValueError("cos and sin must be alike, nonempty [positions, rotary_dim / 2]")
        self = cls.__new__(cls)
        self._shape(2 * cos.shape[1], interleaved)
        self._store(cos, sin)
        return self

    def _shape(self, rotary_dim, interleaved):
        if rotary_dim % 2 or rotary_dim > 256:
            raise ValueError("rotary_dim must be even, at most 256")
        if not isinstance(interleaved, bool):
            raise ValueError("interleaved must be bool")
        self.rotary_dim, self.interleaved = rotary_dim, interleaved

    def _store(self, cos, sin):
        self.cos_sin = torch.stack((cos, sin), dim=-1).detach().to(torch.float32).contiguous()

    @property
    def max_positions(self):
        return self.cos_sin.shape[0]

    @property
    def device(self):
        return self.cos_sin.device

    def _check(self, head_dim, device):
        """Raises what keeps heads of ``head_dim`` on ``device`` from being turned.
        ``cos_sin`` is the caller's to replace (on another device, say): what
        the kernels read is tested at each use."""
        cs = self.cos_sin
        if not isinstance(cs, torch.Tensor) or cs.dtype != torch.float32 or cs.dim() != 3 or \
                cs.layout != torch.strided or not cs.is_contiguous() or cs.data_ptr() & 15 or \
                not 0 < cs.shape[0] < 2 ** 31 or (2 * cs.shape[1], cs.shape[2]) != (self.rotary_dim, 2):
            raise ValueError("rotary.cos_sin must be contiguous, 16-byte aligned fp32 "
                             "[positions, rotary_dim / 2, 2]")
        if self.rotary_dim > head_dim:
            raise ValueError("rotary_dim exceeds head_dim")
        if self.device != device:
            raise ValueError("rotary table must be on the cache's device")


# The checks below name what is wrong with a call.  They are not on the path of
# one that holds: the native host path (csrc/python/calls.cpp) tests the same
# conditions, allocates and launches.

def _check_token_tensor(t, name, n, heads, d, like):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be [N,H,D]")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must match the page pool's device and dtype")
    shape = t.shape
    if shape[0] != n or shape[2] != d or shape[1] < 1 or shape[1] != (heads or shape[1]):
        raise ValueError(f"{name} has an invalid shape")
    if t.stride(2) != 1:
        raise ValueError(f"{name} last dimension must be contiguous")
    if t.requires_grad:
        raise ValueError("KV cache/decode is inference-only; detach Q/K/V")


def _check_pool(k_cache, v_cache, page_table):
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4 or not k_cache.numel():
        raise ValueError("k_cache must be nonempty [pages, page_size, Hkv, D]")
    if k_cache.dtype not in _DTYPES:
        raise ValueError("cache dtype must be BF16 or FP16")
    if not k_cache.is_cuda:
        raise ValueError("cache device must be CUDA")
    if not isinstance(v_cache, torch.Tensor) or v_cache.shape != k_cache.shape or \
            v_cache.dtype != k_cache.dtype or v_cache.device != k_cache.device:
        raise ValueError("v_cache must be like k_cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be contiguous")
    _check_index(page_table, "page_table", 2, k_cache.device)
    if not page_table.numel():
        raise ValueError("page_table must be nonempty")
    pages, page = k_cache.shape[:2]
    if pages * page >= 2 ** 31 or page_table.shape[1] * page >= 2 ** 31:
        raise ValueError("page pool exceeds int32 token capacity")


def _check_index(t, name, dim, device, size=None):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim or \
            t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 {dim}D tensor on the cache's device")
    if size is not None and t.shape[0] != size:
        raise ValueError(f"{name} must have {size} entries")


def _check_append(k, v, k_cache, v_cache, page_table, token_seq, token_pos, rotary, q, offsets):
    """Raises what is wrong with the arguments of an append."""
    _check_pool(k_cache, v_cache, page_table)
    _, _, hkv, d = k_cache.shape
    n = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else 0
    _check_token_tensor(k, "k", n, hkv, d, k_cache)
    _check_token_tensor(v, "v", n, hkv, d, k_cache)
    if n < 1:
        raise ValueError("k has an invalid shape")
    dev = k_cache.device
    _check_index(token_seq, "token_seq", 1, dev, n)
    _check_index(token_pos, "token_pos", 1, dev, n)
    if offsets is not None:
        _check_index(offsets, "offsets", 1, dev, page_table.shape[0])
    if not isinstance(rotary, RotaryTable):
        raise ValueError("rotary must be a RotaryTable")
    rotary._check(d, dev)
    if q is not None:
        _check_token_tensor(q, "q", n, None, d, k_cache)
    if n * ((0 if q is None else q.shape[1]) + 2 * hkv) * d >= 2 ** 31:
        raise ValueError("append exceeds 2^31 elements")


def _span(t):
    """[start, end) addresses of a nonempty tensor's elements."""
    p = t.data_ptr()
    return p, p + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _meet(a, b):
    return a[0] < b[1] and b[0] < a[1]


def append_rotary(k, v, k_cache, v_cache, page_table, token_seq, token_pos, rotary, *, q=None,
                  q_out=None, offsets=None, check=False):
    """Writes N new tokens into a page pool, their keys rotated, and returns
    their queries rotated (None without ``q``).

    k, v [N,Hkv,D] and q [N,Hq,D] may be views (of one projection's output, say)
    with a contiguous last dimension; k_cache, v_cache [pages,page_size,Hkv,D];
    page_table [slots,width] int32 (physical page per logical page, -1 none);
    token_seq, token_pos [N] int32: slot and position of each token.  A token
    turns by its position plus ``offsets[slot]`` ([slots] int32; a sequence
    that goes on behind a shared prefix has the prefix's length there).
    ``q_out`` [N,Hq,D] contiguous receives the queries; it, the inputs and the
    pool must not overlap.

    A token of slot -1 is padding: nothing of it is written.  A token outside
    the table, in an unmapped page or past the rotary table has no key and
    value written either, nor, past the rotary table, its query; with ``check`` such
    tokens, and two tokens of one slot and position, raise RuntimeError after the
    launch (one device-to-host copy).  Two tokens of one cell leave it undefined:
    its key and its value may each hold pieces of both.  A tensor of the call, the
    table's too, that is used on another stream than its own must be kept until
    that work is done, and those of a captured call for as long as it is replayed."""
    if not check:
        done = _lib.calls().append_rotary(k, v, k_cache, v_cache, page_table, token_seq, token_pos,
                                          rotary, q, q_out, offsets)
        if done is not NotImplemented:
            return done
    _check_append(k, v, k_cache, v_cache, page_table, token_seq, token_pos, rotary, q, offsets)
    pages, page, hkv, d = k_cache.shape
    n = k.shape[0]
    pools = _span(k_cache), _span(v_cache)
    if _meet(*pools):
        raise ValueError("k_cache and v_cache must not overlap")
    for t in (k, v, q):
        if t is not None:
            at = _span(t)
            if _meet(at, pools[0]) or _meet(at, pools[1]):
                raise ValueError("append inputs must not alias KV cache storage; clone first")
    hq = 0
    if q is not None:
        hq = q.shape[1]
        if q_out is None:
            q_out = torch.empty((n, hq, d), dtype=q.dtype, device=q.device)
        else:
            _check_token_tensor(q_out, "q_out", n, hq, d, k_cache)
            if not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous")
            at = _span(q_out)
            if any(_meet(at, _span(t)) for t in (q, k, v, k_cache, v_cache)):
                raise ValueError("q_out must not overlap the inputs or the pool")
    elif q_out is not None:
        raise ValueError("q_out without q")
    status = torch.zeros(1, dtype=torch.int32, device=k.device) if check else None
    qa = (None, 0, 0) if q is None else (q.data_ptr(), q.stride(0), q.stride(1))
    _on_device(k_cache.get_device(), "moba_hip_append_rotary", *qa, k.data_ptr(), k.stride(0),
               k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _DTYPES[k.dtype], n, hq, hkv, d,
               rotary.cos_sin.data_ptr(), rotary.max_positions, rotary.rotary_dim,
               rotary.interleaved, k_cache.data_ptr(), v_cache.data_ptr(), pages, page,
               page_table.data_ptr(), page_table.shape[0], page_table.shape[1],
               token_seq.data_ptr(), token_pos.data_ptr(), _lib.ptr(offsets), _lib.ptr(q_out),
               _lib.ptr(status))
    if check:
        _raise_bad(status, token_seq, token_pos, page_table.shape[1] * page)
    return q_out


def _on_device(idx, name, *args):
    """Calls an entry on the current stream of device ``idx``."""
    stream = torch._C._cuda_getCurrentRawStream(idx)
    if torch._C._cuda_getDevice() == idx:
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(idx):
            _lib.call(name, *args, stream)


def _raise_bad(status, token_seq, token_pos, span):
    live = token_seq >= 0
    cells = token_seq[live].long() * span + token_pos[live]
    twice = cells.numel() - torch.unique(cells).numel()
    bad = int(status)
    for bit, message in ((1, "token_seq entries must be slots of page_table, or -1"),
                         (2, "a token's position has no page"),
                         (4, "a token's position lies outside the rotary table")):
        if bad & bit:
            raise RuntimeError(message)
    if twice:
        raise RuntimeError("two tokens of one append share a cell")
