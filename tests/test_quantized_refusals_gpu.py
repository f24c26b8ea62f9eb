"""What an 8-bit cache refuses, it refuses before it stores."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to("cuda", dtype)


@pytest.mark.parametrize("hq,chunk,n,message", [(65, 4, 20, "64 query heads"), (1, 1, 8193, "8192 chunks")])
def test_append_and_attend_refuses_before_it_stores(hq, chunk, n, message):
    """More heads or chunks than are routed: nothing is appended, so that the call can be made
    again in another way."""
    from moba_hip import QuantizedKVCache
    cache = QuantizedKVCache(2, 8300, 1, 64, page_size=16, chunk_size=chunk)
    k = _rand((n, 1, 64), cache.dtype, 1)
    cache.append(k, k, sequence_ids=[1], cu_seqlens=[0, n])
    table, lengths, stored = cache.page_table, cache.lengths, cache.materialize(1)
    q = _rand((2, hq, 64), cache.dtype, 2)
    with pytest.raises(ValueError, match=message):
        cache.append_and_attend(q, k[:2], k[:2], sequence_ids=[1, 0], topk=3)
    assert cache.lengths == lengths and cache.page_table == table
    assert all(torch.equal(a, b) for a, b in zip(stored, cache.materialize(1)))
    result = cache.append_and_attend(q, k[:2], k[:2], sequence_ids=[1, 0], mode="dense")
    assert result.positions == (n, 0) and cache.lengths == (1, n + 1)


def test_the_last_call_that_is_routed():
    """8192 chunks before the one of the token itself, which the call stores."""
    from moba_hip import QuantizedKVCache
    cache = QuantizedKVCache(1, 8300, 1, 64, page_size=16, chunk_size=1)
    k = _rand((8192, 1, 64), cache.dtype, 1)
    cache.append(k, k, sequence_ids=[0], cu_seqlens=[0, 8192])
    q = _rand((1, 64, 64), cache.dtype, 2)
    result = cache.append_and_attend(q, k[:1], k[:1], sequence_ids=[0], topk=3)
    assert result.positions == (8192,) and torch.isfinite(result.output).all()
    with pytest.raises(ValueError, match="8192 chunks"):
        cache.append_and_attend(q, k[:1], k[:1], sequence_ids=[0], topk=3)
    assert cache.lengths == (8193,)


def test_the_most_rows_of_an_attention():
    """Rows of padding, as many as a launch has threads for; one more is refused on both host
    paths, before anything is launched."""
    from moba_hip import QuantizedPages, quantized_attention
    n = (2 ** 23 - 96) // 2
    dev = dict(dtype=torch.int32, device="cuda")
    pages = QuantizedPages.empty(2, 16, 2, 8)
    table, q_seq, lens = torch.zeros(1, 2, **dev), torch.full((n + 1,), -1, **dev), torch.ones(n + 1, **dev)
    q = torch.ones(n + 1, 2, 8, dtype=torch.bfloat16, device="cuda")
    out, lse = quantized_attention(q[:n], pages, table, q_seq[:n], lens[:n])
    assert not out.any() and (lse == -float("inf")).all()
    out.fill_(7.0)
    given = torch.cat([out, out[:1]])
    for kw in ({}, {"out": given}):
        with pytest.raises(ValueError, match="blocks of 16 heads"):
            quantized_attention(q, pages, table, q_seq, lens, **kw)
    assert (given == 7).all()


def test_a_cache_refuses_an_attention_that_is_too_large_before_it_stores(monkeypatch):
    """And a lease of too many rows before it begins."""
    from moba_hip import QuantizedKVCache, quantized_cache
    cache = QuantizedKVCache(1, 40, 2, 64, page_size=16, chunk_size=8)
    k, q = _rand((20, 2, 64), cache.dtype, 1), _rand((1, 4, 64), cache.dtype, 2)
    cache.append(k, k, sequence_ids=[0], cu_seqlens=[0, 20])
    asked = []

    def refuse(*args):
        asked.append(args)
        raise ValueError("too large")

    with monkeypatch.context() as patch:
        patch.setattr(quantized_cache, "_attention_work", refuse)
        for kw in (dict(mode="dense"), dict(topk=3)):
            with pytest.raises(ValueError, match="too large"):
                cache.append_and_attend(q, k[:1], k[:1], sequence_ids=[0], **kw)
            with pytest.raises(ValueError, match="too large"):
                cache.prepare_decode([0], 4, **kw)
    assert asked == [(1, 4, 2, 64, 0, 8, 21), (1, 4, 2, 64, 0, 0, 40), (1, 4, 2, 64, 3, 8, 21), (1, 4, 2, 64, 3, 8, 40)]
    assert cache.lengths == (20,)
    with cache.prepare_decode([0], 4, topk=3) as plan:
        plan.step(q, k[:1], k[:1])
    assert cache.append_and_attend(q, k[:1], k[:1], sequence_ids=[0], topk=3).positions == (21,)
