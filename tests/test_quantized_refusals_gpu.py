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
