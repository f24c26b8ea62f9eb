"""Chunk means of the 8-bit cache: chunks of more than one token a lane, up to the limit,
on pages that divide them and that do not, from appends and from prepared steps."""
import pytest
import torch

from quant_check import numbers, rounded

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "fp8"]
CHUNKS = [63, 64, 65, 100, 128, 512, 1000, 1023, 1024]


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to("cuda", dtype)


def _cache(*args, **kw):
    from moba_hip import QuantizedKVCache
    return QuantizedKVCache(*args, **kw)


def _check_means(cache, slot):
    """Each closed chunk's mean against that of the stored values in 64 bits.  A value is a
    rounded product; of c tokens a lane adds ceil(c / 64), six additions join the lanes, and
    the quotient and the result round once each: in fp32 (ceil(c / 64) + 8) 2^-24 of mean |x|,
    where a token that is left out, or taken twice, changes the mean by |x| / c, 2^-10 at least."""
    n, c = cache.lengths[slot], cache.chunk_size
    k, _, live = numbers(cache.pages, cache._table, slot, torch.arange(n, device="cuda"))
    assert live.all() and n >= c
    x = k[:n // c * c].view(n // c, c, *k.shape[1:])
    want, size = x.mean(1), x.abs().mean(1)
    got = cache._means[slot, :n // c].double()
    assert ((got - want).abs() <= rounded(want, cache.dtype) + size * (-(-c // 64) + 8) * 2.0 ** -24).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("chunk", CHUNKS)
def test_means_of_long_chunks(fmt, dtype, chunk):
    """Chunks that close in one append, two and more of a sequence, and in several appends."""
    hk, dim = 3, 40
    for page in (chunk, 48, 7):
        cache = _cache(2, 3 * chunk + 5, hk, dim, page_size=page, chunk_size=chunk, dtype=dtype, format=fmt)
        for i, (a, b) in enumerate(((2 * chunk + 3, 1), (chunk - 4, chunk - 2), (1, 1), (1, 3))):
            k, v = (_rand((a + b, hk, dim), dtype, 10 * i + x) for x in (1, 2))
            cache.append(k, v, sequence_ids=[1, 0], cu_seqlens=[0, a, a + b])
        assert cache.lengths == (chunk + 3, 3 * chunk + 1)
        for slot in (0, 1):
            _check_means(cache, slot)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [8, 64, 128, 256])
def test_means_at_the_default_chunk(fmt, dim):
    cache = _cache(1, 700, 2, dim, format=fmt)
    k = _rand((700, 2, dim), cache.dtype, dim)
    cache.append(k, k, sequence_ids=[0], cu_seqlens=[0, 700])
    assert cache.chunk_size == 128
    _check_means(cache, 0)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("chunk", [65, 100, 128, 1000, 1024])
def test_steps_that_close_long_chunks(graph, fmt, chunk):
    """The mean that a prepared step takes, of one row and of both at once; routes name the
    chunks of the highest scores by those means."""
    hk, hq, dim, dtype = 2, 6, 64, torch.bfloat16
    cache = _cache(2, 3 * chunk, hk, dim, page_size=48, chunk_size=chunk, dtype=dtype, format=fmt)
    given = 2 * chunk - 3, chunk - 2
    k, v = _rand((sum(given), hk, dim), dtype, 1), _rand((sum(given), hk, dim), dtype, 2)
    cache.append(k, v, sequence_ids=[0, 1], cu_seqlens=[0, given[0], sum(given)])
    with cache.prepare_decode([0, 1], hq, topk=2, check_finite=False) as plan:
        if graph:
            plan.capture()
        for step in range(6):
            q, kn, vn = (_rand((2, h, dim), dtype, 100 * step + x) for x, h in enumerate((hq, hk, hk)))
            result = plan.step(q, kn, vn, use_graph=graph)
            for row in (0, 1):
                closed = result.positions[row] // chunk
                if closed:
                    means = cache._means[row, :closed].double().repeat_interleave(hq // hk, 1)
                    score = (q[row].double()[None] * means).sum(-1)
                    slack = (q[row].double().abs()[None] * means.abs()).sum(-1) * dim * 2.0 ** -23
                    chosen = result.selected_blocks[row, :, 1].long()
                    heads = torch.arange(hq, device="cuda")
                    assert ((score + slack)[chosen, heads] >= (score - slack).amax(0)).all()
    assert cache.lengths == (2 * chunk + 3, chunk + 4)
    for slot in (0, 1):
        _check_means(cache, slot)


def test_more_items_than_a_launch_holds():
    """32 767 items of 64 kv heads of 256 dims fill a launch; of the items around its end, some
    close a chunk, and the others, as a step's rows do, none."""
    from quant_check import cells, make_table
    from moba_hip import QuantizedPages, quantized_append
    from moba_hip.ops import _lib
    hk, dim, page, most = 64, 256, 4, 32767
    table, n_pages = make_table([2] * 5, page, 0)
    pages = QuantizedPages.empty(n_pages, page, hk, dim)
    seq, pos = cells([2] * 5)
    k = _rand((10, hk, dim), torch.bfloat16, 1)
    quantized_append(k, k, pages, table, seq, pos)
    dev = dict(dtype=torch.int32, device="cuda")
    n = most + 100
    item_seq, item_pos = torch.zeros(n, **dev), torch.zeros(n, **dev)
    for slot, at in ((1, most - 1), (2, most), (3, n - 1)):
        item_seq[at], item_pos[at] = slot, 1
    means = torch.full((5, 1, hk, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    _lib.call("moba_hip_quantized_means", 0, pages.k.data_ptr(), pages.k_scale.data_ptr(), n_pages, page, hk, dim,
              table.data_ptr(), 5, 1, item_seq.data_ptr(), item_pos.data_ptr(), n, 1, 2, 0, means.data_ptr(), 1,
              torch.cuda.current_stream().cuda_stream)
    assert (means[[0, 4]] == 7).all()
    for slot in (1, 2, 3):
        x, _, _ = numbers(pages, table, slot, torch.arange(2, device="cuda"))
        want, size = x.mean(0), x.abs().mean(0)
        assert ((means[slot, 0].double() - want).abs() <= rounded(want, means.dtype) + size * 9 * 2.0 ** -24).all()
