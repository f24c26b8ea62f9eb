"""QuantizedKVCache, its prepared decode and Qwen2Session on it: what is stored, routed and
attended, against 64 bits; bounds in quant_check."""
import pytest
import torch

from quant_check import attention, check_attention, numbers, rounded, stored

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "fp8"]


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to("cuda", dtype)


def _cache(*args, **kw):
    from moba_hip import QuantizedKVCache
    return QuantizedKVCache(*args, **kw)


def _check(cache, result, q):
    """A DecodeResult's attention, on the routes that it took, and those routes: they name
    the current chunk and the highest scores of the cache's means (a choice within the
    scores' rounding is as good)."""
    dev = dict(dtype=torch.int32, device="cuda")
    seq = torch.tensor(result.sequence_ids, **dev)
    lens = torch.tensor([p + 1 for p in result.positions], **dev)
    check_attention((result.output, result.lse),
                    attention(q, cache.pages, cache._table, seq, lens, result.selected_blocks,
                              cache.chunk_size))
    if result.selected_blocks is None:
        return
    group = q.shape[1] // cache.num_kv_heads
    for r, (s, p) in enumerate(zip(result.sequence_ids, result.positions)):
        closed = p // cache.chunk_size
        means = cache._means[s, :closed].double().repeat_interleave(group, 1)      # [chunks, heads, d]
        score = (q[r].double()[None] * means).sum(-1)
        slack = (q[r].double().abs()[None] * means.abs()).sum(-1) * q.shape[2] * 2.0 ** -23
        for h in range(q.shape[1]):
            chosen = [c for c in result.selected_blocks[r, h].tolist() if c >= 0]
            assert chosen[0] == closed and len(set(chosen)) == len(chosen)
            want = min(result.selected_blocks.shape[2] - 1, closed)
            assert len(chosen) == 1 + want and all(c < closed for c in chosen[1:])
            if 0 < want < closed:
                rest = [c for c in range(closed) if c not in chosen]
                low = min((score[c, h] + slack[c, h]).item() for c in chosen[1:])
                assert low >= max((score[c, h] - slack[c, h]).item() for c in rest)


def _check_means(cache, slot):
    """Closed chunks' means: those of the stored values, summed in fp32, rounded once."""
    n, c = cache.lengths[slot], cache.chunk_size
    k, _, _ = numbers(cache.pages, cache._table, slot, torch.arange(n, device="cuda"))
    for i in range(n // c):
        x = k[i * c:(i + 1) * c]
        want, size = x.mean(0), x.abs().mean(0)
        got = cache._means[slot, i].double()
        assert ((got - want).abs() <= rounded(want, cache.dtype) + size * (c + 2) * 2.0 ** -24).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,chunk,dim,hq,hk", [(3, 4, 40, 15, 3), (7, 6, 64, 8, 1), (16, 8, 128, 8, 2),
                                                  (5, 64, 256, 6, 2), (100, 32, 96, 40, 1)])
def test_append_attend_and_read_back(fmt, dtype, page, chunk, dim, hq, hk):
    cache = _cache(3, 260, hk, dim, page_size=page, chunk_size=chunk, dtype=dtype, format=fmt)
    given = {2: [], 0: []}
    for i, counts in enumerate(((5, 130), (1, 1), (64, 7), (30, 3))):
        k, v = (_rand((sum(counts), hk, dim), dtype, 10 * i + x) for x in (1, 2))
        cache.append(k, v, sequence_ids=[2, 0], cu_seqlens=[0, counts[0], sum(counts)])
        given[2].append((k[:counts[0]], v[:counts[0]]))
        given[0].append((k[counts[0]:], v[counts[0]:]))
    for s, parts in given.items():
        got = cache.materialize(s)
        for x, y in zip((torch.cat([p[i] for p in parts]) for i in (0, 1)), got):
            c, scale = stored(x, fmt)
            assert y.dtype == dtype
            assert ((y.double() - c * scale[..., None]).abs() <= rounded(c * scale[..., None], dtype)).all()
        _check_means(cache, s)
    assert cache.materialize(1)[0].shape == (0, hk, dim)
    q = _rand((4, hq, dim), dtype, 99)
    ids = [2, 0, 0, 2]
    for mode, topk in (("dense", 4), ("moba", 1), ("moba", 3), ("moba", 9)):
        _check(cache, cache.attend(q, sequence_ids=ids, mode=mode, topk=topk), q)
        _check(cache, cache.attend(q, sequence_ids=ids, positions=[0, 17, 140, 99], mode=mode, topk=topk), q)
    k, v = (_rand((3, hk, dim), dtype, x) for x in (71, 72))
    q = _rand((3, hq, dim), dtype, 73)
    result = cache.append_and_attend(q, k, v, sequence_ids=[1, 2], cu_seqlens=[0, 2, 3], topk=3)
    assert result.sequence_ids == (1, 1, 2) and result.positions == (0, 1, 100)
    _check(cache, result, q)
    cache.reset([2])
    assert cache.lengths == (141, 2, 0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rotary_append(fmt):
    """The cache's append_rotary stores what quantized_append does with the same angles."""
    from moba_hip import QuantizedPages, RotaryTable, quantized_append, quantized_read
    hk, hq, dim, n = 2, 6, 64, 21
    rt = RotaryTable(dim, 100)
    cache = _cache(2, 64, hk, dim, page_size=5, format=fmt)
    k, v, q = _rand((n, hk, dim), cache.dtype, 1), _rand((n, hk, dim), cache.dtype, 2), \
        _rand((n, hq, dim), cache.dtype, 3)
    done = cache.append_rotary(k, v, rt, sequence_ids=[1], cu_seqlens=[0, n], q=q, offsets=[30])
    pages = QuantizedPages.empty(5, 5, hk, dim, format=fmt)
    dev = dict(dtype=torch.int32, device="cuda")
    table, seq, pos = torch.arange(5, **dev)[None], torch.zeros(n, **dev), torch.arange(n, **dev)
    turned = quantized_append(k, v, pages, table, seq, pos, rotary=rt, q=q,
                              offsets=torch.tensor([30], **dev))
    assert torch.equal(done.q, turned)
    for a, b in zip(cache.materialize(1), quantized_read(pages, table, seq, pos)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("mode,topk", [("dense", 4), ("moba", 3)])
@pytest.mark.parametrize("page,chunk,dim,hq,hk", [(3, 4, 40, 15, 3), (16, 8, 128, 8, 2), (5, 8, 256, 34, 2)])
def test_prepared_steps(graph, fmt, mode, topk, page, chunk, dim, hq, hk):
    """Steps and attends of a lease, with eager work between them; chunks close on the
    way, and the cache afterwards goes on from where the lease ended."""
    dtype = torch.bfloat16
    cache = _cache(3, 60, hk, dim, page_size=page, chunk_size=chunk, dtype=dtype, format=fmt)
    k, v = _rand((14, hk, dim), dtype, 501), _rand((14, hk, dim), dtype, 502)
    cache.append(k, v, sequence_ids=[2, 0], cu_seqlens=[0, 5, 14])
    lengths, table = cache.lengths, cache.page_table
    with cache.prepare_decode([2, 0], hq, topk=topk, mode=mode) as plan:
        if graph:
            plan.capture("step").capture("attend")
            assert cache.lengths == lengths and cache.page_table == table
        for step in range(20):
            q = _rand((2, hq, dim), dtype, 510 + step)
            kn, vn = _rand((2, hk, dim), dtype, 530 + step), _rand((2, hk, dim), dtype, 550 + step)
            result = plan.step(q, kn, vn, use_graph=graph)
            _check(cache, result, q)
            for i, sid in enumerate((2, 0)):
                for x, y in zip((kn, vn), cache.materialize(sid)):
                    c, s = stored(x[i], fmt)
                    want = c * s[..., None]
                    assert ((y[-1].double() - want).abs() <= rounded(want, dtype)).all()
            _check(cache, plan.attend(q, use_graph=graph), q)
        with pytest.raises(ValueError, match="owns cache"):
            cache.reset()
        assert plan.delta_uploads <= 20
    assert cache.lengths == (29, 0, 25)
    for s in (0, 2):
        _check_means(cache, s)
    q = _rand((2, hq, dim), dtype, 9)
    _check(cache, cache.attend(q, sequence_ids=[0, 2], topk=3), q)


@pytest.mark.parametrize("graph", [False, True])
def test_prepared_steps_that_turn(graph):
    """A lease with a table of angles does what append_rotary and attend do."""
    from moba_hip import RotaryTable
    hk, hq, dim = 2, 6, 64
    rt = RotaryTable(dim, 40)
    caches = [_cache(2, 32, hk, dim, page_size=4, chunk_size=8, format="int8") for _ in range(2)]
    k, v = _rand((9, hk, dim), caches[0].dtype, 1), _rand((9, hk, dim), caches[0].dtype, 2)
    for c in caches:
        c.append_rotary(k, v, rt, sequence_ids=[1], cu_seqlens=[0, 9])
    with caches[0].prepare_decode([0, 1], hq, mode="dense", rotary=rt) as plan:
        if graph:
            plan.capture()
        for step in range(12):
            q, kn, vn = (_rand((2, h, dim), caches[0].dtype, 100 * step + h + x)
                         for x, h in enumerate((hq, hk, hk)))
            got = plan.step(q, kn, vn, use_graph=graph)
            turned = caches[1].append_rotary(kn, vn, rt, sequence_ids=[0, 1], q=q).q
            assert torch.equal(plan._turned, turned)
            _check(caches[0], got, turned)
        with pytest.raises(ValueError, match="no attend"):
            plan.attend(q)
    for s in (0, 1):
        for a, b in zip(caches[0].materialize(s), caches[1].materialize(s)):
            assert torch.equal(a, b)


def test_lease_lifecycle():
    c = _cache(1, 7, 1, 8, page_size=3, chunk_size=4)
    q = torch.ones((1, 1, 8), device="cuda", dtype=c.dtype)
    with c.prepare_decode([0], 1) as p:
        with pytest.raises(ValueError, match="NaN/Inf"):
            p.step(q * float("nan"), q, q)
        with pytest.raises(ValueError, match="capture"):
            p.step(q, q, q, use_graph=True)
        with pytest.raises(ValueError, match="nonempty"):
            p.attend(q)
        with pytest.raises(ValueError, match="nonempty"):
            p.capture("attend")
        assert c.lengths == [0] or tuple(c.lengths) == (0,)
        for _ in range(7):
            p.step(q, q, q)
        assert p.delta_uploads == 3
        with pytest.raises(ValueError, match="max_seq_len"):
            p.step(q, q, q)
        with torch.cuda.stream(torch.cuda.Stream()):
            with pytest.raises(ValueError, match="cross-stream"):
                p.attend(q)
        p.capture("attend")
        with pytest.raises(ValueError, match="already captured"):
            p.capture("attend")
        _check(c, p.attend(q, use_graph=True), q)
    with pytest.raises(ValueError, match="closed"):
        p.step(q, q, q)
    assert c.lengths == (7,)
    for call in (c.attend_shared, c.prepare_shared_decode):
        with pytest.raises(ValueError, match="16-bit cache"):
            call(q, sequence_ids=[0], prefix_ids=[-1])


def _model(seed, layers=2):
    from transformers import Qwen2Config, Qwen2ForCausalLM
    torch.manual_seed(seed)
    cfg = Qwen2Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=layers,
                      num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=4096,
                      attn_implementation="eager")
    m = Qwen2ForCausalLM(cfg).to("cuda", torch.bfloat16).eval()
    for p in m.parameters():
        p.requires_grad_(False)
    return m


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("mode,topk", [("dense", 4), ("moba", 3)])
def test_qwen2_session_in_8_bits(fmt, mode, topk):
    """Graph and eager steps alike, bit for bit; and the 16-bit session's logits nearly: a
    stored value is off by up to 1/254 (int8) or 1/16 (fp8) of the largest or of itself."""
    from moba_hip.qwen2 import Qwen2Session
    model = _model(3)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 512, (1, 300), generator=g).to("cuda")
    extra = torch.randint(0, 512, (10,), generator=g).tolist()
    logits = {}
    for form, backend in ((None, "eager"), (fmt, "eager"), (fmt, "model_graph")):
        with Qwen2Session(model, 400, mode=mode, chunk=32, topk=topk, page=16, backend=backend,
                          kv_format=form) as s:
            out = [s.prefill(ids)]
            s.prepare()
            for t in extra:
                out.append(s.step(t).clone())
                torch.randn(100, device="cuda").sum().item()   # eager work between replays
            logits[form, backend] = out
    for a, b in zip(logits[fmt, "eager"], logits[fmt, "model_graph"]):
        assert torch.equal(a, b)
    assert torch.equal(logits[None, "eager"][0], logits[fmt, "eager"][0])   # the prompt's own
    if mode == "dense":    # a route may differ where two chunks score alike
        for a, b in zip(logits[None, "eager"][1:], logits[fmt, "eager"][1:]):
            cos = torch.nn.functional.cosine_similarity(a.float().flatten(), b.float().flatten(), dim=0)
            assert cos > 0.99


def test_a_prepared_decode_of_another_cache_is_refused():
    from moba_hip import PagedKVCache, PreparedDecode, PreparedQuantizedDecode, PreparedSharedDecode
    args = (1, 8, 1, 64)
    wide, narrow = PagedKVCache(*args, page_size=4, chunk_size=4), _cache(*args, page_size=4, chunk_size=4)
    with pytest.raises(ValueError, match="8-bit"):
        PreparedDecode(narrow, [0], 1)
    with pytest.raises(ValueError, match="16-bit"):
        PreparedSharedDecode(narrow, [0], [-1], 1)
    with pytest.raises(ValueError, match="QuantizedKVCache"):
        PreparedQuantizedDecode(wide, [0], 1)
    for c in (wide, narrow):
        c.prepare_decode([0], 1).close()    # nothing was leased
