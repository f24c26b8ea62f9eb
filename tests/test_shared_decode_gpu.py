"""The paged-cache operators as a user runs them together: a prompt appended
with its rotation into one slot, sequences that go on behind it, and their
decode, through PagedKVCache, PreparedSharedDecode and Qwen2Branches.

Outputs are compared with the softmax in 64 bits over what the cache holds
(the tolerances of decode_check: bf16 max 2e-2 and mean 2e-3, fp16 4e-3 and
4e-4, the bounds of the other decode paths); what the cache holds is compared
with the rotation in 64 bits at half a step of its type plus fp32 terms."""
import numpy as np
import pytest
import torch

from decode_check import rand
from helpers import TOL
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def _turned(x, table, pos):
    half = table.rotary_dim // 2
    cs = table.cos_sin.double()[torch.as_tensor(pos, device="cuda")][:, None]
    y = x.double().clone()
    a, b = y[..., :half].clone(), y[..., half:2 * half].clone()
    y[..., :half] = a * cs[..., 0] - b * cs[..., 1]
    y[..., half:2 * half] = a * cs[..., 1] + b * cs[..., 0]
    return y


def _near(got, want, dtype):
    """One rounding of the rotated value, and fp32 products of it."""
    step = torch.finfo(dtype).eps / 2
    assert ((got.double() - want).abs() <= step * want.abs() + 2.0 ** -20 * (1 + want.abs().max())).all()


def _attended(cache, q, rows):
    """Exact output of each row: rows = (prefix slot or -1, own slot, own tokens)."""
    out = []
    for r, (prefix, own, n) in enumerate(rows):
        ks, vs = zip(*([cache.materialize(prefix)] if prefix >= 0 else []),
                     tuple(x[:n] for x in cache.materialize(own)))
        k, v = torch.cat(ks).double(), torch.cat(vs).double()
        g = q.shape[1] // k.shape[1]
        k, v = (x.repeat_interleave(g, 1).transpose(0, 1) for x in (k, v))
        s = (q[r].double()[:, None] * k).sum(-1) * q.shape[2] ** -0.5
        out.append((torch.softmax(s, -1)[..., None] * v).sum(1))
    return torch.stack(out)


def _close(got, want, dtype):
    err = (got.double() - want).abs()
    assert err.max() <= TOL[dtype][0] and err.mean() <= TOL[dtype][1]


def _cache(slots, hkv, d, dtype=torch.bfloat16, max_len=600, page=16, chunk=64, **kw):
    from moba_hip import PagedKVCache
    return PagedKVCache(slots, max_len, hkv, d, page_size=page, chunk_size=chunk, dtype=dtype, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 64), (4, 1, 128)])
def test_cache_append_rotary(cuda_device, hq, hkv, d, dtype):
    from moba_hip import RotaryTable
    cache, table = _cache(4, hkv, d, dtype), RotaryTable(d, 800)
    counts = [130, 1, 70]
    n = sum(counts)
    k, v, q = (rand((n, h, d), dtype, s) for s, h in enumerate((hkv, hkv, hq)))
    cu = [0, 130, 131, 201]
    res = cache.append_rotary(k, v, table, sequence_ids=[2, 0, 3], cu_seqlens=cu, q=q,
                              offsets=[0, 17, 300])
    pos = [list(range(130)), [17], list(range(300, 370))]
    assert cache.lengths == (1, 0, 130, 70) and res.positions[:3] == (0, 1, 2)
    _near(res.q, _turned(q, table, sum(pos, [])), dtype)
    for i, slot in enumerate((2, 0, 3)):
        got_k, got_v = cache.materialize(slot)
        _near(got_k, _turned(k[cu[i]:cu[i + 1]], table, pos[i]), dtype)
        assert torch.equal(got_v, v[cu[i]:cu[i + 1]])
        closed = counts[i] // 64
        if closed:   # the means of closed chunks are those of the stored keys
            ref = O.decode_means(O.bits16(got_k), 0 if dtype == torch.bfloat16 else 1, 64)
            np.testing.assert_array_equal(O.bits16(cache._means[slot, :closed]), ref)
    # a second append goes on where the first ended
    more = cache.append_rotary(k[:3], v[:3], table, sequence_ids=[2], cu_seqlens=[0, 3])
    assert more.q is None and more.positions == (130, 131, 132)
    _near(cache.materialize(2)[0][130:], _turned(k[:3], table, [130, 131, 132]), dtype)


def test_attend_shared_against_copies_of_the_prefix(cuda_device):
    """The same attention as dense decode of sequences that each hold a copy
    of the prefix."""
    shared, copies = _cache(5, 2, 128), _cache(4, 2, 128)
    pk, pv = rand((300, 2, 128), torch.bfloat16, 1), rand((300, 2, 128), torch.bfloat16, 2)
    shared.append(pk, pv, sequence_ids=[4], cu_seqlens=[0, 300])
    for s, n in enumerate((1, 64, 90, 33)):
        k, v = rand((n, 2, 128), torch.bfloat16, 10 + s), rand((n, 2, 128), torch.bfloat16, 20 + s)
        shared.append(k, v, sequence_ids=[s], cu_seqlens=[0, n])
        head = (pk, pv) if s != 2 else (pk[:0], pv[:0])     # sequence 2 has no prefix
        copies.append(torch.cat((head[0], k)), torch.cat((head[1], v)), sequence_ids=[s],
                      cu_seqlens=[0, n + len(head[0])])
    q = rand((4, 12, 128), torch.bfloat16, 3)
    got = shared.attend_shared(q, sequence_ids=[0, 1, 2, 3], prefix_ids=[4, 4, -1, 4])
    want = copies.attend(q, sequence_ids=[0, 1, 2, 3], mode="dense")
    exact = _attended(shared, q, [(4, 0, 1), (4, 1, 64), (-1, 2, 90), (4, 3, 33)])
    _close(got.output, exact, torch.bfloat16)
    _close(want.output, exact, torch.bfloat16)
    assert (got.lse - want.lse).abs().max() <= 1e-4 and got.selected_blocks is None
    # rows of one sequence at positions of their own
    q = rand((3, 12, 128), torch.bfloat16, 4)
    got = shared.attend_shared(q, sequence_ids=[1, 1, 1], prefix_ids=[4] * 3, positions=[63, 5, 40])
    _close(got.output, _attended(shared, q, [(4, 1, 64), (4, 1, 6), (4, 1, 41)]), torch.bfloat16)


def _prefilled(dtype, rows, d=128, hq=6, hkv=2, prefix=200, page=16):
    from moba_hip import RotaryTable
    cache, table = _cache(rows + 1, hkv, d, dtype, page=page), RotaryTable(d, 1000)
    k, v = rand((prefix, hkv, d), dtype, 1), rand((prefix, hkv, d), dtype, 2)
    cache.append_rotary(k, v, table, sequence_ids=[rows], cu_seqlens=[0, prefix])
    return cache, table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 48])
def test_prepared_steps(cuda_device, dtype, page):
    """70 steps of 3 rows (pages and chunks begin and end among them), eager
    and replayed: the same bits, the cache's keys turned, every 20th step's
    output exact to the tolerance; the cache serves ordinary calls again after
    the lease."""
    runs = {}
    for graph in (False, True):
        cache, table = _prefilled(dtype, 3, page=page)
        outs = []
        ks, qs = [], []
        with cache.prepare_shared_decode([0, 1, 2], [3, 3, -1], 6, rotary=table, max_length=80) as plan:
            if graph:
                plan.capture()
            for t in range(70):
                q, k, v = (rand((3, h, 128), dtype, 100 * t + h + s) for s, h in enumerate((6, 2, 2)))
                res = plan.step(q, k, v, use_graph=graph)
                assert res.positions == (t, t, t)
                outs.append((res.output.clone(), res.lse.clone()))
                ks.append(k)
                qs.append(q)
                torch.randn(100, device="cuda").sum().item()   # eager work between replays
                if t % 20 == 0:
                    turned = torch.cat([_turned(q[:2], table, [200 + t] * 2), _turned(q[2:], table, [t])])
                    _close(res.output, _attended(cache, turned.to(dtype),
                                                 [(3, 0, t + 1), (3, 1, t + 1), (-1, 2, t + 1)]), dtype)
            assert cache.lengths == (70, 70, 70, 200)
        for row, base in ((0, 200), (2, 0)):
            _near(cache.materialize(row)[0], _turned(torch.stack([k[row] for k in ks]), table,
                                                     list(range(base, base + 70))), dtype)
        ref = O.decode_means(O.bits16(cache.materialize(1)[0]), 0 if dtype == torch.bfloat16 else 1, 64)
        np.testing.assert_array_equal(O.bits16(cache._means[1, :1]), ref)
        after = cache.attend_shared(qs[0], sequence_ids=[0, 1, 2], prefix_ids=[3, 3, -1])
        _close(after.output, _attended(cache, qs[0], [(3, 0, 70), (3, 1, 70), (-1, 2, 70)]), dtype)
        runs[graph] = outs
    for (a, la), (b, lb) in zip(runs[False], runs[True]):
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_prepared_without_rotation_matches_the_dense_step(cuda_device):
    """Inputs that are turned already: the step of PreparedDecode in dense
    mode on sequences without a prefix."""
    a, b = _cache(2, 2, 64), _cache(2, 2, 64)
    with a.prepare_shared_decode([0, 1], [-1, -1], 8) as x, b.prepare_decode([0, 1], 8, mode="dense") as y:
        for t in range(20):
            q, k, v = (rand((2, h, 64), torch.bfloat16, 10 * t + s) for s, h in enumerate((8, 2, 2)))
            got, want = x.step(q, k, v), y.step(q, k, v)
            assert (got.lse - want.lse).abs().max() <= 1e-4
            assert (got.output - want.output).abs().max() <= 2e-2
    for s in (0, 1):
        for u, w in zip(a.materialize(s), b.materialize(s)):
            assert torch.equal(u, w)


def test_refused_steps_change_nothing(cuda_device):
    from moba_hip import RotaryTable
    cache, _ = _prefilled(torch.bfloat16, 2)
    short = RotaryTable(128, 203)
    q, k, v = (rand((2, h, 128), torch.bfloat16, h) for h in (6, 2, 2))
    with cache.prepare_shared_decode([0, 1], [2, 2], 6, rotary=short) as plan:
        for _ in range(3):
            plan.step(q, k, v)
        before = cache.k_cache.view(torch.int16).clone()   # bits: unused cells may hold NaN
        with pytest.raises(ValueError, match="rotary table"):
            plan.step(q, k, v)
        with pytest.raises(ValueError, match="capture"):
            plan.step(q, k, v, use_graph=True)
        with pytest.raises(ValueError, match="fixed shape"):
            plan.step(q[:1], k, v)
        with pytest.raises(ValueError, match="no attend"):
            plan.attend(q)
        assert torch.equal(cache.k_cache.view(torch.int16), before) and cache.lengths == (3, 3, 200)
    with cache.prepare_shared_decode([0, 1], [2, 2], 6, rotary=RotaryTable(128, 999), max_length=4) as plan:
        plan.step(q, k, v)
        with pytest.raises(ValueError, match="max_length"):
            plan.step(q, k, v)
    assert cache.lengths == (4, 4, 200)


def test_cache_refusals(cuda_device):
    from moba_hip import RotaryTable
    cache, table = _prefilled(torch.bfloat16, 2)
    q, k, v = (rand((2, h, 128), torch.bfloat16, h) for h in (6, 2, 2))
    cache.append(k, v, sequence_ids=[0, 1])
    state = cache.k_cache.view(torch.int16).clone(), cache.lengths

    def bad(match, f):
        with pytest.raises(ValueError, match=match):
            f()
    app = dict(sequence_ids=[0, 1])
    bad("RotaryTable", lambda: cache.append_rotary(k, v, None, **app))
    bad("exceeds head_dim", lambda: cache.append_rotary(k, v, RotaryTable(256, 10), **app))
    bad("rotary table", lambda: cache.append_rotary(k, v, RotaryTable(128, 1), **app))
    bad("rotary table", lambda: cache.append_rotary(k, v, table, offsets=[0, 999], **app))
    bad("offset", lambda: cache.append_rotary(k, v, table, offsets=[0], **app))
    bad("offset", lambda: cache.append_rotary(k, v, table, offsets=[0, -1], **app))
    bad("q token count", lambda: cache.append_rotary(k, v, table, q=q[:1], **app))
    bad("NaN/Inf", lambda: cache.append_rotary(k * float("nan"), v, table, **app))
    bad("alias", lambda: cache.append_rotary(cache.k_cache[0, :2], v, table, **app))
    att = dict(sequence_ids=[0, 1])
    bad("one prefix ID", lambda: cache.attend_shared(q, prefix_ids=[2], **att))
    bad("as well", lambda: cache.attend_shared(q, prefix_ids=[2, 0], **att))
    bad("range|ID", lambda: cache.attend_shared(q, prefix_ids=[2, 7], **att))
    bad("cached tokens", lambda: cache.attend_shared(q, prefix_ids=[2, 2], positions=[0, 1], **att))
    bad("scale", lambda: cache.attend_shared(q, prefix_ids=[2, 2], scale=-1.0, **att))
    bad("multiple of Hkv", lambda: cache.attend_shared(q[:, :5], prefix_ids=[2, 2], **att))
    bad("max_length", lambda: cache.prepare_shared_decode([0], [2], 6, max_length=601))
    bad("as well", lambda: cache.prepare_shared_decode([0, 2], [2, -1], 6))
    assert torch.equal(cache.k_cache.view(torch.int16), state[0]) and cache.lengths == state[1]
    odd = _cache(2, 1, 20)
    odd.append(*(rand((1, 1, 20), torch.bfloat16, s) for s in (1, 2)), sequence_ids=[0])
    bad("multiple of 8", lambda: odd.attend_shared(rand((1, 2, 20), torch.bfloat16, 3),
                                                   sequence_ids=[0], prefix_ids=[-1]))
    with cache.prepare_shared_decode([0, 1], [2, 2], 6, rotary=table):
        bad("owns cache", lambda: cache.attend_shared(q, prefix_ids=[2, 2], **att))
        bad("owns cache", lambda: cache.append_rotary(k, v, table, **app))


def _model(seed=0):
    from transformers import Qwen2Config, Qwen2ForCausalLM
    torch.manual_seed(seed)
    cfg = Qwen2Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=4096,
                      attn_implementation="eager")
    m = Qwen2ForCausalLM(cfg).to("cuda", torch.bfloat16).eval()
    for p in m.parameters():
        p.requires_grad_(False)
    return m


def test_qwen2_branches(cuda_device):
    """Three continuations of one prompt against the transformers model on
    each full sequence; graph replays equal eager steps bit for bit."""
    from moba_hip.qwen2 import Qwen2Branches
    model = _model()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 512, (1, 150), generator=g).to("cuda")
    extra = torch.randint(0, 512, (20, 3), generator=g).tolist()
    logits = {}
    for backend in ("eager", "model_graph"):
        with Qwen2Branches(model, 160, 3, 24, chunk=64, backend=backend) as s:
            out = [s.prefill(ids)]
            s.prepare()
            for t in extra:
                out.append(s.step(t).clone())
                torch.randn(100, device="cuda").sum().item()
            with pytest.raises(ValueError):
                s.step([0, 0])
            logits[backend] = out
    for a, b in zip(*logits.values()):
        assert torch.equal(a, b)
    for b in range(3):
        full = torch.cat([ids, torch.tensor([[t[b] for t in extra]], device="cuda")], 1)
        with torch.no_grad():
            ref = model(full).logits[0].float()
        for i, got in enumerate(logits["eager"]):
            x, y = got[b if i else 0].float(), ref[149 + i]
            assert torch.nn.functional.cosine_similarity(x, y, dim=0) > 0.999, (b, i)
            assert (x - y).abs().max() < 0.05 * y.abs().max(), (b, i)
