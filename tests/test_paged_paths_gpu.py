"""Calls of the paged-cache operators beside the ordinary ones: replaced tables
and plans, failures inside a step, and the kernels that only far pools, unmapped
pages or long lookups reach."""
import math

import numpy as np
import pytest
import torch

from test_paged_contract import RECORDS, REPLACED, SCALES, qwen2_model
from test_rotary_append_gpu import SENTINEL, _case, _run
from test_shared_prefix_gpu import _exact, _pool
from test_shared_prefix_gpu import _run as _attend

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- rotary tables
@pytest.mark.parametrize("how", REPLACED)
@pytest.mark.parametrize("check", [False, True])
def test_append_refuses_a_replaced_table(cuda_device, how, check):
    st = _case([4, 9], 4, 2, 64, 64, 16, torch.bfloat16)
    st["rotary"].cos_sin = REPLACED[how](st["rotary"].cos_sin)
    with pytest.raises(ValueError, match="cos_sin must be"):
        _run(st, check=check)
    torch.cuda.synchronize()
    assert (st["k_cache"] == SENTINEL).all() and (st["v_cache"] == SENTINEL).all()


def test_append_uses_the_rows_a_replaced_table_has(cuda_device):
    """A shorter table: tokens past its end are dropped as past any table's."""
    st = _case([9], 4, 2, 64, 64, 16, torch.bfloat16, context=[0])
    whole = _run(st)
    st["rotary"].cos_sin = st["rotary"].cos_sin[:5]
    st["k_cache"].fill_(SENTINEL)
    out = torch.full_like(whole, SENTINEL)
    _run(st, q_out=out)
    assert torch.equal(out[:5], whole[:5]) and (out[5:] == SENTINEL).all()
    with pytest.raises(RuntimeError, match="rotary table"):
        _run(st, check=True)


@pytest.mark.parametrize("how", REPLACED)
def test_cache_and_lease_refuse_a_replaced_table(cuda_device, how):
    from moba_hip import PagedKVCache, RotaryTable
    cache, table = PagedKVCache(2, 64, 2, 64, chunk_size=32), RotaryTable(64, 100)
    table.cos_sin = REPLACED[how](table.cos_sin)
    k = torch.randn(3, 2, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="cos_sin must be"):
        cache.append_rotary(k, k, table, sequence_ids=[0], cu_seqlens=[0, 3])
    with pytest.raises(ValueError, match="cos_sin must be"):
        cache.prepare_shared_decode([0], [-1], 4, rotary=table)
    assert cache.lengths == (0, 0)


def test_lease_keeps_the_table_it_was_made_with(cuda_device):
    """The launches hold the address of the angles: replacing the attribute
    later changes nothing of them."""
    from moba_hip import PagedKVCache, RotaryTable
    outs = []
    for replace in (False, True):
        cache, table = PagedKVCache(2, 64, 2, 64, chunk_size=32), RotaryTable(64, 100)
        with cache.prepare_shared_decode([0, 1], [-1, -1], 4, rotary=table) as plan:
            if replace:
                table.cos_sin = None
                torch.cuda.empty_cache()
                junk = [torch.full((100, 32, 2), 9.0, device="cuda") for _ in range(8)]
            for t in range(3):
                g = torch.Generator().manual_seed(t)
                q, k, v = (torch.randn(2, h, 64, generator=g).to("cuda", torch.bfloat16) for h in (4, 2, 2))
                out = plan.step(q, k, v).output.clone()
            torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(*outs) and len(junk) == 8


# ------------------------------------------------------------------ the plan
@pytest.mark.parametrize("how", [*RECORDS, "host"])
@pytest.mark.parametrize("given", [False, True])
def test_attention_refuses_replaced_records(cuda_device, how, given):
    """Without outputs of the caller's (the native entry's calls) and with them."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([100, 5], 2, 64, 16, torch.bfloat16, 2)
    plan = SharedPrefixPlan([0], [100], [1], 4, 2, 64, max_suffix=5)
    plan.meta = plan.meta.cpu() if how == "host" else RECORDS[how](plan.meta)
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    own = torch.tensor([5], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="the plan on it" if how == "host" else "plan.meta must be"):
        shared_prefix_attention(q, kc, vc, table, own, plan, out=torch.empty_like(q) if given else None)


@pytest.mark.parametrize("scale", [*SCALES, 2e30, 2])
def test_scales(cuda_device, scale):
    """Refused in one way by calls with and without an output of the caller's;
    a whole number is a scale."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([100, 5], 2, 64, 16, torch.bfloat16, 2)
    plan = SharedPrefixPlan([0], [100], [1], 4, 2, 64, max_suffix=5)
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    own = torch.tensor([5], dtype=torch.int32, device="cuda")
    for out in (None, torch.empty_like(q)):
        def call(scale):
            return shared_prefix_attention(q, kc, vc, table, own, plan, scale=scale, out=out)
        if scale == 2:
            assert torch.equal(call(2)[0].clone(), call(2.0)[0])
        else:
            with pytest.raises(ValueError, match="scale must be"):
                call(scale)


def test_smallest_scale_with_masked_tiles(cuda_device):
    """All scores near 0: the mean of the attended values, whatever is masked."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, vs = _pool([100, 70], 1, 64, 16, torch.bfloat16, 2)
    plan = SharedPrefixPlan([-1] * 3, [0] * 3, [1] * 3, 2, 1, 64, max_suffix=70)
    q = torch.randn(3, 2, 64, device="cuda").bfloat16()
    own = torch.tensor([1, 70, 0], dtype=torch.int32, device="cuda")
    out, lse = shared_prefix_attention(q, kc, vc, table, own, plan, scale=2.0 ** -126)
    assert torch.equal(out[0], vs[1][0].cuda().expand(2, 64)) and (out[2] == 0).all()
    mean = vs[1].double().mean(0)
    # weights of 1 exactly; sums of 70 terms in fp32, one rounding
    tol = 2.0 ** -8 * mean.abs() + 70 * 2.0 ** -24 * vs[1].double().abs().mean(0) + 2.0 ** -20
    assert ((out[1].double().cpu() - mean).abs() <= tol).all()
    assert (lse[1] - math.log(70)).abs().max() < 1e-5 and (lse[2] == float("-inf")).all()


# ------------------------------------------------------ failures inside a step
def test_a_failed_replay_ends_the_lease(cuda_device):
    from moba_hip import PagedKVCache
    cache = PagedKVCache(2, 64, 2, 64, chunk_size=32)
    q, k, v = (torch.randn(2, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    plan = cache.prepare_shared_decode([0, 1], [-1, -1], 4)
    plan.capture()
    plan.step(q, k, v, use_graph=True)

    class Broken:
        def replay(self):
            raise RuntimeError("replay")
    plan._graph = Broken()
    with pytest.raises(RuntimeError, match="replay"):
        plan.step(q, k, v, use_graph=True)
    with pytest.raises(RuntimeError, match="discard prepared decode"):
        plan.step(q, k, v)
    plan.close()
    with pytest.raises(RuntimeError, match="discard this cache"):
        cache.attend_shared(q, sequence_ids=[0, 1], prefix_ids=[-1, -1])


def test_page_grants_are_uploaded_when_a_page_begins(cuda_device):
    """delta_uploads counts as PreparedDecode's does: rows of 0 and 5 tokens on
    pages of 16, 40 steps."""
    from moba_hip import PagedKVCache
    counts = []
    for shared in (False, True):
        cache = PagedKVCache(2, 64, 2, 64, page_size=16, chunk_size=32)
        k = torch.randn(5, 2, 64, device="cuda").bfloat16()
        cache.append(k, k, sequence_ids=[1], cu_seqlens=[0, 5])
        q, k, v = (torch.randn(2, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
        with (cache.prepare_shared_decode([0, 1], [-1, -1], 4) if shared else
              cache.prepare_decode([0, 1], 4, mode="dense")) as plan:
            assert plan.delta_uploads == 0
            seen = []
            for _ in range(40):
                plan.step(q, k, v)
                seen.append(plan.delta_uploads)
            counts.append(seen)
    assert counts[0] == counts[1]
    assert counts[1][0] == 1 and counts[1][-1] == 5   # at tokens 0, 16, 32 and 16, 32 of the rows


@pytest.mark.parametrize("graph", [False, True])
def test_rows_that_begin_their_pages_at_steps_of_their_own(cuda_device, graph):
    """Rows of 0, 5, 16 and 31 tokens behind prefixes of 40, 0 and 77: the grant of
    one row's page is replayed with the steps after it and changes no other row's.
    Outputs against 64 bits over what the cache holds, within half a bf16 step of
    the weights' sum and of the result, and fp32's 2^-12 of it."""
    from moba_hip import PagedKVCache, RotaryTable
    hq, hkv, d, starts = 4, 2, 64, (0, 5, 16, 31)
    cache, rt = PagedKVCache(7, 160, hkv, d, page_size=16, chunk_size=32), RotaryTable(d, 300)
    g = torch.Generator().manual_seed(3)

    def rand(*shape):
        return torch.randn(*shape, generator=g).to("cuda", torch.bfloat16)
    for slot, n in [(4, 40), (6, 77), *((i, n) for i, n in enumerate(starts) if n)]:
        cache.append_rotary(rand(n, hkv, d), rand(n, hkv, d), rt, sequence_ids=[slot], cu_seqlens=[0, n])
    prefix = [4, -1, 6, 6]
    with cache.prepare_shared_decode([0, 1, 2, 3], prefix, hq, rotary=rt, max_length=100) as plan:
        if graph:
            plan.capture()
        for t in range(45):
            q, k, v = rand(4, hq, d), rand(4, hkv, d), rand(4, hkv, d)
            res = plan.step(q, k, v, use_graph=graph)
            assert res.positions == tuple(n + t for n in starts)
            if t % 4:
                continue
            for r, own in enumerate(starts):
                ks, vs = zip(*(cache.materialize(s) for s in ([prefix[r]] if prefix[r] >= 0 else []) + [r]))
                kk, vv = (torch.cat(x).double().repeat_interleave(hq // hkv, 1) for x in (ks, vs))
                assert len(kk) == own + t + 1 + (cache.lengths[prefix[r]] if prefix[r] >= 0 else 0)
                x = plan._turned[r].double()
                p = torch.softmax((x * kk).sum(-1) * d ** -0.5, 0)[..., None]
                want, A = (p * vv).sum(0), (p * vv.abs()).sum(0)
                tol = 2.0 ** -8 * (A + want.abs()) * (1 + 2.0 ** -6) + 2.0 ** -12 * A
                assert ((res.output[r].double() - want).abs() <= tol).all(), (t, r)
    assert cache.lengths[:4] == tuple(n + 45 for n in starts)


def test_a_failed_capture_leaves_the_lease(cuda_device, monkeypatch):
    """Nothing runs in a capture: the lease goes on, and can be captured later."""
    from moba_hip import PagedKVCache
    cache = PagedKVCache(2, 64, 2, 64, chunk_size=32)
    q, k, v = (torch.randn(2, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    with cache.prepare_shared_decode([0, 1], [-1, -1], 4) as plan:
        calls = plan._calls
        plan._calls = [calls[0], ("moba_hip_no_such_entry", ())]
        with pytest.raises(Exception):
            plan.capture()
        plan._calls = calls
        a = plan.step(q, k, v).output.clone()
        plan.capture()
        b = plan.step(q, k, v, use_graph=True).output.clone()
    assert cache.lengths == (2, 2)
    # the second token's key and value are the first's: the same average
    assert torch.equal(a, b)


# ------------------------------------------- every kernel against 64 bits
@pytest.fixture(scope="module")
def far_memory(cuda_device):
    """Room for a K and a V pool of more than 4 GiB (and 2^31 elements) each."""
    flat = [torch.empty(2400 << 20, dtype=torch.int16, device="cuda") for _ in range(2)]
    yield flat
    flat.clear()
    torch.cuda.empty_cache()


def _laid_out(lengths, holes, hkv, d, page, dtype, far, seed):
    """Pools and table of sequences, whose logical pages `holes` (slot, page) are
    unmapped; (k_cache, v_cache, table, cells, ks, vs): tensors of the mapped
    tokens alone, and their cells.  Cells of no token hold NaN."""
    g = torch.Generator().manual_seed(seed)
    width = max(-(-n // page) for n in lengths) + 1
    need = sum(-(-n // page) for n in lengths) + 2
    if far is None:
        pages = need
        kc, vc = (torch.empty((pages, page, hkv, d), dtype=dtype, device="cuda") for _ in range(2))
        ids = torch.randperm(pages, generator=g).tolist()
    else:   # over the whole of the pool, its first and last pages among them
        pages = far[0].numel() // (page * hkv * d)
        kc, vc = (t[:pages * page * hkv * d].view(dtype).view(pages, page, hkv, d) for t in far)
        assert kc.numel() * 2 > 2 ** 32
        ids = torch.linspace(0, pages - 1, need, dtype=torch.float64).long()
        ids = ids[torch.randperm(need, generator=g)].tolist()
    used = torch.tensor(ids, device="cuda")
    kc[used], vc[used] = float("nan"), float("nan")
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at, cells, ks, vs = 0, [], [], []
    for slot, n in enumerate(lengths):
        for lp in range(-(-n // page)):
            if (slot, lp) not in holes:
                table[slot, lp] = ids[at]
            elif lp % 2:
                table[slot, lp] = pages + 5     # no page of the pool either
            at += 1
        i = torch.tensor([t for t in range(n) if (slot, t // page) not in holes], dtype=torch.long)
        cell = (table[slot].long()[i // page] * page + i % page).cuda()
        k, v = (torch.randn(len(i), hkv, d, generator=g).to("cuda", dtype) for _ in range(2))
        kc.view(-1, hkv, d)[cell], vc.view(-1, hkv, d)[cell] = k, v
        cells.append(cell), ks.append(k), vs.append(v)
    return kc, vc, table.cuda(), cells, ks, vs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [40, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("form,rows", [("wide", 20), ("narrow", 6), ("solo", 6)])
@pytest.mark.parametrize("slots", ["each", "one"])
@pytest.mark.parametrize("where", ["near", "far"])
def test_every_kernel_against_64_bits(far_memory, monkeypatch, where, slots, form, rows, d, dtype):
    """Items of four waves with 32 pairs each, of four with the same pairs and of
    single waves, each with more keys than one lookup holds (1024, 256) and
    unmapped pages among them; rows with an own slot each, and all with one at
    lengths of their own; pools below and above 4 GiB.

    Allowed, with A = sum_j p_j |v_j| / z: half a step of A for the weights and
    of the result; scores and their scale 2 (D + 4) 2^-24 S of A, S the largest
    sum of |q_d k_d| scale; 2^-15 of A for fp32 sums of at most 3800 / 16 + 16 < 2^8
    additions in numerator and z; in fp16 2^-32 of the largest weight for weights
    and 2^-25 for results below the normal ones.  Values that are not finite then go
    in at two tokens of the one slot, and reach the rows that attend them."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    monkeypatch.setattr(SharedPrefixPlan, "_ranges",
                        lambda self, blocks, *a: (np.full(len(blocks), 1), form == "solo"))
    hq, hkv, page, plen = 4, 2, 64 if where == "far" else 16, 2500
    own = [[1300, 700, 1, 1201, 64, 1025, 0, 1024, 701, 1100][i % 10] for i in range(rows)]
    suffix = [1 + i if slots == "each" else 1 for i in range(rows)]
    lengths = [plen] + (own if slots == "each" else [1300])
    holes = {(0, 3), (0, 1100 // page), (1, 2)}
    kc, vc, table, cells, ks, vs = _laid_out(lengths, holes, hkv, d, page, dtype,
                                             far_memory if where == "far" else None, d + rows)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(rows, hq, d, generator=g).to("cuda", dtype)
    plan = SharedPrefixPlan([0] * rows, [plen] * rows, suffix, hq, hkv, d, max_suffix=1300)
    dev_own = torch.tensor(own, dtype=torch.int32, device="cuda")
    out, lse = shared_prefix_attention(q, kc, vc, table, dev_own, plan)

    mapped = [sum((s, t // page) not in holes for t in range(n)) for s, n in zip(suffix, own)]
    want, wl, A, S, V = [t.cuda() for t in _exact(q, ks, vs, [0] * rows, [len(ks[0])] * rows, suffix,
                                                  mapped, d ** -0.5)]
    eps = torch.finfo(dtype).eps
    rel = 2 * (d + 4) * 2.0 ** -24 * S + 2.0 ** -15
    tol = eps / 2 * (A + want.abs()) * (1 + 2.0 ** -6) + rel[..., None] * A
    if dtype == torch.float16:
        tol = tol + 2.0 ** -32 * V + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()
    assert ((lse.double() - wl).abs() <= rel + 2.0 ** -22 * wl.abs()).all()

    if slots == "one":
        inf, nan = float("inf"), float("nan")
        before = sum((1, t // page) not in holes for t in range(700))
        later = sum((1, t // page) not in holes for t in range(1200))
        flat = vc.view(-1, hkv, d)
        flat[cells[1][before], 0, :2] = torch.tensor([-inf, inf], dtype=dtype, device="cuda")
        flat[cells[1][later], 0, :3] = torch.tensor([inf, inf, nan], dtype=dtype, device="cuda")
        odd, odd_lse = shared_prefix_attention(q, kc, vc, table, dev_own, plan)
        want = out.clone()
        for i, n in enumerate(own):
            if n > 700:    # the heads of kv head 0
                want[i, :2, :2] = torch.tensor([-inf, inf], dtype=dtype, device="cuda")
            if n > 1200:   # -inf and inf; inf twice; NaN
                want[i, :2, :3] = torch.tensor([nan, inf, nan], dtype=dtype, device="cuda")
        assert torch.equal(odd_lse, lse)
        assert torch.equal(torch.nan_to_num(odd, nan=123.0), torch.nan_to_num(want, nan=123.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,d", [(513, 64), (300, 256)])
def test_long_extension_of_one_sequence(cuda_device, tokens, d, dtype):
    """Several hundred new tokens behind a prefix: blocks of one sequence's rows
    whose lengths end in tiles of their own."""
    n = tokens + 150
    _attend([200, n], [0] * tokens, [200] * tokens, [1] * tokens, list(range(n - tokens + 1, n + 1)),
            2, 1, d, 16, dtype)


# ------------------------------------------------------ small weights in fp16
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("nats", [12.0, 17.0, 17.5, 19.0])
@pytest.mark.parametrize("rows,d", [(1, 64), (1, 128), (1, 256), (40, 64), (40, 128), (40, 256)])
def test_flat_tail_behind_one_strong_key_in_fp16(cuda_device, monkeypatch, rows, d, nats, first):
    """One key of a value of 0 and 16000 keys `nats` below it of values of 1, in
    one range: the output is the tail's share.  first: the strong key comes
    before the others; else behind them, when the tail's sums are scaled down.

    A weight lies in fp16 relative to its wave's largest, which is at least 2^7
    there (at most 2^15), so that it is off by at most half a step, 2^-11 of
    itself, or below 2^-14 by 2^-25: 2^-32 of the largest weight.  Numerator and z
    are fp32 sums of positive terms: a lane adds to them at most 16001 / 16 + 16 <
    2^10 times, each off by at most 2^-24 of the sum (equal terms round alike, so
    that these add up), 2^-14 in all for each.  The result is rounded by 2^-11 of
    itself or 2^-25.  Scores are sums of exact products; scaled they are below 2^5,
    off by 2^-19 at most, 2^-18 of a weight."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    monkeypatch.setattr(SharedPrefixPlan, "_ranges",
                        lambda self, blocks, *a: (np.full(len(blocks), 1), False))
    n, page = 16001, 64
    pages = -(-n // page)
    kc = torch.zeros((pages, page, 1, d), dtype=torch.float16)
    vc = torch.ones_like(kc)
    at = 0 if first else n - 1
    kc.view(-1, d)[at, 0], vc.view(-1, d)[at] = nats, 0.0
    q = torch.zeros((rows, 1, d), dtype=torch.float16)
    q[..., 0] = 1.0
    table = torch.arange(pages, dtype=torch.int32)[None].cuda()
    plan = SharedPrefixPlan([0] * rows, [n] * rows, [-1] * rows, 1, 1, d, max_suffix=0)
    own = torch.zeros(rows, dtype=torch.int32, device="cuda")
    out, lse = shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), table, own, plan, scale=1.0)
    tail = (n - 1) * math.exp(-nats)           # relative to the strong key
    share = tail / (1 + tail)
    allowed = (2.0 ** -10 + 2.0 ** -13 + 2.0 ** -17) * share + 2.0 ** -25 + (n - 1) * 2.0 ** -32 / (1 + tail)
    assert (out.double().cpu() - share).abs().max() <= allowed
    want = nats + math.log1p(tail)
    assert (lse.double().cpu() - want).abs().max() <= 2.0 ** -14 + 2.0 ** -18 + 2.0 ** -22 * want


# -------------------------------------------------------------- Qwen2 session
@pytest.mark.parametrize("rope", ["linear", "yarn", "llama3"])
def test_branches_of_models_with_fixed_frequencies(cuda_device, rope):
    """Angles, and the attention factor of yarn, past the original length."""
    from moba_hip.qwen2 import Qwen2Branches
    model = qwen2_model(rope, "cuda")
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 256, (1, 300), generator=g).to("cuda")
    extra = torch.randint(0, 256, (6, 2), generator=g).tolist()
    with Qwen2Branches(model, 300, 2, 8, chunk=64) as s:
        out = [s.prefill(ids)]
        s.prepare()
        out += [s.step(t).clone() for t in extra]
    for b in range(2):
        full = torch.cat([ids, torch.tensor([[t[b] for t in extra]], device="cuda")], 1)
        with torch.no_grad():
            ref = model(full).logits[0].float()
        for i, got in enumerate(out):
            x, y = got[b if i else 0].float(), ref[299 + i]
            assert torch.nn.functional.cosine_similarity(x, y, dim=0) > 0.999, (b, i)


def test_branches_prepared_again_after_a_failure(cuda_device, monkeypatch):
    """A capture that fails in the second layer's launches, then one that holds:
    the steps are those of a session that never failed."""
    from moba_hip.qwen2 import Qwen2Branches
    model = qwen2_model("default", "cuda")
    ids = torch.randint(0, 256, (1, 100), generator=torch.Generator().manual_seed(2)).to("cuda")
    outs = []
    for failing in (False, True):
        with Qwen2Branches(model, 100, 2, 8, chunk=64, backend="model_graph") as s:
            s.prefill(ids)
            if failing:
                with monkeypatch.context() as m:
                    def broken(self, stream):
                        if self is s.plans[1]:
                            raise RuntimeError("launch")
                        launch(self, stream)
                    from moba_hip import PreparedSharedDecode
                    launch = PreparedSharedDecode._launch_step
                    m.setattr(PreparedSharedDecode, "_launch_step", broken)
                    with pytest.raises(RuntimeError):
                        s.prepare()
                assert not s.plans and s.graph is None
            s.prepare()
            outs.append([s.step([3 + i, 7 * i]).clone() for i in range(4)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
