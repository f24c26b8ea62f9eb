"""Calls of the paged-cache operators beside the ordinary ones: replaced tables
and plans, failures inside a step, and the kernels that only far pools, unmapped
pages or long lookups reach."""
import math

import numpy as np
import pytest
import torch

from test_paged_contract import RECORDS, REPLACED, SCALES, qwen2_model
from test_rotary_append_gpu import SENTINEL, _case, _run
from test_shared_prefix_gpu import _pool

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


def test_a_failed_capture_leaves_the_lease(cuda_device, monkeypatch):
    """Nothing runs in a capture: the lease goes on, and can be captured later."""
    from moba_hip import PagedKVCache
    cache = PagedKVCache(2, 64, 2, 64, chunk_size=32)
    q, k, v = (torch.randn(2, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    with cache.prepare_shared_decode([0, 1], [-1, -1], 4) as plan:
        calls, plan._calls = plan._calls, [("moba_hip_no_such_entry", ())]
        with pytest.raises(Exception):
            plan.capture()
        plan._calls = calls
        a = plan.step(q, k, v).output.clone()
        plan.capture()
        b = plan.step(q, k, v, use_graph=True).output.clone()
    assert cache.lengths == (2, 2)
    # the second token's key and value are the first's: the same average
    assert torch.equal(a, b)


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
