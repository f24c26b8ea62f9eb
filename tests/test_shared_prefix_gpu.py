"""Shared-prefix attention (moba_hip.shared_prefix_attention) against the
softmax in 64 bits, row by row.

Allowed error of an output element, with A = sum_j p_j |v_j| / z:
* weights are rounded to the 16-bit type before the product with V: half a
  step, eps/2 * A (fp16 weights below 2^-14 of a range's largest: 2^-25 each);
* scores carry the fp32 sum of D exact products and their scaling, at most
  (D + 4) 2^-24 S with S the largest sum of |q_d k_d| * scale, a relative
  error of the weights, in numerator and denominator; exp2 and the sums of
  fp32 add 2^-20 (the sums run over at most 2^12 terms per lane, with errors
  of 2^-24 each that add up as their root in practice and 2^-12 at worst: the
  test's sums are below 2^4 terms per step of that bound);
* the result is rounded once: eps/2 * |out|."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pool(lengths, hkv, d, page, dtype, seed, spare=3):
    """Page pool whose cells outside the sequences hold NaN."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    width = max(1, max(counts)) + 1
    pages = sum(counts) + spare
    perm = torch.randperm(pages, generator=g).tolist()
    kc, vc = (torch.full((pages, page, hkv, d), float("nan"), dtype=dtype) for _ in range(2))
    table, at, ks, vs = [], 0, [], []
    for n, c in zip(lengths, counts):
        own = perm[at:at + c]
        at += c
        table.append(own + [-1] * (width - c))
        k, v = (torch.randn(n, hkv, d, generator=g).to(dtype) for _ in range(2))
        cell = torch.tensor([own[i // page] * page + i % page for i in range(n)], dtype=torch.long)
        kc.view(-1, hkv, d)[cell], vc.view(-1, hkv, d)[cell] = k, v
        ks.append(k)
        vs.append(v)
    return (kc.cuda(), vc.cuda(), torch.tensor(table, dtype=torch.int32, device="cuda"), ks, vs)


def _exact(q, ks, vs, prefix, length, suffix, own, scale):
    """(out, lse, A, S, sum |v| / z) of every row in 64 bits."""
    res = []
    for r in range(q.shape[0]):
        pk = ks[prefix[r]][:length[r]] if length[r] else ks[0][:0]
        pv = vs[prefix[r]][:length[r]] if length[r] else vs[0][:0]
        sk = ks[suffix[r]][:own[r]] if suffix[r] >= 0 else ks[0][:0]
        sv = vs[suffix[r]][:own[r]] if suffix[r] >= 0 else vs[0][:0]
        k, v = torch.cat((pk, sk)).double(), torch.cat((pv, sv)).double()
        hq, d = q.shape[1:]
        g = hq // k.shape[1]
        k, v = (x.repeat_interleave(g, dim=1).transpose(0, 1) for x in (k, v))
        x = q[r].double()[:, None]
        if not k.shape[1]:
            zero = torch.zeros(hq, d, dtype=torch.float64)
            res.append((zero, torch.full((hq,), float("-inf"), dtype=torch.float64), zero,
                        torch.zeros(hq, dtype=torch.float64), zero))
            continue
        s = (x * k).sum(-1) * scale
        S = ((x * k).abs().sum(-1) * scale).amax(-1)
        p = torch.softmax(s, -1)[..., None]
        z = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1)
        res.append(((p * v).sum(1), torch.logsumexp(s, -1), (p * v.abs()).sum(1), S,
                    v.abs().sum(1) / z[:, None]))
    return [torch.stack(t) for t in zip(*res)]


def _compare(out, lse, q, ks, vs, prefix, length, suffix, own, scale):
    want, wl, A, S, V = _exact(q.cpu(), ks, vs, prefix, length, suffix, own, scale)
    eps, d = torch.finfo(q.dtype).eps, q.shape[2]
    rel = 2 * (d + 4) * 2.0 ** -24 * S + 2.0 ** -20
    tol = eps / 2 * (A + want.abs()) * (1 + 2.0 ** -6) + rel[..., None] * A
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (V + 1)
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), f"out off by up to {(err / tol.clamp_min(1e-30)).max():.2f} of the allowed error"
    dead = torch.isinf(wl)
    got = lse.cpu().double()
    assert torch.equal(torch.isinf(got), dead) and (out.cpu()[dead] == 0).all()
    ltol = rel + 2.0 ** -22 * wl.abs()
    assert ((got - wl).abs() <= ltol)[~dead].all()


def _run(lengths, prefix, plen, suffix, own, hq, hkv, d, page, dtype, *, scale=None, max_suffix=None,
         seed=0, qscale=1.0):
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, ks, vs = _pool(lengths, hkv, d, page, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(len(prefix), hq, d, generator=g) * qscale).to("cuda", dtype)
    bound = max(own) if max_suffix is None else max_suffix
    plan = SharedPrefixPlan(prefix, plen, suffix, hq, hkv, d, max_suffix=bound)
    dl = torch.tensor(own, dtype=torch.int32, device="cuda")
    out, lse = shared_prefix_attention(q, kc, vc, table, dl, plan, scale=scale)
    again = shared_prefix_attention(q, kc, vc, table, dl, plan, scale=scale)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    own = [max(0, min(n, bound)) for n in own]
    _compare(out, lse, q, ks, vs, prefix, plen, suffix, own, scale or d ** -0.5)
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (16, 1, 96), (14, 2, 64), (8, 8, 64), (6, 3, 40),
                                      (4, 1, 256), (2, 2, 192), (4, 2, 8), (3, 1, 72), (48, 1, 128)])
def test_heads_and_types(cuda_device, hq, hkv, d, dtype):
    own = [1, 30, 64, 100, 7]
    _run([333] + own, [0] * 5, [333] * 5, [1, 2, 3, 4, 5], own, hq, hkv, d, 16, dtype, seed=d)


@pytest.mark.parametrize("page", [1, 3, 16, 48, 500])
@pytest.mark.parametrize("plen", [1, 31, 32, 33, 64, 65, 257, 1500])
def test_prefix_lengths_and_pages(cuda_device, plen, page):
    own = [1, 0, 129]
    _run([plen] + own, [0] * 3, [plen] * 3, [1, 2, 3], own, 4, 2, 128, page, torch.bfloat16, seed=plen)


@pytest.mark.parametrize("rows", [1, 2, 11, 43, 130])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_row_counts(cuda_device, rows, d):
    own = [(17 * i) % 90 for i in range(rows)]
    _run([700] + own, [0] * rows, [700] * rows, list(range(1, rows + 1)), own, 6, 2, d, 16,
         torch.bfloat16, seed=rows)


@pytest.mark.parametrize("solo", [False, True])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 8, 64, torch.bfloat16), (32, 4, 128, torch.float16),
                                            (40, 1, 96, torch.bfloat16), (6, 3, 40, torch.float16),
                                            (4, 2, 256, torch.bfloat16), (3, 1, 192, torch.bfloat16)])
def test_ways_to_cut_the_work(cuda_device, monkeypatch, hq, hkv, d, dtype, splits, solo):
    """Own tokens by whole workgroups and by single waves, in one and several
    ranges, with own lengths from none to more than a lookup's 256 and 1024."""
    from moba_hip.shared_prefix import SharedPrefixPlan
    monkeypatch.setattr(SharedPrefixPlan, "_ranges",
                        lambda self, blocks, *a: (np.full(len(blocks), splits), solo))
    own = [0, 1, 15, 16, 17, 255, 257, 1, 1100, 64, 300]
    n = len(own)
    _run([500] + own, [0] * n, [500] * n, list(range(1, n + 1)), own, hq, hkv, d, 16, dtype,
         seed=d + splits)


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 4, 128), (48, 1, 80)])
def test_many_short_sequences(cuda_device, hq, hkv, d):
    own = [(7 * i) % 23 for i in range(300)]
    _run([70] + own, [0] * 300, [70] * 300, list(range(1, 301)), own, hq, hkv, d, 16, torch.bfloat16)


def test_groups_of_unlike_prefixes_and_rows_of_nothing(cuda_device):
    """Rows in mixed order: two prefixes, one of them at two lengths, rows
    without a prefix, without own tokens, and without either."""
    lengths = [400, 90, 33, 70, 1, 200]
    prefix = [0, 1, -1, 0, 1, 0, -1, -1, 0]
    plen = [400, 90, 0, 100, 90, 400, 0, 0, 100]
    suffix = [2, 3, 4, -1, 5, 2, -1, 5, 3]
    own = [33, 70, 1, 9, 0, 20, 5, 200, 64]
    out, lse = _run(lengths, prefix, plen, suffix, own, 8, 2, 64, 16, torch.float16)
    assert (out[6] == 0).all() and torch.isinf(lse[6]).all()


def test_several_query_tokens_of_a_sequence(cuda_device):
    """A causal block of 50 tokens of each of three sequences, in scattered
    order."""
    n = [50, 80, 131]
    rows = [(s, t) for t in range(50) for s in (2, 0, 1)]
    _run([600] + n, [0] * 150, [600] * 150, [1 + s for s, _ in rows],
         [n[s] - 49 + t for s, t in rows], 4, 1, 128, 16, torch.bfloat16)


def test_own_lengths_are_cut_to_the_bound(cuda_device):
    _run([90, 300, 300], [0, 0], [90, 90], [1, 2], [300, -4], 4, 2, 64, 16, torch.bfloat16,
         max_suffix=130)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_prefix_and_sharp_scores(cuda_device, dtype):
    """Many ranges; scores of deviation 6, whose largest arrive late and early."""
    _run([9001, 2], [0] * 3, [9001] * 3, [1, 1, 1], [2, 1, 0], 2, 1, 64, 48, dtype, qscale=6.0)


def test_scale_argument(cuda_device):
    _run([100, 9], [0], [100], [1], [9], 2, 2, 64, 16, torch.bfloat16, scale=0.5)


def test_unmapped_pages_are_not_attended(cuda_device):
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, ks, vs = _pool([200, 100], 1, 64, 16, torch.bfloat16, 3)
    q = torch.randn(1, 2, 64, device="cuda").bfloat16()
    plan = SharedPrefixPlan([0], [200], [1], 2, 1, 64, max_suffix=100)
    table[0, 2] = -1
    table[0, 12] = kc.shape[0]
    table[1, 0] = -7
    own = torch.tensor([100], dtype=torch.int32, device="cuda")
    out, lse = shared_prefix_attention(q, kc, vc, table, own, plan)
    keep0 = [i for i in range(200) if i // 16 not in (2, 12)]
    ks, vs = [[x[0][keep0], x[1][16:]] for x in (ks, vs)]
    _compare(out, lse, q, ks, vs, [0], [len(keep0)], [1], [84], 64 ** -0.5)


def test_infinities_and_nan_stay_in_their_rows(cuda_device):
    """A NaN or infinite key of one sequence reaches only the rows that
    attend it, and there as the softmax has it."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([64, 40, 40, 40, 40], 1, 64, 16, torch.bfloat16, 5)
    q = torch.ones(4, 1, 64, device="cuda").bfloat16()
    plan = SharedPrefixPlan([0] * 4, [64] * 4, [1, 2, 3, 4], 1, 1, 64, max_suffix=40)
    own = torch.full((4,), 40, dtype=torch.int32, device="cuda")
    clean, _ = shared_prefix_attention(q, kc, vc, table, own, plan)

    def cell(slot, i):
        return int(table[slot, i // 16]), i % 16
    kc[cell(2, 5)] = float("nan")
    kc[cell(3, 5)] = float("-inf")     # a weight of zero
    vc[cell(3, 5)] = 1.0
    kc[cell(4, 5)] = float("inf")
    out, lse = shared_prefix_attention(q, kc, vc, table, own, plan)
    assert torch.equal(out[0], clean[0])
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    assert torch.isfinite(out[2]).all()
    assert torch.isnan(out[3]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,tokens,solo", [(4, 2, 128, 60, False), (8, 1, 96, 3, False),
                                                  (8, 1, 96, 3, True), (2, 2, 64, 40, False),
                                                  (4, 4, 40, 7, True), (2, 1, 256, 40, False),
                                                  (4, 1, 192, 9, False), (5, 1, 200, 3, True)])
def test_values_behind_a_row_do_not_reach_it(cuda_device, monkeypatch, hq, hkv, d, tokens, solo, dtype):
    """Several query tokens of a sequence: an infinite or NaN value reaches the
    rows at and behind its position, as the sum has it, and no row before."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    monkeypatch.setattr(SharedPrefixPlan, "_ranges",
                        lambda self, blocks, *a: (np.full(len(blocks), 1), solo))
    n = 1500
    kc, vc, table, ks, vs = _pool([50, n], hkv, d, 16, dtype, 4)
    rows = list(range(n - tokens, n))          # row r attends r + 1 tokens
    q = torch.randn(tokens, hq, d, generator=torch.Generator().manual_seed(2)).to("cuda", dtype)
    plan = SharedPrefixPlan([0] * tokens, [50] * tokens, [1] * tokens, hq, hkv, d, max_suffix=n)
    own = torch.tensor([r + 1 for r in rows], dtype=torch.int32, device="cuda")
    clean, clean_lse = shared_prefix_attention(q, kc, vc, table, own, plan)
    inf, nan = float("inf"), float("nan")
    odd = {n - 1: [(0, nan), (1, inf)], n - 2: [(1, -inf), (2, inf)]}
    for at, values in odd.items():
        for dim, x in values:
            vc[int(table[1, at // 16]), at % 16, 0, dim] = x
    out, lse = shared_prefix_attention(q, kc, vc, table, own, plan)
    assert torch.equal(lse, clean_lse)
    g = hq // hkv
    want = clean.clone()
    want[tokens - 2:, :g, 1:3] = torch.tensor([-inf, inf], device="cuda", dtype=dtype)
    want[tokens - 1, :g, :2] = nan             # NaN alone; -inf and inf together
    assert torch.equal(torch.nan_to_num(out, nan=123.0), torch.nan_to_num(want, nan=123.0))


def test_plan_of_nothing_runs(cuda_device):
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([20], 1, 64, 16, torch.bfloat16, 1)
    plan = SharedPrefixPlan([-1, -1], [0, 0], [-1, -1], 2, 1, 64, max_suffix=5)
    out, lse = shared_prefix_attention(torch.ones(2, 2, 64, device="cuda").bfloat16(), kc, vc, table,
                                       torch.tensor([3, 4], dtype=torch.int32, device="cuda"), plan)
    assert (out == 0).all() and (lse == float("-inf")).all()


def test_far_cells(cuda_device):
    """Pages behind 2^31 elements of the pool."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    pages, page, hkv, d = 70000, 64, 4, 128
    kc = torch.empty((pages, page, hkv, d), dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    ids = [[pages - 1, 0, 40000], [69000, 33000, -1]]
    table = torch.tensor(ids, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    ks, vs = ([torch.randn(n, hkv, d, generator=g).bfloat16() for n in (150, 100)] for _ in range(2))
    for s, n in enumerate((150, 100)):
        for i in range(0, n, page):
            m = min(page, n - i)
            kc[ids[s][i // page], :m], vc[ids[s][i // page], :m] = ks[s][i:i + m].cuda(), vs[s][i:i + m].cuda()
    q = torch.randn(3, 8, d, generator=g).to("cuda", torch.bfloat16)
    plan = SharedPrefixPlan([0] * 3, [150] * 3, [1] * 3, 8, hkv, d, max_suffix=100)
    own = [100, 64, 3]
    out, lse = shared_prefix_attention(q, kc, vc, table, torch.tensor(own, dtype=torch.int32, device="cuda"), plan)
    _compare(out, lse, q, ks, vs, [0] * 3, [150] * 3, [1] * 3, own, d ** -0.5)


def test_graph_replays_and_other_streams(cuda_device):
    """A captured call follows the lengths, queries and cache it finds; two
    captured calls of one plan and eager calls do not share anything."""
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([300, 90, 90], 2, 128, 16, torch.bfloat16, 9)
    plan = SharedPrefixPlan([0, 0], [300, 300], [1, 2], 12, 2, 128, max_suffix=90)
    qs = [torch.randn(2, 12, 128, device="cuda").bfloat16() for _ in range(2)]
    own = torch.tensor([1, 40], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    outs, graphs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(shared_prefix_attention(q, kc, vc, table, own, plan))
        graphs.append(graph)
    for step in range(4):
        own.add_(7)
        for q in qs:
            q.copy_(torch.randn_like(q))
        for graph in graphs:
            graph.replay()
        torch.randn(1000, device="cuda").sum().item()
        for q, (out, lse) in zip(qs, outs):
            want = shared_prefix_attention(q, kc, vc, table, own, plan)
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = shared_prefix_attention(qs[0], kc, vc, table, own, plan)
    side.synchronize()
    assert torch.equal(got[0], outs[0][0])


def test_strided_queries_and_own_outputs(cuda_device):
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([100, 5], 2, 64, 16, torch.bfloat16, 2)
    plan = SharedPrefixPlan([0], [100], [1], 4, 2, 64, max_suffix=5)
    own = torch.tensor([5], dtype=torch.int32, device="cuda")
    wide = torch.randn(1, 8, 64, device="cuda").bfloat16()
    want = shared_prefix_attention(wide[:, ::2].contiguous(), kc, vc, table, own, plan)
    out, lse = torch.empty(1, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 4, device="cuda")
    got = shared_prefix_attention(wide[:, ::2], kc, vc, table, own, plan, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_shared_refusals(cuda_device):
    from moba_hip import SharedPrefixPlan, shared_prefix_attention
    kc, vc, table, _, _ = _pool([100, 5], 2, 64, 16, torch.bfloat16, 2)
    plan = SharedPrefixPlan([0], [100], [1], 4, 2, 64, max_suffix=5)
    own = torch.tensor([5], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()

    def bad(match, q=q, kc=kc, vc=vc, table=table, own=own, plan=plan, **kw):
        with pytest.raises(ValueError, match=match):
            shared_prefix_attention(q, kc, vc, table, own, plan, **kw)

    bad("plan must be", plan=None)
    bad("the plan on it", plan=SharedPrefixPlan([0], [9], [1], 4, 2, 64, max_suffix=5, device="cpu"))
    bad("device and dtype", q=q.half())
    bad("plan's rows", q=torch.cat((q, q)))
    bad("plan's rows", q=q[:, :2])
    bad("plan's rows", plan=SharedPrefixPlan([0], [9], [1], 4, 1, 64, max_suffix=5))
    bad("fit page_table", plan=SharedPrefixPlan([0], [9], [2], 4, 2, 64, max_suffix=5))
    bad("fit page_table", plan=SharedPrefixPlan([0], [129], [1], 4, 2, 64, max_suffix=5))
    bad("suffix_lengths", own=own.long())
    bad("suffix_lengths must have", own=torch.cat((own, own)))
    bad("scale", scale=0.0)
    bad("scale", scale=float("inf"))
    bad("out must be", out=q.float())
    bad("lse must be", lse=torch.empty(1, 4, 2, device="cuda"))
    bad("out must not overlap", out=kc.view(-1)[:256].view(1, 4, 64))
    bad("lse must not overlap", lse=vc.view(-1)[:8].view(torch.float32).view(1, 4))
    bad("page_table", table=table.t())
    bad("cache dtype", kc=kc.float(), vc=vc.float())
    wide = torch.empty(4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    bad("aligned", q=wide[1:257].view(1, 4, 64))
    with pytest.raises(ValueError, match="inference-only"):
        shared_prefix_attention(q.clone().requires_grad_(True), kc, vc, table, own, plan)
