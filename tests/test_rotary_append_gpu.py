"""Rotary append (moba_hip.append_rotary) against the rotation in 64 bits.

A rotated value is formed in fp32 from two products and rounded once, so it is
off by at most half a step of its type plus 3 roundings of 2^-24 of
|a| + |b| (a fused and a plain product, one sum; |cos|, |sin| <= 1 as fp32
values); fp16 results below 2^-14 by half the subnormal step 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SENTINEL = 7.0


def _tokens(lengths, context):
    seq = [s for s, n in enumerate(lengths) for _ in range(n)]
    pos = [c + i for c, n in zip(context, lengths) for i in range(n)]
    return seq, pos


def _case(lengths, hq, hkv, d, rotary, page, dtype, *, interleaved=False, context=None, seed=0,
          offsets=None, contiguous=False):
    from moba_hip import RotaryTable
    g = torch.Generator().manual_seed(seed)
    context = context or [(5 * i) % 11 for i in range(len(lengths))]
    total = [c + n for c, n in zip(context, lengths)]
    width = -(-max(total) // page) + 1
    pages = sum(-(-t // page) for t in total) + 2
    perm = torch.randperm(pages, generator=g).tolist()
    table, at = [], 0
    for t in total:
        n = -(-t // page)
        table.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    n = sum(lengths)
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g).to("cuda", dtype)
    q, k, v = qkv.split([hq, hkv, hkv], dim=1)
    if contiguous:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    seq, pos = _tokens(lengths, context)
    dev = dict(dtype=torch.int32, device="cuda")
    st = dict(q=q, k=k, v=v, table=torch.tensor(table, **dev), seq=torch.tensor(seq, **dev),
              pos=torch.tensor(pos, **dev),
              offsets=None if offsets is None else torch.tensor(offsets, **dev))
    span = max(total) + (max(offsets) if offsets else 0)
    st["rotary"] = RotaryTable(rotary, span, interleaved=interleaved)
    for name in ("k_cache", "v_cache"):
        st[name] = torch.full((pages, page, hkv, d), SENTINEL, dtype=dtype, device="cuda")
    return st


def _run(st, **kw):
    from moba_hip import append_rotary
    return append_rotary(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["seq"],
                         st["pos"], st["rotary"], offsets=st["offsets"],
                         **{"q": st["q"], **kw})


def _turned(x, st, dtype):
    """(rotation in 64 bits, allowed error) of x [n,h,d]."""
    rt = st["rotary"]
    half = rt.rotary_dim // 2
    pos = st["pos"].long()
    if st["offsets"] is not None:
        pos = pos + st["offsets"].long()[st["seq"].long()]
    cs = rt.cos_sin.double()[pos][:, None]
    i = torch.arange(half, device="cuda")
    ia, ib = (2 * i, 2 * i + 1) if rt.interleaved else (i, i + half)
    y, tol = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia] = a * cs[..., 0] - b * cs[..., 1]
    y[..., ib] = a * cs[..., 1] + b * cs[..., 0]
    extra = 3 * 2.0 ** -24 * (a.abs() + b.abs()) + (2.0 ** -25 if dtype == torch.float16 else 0)
    for idx in (ia, ib):
        tol[..., idx] = torch.finfo(dtype).eps / 2 * (y[..., idx].abs() + extra) + extra
    return y, tol


def _check(st, got_q, dtype, live=None):
    n = st["k"].shape[0]
    live = torch.ones(n, dtype=torch.bool, device="cuda") if live is None else live
    page = st["k_cache"].shape[1]
    if got_q is not None:
        want, tol = _turned(st["q"], st, dtype)
        assert ((got_q.double() - want).abs() <= tol)[live].all()
    kc, vc = (torch.full_like(st["k_cache"], SENTINEL) for _ in range(2))
    seq, pos = st["seq"].long()[live], st["pos"].long()[live]
    phys, off = st["table"][seq, pos // page].long(), pos % page
    want, tol = _turned(st["k"], st, dtype)
    got = st["k_cache"][phys, off].double()
    assert ((got - want[live]).abs() <= tol[live]).all()
    vc[phys, off] = st["v"][live]
    assert torch.equal(st["v_cache"], vc)
    kc[phys, off] = st["k_cache"][phys, off]      # every other cell as it was
    assert torch.equal(st["k_cache"], kc)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d,rotary", [
    (4, 2, 256, 24), (3, 1, 96, 24), (2, 2, 80, 40), (2, 1, 72, 8),  # copied in wider pieces than turned
    (12, 2, 128, 128), (16, 1, 96, 96), (14, 2, 64, 64), (4, 4, 256, 64), (3, 1, 40, 40),
    (4, 2, 40, 10), (2, 2, 64, 2), (6, 3, 72, 36), (1, 1, 8, 8), (5, 1, 24, 16), (3, 3, 20, 6), (2, 1, 96, 24), (3, 1, 80, 20),
    (2, 1, 7, 4)])
def test_append_matches_fp64(cuda_device, hq, hkv, d, rotary, interleaved, dtype):
    st = _case([1, 37, 5, 64], hq, hkv, d, rotary, 16, dtype, interleaved=interleaved, seed=d)
    _check(st, _run(st, check=True), dtype)


@pytest.mark.parametrize("page", [1, 3, 48, 1000])
@pytest.mark.parametrize("lengths", [[1], [1] * 33, [257, 1, 90]])
def test_append_pages(cuda_device, lengths, page):
    st = _case(lengths, 4, 2, 64, 64, page, torch.bfloat16, seed=page)
    _check(st, _run(st), torch.bfloat16)


def test_append_without_queries_offsets_and_own_output(cuda_device):
    st = _case([3, 20], 4, 2, 128, 128, 16, torch.bfloat16, offsets=[1000, 77])
    assert _run(st, q=None) is None
    _check(st, None, torch.bfloat16)
    out = torch.full(st["q"].shape, SENTINEL, dtype=torch.bfloat16, device="cuda")
    st["k_cache"].fill_(SENTINEL), st["v_cache"].fill_(SENTINEL)
    assert _run(st, q_out=out) is out
    _check(st, out, torch.bfloat16)


@pytest.mark.parametrize("rotary,interleaved", [(64, False), (64, True), (24, False), (20, True), (6, False)])
@pytest.mark.parametrize("start,pad", [(1, 3), (2, 2), (4, 4), (8, 4), (2, 8)])
def test_misaligned_views(cuda_device, start, pad, rotary, interleaved):
    """Rows that are whole pieces of 8, 4 and 2 bytes only: odd starts and
    token strides."""
    st = _case([50], 2, 1, 64, rotary, 16, torch.float16, interleaved=interleaved)
    wide = torch.randn(50, 4 * 64 + start + pad, device="cuda").half()
    st["q"] = wide[:, start:start + 128].unflatten(1, (2, 64))
    st["k"] = wide[:, start + 128:start + 192].unflatten(1, (1, 64))
    st["v"] = wide[:, start + 192:start + 256].unflatten(1, (1, 64))
    _check(st, _run(st), torch.float16)


def test_padding_and_bad_tokens_are_left_alone(cuda_device):
    st = _case([40, 9], 4, 2, 64, 64, 16, torch.bfloat16)
    live = torch.ones(49, dtype=torch.bool, device="cuda")
    q = torch.full(st["q"].shape, SENTINEL, dtype=torch.bfloat16, device="cuda")
    pad = [3, 17, 48]
    for i in pad:
        st["seq"][i] = -1
        live[i] = False
    _run(st, q_out=q, check=True)     # padding is no error
    rows = torch.tensor(pad, device="cuda")
    assert (q[rows] == SENTINEL).all()
    seq = st["seq"].clone()
    st["seq"].clamp_min_(0)           # the reference indexes with it
    _check(st, q, torch.bfloat16, live)
    st["seq"] = seq
    for name, at, value, message in (
            ("seq", 5, 2, "slots of page_table"), ("seq", 5, -2, "slots of page_table"),
            ("pos", 6, 16 * st["table"].shape[1], "no page"), ("pos", 6, -1, "no page|rotary table"),
            ("pos", 7, 2 ** 31 - 1, "no page|rotary table"), ("pos", 8, 60, "no page|rotary table")):
        before = st["k_cache"].clone(), st["v_cache"].clone()
        keep = st[name][at].clone()
        st[name][at] = value
        with pytest.raises(RuntimeError, match=message):
            _run(st, check=True)
        _run(st)                      # unchecked: the token is dropped
        st[name][at] = keep
        assert torch.equal(st["k_cache"], before[0]) and torch.equal(st["v_cache"], before[1])
    st["table"][0, 1] = st["k_cache"].shape[0]    # a page outside the pool
    before = st["k_cache"].clone()
    with pytest.raises(RuntimeError, match="no page"):
        _run(st, check=True)
    assert torch.equal(st["k_cache"], before)


def test_two_tokens_of_one_cell(cuda_device):
    st = _case([8], 2, 1, 64, 64, 16, torch.bfloat16)
    st["pos"][3] = st["pos"][4]
    with pytest.raises(RuntimeError, match="share a cell"):
        _run(st, check=True)


def test_far_cells_and_positions(cuda_device):
    """A pool of more than 2^31 elements, and positions whose 32-bit angles
    would be off."""
    from moba_hip import RotaryTable, append_rotary
    pages, page, hkv, d = 70000, 64, 4, 128
    kc = torch.empty((pages, page, hkv, d), dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 31
    cells = [(pages - 1, 63), (pages - 2, 0), (0, 5), (33000, 31)]
    width = 4000
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    pos = [199 * page + 63, 200 * page, 5, 3999 * page + 31]
    for (pg, _), p in zip(cells, pos):
        table[0, p // page] = pg
    dev = dict(dtype=torch.int32, device="cuda")
    k, v, q = (torch.randn(4, h, d, device="cuda").bfloat16() for h in (hkv, hkv, 8))
    st = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, table=table,
              seq=torch.zeros(4, **dev), pos=torch.tensor(pos, **dev), offsets=None,
              rotary=RotaryTable(d, width * page))
    got = append_rotary(k, v, kc, vc, table, st["seq"], st["pos"], st["rotary"], q=q, check=True)
    for x, y in ((q, got), (k, torch.stack([kc[a, b] for a, b in cells]))):
        want, tol = _turned(x, st, torch.bfloat16)
        assert ((y.double() - want).abs() <= tol).all()
    assert torch.equal(torch.stack([vc[a, b] for a, b in cells]), v)


def test_append_on_another_stream_and_in_a_graph(cuda_device):
    from moba_hip import RotaryTable
    st = _case([1] * 40, 12, 2, 128, 128, 48, torch.bfloat16)
    st["rotary"] = RotaryTable(128, 48)
    want = _run(st)
    kc, vc = st["k_cache"].clone(), st["v_cache"].clone()
    side = torch.cuda.Stream()
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        st["k_cache"].fill_(SENTINEL), st["v_cache"].fill_(SENTINEL)
        got = _run(st)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(st["k_cache"], kc)
    with torch.cuda.graph(graph, stream=side):
        _run(st, q_out=out)
    for step in range(4):
        st["q"].copy_(torch.randn_like(st["q"]))
        st["k"].copy_(torch.randn_like(st["k"]))
        st["pos"].add_(step and 1)   # moves on as a decode does
        graph.replay()
        torch.randn(1000, device="cuda").sum().item()
        torch.cuda.synchronize()
        kc, vc = st["k_cache"].clone(), st["v_cache"].clone()
        assert torch.equal(out, _run(st))
        assert torch.equal(st["k_cache"], kc) and torch.equal(st["v_cache"], vc)


def test_append_refusals(cuda_device):
    from moba_hip import RotaryTable
    st = _case([4], 4, 2, 64, 64, 16, torch.bfloat16)

    def bad(match, **change):
        with pytest.raises(ValueError, match=match):
            _run({**st, **{k: v for k, v in change.items() if k in st}},
                 **{k: v for k, v in change.items() if k not in st or k == "q"})

    q, k = st["q"], st["k"]
    bad("k must match", k=k.half())
    bad("k must be", k=k[0])
    bad("v has an invalid shape", v=st["v"][:3])
    bad("q must match", q=q.float())
    bad("last dimension", k=torch.randn(4, 64, 2, device="cuda").bfloat16().transpose(1, 2))
    bad("token_seq", seq=st["seq"].long())
    bad("token_pos must have", pos=st["pos"][:3].clone())
    bad("page_table", table=st["table"].cpu())
    bad("offsets", offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    bad("RotaryTable", rotary=st["rotary"].cos_sin)
    bad("exceeds head_dim", rotary=RotaryTable(128, 8))
    bad("cache's device", rotary=RotaryTable(64, 8, device="cpu"))
    bad("q_out without q", q=None, q_out=torch.empty_like(q))
    bad("must not overlap", q_out=st["k_cache"].view(-1)[:4 * 4 * 64].view(4, 4, 64))
    bad("alias", k=st["k_cache"].view(-1)[:4 * 2 * 64].view(4, 2, 64))
    bad("v_cache must be like", v_cache=st["v_cache"][:1])
    bad("must not overlap", v_cache=st["k_cache"])
    bad("contiguous", k_cache=st["k_cache"].transpose(0, 1), v_cache=st["v_cache"].transpose(0, 1))
    own = q.contiguous()
    bad("must not overlap", q=own, q_out=own)
    with pytest.raises(ValueError, match="inference-only"):
        _run({**st, "k": k.detach().clone().requires_grad_(True)})
