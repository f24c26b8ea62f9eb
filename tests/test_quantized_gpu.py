"""The operators of the 8-bit paged cache (moba_hip.quantized_append, quantized_read,
quantized_attention) against their formulas in 64 bits; bounds in quant_check."""
import pytest
import torch

from quant_check import (LEAST, TOP, attention, cells, check_attention, half_step, make_table, nearest,
                         numbers, rounded, stored)

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "fp8"]
TYPES = [torch.bfloat16, torch.float16]


def _pool(pages, page, hkv, d, fmt, fill=None):
    from moba_hip import QuantizedPages
    pool = QuantizedPages.empty(pages, page, hkv, d, format=fmt)
    if fill is not None:   # every code and scale of a cell that is not written
        for t in pool[:2]:
            t.view(torch.uint8).fill_(fill)
        for t in pool[2:4]:
            t.fill_(float("nan"))
    return pool


def _randn(*shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to("cuda", dtype)


def _filled(lengths, page, hkv, d, fmt, dtype, seed=0, **kw):
    """(pages, table) whose slots hold random tokens; other cells hold NaN codes and scales."""
    from moba_hip import quantized_append
    table, n_pages = make_table(lengths, page, seed, **kw)
    pages = _pool(n_pages, page, hkv, d, fmt, fill=0x7f)
    if sum(lengths):
        seq, pos = cells(lengths)
        n = len(seq)
        quantized_append(_randn(n, hkv, d, dtype=dtype, seed=seed + 1),
                         _randn(n, hkv, d, dtype=dtype, seed=seed + 2), pages, table, seq, pos, check=True)
    return pages, table


# ------------------------------------------------------------ append and read
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page,lengths", [(8, 1, [3]), (40, 5, [7, 1, 12]), (64, 16, [33, 2]),
                                            (96, 48, [100]), (128, 16, [17, 64]), (136, 7, [9]),
                                            (192, 3, [5, 4]), (256, 100, [130])])
def test_stored_values_are_those_of_the_formulas(fmt, dtype, d, page, lengths):
    """Codes and scales of tokens that do not turn: the nearest code, ties (which 16-bit
    values meet often) to the even one, exactly."""
    from moba_hip import quantized_append, quantized_read
    table, n_pages = make_table(lengths, page, 1)
    pages = _pool(n_pages, page, 3, d, fmt, fill=0x7f)
    seq, pos = cells(lengths)
    n = len(seq)
    k, v = (_randn(n, 3, d, dtype=dtype, seed=s, scale=3.0) for s in (1, 2))
    k[0] = 0
    v[-1, 1] = torch.arange(d, device="cuda").to(dtype) - d // 2
    assert quantized_append(k, v, pages, table, seq, pos, check=True) is None
    got = quantized_read(pages, table, seq, pos, dtype=dtype, check=True)
    for x, y, codes, scales in ((k, got[0], pages.k, pages.k_scale), (v, got[1], pages.v, pages.v_scale)):
        c, s = stored(x, fmt)
        phys = table[seq.long(), pos.long() // page].long()
        mine = codes.view(torch.uint8)[phys, :, pos.long() % page].view(codes.dtype).float().double()
        assert torch.equal(mine[..., :d], c)
        assert (mine[..., d:] == 0).all()    # behind D
        s32 = scales[phys, :, pos.long() % page].double()
        assert ((s32 - s).abs() <= s * 2.0 ** -24).all()
        assert ((y.double() - c * s[..., None]).abs() <= rounded(c * s[..., None], dtype)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rotary,inter", [(128, 128, False), (128, 128, True), (64, 16, False),
                                            (96, 96, False), (96, 24, False), (40, 40, True),
                                            (256, 64, False), (72, 2, False), (80, 80, False),
                                            (200, 100, True), (8, 8, False)])
def test_turned_keys_and_queries(fmt, dtype, d, rotary, inter):
    """A turned key is the nearest code of the fp32 rotation, which is within three
    roundings of 2^-24 (|a| + |b|) of the 64-bit one: it is off by half a step and
    that, and by it times 1 + 2^-20 where the scale follows it."""
    from moba_hip import RotaryTable, quantized_append, quantized_read
    lengths, first, page = [5, 1, 19], [0, 13, 2], 7
    table, n_pages = make_table([f + n for f, n in zip(first, lengths)], page, 3)
    pages = _pool(n_pages, page, 2, d, fmt, fill=0x7f)
    seq, pos = cells(lengths, first)
    n, hq = len(seq), 6
    qkv = _randn(n, hq + 4, d, dtype=dtype, seed=4, scale=2.0)
    q, k, v = qkv.split([hq, 2, 2], dim=1)
    offsets = torch.tensor([0, 40, 7], dtype=torch.int32, device="cuda")
    rt = RotaryTable(rotary, 80, interleaved=inter)
    turned = quantized_append(k, v, pages, table, seq, pos, rotary=rt, q=q, offsets=offsets, check=True)
    got_k, got_v = quantized_read(pages, table, seq, pos, dtype=dtype)
    at = pos.long() + offsets.long()[seq.long()]
    cs = rt.cos_sin.double()[at][:, None]
    i = torch.arange(rotary // 2, device="cuda")
    ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + rotary // 2)

    def turn(x):
        y, err = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        a, b = y[..., ia].clone(), y[..., ib].clone()
        y[..., ia], y[..., ib] = a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]
        err[..., ia] = err[..., ib] = 3 * 2.0 ** -24 * (a.abs() + b.abs())
        return y, err

    want, err = turn(q)
    assert ((turned.double() - want).abs() <= rounded(want, dtype) + err * 1.01).all()
    want, err = turn(k)
    step = half_step(want, fmt) * (1 + 2.0 ** -10) + err.amax(-1, keepdim=True) * 2
    assert ((got_k.double() - want).abs() <= step + rounded(want.abs() + step, dtype)).all()
    c, s = stored(v, fmt)
    assert ((got_v.double() - c * s[..., None]).abs() <= rounded(c * s[..., None], dtype)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,big,small", [(torch.bfloat16, 3.3e38, 1e-38), (torch.float16, 65504.0, 6e-8)])
def test_largest_and_smallest_rows(fmt, dtype, big, small):
    """Rows at the ends of a type's range: no overflow on the way, and a row below
    2^-100 keeps the scale of 2^-100."""
    from moba_hip import quantized_append, quantized_read
    table, n_pages = make_table([6], 4, 0)
    pages = _pool(n_pages, 4, 1, 64, fmt)
    seq, pos = cells([6])
    x = _randn(6, 1, 64, dtype=torch.float64, seed=5)
    x = x / x.abs().amax(-1, keepdim=True)
    scale = torch.tensor([big, small, 0.0, 1.0, big / 3, small * 5], dtype=torch.float64, device="cuda")
    x = (x * scale[:, None, None]).to(dtype)
    quantized_append(x, x, pages, table, seq, pos, check=True)
    k, v = quantized_read(pages, table, seq, pos, dtype=dtype)
    c, s = stored(x, fmt)
    assert torch.equal(k, v) and torch.isfinite(k).all()
    assert ((k.double() - c * s[..., None]).abs() <= rounded(c * s[..., None], dtype)).all()
    assert (k[2] == 0).all() and s[2, 0] == LEAST / TOP[fmt]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [128, 40])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rows_that_are_not_finite_read_as_nan(fmt, d, bad):
    from moba_hip import quantized_append, quantized_read
    table, n_pages = make_table([4], 4, 0)
    pages = _pool(n_pages, 4, 2, d, fmt)
    seq, pos = cells([4])
    k, v = (_randn(4, 2, d, dtype=torch.bfloat16, seed=s) for s in (6, 7))
    k[1, 0, 5], v[2, 1, d - 1] = bad, bad
    quantized_append(k, v, pages, table, seq, pos)
    got_k, got_v = quantized_read(pages, table, seq, pos)
    nan_k, nan_v = (torch.zeros(4, 2, dtype=torch.bool, device="cuda") for _ in range(2))
    nan_k[1, 0] = nan_v[2, 1] = True
    assert torch.equal(torch.isnan(got_k).all(-1), nan_k) and torch.equal(torch.isnan(got_k).any(-1), nan_k)
    assert torch.equal(torch.isnan(got_v).all(-1), nan_v) and torch.equal(torch.isnan(got_v).any(-1), nan_v)
    phys = table[0, 0].long()    # a code of such a row is 0: it harms no masked product
    assert (pages.k.view(torch.uint8)[phys, 0, 1] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_strided_and_misaligned_inputs(fmt):
    """Views of every kind give what packed copies give."""
    from moba_hip import RotaryTable, quantized_append, quantized_read
    d, page, n = 64, 5, 23
    rt = RotaryTable(d, 40)
    seq, pos = cells([n])
    base = _randn(n, 9, d + 3, dtype=torch.bfloat16, seed=8)
    views = [base[:, 2:4, 1:d + 1], base[:, 5:7, 2:d + 2], base[:, 4:8, 3:d + 3]]
    views += [base[:, :1, :d].expand(n, 2, d), base[:1, 5:7, :d].expand(n, 2, d), base[:, 4:8, :d]]
    for k, v, q in (views[:3], views[3:]):
        kept = []
        for packed in (False, True):
            table, n_pages = make_table([n], page, 2)
            pages = _pool(n_pages, page, 2, d, fmt, fill=0x7f)
            a, b, c = (x.contiguous() for x in (k, v, q)) if packed else (k, v, q)
            turned = quantized_append(a, b, pages, table, seq, pos, rotary=rt, q=c, check=True)
            kept.append((turned, *quantized_read(pages, table, seq, pos)))
        assert all(torch.equal(x, y) for x, y in zip(*kept))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 40])
def test_what_has_no_cell_is_left_alone(fmt, d):
    """Padding, slots and positions outside the table, unmapped pages, angles past the
    table: no other byte of the pool changes, a query without slot or angle is not
    written, and a read gives zeros."""
    from moba_hip import RotaryTable, quantized_append, quantized_read
    page, dev = 4, dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[2, -1, 0], [1, 99, 3]], **dev)
    pages = _pool(5, page, 2, d, fmt, fill=0x35)
    pages.k_scale.fill_(5.0), pages.v_scale.fill_(6.0)
    before = [t.clone() for t in pages[:4]]
    seq = torch.tensor([-1, 0, 2, -7, 0, 0, 1, 1, 0, 1], **dev)
    pos = torch.tensor([0, 1, 0, 0, 5, 12, 4, 8, -1, 1], **dev)
    n = len(seq)
    q, k, v = (_randn(n, 2, d, dtype=torch.float16, seed=s) for s in (1, 2, 3))
    rt = RotaryTable(d, 8)
    out = torch.full((n, 2, d), 7.0, dtype=torch.float16, device="cuda")
    assert quantized_append(k, v, pages, table, seq, pos, rotary=rt, q=q, q_out=out) is out
    written = {(2, 1), (1, 1)}     # (page, place) of tokens 1 and 9; 7's position has no angle
    for t, old in zip(pages[:4], before):
        a, b = (x.view(torch.uint8) if x.element_size() == 1 else x for x in (t, old))
        for p in range(5):
            for i in range(page):
                same = torch.equal(a[p, :, i], b[p, :, i])
                assert same != ((p, i) in written), (p, i)
    kept = [i for i in range(n) if bool((out[i] == 7).all())]
    assert kept == [0, 2, 3, 5, 7, 8]
    rk, rv = quantized_read(pages, table, seq, pos, dtype=torch.float16)
    for i in range(n):
        held = i in (1, 7, 9)
        assert bool((rk[i] != 0).any()) == held and bool((rv[i] != 0).any()) == held
    for s, p, message in ((2, 0, "slots"), (0, 5, "no page"), (1, 4, "no page"), (0, 12, "no page")):
        one = torch.tensor([s], **dev), torch.tensor([p], **dev)
        with pytest.raises(RuntimeError, match=message):
            quantized_append(k[:1], v[:1], pages, table, *one, check=True)
        with pytest.raises(RuntimeError, match=message):
            quantized_read(pages, table, *one, check=True)
    one = torch.tensor([1], **dev), torch.tensor([8], **dev)
    with pytest.raises(RuntimeError, match="rotary"):
        quantized_append(k[:1], v[:1], pages, table, *one, rotary=rt, check=True)
    two = torch.tensor([0, 0], **dev), torch.tensor([1, 1], **dev)
    with pytest.raises(RuntimeError, match="share a cell"):
        quantized_append(k[:2], v[:2], pages, table, *two, check=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_without_keys_turning_needs_no_angles(fmt):
    """An append without a table, twice to the same cells: the last one's tokens stay."""
    from moba_hip import quantized_append, quantized_read
    pages, table = _filled([9, 4], 4, 2, 48, fmt, torch.bfloat16)
    seq, pos = cells([9, 4])
    k, v = (_randn(13, 2, 48, dtype=torch.float16, seed=s) for s in (21, 22))   # another type than before
    quantized_append(k, v, pages, table, seq, pos)
    got = quantized_read(pages, table, seq, pos, dtype=torch.float16)
    for x, y in zip((k, v), got):
        c, s = stored(x, fmt)
        assert ((y.double() - c * s[..., None]).abs() <= rounded(c * s[..., None], torch.float16)).all()


def test_reads_of_one_cell_many_times():
    from moba_hip import quantized_read
    pages, table = _filled([40], 16, 2, 64, "fp8", torch.bfloat16)
    pos = torch.tensor([5, 5, 39, 0, 5] * 100, dtype=torch.int32, device="cuda")
    k, v = quantized_read(pages, table, torch.zeros_like(pos), pos)
    want = numbers(pages, table, 0, pos.long())
    assert torch.equal(k[0::5], k[1::5]) and torch.equal(v[0::5], v[4::5])
    assert ((k.double() - want[0]).abs() <= rounded(want[0], torch.bfloat16)).all()


# ------------------------------------------------------------------ attention
def _attend(lengths, hq, hkv, d, page, fmt, dtype, *, rows=None, chunk=None, slots=4, seed=0, qscale=2.0,
            **kw):
    """Runs and checks a call; rows: (slot, length) pairs, default each slot's whole length."""
    from moba_hip import quantized_attention
    pages, table = _filled(lengths, page, hkv, d, fmt, dtype, seed)
    rows = list(enumerate(lengths)) if rows is None else rows
    dev = dict(dtype=torch.int32, device="cuda")
    q_seq = torch.tensor([s for s, _ in rows], **dev)
    lens = torch.tensor([n for _, n in rows], **dev)
    q = _randn(len(rows), hq, d, dtype=dtype, seed=seed + 9, scale=qscale)
    selected = None
    if chunk:
        g = torch.Generator().manual_seed(seed)
        top = max(1, -(-max(n for _, n in rows) // chunk))
        selected = torch.randint(-1, top + 1, (len(rows), hq, slots), generator=g).to("cuda", torch.int32)
    got = quantized_attention(q, pages, table, q_seq, lens, selected=selected, chunk_size=chunk, **kw)
    check_attention(got, attention(q, pages, table, q_seq, lens, selected, chunk))
    return q, pages, table, q_seq, lens, selected, got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 8), (12, 2, 128), (14, 2, 64), (16, 1, 96), (8, 8, 40),
                                      (16, 4, 256), (6, 3, 136), (7, 1, 200), (17, 1, 64), (32, 1, 80),
                                      (48, 1, 128), (66, 2, 64), (40, 1, 256)])
def test_attention_of_every_head_layout(fmt, dtype, hq, hkv, d):
    _attend([1, 31, 32, 33, 127, 128, 129, 700], hq, hkv, d, 16, fmt, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", [1, 3, 16, 31, 48, 64, 100, 5000])
def test_attention_of_every_page_size(fmt, page):
    """Pages that end inside a step; lengths that end inside a page."""
    _attend([257, 95, 1, 1500], 6, 2, 64, page, fmt, torch.bfloat16)


@pytest.mark.parametrize("chunk,slots", [(1, 16), (7, 3), (32, 1), (64, 9), (100, 4), (512, 4), (10 ** 9, 2)])
@pytest.mark.parametrize("hq,hkv,d,fmt", [(12, 2, 128, "int8"), (32, 1, 64, "fp8"), (48, 1, 40, "int8"),
                                          (4, 4, 256, "fp8")])
def test_attention_of_selected_chunks(chunk, slots, hq, hkv, d, fmt):
    """Each head's own chunks: -1 entries, chunks named twice, chunks behind the length, heads
    that select nothing."""
    _attend([1500, 33, 640, 7, 200], hq, hkv, d, 16, fmt, torch.float16, chunk=chunk, slots=slots,
            rows=[(0, 1500), (1, 33), (2, 640), (3, 7), (4, 0), (4, 129), (-1, 5), (0, 513)])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("chunk", [None, 64])
@pytest.mark.parametrize("hq,hkv,d", [(17, 1, 64), (32, 1, 128), (64, 2, 40), (64, 1, 96), (30, 1, 256)])
def test_two_blocks_of_heads_in_an_entry(fmt, chunk, hq, hkv, d):
    """Tables that could map more than the last-level cache holds: more than 16 heads of a kv
    head read its tokens together.  (Most of the table has no page.)"""
    from moba_hip import quantized_attention
    lengths, page = [700, 33, 1, 129], 16
    pages, table = _filled(lengths, page, hkv, d, fmt, torch.bfloat16, width=2 ** 18 // page)
    rows = list(enumerate(lengths)) * 4
    assert 2 * len(rows) * hkv * 2 ** 18 * d > 256 << 20
    dev = dict(dtype=torch.int32, device="cuda")
    q_seq, lens = torch.tensor([s for s, _ in rows], **dev), torch.tensor([n for _, n in rows], **dev)
    q = _randn(len(rows), hq, d, dtype=torch.bfloat16, seed=3, scale=2.0)
    selected = None
    if chunk:
        g = torch.Generator().manual_seed(1)
        selected = torch.randint(-1, 12, (len(rows), hq, 4), generator=g).to("cuda", torch.int32)
    got = quantized_attention(q, pages, table, q_seq, lens, selected=selected, chunk_size=chunk)
    check_attention(got, attention(q, pages, table, q_seq, lens, selected, chunk))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_of_unlike_lengths_share_the_card(fmt):
    """One long row among short and empty ones, and several rows of one slot: entries that
    span many workgroups, workgroups that hold many entries."""
    lengths = [20011, 1, 130, 64, 3, 999, 5, 0, 17]
    rows = [(0, 20011), (1, 1), (7, 0), (2, 130), (0, 1), (0, 12345), (3, 64), (4, 0), (5, 999), (6, 5),
            (8, 17), (5, 500)] + [(2, i) for i in range(40)]
    _attend(lengths, 4, 2, 64, 16, fmt, torch.bfloat16, rows=rows)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq", [4, 20])
def test_many_short_rows(d, hq):
    """More rows than workgroups, so that a workgroup walks through several whole entries."""
    n = 900
    _attend([5, 140], hq, 2, d, 16, "int8", torch.float16,
            rows=[(i % 2, (i * 7) % (6 if i % 2 == 0 else 141)) for i in range(n)])


@pytest.mark.parametrize("fmt", FORMATS)
def test_unmapped_pages_and_lengths_behind_the_table(fmt):
    """Tokens of an unmapped page are not attended, in whole steps and inside one; a
    length is cut to what the table and max_length allow, a negative one is none."""
    from moba_hip import quantized_attention
    pages, table = _filled([304, 304, 48], 16, 2, 64, fmt, torch.bfloat16)   # every cell of a page
    table[0, 3:9] = -1
    table[1, :] = -1
    table[2, 2] = 10 ** 6
    dev = dict(dtype=torch.int32, device="cuda")
    q_seq = torch.tensor([0, 1, 2, 0, 2, 0, 3, 2 ** 31 - 1], **dev)
    lens = torch.tensor([300, 300, 40, 2 ** 31 - 1, -5, 50, 9, 9], **dev)
    q = _randn(8, 8, 64, dtype=torch.bfloat16, seed=3)
    for limit in (None, 1, 77, 10 ** 6):
        got = quantized_attention(q, pages, table, q_seq, lens, max_length=limit)
        check_attention(got, attention(q, pages, table, q_seq, lens, limit=limit))


@pytest.mark.parametrize("scale", [2.0 ** -126, 1e-3, 1.0, 30.0])
def test_scales(scale):
    """Flat and all but one-hot weights."""
    from moba_hip import quantized_attention
    pages, table = _filled([500], 16, 1, 64, "int8", torch.float16)
    dev = dict(dtype=torch.int32, device="cuda")
    q = _randn(1, 8, 64, dtype=torch.float16, seed=3)
    args = q, pages, table, torch.tensor([0], **dev), torch.tensor([500], **dev)
    check_attention(quantized_attention(*args, scale=scale), attention(*args, scale=scale))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,spread", [(torch.bfloat16, 30), (torch.float16, 10)])
def test_values_of_unlike_scales(fmt, dtype, spread):
    """Rows of 2^-spread to 2^spread: the weights keep the range of the values' scales, and a
    small value next to large ones its share."""
    from moba_hip import quantized_append, quantized_attention
    n, hkv, d = 400, 2, 64
    table, n_pages = make_table([n], 16, 0)
    pages = _pool(n_pages, 16, hkv, d, fmt, fill=0x7f)
    seq, pos = cells([n])
    k, v = (_randn(n, hkv, d, dtype=torch.float32, seed=s) for s in (1, 2))
    power = torch.linspace(-spread, spread, n, device="cuda").round()
    v = v * 2.0 ** power[torch.randperm(n, generator=torch.Generator().manual_seed(0))][:, None, None]
    quantized_append(k.to(dtype), v.to(dtype), pages, table, seq, pos)
    q = _randn(1, 8, d, dtype=dtype, seed=3, scale=0.5)
    dev = dict(dtype=torch.int32, device="cuda")
    args = q, pages, table, torch.tensor([0], **dev), torch.tensor([n], **dev)
    check_attention(quantized_attention(*args), attention(*args))


def test_scores_that_rise_token_by_token():
    """The running maximum moves again and again, by more and by less than its margin."""
    from moba_hip import quantized_append, quantized_attention
    n, d = 2000, 64
    table, n_pages = make_table([n], 16, 0)
    pages = _pool(n_pages, 16, 1, d, "int8")
    seq, pos = cells([n])
    k = torch.zeros(n, 1, d, device="cuda")
    k[:, 0, 0] = torch.arange(n, device="cuda") / 50 - 20
    quantized_append(k.bfloat16(), _randn(n, 1, d, dtype=torch.bfloat16, seed=2), pages, table, seq, pos)
    q = torch.zeros(3, 4, d, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = torch.tensor([[8.0], [-8.0], [0.5]], device="cuda")
    dev = dict(dtype=torch.int32, device="cuda")
    args = q, pages, table, torch.zeros(3, **dev), torch.full((3,), n, **dev)
    check_attention(quantized_attention(*args), attention(*args))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_reaches_who_attends_it_alone(fmt, d):
    """Tokens with an infinity or a NaN: a row behind whose length they lie, and a head that
    did not select their chunk, keep finite results; the others get NaN."""
    from moba_hip import quantized_append, quantized_attention
    n, hkv = 200, 2
    table, n_pages = make_table([n], 16, 0)
    pages = _pool(n_pages, 16, hkv, d, fmt, fill=0x7f)
    seq, pos = cells([n])
    k, v = (_randn(n, hkv, d, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    k[150, 0, 3], v[150, 1, 5] = float("nan"), float("inf")
    quantized_append(k, v, pages, table, seq, pos)
    dev = dict(dtype=torch.int32, device="cuda")
    q = _randn(2, 4, d, dtype=torch.bfloat16, seed=3)
    q_seq, lens = torch.zeros(2, **dev), torch.tensor([150, 151], **dev)
    out, lse = quantized_attention(q, pages, table, q_seq, lens)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()
    assert torch.isnan(lse[1, :2]).all() and torch.isfinite(lse[1, 2:]).all()
    selected = torch.tensor([0, 3], **dev).repeat(2, 4, 1)
    selected[1, 1::2, 1] = 2          # heads 1 and 3 read another chunk than that of token 150
    clean = [t.clone() for t in pages[2:4]]
    got = quantized_attention(q, pages, table, q_seq, torch.full((2,), 190, **dev), selected=selected,
                              chunk_size=50)
    assert torch.isnan(got[0][0]).all() and torch.isnan(got[0][1, ::2]).all()
    for s in (pages.k_scale, pages.v_scale):
        s.nan_to_num_(nan=1.0)
    want = attention(q, pages, table, q_seq, torch.full((2,), 190, **dev), selected, 50)
    for s, old in zip(pages[2:4], clean):
        s.copy_(old)
    kept = torch.tensor([[False] * 4, [False, True, False, True]], device="cuda")
    assert ((got[0].double() - want[0]).abs() <= want[2])[kept].all()
    assert ((got[1].double() - want[1]).abs() <= want[3])[kept].all()


@pytest.mark.parametrize("chunk", [None, 64])
def test_results_do_not_depend_on_the_run(chunk):
    from moba_hip import quantized_attention
    q, pages, table, q_seq, lens, selected, got = _attend([3000, 1, 500], 12, 2, 128, 16, "int8",
                                                          torch.bfloat16, chunk=chunk)
    for _ in range(3):
        again = quantized_attention(q, pages, table, q_seq, lens, selected=selected, chunk_size=chunk)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_given_outputs_and_a_batch_padded_at_its_end():
    """out and lse of the caller; padded rows give zeros and -inf."""
    from moba_hip import quantized_attention
    pages, table = _filled([70, 9], 16, 2, 64, "fp8", torch.float16)
    dev = dict(dtype=torch.int32, device="cuda")
    q = _randn(4, 4, 64, dtype=torch.float16, seed=1)
    q_seq, lens = torch.tensor([0, 1, -1, -1], **dev), torch.tensor([70, 9, 70, 0], **dev)
    out, lse = torch.full_like(q, 7.0), torch.full((4, 4), 7.0, device="cuda")
    got = quantized_attention(q, pages, table, q_seq, lens, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    check_attention(got, attention(q, pages, table, q_seq, lens))


def test_a_long_context():
    """One row of 131071 tokens: every workgroup has a part of it."""
    _attend([131071], 14, 2, 64, 16, "fp8", torch.bfloat16)


def test_more_rows_than_a_workgroup_has_threads():
    """Each thread sums the shares of several rows; some rows are padding, some empty."""
    _attend([40, 9], 2, 1, 64, 16, "fp8", torch.bfloat16,
            rows=[(i % 3 if i % 3 < 2 else -1, (i * 11) % (41 if i % 3 == 0 else 10)) for i in range(3001)])


def test_offsets_behind_32_bits():
    """A pool of 2 x 36 GiB of codes whose last pages are used: bytes pass 2^35, pieces 2^31."""
    from moba_hip import QuantizedPages, quantized_append, quantized_attention, quantized_read
    n_pages, page, hkv, d = 36 << 16, 16, 8, 128
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GiB of device memory")
    pages = QuantizedPages.empty(n_pages, page, hkv, d, format="int8")
    first = n_pages - 6
    table = torch.tensor([[first + 4, first, first + 5], [first + 2, first + 3, first + 1]],
                         dtype=torch.int32, device="cuda")
    lengths = [40, 33]
    seq, pos = cells(lengths)
    k, v = (_randn(len(seq), hkv, d, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    quantized_append(k, v, pages, table, seq, pos, check=True)
    for x, y in zip((k, v), quantized_read(pages, table, seq, pos, check=True)):
        c, s = stored(x, "int8")
        want = c * s[..., None]
        assert ((y.double() - want).abs() <= rounded(want, torch.bfloat16)).all()
    q = _randn(2, 16, d, dtype=torch.bfloat16, seed=3)
    rows = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for selected, chunk in ((None, None), (torch.tensor([1, 4, -1], dtype=torch.int32, device="cuda")
                                           .expand(2, 16, 3).contiguous(), 8)):
        got = quantized_attention(q, pages, table, rows, lens, selected=selected, chunk_size=chunk)
        check_attention(got, attention(q, pages, table, rows, lens, selected, chunk))


@pytest.mark.parametrize("turn", [False, True])
def test_an_append_of_more_than_2_to_the_31_elements(turn):
    """A prompt of a million tokens of 8 heads of 128 dims, all alike before they turn."""
    from moba_hip import RotaryTable, quantized_append, quantized_read
    n, page, hkv, d = 2 ** 20 + 40, 64, 8, 128
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GiB of device memory")
    pages = _pool(-(-n // page), page, hkv, d, "int8")
    table = torch.arange(pages.k.shape[0], dtype=torch.int32, device="cuda")[None]
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    k, v = (_randn(1, hkv, d, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    rotary = RotaryTable(64, n) if turn else None
    quantized_append(k.expand(n, hkv, d), v.expand(n, hkv, d), pages, table, torch.zeros_like(pos), pos,
                     rotary=rotary)
    small = _pool(1, 64, hkv, d, "int8")
    for at in (0, n - 64, n // 2):
        few = pos[at:at + 64]
        got = quantized_read(pages, table, torch.zeros_like(few), few)
        quantized_append(k.expand(64, hkv, d), v.expand(64, hkv, d), small, table[:, :1], torch.zeros_like(few),
                         pos[:64], rotary=rotary,
                         offsets=torch.tensor([at], dtype=torch.int32, device="cuda") if turn else None)
        want = quantized_read(small, table[:, :1], torch.zeros_like(few), pos[:64])
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_read_of_more_than_2_to_the_31_elements():
    """A context of 2.1 million tokens of 8 heads of 128 dims, whose cells are a few."""
    from moba_hip import quantized_read
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GiB of device memory")
    pages, table = _filled([16], 16, 8, 128, "fp8", torch.bfloat16)
    n = (2 ** 31 + 2 ** 20) // 1024
    pos = torch.arange(n, dtype=torch.int32, device="cuda") % 16
    k, v = quantized_read(pages, table, torch.zeros_like(pos), pos)
    few = quantized_read(pages, table, torch.zeros_like(pos[:16]), pos[:16])
    for x, y in zip((k, v), few):
        assert torch.equal(x.view(-1, 16, 8, 128)[-5:], y.expand(5, 16, 8, 128))
        assert torch.equal(x.view(-1, 16, 8, 128)[:5], y.expand(5, 16, 8, 128))


# ------------------------------------------------------------------- refusals
def _refusal_state():
    from moba_hip import QuantizedPages, RotaryTable
    dev = dict(dtype=torch.int32, device="cuda")
    pages = QuantizedPages.empty(4, 8, 2, 64, format="int8")
    return dict(pages=pages, table=torch.zeros(2, 2, **dev), seq=torch.zeros(3, **dev), pos=torch.arange(3, **dev),
                k=torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda"),
                v=torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda"),
                q=torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda"), rotary=RotaryTable(64, 9),
                lengths=torch.ones(3, **dev))


BAD_PAGES = {
    "no pool": lambda p: tuple(p),
    "codes of 16 bits": lambda p: p._replace(k=p.k.to(torch.int16)),
    "fp8 beside int8": lambda p: p._replace(v=p.v.view(torch.float8_e4m3fn)),
    "narrow rows": lambda p: p._replace(k=p.k[..., :48], v=p.v[..., :48]),
    "another head_dim": lambda p: p._replace(head_dim=80),
    "odd head_dim": lambda p: p._replace(head_dim=60),
    "bool head_dim": lambda p: p._replace(head_dim=True),
    "fewer values": lambda p: p._replace(v=p.v[:3]),
    "scales of 16 bits": lambda p: p._replace(k_scale=p.k_scale.half()),
    "scales of fewer pages": lambda p: p._replace(v_scale=p.v_scale[:2]),
    "strided": lambda p: p._replace(k=p.k.transpose(1, 2).contiguous().transpose(1, 2)),
    "one pool twice": lambda p: p._replace(v=p.k),
    "on the CPU": lambda p: p._replace(k_scale=p.k_scale.cpu()),
    "misaligned": lambda p: p._replace(k=torch.empty(p.k.numel() + 8, dtype=torch.int8, device="cuda")[8:].view(p.k.shape)),
    "no tensor": lambda p: p._replace(v_scale=None),
}


@pytest.mark.parametrize("how", BAD_PAGES)
def test_pools_that_are_refused(how):
    from moba_hip import quantized_append, quantized_attention, quantized_read
    st = _refusal_state()
    bad = BAD_PAGES[how](st["pages"])
    for call in (lambda: quantized_append(st["k"], st["v"], bad, st["table"], st["seq"], st["pos"]),
                 lambda: quantized_read(bad, st["table"], st["seq"], st["pos"]),
                 lambda: quantized_attention(st["q"], bad, st["table"], st["seq"], st["lengths"])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("change,message", [
    (dict(k=lambda st: st["k"][:2]), "invalid shape"), (dict(k=lambda st: st["k"].float()), "BF16 or FP16"),
    (dict(k=lambda st: st["k"].half()), "match"), (dict(v=lambda st: st["v"][..., :32]), "invalid shape"),
    (dict(k=lambda st: st["k"].requires_grad_(True)), "inference-only"),
    (dict(k=lambda st: st["k"][:0], v=lambda st: st["v"][:0], seq=lambda st: st["seq"][:0],
          pos=lambda st: st["pos"][:0], q=lambda st: None), "invalid shape"),
    (dict(k=lambda st: st["k"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
    (dict(seq=lambda st: st["seq"].long()), "token_seq"), (dict(pos=lambda st: st["pos"][:2]), "token_pos"),
    (dict(table=lambda st: st["table"].t()), "page_table"), (dict(table=lambda st: st["table"][:0]), "page_table"),
    (dict(rotary=lambda st: None), "without rotary"), (dict(rotary=lambda st: 3), "RotaryTable"),
    (dict(offsets=lambda st: st["seq"]), "offsets"), (dict(q=lambda st: st["q"][:, :0]), "invalid shape"),
    (dict(q=lambda st: None, q_out=lambda st: st["q"]), "q_out without q"),
    (dict(q_out=lambda st: st["q"]), "overlap"), (dict(q_out=lambda st: st["q"][:2]), "invalid shape"),
    (dict(k=lambda st: st["pages"].k.view(torch.bfloat16).reshape(-1)[:384].view(3, 2, 64)), "alias"),
])
def test_appends_that_are_refused(change, message):
    from moba_hip import quantized_append
    st = _refusal_state()
    args = {"q_out": None, "offsets": None, **st, **{n: f(st) for n, f in change.items()}}
    with pytest.raises(ValueError, match=message):
        quantized_append(args["k"], args["v"], args["pages"], args["table"], args["seq"], args["pos"],
                         rotary=args["rotary"], q=args["q"], q_out=args["q_out"], offsets=args["offsets"])


def test_a_replaced_table_of_angles_is_checked():
    from moba_hip import quantized_append
    st = _refusal_state()
    st["rotary"].cos_sin = st["rotary"].cos_sin[:, :16].contiguous()
    with pytest.raises(ValueError, match="cos_sin"):
        quantized_append(st["k"], st["v"], st["pages"], st["table"], st["seq"], st["pos"], rotary=st["rotary"])


@pytest.mark.parametrize("kw", [dict(dtype=torch.float32), dict(seq=lambda t: t[:0]), dict(seq=lambda t: t.long()),
                                dict(pos=lambda t: t[:1]), dict(seq=lambda t: t[None])])
def test_reads_that_are_refused(kw):
    from moba_hip import quantized_read
    st = _refusal_state()
    seq, pos = (kw.get(n, lambda t: t)(st[n]) for n in ("seq", "pos"))
    with pytest.raises(ValueError):
        quantized_read(st["pages"], st["table"], seq, pos, dtype=kw.get("dtype", torch.bfloat16))


@pytest.mark.parametrize("kw,message", [
    (dict(scale=0.0), "scale"), (dict(scale=1e31), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(max_length=0), "max_length"), (dict(max_length=2.5), "max_length"), (dict(chunk_size=8), "without selected"),
    (dict(selected=lambda st: torch.zeros(3, 4, 2, dtype=torch.int32, device="cuda")), "chunk_size"),
    (dict(selected=lambda st: torch.zeros(3, 4, 17, dtype=torch.int32, device="cuda"), chunk_size=8), "1 to 16"),
    (dict(selected=lambda st: torch.zeros(3, 2, 2, dtype=torch.int32, device="cuda"), chunk_size=8), "selected"),
    (dict(selected=lambda st: torch.zeros(3, 4, 2, device="cuda"), chunk_size=8), "selected"),
    (dict(selected=lambda st: torch.zeros(3, 4, 2, dtype=torch.int32, device="cuda"), chunk_size=0), "chunk_size"),
    (dict(q=lambda st: st["q"][:, :3]), "multiple of Hkv"), (dict(q=lambda st: st["q"][:2]), "q_seq"),
    (dict(q=lambda st: st["q"].float()), "BF16 or FP16"),
    (dict(q=lambda st: torch.zeros(3 * 256 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(3, 4, 64)), "16-byte"),
    (dict(q=lambda st: st["q"].transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
    (dict(lengths=lambda st: st["lengths"].long()), "lengths"), (dict(lengths=lambda st: st["lengths"][:1]), "lengths"),
    (dict(out=lambda st: st["q"]), "overlap"), (dict(out=lambda st: st["q"].half()), "out must be"),
    (dict(lse=lambda st: torch.zeros(3, 4, dtype=torch.float64, device="cuda")), "lse"),
    (dict(lse=lambda st: st["pages"].k_scale.view(-1)[:12].view(3, 4)), "overlap"),
])
def test_attentions_that_are_refused(kw, message):
    from moba_hip import quantized_attention
    st = _refusal_state()
    kw = {n: f(st) if callable(f) else f for n, f in kw.items()}
    q, lengths = kw.pop("q", st["q"]), kw.pop("lengths", st["lengths"])
    with pytest.raises(ValueError, match=message):
        quantized_attention(q, st["pages"], st["table"], st["seq"], lengths, **kw)


# --------------------------------------------------------- streams and graphs
def _step(pages, table, rt, n, hq, hkv, d, seed):
    """State of a decode step of n slots, one token each."""
    dev = dict(dtype=torch.int32, device="cuda")
    return dict(q=_randn(n, hq, d, dtype=torch.bfloat16, seed=seed), k=_randn(n, hkv, d, dtype=torch.bfloat16, seed=seed + 1),
                v=_randn(n, hkv, d, dtype=torch.bfloat16, seed=seed + 2), seq=torch.arange(n, **dev))


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_then_attend_captured_and_replayed(fmt):
    """A run of the operators as a decode step has them, in one graph: positions move on
    the device, several replays, eager work between them, each like the eager step."""
    from moba_hip import RotaryTable, quantized_append, quantized_attention
    hq, hkv, d, page, lengths = 6, 2, 64, 16, [30, 1, 90]
    full = [n + 8 for n in lengths]
    table, n_pages = make_table(full, page, 5)
    rt = RotaryTable(d, 200)
    seq, pos0 = cells(lengths)
    k0, v0 = (_randn(len(seq), hkv, d, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    pools = []
    for _ in range(2):
        pages = _pool(n_pages, page, hkv, d, fmt, fill=0x7f)
        quantized_append(k0, v0, pages, table, seq, pos0, rotary=rt)
        pools.append(pages)
    st = _step(pools[0], table, rt, 3, hq, hkv, d, 10)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def step(pages, pos):
        turned = quantized_append(st["k"], st["v"], pages, table, st["seq"], pos, rotary=rt, q=st["q"])
        return quantized_attention(turned, pages, table, st["seq"], pos + 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pools[0], pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(pools[0], pos)
        pos.add_(1)
    for i in range(6):
        for x, s in (("q", 30), ("k", 31), ("v", 32)):
            st[x].copy_(_randn(*st[x].shape, dtype=torch.bfloat16, seed=s + 3 * i))
        at = pos.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = step(pools[1], at)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert torch.equal(pos, at + 1)
    for a, b in zip(pools[0][:4], pools[1][:4]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_calls_at_once_on_streams_of_their_own():
    """Each call has a workspace of its own."""
    from moba_hip import quantized_attention
    a = _attend([5000, 77], 12, 2, 128, 16, "int8", torch.bfloat16, seed=1)
    b = _attend([900, 4000, 3], 8, 2, 64, 16, "fp8", torch.float16, chunk=64, seed=2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, x, chunk) in enumerate(zip(streams, (a, b), (None, 64))):
            with torch.cuda.stream(s):
                got[i].append(quantized_attention(*x[:5], selected=x[5], chunk_size=chunk))
    torch.cuda.synchronize()
    for results, x in zip(got, (a, b)):
        for r in results:
            assert all(torch.equal(p, w) for p, w in zip(r, x[6]))
