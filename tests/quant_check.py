"""The 8-bit cache in 64 bits: codes, stored values, attention over them, and how far
the kernels may be from each."""
import torch

TOP = {"int8": 127.0, "fp8": 448.0}
LEAST = 2.0 ** -100


def nearest(y, fmt):
    """y (64 bits) at its nearest code's number, ties to the even code."""
    if fmt == "int8":
        return y.round().clamp(-127, 127)
    e = torch.frexp(y).exponent.clamp_min(-5) - 1     # 4 significant bits, exponents from -6 on
    step = ((e.long() - 3 + 1023) << 52).view(torch.float64)     # 2^(e - 3), exactly
    return (torch.round(y / step) * step).clamp(-448, 448)


def stored(x, fmt):
    """(codes' numbers, scale) of rows x [..., D] by the formulas, in 64 bits."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    return nearest(x * TOP[fmt] / a, fmt), (a / TOP[fmt])[..., 0]


def half_step(x, fmt):
    """What the nearest code may be off by, as values of x [..., D] in 64 bits."""
    a = x.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    if fmt == "int8":
        return (a / 254).expand_as(x)
    return torch.maximum(x.abs() * 2.0 ** -4, a / 448 * 2.0 ** -10)


def rounded(want, dtype):
    """What one rounding of `want` to a 16-bit type may be off by: half a step, or half
    the smallest subnormal of fp16; and 3 x 2^-24 for the scale and the product in fp32."""
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    return want.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + 3 * 2.0 ** -24) + least


def make_table(lengths, page, seed, spare=2, width=None):
    """(table, pages): pages in random order, dealt to slots of the given lengths."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    width = max(1, max(counts)) if width is None else width
    perm = torch.randperm(sum(counts) + spare, generator=g).tolist()
    rows, at = [], 0
    for c in counts:
        rows.append(perm[at:at + c] + [-1] * (width - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), len(perm)


def cells(lengths, first=None):
    """Device (slot, position) of every token of sequences that begin at `first`."""
    first = first or [0] * len(lengths)
    seq = [s for s, n in enumerate(lengths) for _ in range(n)]
    pos = [f + i for f, n in zip(first, lengths) for i in range(n)]
    return (torch.tensor(seq, dtype=torch.int32, device="cuda"),
            torch.tensor(pos, dtype=torch.int32, device="cuda"))


def numbers(pages, page_table, slot, pos):
    """(k, v, live): the stored values of one slot's positions in 64 bits, [n,Hkv,D], and
    which of them have a page."""
    page = pages.k.shape[2]
    phys = page_table[slot].long()[pos // page]
    live = (phys >= 0) & (phys < pages.k.shape[0])
    phys = torch.where(live, phys, 0)

    def of(codes, scale):
        x = codes.view(torch.uint8)[phys, :, pos % page].contiguous().view(codes.dtype).float().double()
        return x[..., :pages.head_dim] * scale[phys, :, pos % page].double()[..., None]
    return of(pages.k, pages.k_scale), of(pages.v, pages.v_scale), live


def attention(q, pages, page_table, q_seq, lengths, selected=None, chunk=None, scale=None,
              limit=None):
    """(out, lse, allowed error of out, of lse) in 64 bits, row by row.

    A score is a sum of D exact products in fp32 and three products more, off by at most
    (D + 8) 2^-24 of A = max_t scale sum_d |q_d k_td|; an exponential by that and 2^-22, a
    weight by 2^-16 more (two bf16 parts), and sums of T of them in fp32 by (T / 16 + 64)
    2^-24; the result by half a step of its type."""
    n, hq, d = q.shape
    hkv, page = pages.k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    span = page_table.shape[1] * page
    limit = span if limit is None else min(limit, span)
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((n, hq), -float("inf"), dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for r, (slot, length) in enumerate(zip(q_seq.tolist(), lengths.tolist())):
        length = max(0, min(length, limit))
        if not 0 <= slot < page_table.shape[0] or not length:
            continue
        t = torch.arange(length, device=q.device)
        k, v, live = numbers(pages, page_table, slot, t)
        # [heads, tokens]; what is not attended must not count, whatever it holds
        k, v = (torch.where(live[:, None, None], x, 0.0).repeat_interleave(hq // hkv, 1) for x in (k, v))
        qr = q[r].double()
        s = (qr[:, None] * k.transpose(0, 1)).sum(-1) * scale
        big = (qr.abs()[:, None] * k.transpose(0, 1).abs()).sum(-1) * scale
        on = live[None].expand(hq, length)     # an unmapped page is not attended
        if selected is not None:
            on = on & (selected[r][:, :, None] == (t // chunk)).any(1)
        s = torch.where(on, s, -float("inf"))
        big = torch.where(on, big, 0.0).amax(-1)
        lse[r] = torch.logsumexp(s, -1)
        some = on.any(-1)
        p = torch.where(on, torch.exp(s - torch.where(some, lse[r], 0.0)[:, None]), 0.0)
        # a weight of 0 takes nothing, unless the token is attended
        vt = v.transpose(0, 1)
        out[r] = (p[..., None] * torch.where(on[..., None], vt, 0.0)).sum(1)
        flat = (p[..., None] * torch.where(on[..., None], vt.abs(), 0.0)).sum(1)
        delta = (d + 8) * 2.0 ** -24 * big + 2.0 ** -20
        tol[r] = flat * (2 * delta + 2.0 ** -15 + (length / 16 + 64) * 2.0 ** -23)[:, None]
        ltol[r] = delta + torch.where(some, lse[r], 0.0).abs() * 2.0 ** -22 + (length / 16 + 64) * 2.0 ** -23
    least = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134
    tol = tol + torch.finfo(q.dtype).eps / 2 * (out.abs() + tol) + least
    return out, lse, tol, ltol


def check_attention(got, want):
    out, lse, tol, ltol = want
    got_out, got_lse = (x.double() for x in got)
    empty = torch.isinf(lse) & (lse < 0)
    assert torch.equal(torch.isinf(got_lse) & (got_lse < 0), empty)
    assert torch.equal(got_out[empty], torch.zeros_like(got_out[empty]))
    off = (got_out - out).abs() - tol
    assert (off <= 0).all(), f"out: {off.max():.3g} over its bound"
    off = torch.where(empty, -1.0, (got_lse - lse).abs() - ltol)
    assert (off <= 0).all(), f"lse: {off.max():.3g} over its bound"
