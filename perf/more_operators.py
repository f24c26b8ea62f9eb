"""Operators of an 8-bit paged KV cache: their cases, their plain forms and the
calls a user's program makes of them.

A pool holds codes ``[pages, Hkv, page, Dp]`` (int8, or 8-bit floats e4m3; Dp: the
head dims rounded up to 16) and one fp32 scale per token and kv head
``[pages, Hkv, page]``, for keys and for values.  A row of D values x stands as
codes c and a scale s with x ~ c s:  a = max(|x|, 2^-100), s = a / top, c = x / s
rounded to the nearest code (ties to even), top = 127 (int8) or 448 (fp8).

Kinds of case (``case["kind"]``):

* ``store``   new keys and values are quantised into the pool, the keys turned by
              their positions first and the queries of the same tokens with them;
              what the cells then hold is read back in the inputs' type.  Inputs
              are views of one projection's output ``[tokens, (Hq + 2 Hkv) D]``.
* ``read``    stored tokens of several sequences, read back in 16 bits.
* ``attend``  one new query per row attends its sequence's tokens in the pool:
              all of them, or (``chunk`` > 0) those of the chunks that each of its
              heads selected.

``lengths`` (store, read) holds each sequence's tokens as text; the rows of an
attend case have lengths from ``lo`` to ``hi``, even in their logarithm, dealt by
``mix``.  ``own`` selects the framework's kernels; the plain forms need torch alone.
"""
import math
import os
import random
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "moba-merge-cuda_amd")
_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
_TOP = {"int8": 127.0, "fp8": 448.0}
_LEAST = 2.0 ** -100


def _framework():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import moba_hip
    return moba_hip


def listed():
    return [
        # One decode step of 8 requests (Qwen2-1.5B attention shape), pages of 48
        # tokens: latency.
        dict(name="store_step_b8", kind="store", format="int8", lengths=",".join(["1"] * 8),
             context=2000, hq=12, hkv=2, d=128, rotary=128, interleaved=False, page=48,
             dtype="bf16"),
        # One decode step of a full serving batch, one kv head of 96 dims.
        dict(name="store_step_mqa_b256", kind="store", format="fp8", lengths=",".join(["1"] * 256),
             context=500, hq=16, hkv=1, d=96, rotary=96, interleaved=False, page=64, dtype="fp16"),
        # A 32K-token prompt written into an empty slot, 8 kv heads.
        dict(name="store_prompt_32k", kind="store", format="int8", lengths="32768", context=0,
             hq=32, hkv=8, d=128, rotary=128, interleaved=False, page=16, dtype="bf16"),
        # A packed batch of prompts of ragged lengths (Qwen2-0.5B heads), pairs of
        # neighbouring dims turned.
        dict(name="store_ragged", kind="store", format="fp8", lengths="5003,311,4097,1,2049,777",
             context=30, hq=14, hkv=2, d=64, rotary=64, interleaved=True, page=16, dtype="fp16"),
        # The chunks that four sequences close in a step, for their key means.
        dict(name="read_chunks", kind="read", format="int8", lengths="512,512,512,512", hkv=2, d=128,
             page=48, dtype="bf16"),
        # A whole 32K context, for a prefill that goes on behind it.
        dict(name="read_context_32k", kind="read", format="fp8", lengths="32768", hkv=8, d=128,
             page=16, dtype="bf16"),
        # Contexts of ragged lengths, wide heads.
        dict(name="read_ragged", kind="read", format="int8", lengths="12289,1,5003,311", hkv=4, d=256,
             page=100, dtype="fp16"),
        # Decode of 8 requests of up to 2K tokens: latency.
        dict(name="attend_b8_2k", kind="attend", format="int8", rows=8, lo=200, hi=2048, mix=1, chunk=0,
             topk=1, hq=12, hkv=2, d=128, page=48, dtype="bf16"),
        # One request of a very long context: one row, a long axis.
        dict(name="attend_b1_128k", kind="attend", format="fp8", rows=1, lo=131071, hi=131071, mix=2,
             chunk=0, topk=1, hq=14, hkv=2, d=64, page=16, dtype="bf16"),
        # A full serving batch, one kv head.
        dict(name="attend_mqa_b256", kind="attend", format="fp8", rows=256, lo=64, hi=4096, mix=3,
             chunk=0, topk=1, hq=16, hkv=1, d=96, page=64, dtype="fp16"),
        # Requests of unlike lengths up to 32K, 8 kv heads: bound by the reads.
        dict(name="attend_b64_ragged", kind="attend", format="int8", rows=64, lo=256, hi=32768, mix=4,
             chunk=0, topk=1, hq=32, hkv=8, d=128, page=16, dtype="bf16"),
        # The same heads, each reading its own and three more chunks of 512 tokens.
        dict(name="attend_moba_b16_32k", kind="attend", format="int8", rows=16, lo=20000, hi=32768,
             mix=5, chunk=512, topk=4, hq=32, hkv=8, d=128, page=16, dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hq, hkv = rng.choice([(12, 2), (16, 1), (32, 8), (14, 2), (28, 4), (16, 4), (8, 8), (32, 32),
                          (6, 3), (48, 1)])
    d = rng.choice([64, 64, 96, 128, 128, 128, 192, 256, 40, 80])
    page = rng.choice([16, 16, 48, 64, 1, 100, 256])
    base = dict(format=rng.choice(["int8", "fp8"]), hkv=hkv, d=d, page=page,
                dtype=rng.choice(["bf16", "bf16", "fp16"]))
    while True:
        kind = rng.choice(["store", "store", "read", "attend", "attend", "attend"])
        if kind == "attend":
            hi = log(1, 131072)
            chunk = rng.choice([0, 0, 0, 64, 128, 512, 1000])
            case = dict(base, kind=kind, rows=log(1, 256), lo=rng.choice([1, hi, max(1, hi // 8)]), hi=hi,
                        mix=rng.randrange(1 << 20), chunk=chunk,
                        topk=rng.choice([2, 3, 4, 9]) if chunk else 1, hq=hq)
            # within the largest listed case, for the plain form's padded copies too
            if work(case)["bytes"] <= 2e9 and case["rows"] * hi * hkv * d <= 1 << 31:
                return case
            continue
        if rng.random() < 0.5:
            lengths = [rng.choice([1, 1, 1, 2, 5]) for _ in range(log(1, 512))]
        else:
            tokens = log(16, 32768)
            cuts = sorted(rng.sample(range(1, tokens), min(tokens - 1, rng.choice([0, 1, 5]))))
            lengths = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
        case = dict(base, kind=kind, lengths=",".join(map(str, lengths)))
        if kind == "store":
            case.update(hq=hq, context=rng.choice([0, log(1, 1000)]), interleaved=rng.random() < 0.4,
                        rotary=rng.choice([d, d, d, d // 2, d // 4 - d // 4 % 2, 2]))
        if work(case)["bytes"] <= 8e8:
            return case


def _ints(text):
    return [int(x) for x in text.split(",")]


def _rows(case):
    """Lengths of the rows of an attend case and, with chunks, what each head
    selected: [rows][hq][topk], its current chunk first, -1 where there are not so
    many.  The heads of a model agree on some chunks: half the picks are the row's."""
    rng = random.Random(case["mix"])
    lo, hi = math.log(case["lo"]), math.log(case["hi"])
    lengths = [min(case["hi"], max(case["lo"], round(math.exp(rng.uniform(lo, hi)))))
               for _ in range(case["rows"])]
    if not case["chunk"]:
        return lengths, None
    picked = []
    for n in lengths:
        closed, want = (n - 1) // case["chunk"], case["topk"] - 1
        common = rng.sample(range(closed), min(want, closed))
        heads = []
        for _ in range(case["hq"]):
            mine = set(common[:len(common) // 2])
            while len(mine) < min(want, closed):
                mine.add(rng.randrange(closed))
            heads.append([closed] + sorted(mine) + [-1] * (want - len(mine)))
        picked.append(heads)
    return lengths, picked


def work(case):
    hkv, d = case["hkv"], case["d"]
    stored = 2 * hkv * (d + 4)   # codes and scales of a token
    if case["kind"] == "read":
        n = sum(_ints(case["lengths"]))
        return {"bytes": n * (stored + 4 * hkv * d + 8), "flops": 2 * n * hkv * d}
    hq = case["hq"]
    if case["kind"] == "store":
        lengths = _ints(case["lengths"])
        n, r = sum(lengths), case["rotary"]
        # q, k and v in; q, codes and scales out; those in and the values out; the
        # table's rows of the distinct positions; (sequence, position) of each token
        rows = max(lengths) if max(lengths) > 1 else n
        return {"bytes": n * ((2 * hq + 4 * hkv) * d * 2 + 2 * stored) + rows * r * 4 + n * 8,
                "flops": n * ((hq + hkv) * r * 3 + hkv * d * 8)}
    lengths, picked = _rows(case)
    read = pairs = 0
    if picked is None:
        read, pairs = sum(lengths) * hkv, sum(lengths) * hq
    else:
        g = hq // hkv
        for n, heads in zip(lengths, picked):
            def size(c, n=n):
                return min(case["chunk"], n - c * case["chunk"])
            pairs += sum(size(c) for h in heads for c in h if c >= 0)
            read += sum(size(c) for k in range(hkv)
                        for c in set(c for h in heads[k * g:(k + 1) * g] for c in h if c >= 0))
    rows = case["rows"]
    return {"bytes": 2 * read * (d + 4) + rows * hq * (4 * d + 4), "flops": 4 * pairs * d}


def _randn(gen, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _quantised(x, form):
    """Codes (as bytes) and scales of rows x [..., D] in 32 bits."""
    top = _TOP[form]
    a = x.abs().amax(-1, keepdim=True).clamp_min(_LEAST)
    y = x * top / a
    code = y.round().clamp(-top, top).to(torch.int8) if form == "int8" else y.to(torch.float8_e4m3fn)
    return code.view(torch.uint8), (a / top)[..., 0]


def _numbers(code, form):
    """The numbers that codes (bytes) stand for before their scale."""
    return code.view(torch.int8 if form == "int8" else torch.float8_e4m3fn).float()


def _page_table(lengths, page, seed):
    """Pages of a pool in random order, dealt to the sequences; -1: no page."""
    counts = [-(-n // page) for n in lengths]
    pages = list(range(sum(counts)))
    random.Random(seed).shuffle(pages)
    table, at = [], 0
    for c in counts:
        table.append(pages[at:at + c] + [-1] * (max(counts) - c))
        at += c
    return torch.tensor(table, dtype=torch.int32, device="cuda"), at


def _cells(sequences, device="cuda"):
    """(slot, position) of every token of [(first position, tokens)] sequences."""
    seq = [s for s, (_, n) in enumerate(sequences) for _ in range(n)]
    pos = [first + i for first, n in sequences for i in range(n)]
    return (torch.tensor(seq, dtype=torch.int32, device=device),
            torch.tensor(pos, dtype=torch.int32, device=device))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, form = _DTYPE[case["dtype"]], case["format"]
    hkv, d, page = case["hkv"], case["d"], case["page"]
    wide = -(-d // 16) * 16
    st = dict(case=case)
    if case["kind"] == "attend":
        lengths, picked = _rows(case)
        capacity = lengths
    else:
        lengths = _ints(case["lengths"])
        first = [rng.randint(0, case.get("context", 0)) for _ in lengths]
        capacity = [case.get("context", 0) + n for n in lengths]
        st["seq"], st["pos"] = _cells(list(zip(first, lengths)))
    st["table"], pages = _page_table(capacity, page, seed)
    for name in ("k", "v"):
        code = torch.zeros((pages, hkv, page, wide), dtype=torch.uint8, device="cuda")
        scale = torch.ones((pages, hkv, page), device="cuda")
        if case["kind"] != "store":
            step = max(1, (1 << 26) // (hkv * page * wide))   # pages at once
            for i in range(0, pages, step):
                x = torch.randn((min(step, pages - i), hkv, page, d), generator=gen, device="cuda")
                code[i:i + step, ..., :d], scale[i:i + step] = _quantised(x, form)
        st[name + "_code"], st[name + "_scale"] = code, scale
    if case["kind"] == "store":
        hq, n = case["hq"], sum(lengths)
        qkv = _randn(gen, n, hq + 2 * hkv, d, dtype=dtype)
        st["q"], st["k"], st["v"] = qkv.split([hq, hkv, hkv], dim=1)
        half = case["rotary"] // 2
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(max(capacity), dtype=torch.float64, device="cuda")[:, None] * inv
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    elif case["kind"] == "attend":
        # scores of deviation 2: a few keys of thousands hold most of the weight
        st["q"] = _randn(gen, case["rows"], case["hq"], d, dtype=dtype, scale=2.0)
        st["q_seq"] = torch.arange(case["rows"], dtype=torch.int32, device="cuda")
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        st["selected"] = None if picked is None else torch.tensor(picked, dtype=torch.int32,
                                                                  device="cuda")
    if own:
        kind = torch.int8 if form == "int8" else torch.float8_e4m3fn
        st["pages"] = _framework().QuantizedPages(st["k_code"].view(kind), st["v_code"].view(kind),
                                                  st["k_scale"], st["v_scale"], d)
        if case["kind"] == "store":
            st["rotary"] = _framework().RotaryTable.from_cos_sin(st["cos"], st["sin"],
                                                                 interleaved=case["interleaved"])
    return st


def run(state):
    kind = state["case"]["kind"]
    if kind == "attend":
        return _attend_own(state) if own else _attend_plain(state)
    out = {}
    if kind == "store":
        out["q"] = _store_own(state) if own else _store_plain(state)
    out["k"], out["v"] = _read_own(state) if own else _read_plain(state)
    return out


def _store_own(st):
    return _framework().quantized_append(st["k"], st["v"], st["pages"], st["table"], st["seq"],
                                         st["pos"], rotary=st["rotary"], q=st["q"])


def _read_own(st):
    return _framework().quantized_read(st["pages"], st["table"], st["seq"], st["pos"],
                                       dtype=_DTYPE[st["case"]["dtype"]])


def _attend_own(st):
    case = st["case"]
    out, lse = _framework().quantized_attention(
        st["q"], st["pages"], st["table"], st["q_seq"], st["lengths"], selected=st["selected"],
        chunk_size=case["chunk"] or None)
    return {"out": out, "lse": lse}


def _where(st):
    """Physical page and place in it of the tokens of a store or read case."""
    seq, pos, page = st["seq"].long(), st["pos"].long(), st["case"]["page"]
    return st["table"][seq, pos // page].long(), pos % page


def _rotated(x, cos, sin, interleaved):
    """x [n, heads, d] with its first 2 * half dims rotated, pair by pair."""
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((y, x[..., 2 * half:]), dim=-1)


def _store_plain(st):
    case, pos = st["case"], st["pos"].long()
    d, dtype = case["d"], st["q"].dtype
    phys, at = _where(st)
    cos, sin = st["cos"][pos], st["sin"][pos]
    rows = {"k": _rotated(st["k"].float(), cos, sin, case["interleaved"]), "v": st["v"].float()}
    for name in ("k", "v"):
        code, scale = _quantised(rows[name], case["format"])
        st[name + "_code"][phys, :, at, :d] = code
        st[name + "_scale"][phys, :, at] = scale
    return _rotated(st["q"].float(), cos, sin, case["interleaved"]).to(dtype)


def _read_plain(st):
    case = st["case"]
    phys, at = _where(st)
    return tuple((_numbers(st[name + "_code"][phys, :, at, :case["d"]].contiguous(), case["format"])
                  * st[name + "_scale"][phys, :, at][..., None]).to(_DTYPE[case["dtype"]])
                 for name in ("k", "v"))


def _attend_plain(st):
    case, q = st["case"], st["q"]
    n, hq, d = q.shape
    hkv, page = case["hkv"], case["page"]
    width = st["table"].shape[1]
    phys = st["table"][st["q_seq"].long()].long().clamp_min(0)            # [n, pages]

    def gathered(name):   # [n, hkv, tokens, d]
        code = _numbers(st[name + "_code"][phys][..., :d].contiguous(), case["format"])
        x = code * st[name + "_scale"][phys][..., None]
        return x.transpose(1, 2).reshape(n * hkv, width * page, d)

    qs = (q.float() * d ** -0.5).view(n * hkv, hq // hkv, d)
    s = torch.bmm(qs, gathered("k").transpose(1, 2).contiguous()).view(n, hq, -1)
    token = torch.arange(width * page, device=q.device)
    live = (token < st["lengths"][:, None])[:, None]
    if st["selected"] is not None:
        chunk = (token // case["chunk"]).int()
        # a head's chunks as a table of truth values, then looked up by token
        count = int(chunk[-1]) + 1
        takes = torch.zeros((n, hq, count + 1), dtype=torch.bool, device=q.device)
        takes.scatter_(2, torch.where(st["selected"] >= 0, st["selected"], count).long(), True)
        live = live & takes[:, :, chunk.long()]
    s = s.masked_fill(~live, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(n * hkv, hq // hkv, -1), gathered("v")).view(n, hq, d)
    return {"out": (o / z).to(q.dtype), "lse": (m + z.log())[..., 0]}


def _nearest(y, form):
    """y in 64 bits at its nearest code's number, ties to the even code."""
    if form == "int8":
        return y.round().clamp(-127, 127)
    # 8-bit floats: 4 significant bits, exponents from -6 on
    exponent = torch.frexp(y).exponent.clamp_min(-5) - 1
    step = torch.ldexp(torch.ones_like(y), exponent - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def exact(case, seed):
    st = prepare(case, seed)
    form, page, d, hkv = case["format"], case["page"], case["d"], case["hkv"]
    if case["kind"] == "store":
        # the rotation of a pair as the product of complex numbers
        pos = st["pos"].long()
        turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, None]
        half = case["rotary"] // 2
        even = torch.arange(half, device="cuda")
        first, second = (2 * even, 2 * even + 1) if case["interleaved"] else (even, even + half)
        outs = {}
        for name in ("q", "k"):
            x = st[name].double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            outs[name] = x
        outs["v"] = st["v"].double()
        for name in ("k", "v"):
            x = outs[name]
            a = x.abs().amax(-1, keepdim=True)
            outs[name] = _nearest(x * _TOP[form] / a, form) * a / _TOP[form]
        return outs

    # the pool cell by cell: [cells, hkv, d]
    wide = st["k_code"].shape[-1]
    codes = {x: st[x + "_code"].transpose(1, 2).reshape(-1, hkv, wide) for x in ("k", "v")}
    scales = {x: st[x + "_scale"].transpose(1, 2).reshape(-1, hkv) for x in ("k", "v")}

    def stored(name, slot, token):
        """[tokens, hkv, d] of one sequence."""
        where = st["table"][slot].long()[token // page] * page + token % page
        return _numbers(codes[name][where], form)[..., :d].double() * scales[name][where].double()[..., None]

    if case["kind"] == "read":
        own_tokens = st["pos"].long().split(_ints(case["lengths"]))
        return {x: torch.cat([stored(x, slot, token) for slot, token in enumerate(own_tokens)])
                for x in ("k", "v")}
    # one row after another: the codes of its keys laid end to end, one softmax
    n, hq, _ = st["q"].shape
    outs, lses = [], []
    for row, length in enumerate(st["lengths"].tolist()):
        token = torch.arange(length, device="cuda")
        k, v = (stored(x, row, token).transpose(0, 1) for x in ("k", "v"))
        q = st["q"][row].double().view(hkv, -1, d)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()).view(hq, length) / math.sqrt(d)
        if st["selected"] is not None:
            mine = (st["selected"][row][:, :, None] == (token // case["chunk"])).any(1)
            s = torch.where(mine, s, float("-inf"))
        p = torch.softmax(s, dim=-1)
        outs.append(torch.bmm(p.view(hkv, -1, length), v.contiguous()).view(hq, d))
        lses.append(torch.logsumexp(s, dim=-1))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}
