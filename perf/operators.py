"""Operators of serving from a paged KV cache: their cases, their plain forms
and the calls a user's program makes of them.

Kinds of case (``case["kind"]``):

* ``append``  new keys and values are rotated by their positions and written
              into the page pool; the queries of the same tokens are rotated on
              the way.  The inputs are views of one projection's output
              ``[tokens, (Hq + 2 Hkv) D]``.
* ``attend``  every query attends the prefix that its batch shares and then
              its own sequence's tokens up to its position; both lie in the
              page pool.

``lengths`` (append) holds the new tokens of each sequence as text;
``prefixes`` and ``rows`` (attend) hold the length of each shared prefix and
the number of sequences behind it (length 0: sequences with no prefix).
``own`` selects the framework's kernels; the plain forms need torch alone.
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


def _framework():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import moba_hip
    return moba_hip


def listed():
    return [
        # One decode step of 8 requests, Qwen2-1.5B attention shape, pages of 48
        # tokens: a launch's latency is what the step pays.
        dict(name="append_step_b8", kind="append", lengths=",".join(["1"] * 8), context=2000,
             hq=12, hkv=2, d=128, rotary=128, interleaved=False, page=48, dtype="bf16"),
        # One decode step of a full serving batch, fp16, 96-dim heads of one
        # kv head.
        dict(name="append_step_mqa_b256", kind="append", lengths=",".join(["1"] * 256),
             context=500, hq=16, hkv=1, d=96, rotary=96, interleaved=False, page=64,
             dtype="fp16"),
        # A 32K-token prompt written into an empty slot, 8 kv heads.
        dict(name="append_prompt_32k", kind="append", lengths="32768", context=0, hq=32, hkv=8,
             d=128, rotary=128, interleaved=False, page=16, dtype="bf16"),
        # A packed batch of prompts of ragged lengths (Qwen2-0.5B heads), pairs
        # of neighbouring dims rotated.
        dict(name="append_ragged", kind="append", lengths="5003,311,4097,1,2049,777", context=30,
             hq=14, hkv=2, d=64, rotary=64, interleaved=True, page=16, dtype="fp16"),
        # Wide heads of which the first quarter is rotated.
        dict(name="append_partial_8k", kind="append", lengths="4099,4093", context=0, hq=16,
             hkv=4, d=256, rotary=64, interleaved=False, page=64, dtype="bf16"),
        # Decode of 8 continuations of one 2K prompt, first tokens: latency.
        dict(name="shared_b8_2k", kind="attend", prefixes="2048", rows="8", tokens=1, lo=1,
             hi=200, mix=1, hq=12, hkv=2, d=128, page=48, dtype="bf16"),
        # A system prompt of 16K tokens before 32 conversations, one kv head.
        dict(name="shared_mqa_b32_16k", kind="attend", prefixes="16384", rows="32", tokens=1,
             lo=64, hi=2048, mix=2, hq=16, hkv=1, d=96, page=64, dtype="fp16"),
        # A long document before 64 conversations, 8 kv heads: cache reads of
        # the conversations and products of the document are alike in weight.
        dict(name="shared_b64_32k", kind="attend", prefixes="32768", rows="64", tokens=1, lo=64,
             hi=2048, mix=3, hq=32, hkv=8, d=128, page=16, dtype="bf16"),
        # Sampling at scale: 256 continuations of one document, bound by the
        # products.
        dict(name="shared_b256_32k", kind="attend", prefixes="32768", rows="256", tokens=1, lo=1,
             hi=512, mix=4, hq=32, hkv=8, d=128, page=16, dtype="bf16"),
        # Two continuations of a very long context: one long read, few rows.
        dict(name="shared_b2_128k", kind="attend", prefixes="131071", rows="2", tokens=1, lo=1,
             hi=300, mix=5, hq=14, hkv=2, d=64, page=16, dtype="bf16"),
        # Five prompts shared by unequal parts of a batch, some requests on
        # their own.
        dict(name="shared_groups", kind="attend", prefixes="5003,311,12289,1,0,2049",
             rows="7,13,21,3,9,1", tokens=1, lo=1, hi=1500, mix=6, hq=28, hkv=4, d=64, page=16,
             dtype="fp16"),
        # 8 questions of 128 tokens put to one document at once, wide heads.
        dict(name="shared_extend_d256", kind="attend", prefixes="8192", rows="8", tokens=128,
             lo=128, hi=128, mix=7, hq=16, hkv=4, d=256, page=64, dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hq, hkv = rng.choice([(12, 2), (16, 1), (32, 8), (14, 2), (28, 4), (16, 4), (8, 8), (32, 32),
                          (6, 3), (48, 1)])
    d = rng.choice([64, 64, 96, 128, 128, 128, 192, 256, 40, 80])
    page = rng.choice([16, 16, 48, 64, 1, 100, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if rng.random() < 0.4:
            if rng.random() < 0.5:
                lengths = [rng.choice([1, 1, 1, 2, 5]) for _ in range(log(1, 512))]
            else:
                tokens = log(16, 32768)
                cuts = sorted(rng.sample(range(1, tokens), min(tokens - 1, rng.choice([0, 1, 5]))))
                lengths = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
            rotary = rng.choice([d, d, d, d // 2, d // 4 - d // 4 % 2, 2])
            case = dict(kind="append", lengths=",".join(map(str, lengths)),
                        context=rng.choice([0, log(1, 1000)]), hq=hq, hkv=hkv, d=d, rotary=rotary,
                        interleaved=rng.random() < 0.4, page=page, dtype=dtype)
            if work(case)["bytes"] <= 8e8:
                return case
            continue
        groups = rng.choice([1, 1, 1, 2, 5])
        tokens = rng.choice([1, 1, 1, 1, 3, 64])
        prefixes = [rng.choice([log(16, 131072), log(16, 131072), 0, 1]) for _ in range(groups)]
        if not any(prefixes):
            prefixes[0] = log(16, 131072)
        rows = [log(1, 256) for _ in range(groups)]
        hi = max(tokens, log(1, 2048))
        case = dict(kind="attend", prefixes=",".join(map(str, prefixes)),
                    rows=",".join(map(str, rows)), tokens=tokens, lo=min(hi, tokens), hi=hi,
                    mix=rng.randrange(1 << 20), hq=hq, hkv=hkv, d=d, page=page, dtype=dtype)
        w = work(case)
        # within the largest listed cases: operations, bytes of the pool, rows
        if w["flops"] <= 1.3e11 and w["bytes"] <= 5e8 and sum(rows) * tokens * hq <= 1 << 15:
            return case


def _ints(text):
    return [int(x) for x in text.split(",")]


def _sequences(case):
    """(prefix index, own length) of every sequence of an attend case."""
    rng = random.Random(case["mix"])
    return [(g if p else -1, rng.randint(case["lo"], case["hi"]))
            for g, (p, n) in enumerate(zip(_ints(case["prefixes"]), _ints(case["rows"])))
            for _ in range(n)]


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "append":
        lengths = _ints(case["lengths"])
        n, r = sum(lengths), case["rotary"]
        # q, k and v in and out, the table's rows of the distinct positions,
        # (sequence, position) of each token
        rows = max(lengths) if max(lengths) > 1 else n
        return {"bytes": n * (2 * hq + 4 * hkv) * d * 2 + rows * r * 4 + n * 8,
                "flops": n * (hq + hkv) * r * 3}
    prefixes, seqs, t = _ints(case["prefixes"]), _sequences(case), case["tokens"]
    rows = len(seqs) * t
    pairs = sum(t * (prefixes[g] if g >= 0 else 0) + t * n - t * (t - 1) // 2 for g, n in seqs)
    keys = sum(prefixes) + sum(n for _, n in seqs)
    return {"bytes": 2 * rows * hq * d * 2 + rows * hq * 4 + keys * hkv * d * 4,
            "flops": 4 * pairs * hq * d}


def _randn(gen, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _page_table(lengths, page, width, seed):
    """Pages of a pool in random order, dealt to the sequences; -1: no page."""
    counts = [-(-n // page) for n in lengths]
    pages = list(range(sum(counts)))
    random.Random(seed).shuffle(pages)
    table, at = [], 0
    for c in counts:
        table.append(pages[at:at + c] + [-1] * (width - c))
        at += c
    return torch.tensor(table, dtype=torch.int32, device="cuda"), at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPE[case["dtype"]]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    st = dict(case=case)
    if case["kind"] == "append":
        lengths = _ints(case["lengths"])
        rng = random.Random(seed)
        context = [rng.randint(0, case["context"]) for _ in lengths]
        capacity = [case["context"] + n for n in lengths]
        st["table"], pages = _page_table(capacity, page, -(-max(capacity) // page), seed)
        st["k_cache"] = _randn(gen, pages, page, hkv, d, dtype=dtype)
        st["v_cache"] = _randn(gen, pages, page, hkv, d, dtype=dtype)
        n = sum(lengths)
        qkv = _randn(gen, n, hq + 2 * hkv, d, dtype=dtype)
        st["q"], st["k"], st["v"] = qkv.split([hq, hkv, hkv], dim=1)
        st["seq"] = torch.tensor([s for s, m in enumerate(lengths) for _ in range(m)],
                                 dtype=torch.int32, device="cuda")
        st["pos"] = torch.tensor([c + i for c, m in zip(context, lengths) for i in range(m)],
                                 dtype=torch.int32, device="cuda")
        half = case["rotary"] // 2
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(max(capacity), dtype=torch.float64, device="cuda")[:, None] * inv
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        if own:
            st["rotary"] = _framework().RotaryTable.from_cos_sin(
                st["cos"], st["sin"], interleaved=case["interleaved"])
        return st
    prefixes, seqs, t = _ints(case["prefixes"]), _sequences(case), case["tokens"]
    lengths = prefixes + [n for _, n in seqs]
    st["table"], pages = _page_table(lengths, page, -(-max(lengths) // page), seed)
    st["k_cache"] = _randn(gen, pages, page, hkv, d, dtype=dtype)
    st["v_cache"] = _randn(gen, pages, page, hkv, d, dtype=dtype)
    # scores of deviation 2: a few keys of thousands hold most of the weight
    st["q"] = _randn(gen, len(seqs) * t, hq, d, dtype=dtype, scale=2.0)
    st["prefix_ids"] = [g for g, _ in seqs for _ in range(t)]
    st["prefix_lengths"] = [prefixes[g] if g >= 0 else 0 for g in st["prefix_ids"]]
    st["suffix_ids"] = [len(prefixes) + i for i in range(len(seqs)) for _ in range(t)]
    st["limits"] = [n - t + 1 + i for _, n in seqs for i in range(t)]
    st["suffix_lengths"] = torch.tensor(st["limits"], dtype=torch.int32, device="cuda")
    if own:
        st["plan"] = _framework().SharedPrefixPlan(
            st["prefix_ids"], st["prefix_lengths"], st["suffix_ids"], hq, hkv, d,
            max_suffix=case["hi"], device="cuda")
    return st


def run(state):
    if state["case"]["kind"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def _append_own(st):
    q = _framework().append_rotary(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"],
                                   st["seq"], st["pos"], st["rotary"], q=st["q"])
    return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


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


def _append_plain(st):
    pos, seq = st["pos"].long(), st["seq"].long()
    page = st["k_cache"].shape[1]
    phys, off = st["table"][seq, pos // page].long(), pos % page
    cos, sin = st["cos"][pos], st["sin"][pos]
    inter = st["case"]["interleaved"]
    st["k_cache"][phys, off] = _rotated(st["k"].float(), cos, sin, inter).to(st["k"].dtype)
    st["v_cache"][phys, off] = st["v"]
    q = _rotated(st["q"].float(), cos, sin, inter).to(st["q"].dtype)
    return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _attend_own(st):
    out, lse = _framework().shared_prefix_attention(
        st["q"], st["k_cache"], st["v_cache"], st["table"], st["suffix_lengths"], st["plan"])
    return {"out": out, "lse": lse}


def _gather(cache, table, slots, tokens):
    """[slots, tokens, heads, d] of the pool in 32 bits (masked tokens: any)."""
    page = cache.shape[1]
    t = torch.arange(tokens, device=cache.device)
    phys = table[slots][:, t // page].long().clamp_min(0)
    return cache[phys, t % page].float()


def _attend_plain(st):
    case, q = st["case"], st["q"]
    n, hq, d = q.shape
    hkv = case["hkv"]
    g = hq // hkv
    qs = (q.float() * d ** -0.5).view(n, hkv, g, d)
    # scores of each row's own tokens, masked behind its length
    hi = max(st["limits"])
    slots = torch.tensor(st["suffix_ids"], device="cuda")
    ks = _gather(st["k_cache"], st["table"], slots, hi).permute(0, 2, 3, 1)   # [n, hkv, d, hi]
    ss = torch.matmul(qs, ks)
    dead = torch.arange(hi, device="cuda") >= st["suffix_lengths"][:, None]
    ss = ss.masked_fill(dead[:, None, None], float("-inf"))
    vs = _gather(st["v_cache"], st["table"], slots, hi).transpose(1, 2)       # [n, hkv, hi, d]
    out = torch.empty((n, hkv, g, d), device="cuda")
    lse = torch.empty((n, hkv, g), device="cuda")
    groups = {}
    for row, key in enumerate(zip(st["prefix_ids"], st["prefix_lengths"])):
        groups.setdefault(key, []).append(row)
    for (slot, length), rows in groups.items():
        rows = torch.tensor(rows, device="cuda")
        own_s, own_v = ss[rows], vs[rows]
        if length:
            one = torch.tensor([slot], device="cuda")
            kp = _gather(st["k_cache"], st["table"], one, length)[0]
            vp = _gather(st["v_cache"], st["table"], one, length)[0]
        for h in range(hkv):
            s = own_s[:, h]                                                   # [rows, g, hi]
            m = s.amax(-1)
            if length:
                sp = torch.matmul(qs[rows, h].reshape(-1, d), kp[:, h].t().contiguous())
                m = torch.maximum(m, sp.amax(-1).view(m.shape))
            p = torch.exp(s - m[..., None])
            z, o = p.sum(-1), torch.matmul(p, own_v[:, h])
            if length:
                pp = torch.exp(sp - m.view(-1, 1))
                z = z + pp.sum(-1).view(z.shape)
                o = o + torch.matmul(pp, vp[:, h]).view(o.shape)
            out[rows, h] = o / z[..., None]
            lse[rows, h] = m + z.log()
    return {"out": out.view(n, hq, d).to(q.dtype), "lse": lse.view(n, hq)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
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
        page = case["page"]
        cell = st["table"][st["seq"].long(), pos // page].long() * page + pos % page
        caches = {}
        for name, x in (("k_cache", outs["k"]), ("v_cache", st["v"].double())):
            c = st[name].double()
            c.view(-1, case["hkv"], case["d"]).index_copy_(0, cell, x)
            caches[name] = c
        return {"q": outs["q"], **caches}
    # one row after another: its keys laid end to end, one softmax over them
    page, table = case["page"], st["table"].long()
    flat_k = st["k_cache"].view(-1, case["hkv"], case["d"])
    flat_v = st["v_cache"].view(-1, case["hkv"], case["d"])

    def cells(slot, length):
        t = torch.arange(length, device="cuda")
        return table[slot, t // page] * page + t % page

    n, hq, d = st["q"].shape
    outs, lses, last, cached = [], [], None, None
    for row in range(n):
        key = (st["prefix_ids"][row], st["prefix_lengths"][row])
        if key != last:
            c = cells(*key) if key[1] else torch.zeros(0, dtype=torch.long, device="cuda")
            cached = (flat_k[c].double().permute(1, 2, 0).contiguous(),
                      flat_v[c].double().transpose(0, 1).contiguous())
            last = key
        c = cells(st["suffix_ids"][row], st["limits"][row])
        q = st["q"][row].double().view(case["hkv"], -1, d)
        own_k = flat_k[c].double().permute(1, 2, 0).contiguous()
        s = torch.cat((torch.bmm(q, cached[0]), torch.bmm(q, own_k)), dim=-1) / math.sqrt(d)
        p = torch.softmax(s, dim=-1)
        m = key[1]
        own_v = flat_v[c].double().transpose(0, 1).contiguous()
        o = torch.bmm(p[..., :m].contiguous(), cached[1]) + torch.bmm(p[..., m:].contiguous(), own_v)
        outs.append(o.view(hq, d))
        lses.append(torch.logsumexp(s, dim=-1).view(hq))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}
