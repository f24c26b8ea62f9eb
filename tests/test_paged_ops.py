"""CPU tests of the paged-cache operators: rotary tables, the work plan of
shared-prefix attention, and the refusals that need no device."""
import ctypes
import random

import numpy as np
import pytest
import torch

from moba_hip import RotaryTable, SharedPrefixPlan, append_rotary, shared_prefix_attention
from moba_hip.ops import _lib


# ------------------------------------------------------------- rotary tables
@pytest.mark.parametrize("dim,base,scaling", [(2, 10000.0, 1.0), (64, 1e6, 1.0), (96, 10000.0, 0.5)])
def test_table_angles_are_rounded_once(dim, base, scaling):
    """cos and sin within half an fp32 step of the 64-bit values, also where a
    32-bit angle would be far off."""
    t = RotaryTable(dim, 200001, base=base, scaling=scaling, device="cpu")
    assert t.cos_sin.shape == (200001, dim // 2, 2) and t.cos_sin.dtype == torch.float32
    p = np.array([0, 1, 77, 199999, 200000], dtype=np.float64)
    angle = p[:, None] * base ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    want = np.stack((np.cos(angle), np.sin(angle)), -1) * scaling
    got = t.cos_sin[torch.from_numpy(p).long()].double().numpy()
    # half a step of the value, and 2^-52 of the angle
    assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -50 * angle[..., None] + 1e-30).all()


def test_table_from_tensors_and_frequencies():
    inv = [1.0, 0.25, 0.0625]
    a = RotaryTable(6, 10, inv_freq=inv, device="cpu", interleaved=True)
    ang = torch.arange(10, dtype=torch.float64)[:, None] * torch.tensor(inv, dtype=torch.float64)
    b = RotaryTable.from_cos_sin(ang.cos(), ang.sin(), interleaved=True)
    assert torch.equal(a.cos_sin, b.cos_sin) and b.rotary_dim == 6 and b.interleaved
    assert b.max_positions == 10
    c = RotaryTable.from_cos_sin(ang.cos().requires_grad_(True), ang.sin(), interleaved=True)
    assert torch.equal(c.cos_sin, b.cos_sin) and not c.cos_sin.requires_grad


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=258),
                                dict(max_positions=0), dict(max_positions=2 ** 31), dict(interleaved=1),
                                dict(inv_freq=[1.0, 2.0])])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        RotaryTable(**{"rotary_dim": 8, "max_positions": 4, "device": "cpu", **kw})


@pytest.mark.parametrize("cos,sin", [(torch.ones(3, 2), torch.ones(3, 3)), (None, torch.ones(3, 2)),
                                     (torch.ones(3), torch.ones(3)), (torch.ones(0, 2),) * 2,
                                     (torch.ones(3, 2, dtype=torch.int32),) * 2,
                                     (torch.ones(1, 1).expand(2 ** 31, 1),) * 2])
def test_table_from_tensors_refusals(cos, sin):
    with pytest.raises(ValueError, match="alike"):
        RotaryTable.from_cos_sin(cos, sin)


# ------------------------------------------------------------------ the plan
def _covered(plan, prefix, length, suffix):
    """Checks that every range of every (row, head) is one item's, that a
    row's partials are dense, and that an item's rows share its keys."""
    flat = plan.meta.numpy()
    every = flat[:plan._rows_at // 4].reshape(-1, 8)
    items = list(every[:plan.n_items])
    used = set()
    for x in list(items):     # the items of single waves
        if x[2] < 0:
            mine = range(x[0], x[0] + 4)
            assert x[0] >= plan.n_items and not used.intersection(mine)
            used.update(mine)
            items += list(every[mine.start:mine.stop])
    assert len(used) == len(every) - plan.n_items
    n, hkv = plan.rows, plan.num_kv_heads
    g = plan.num_q_heads // hkv
    rows = flat[plan._rows_at // 4:plan._parts_at // 4]
    part_at, own_at, n_part = flat[plan._parts_at // 4:].reshape(3, n)
    n_prefix = own_at - part_at
    assert part_at[0] == 0 and (np.diff(part_at) == n_part[:-1]).all()
    assert part_at[-1] + n_part[-1] == plan.parts
    seen = np.zeros((plan.parts, plan.num_q_heads), np.int64)
    for row_at, m0, n_m, slot, kh, packed, tokens, only in items:
        if n_m <= 0:
            continue
        split, splits = packed & 0xffff, packed >> 16
        its = {rows[row_at + m // g] for m in range(m0, m0 + n_m)}
        assert its == {only} if only >= 0 else len(its) > 1
        assert n_m <= 128 and 0 <= split < splits and 0 <= kh < hkv
        for m in range(m0, m0 + n_m):
            row, h = rows[row_at + m // g], kh * g + m % g
            if tokens >= 0:
                assert (slot, tokens) == (prefix[row], length[row]) and splits == n_prefix[row]
                at = part_at[row] + split
            else:
                assert slot == suffix[row] and splits == n_part[row] - n_prefix[row]
                at = part_at[row] + n_prefix[row] + split
            seen[at, h] += 1
    assert (seen == 1).all()
    for r in range(n):
        assert (n_prefix[r] > 0) == (length[r] > 0)
        assert (n_part[r] > n_prefix[r]) == (suffix[r] >= 0 and plan.max_suffix > 0)


@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (16, 1, 96), (8, 8, 64), (96, 1, 40), (16, 4, 256)])
@pytest.mark.parametrize("seed", range(10))
def test_plan_covers_every_range_once(hq, hkv, d, seed):
    rng = random.Random(seed)
    n = rng.choice([1, 2, 7, 40, 130, 600])
    prefix = [rng.choice([-1, 0, 1, 1]) for _ in range(n)]
    length = [0 if p < 0 else rng.choice([0, 1, 63, 64, 65, 5000, 40000]) for p in prefix]
    suffix = [rng.choice([-1, 3, 4 + i, 4 + i, 4 + i]) for i in range(n)]
    plan = SharedPrefixPlan(prefix, length, suffix, hq, hkv, d,
                            max_suffix=rng.choice([0, 1, 64, 3000]), device="cpu")
    _covered(plan, prefix, length, suffix)
    assert plan.max_prefix == max(length)


def test_plan_of_nothing():
    plan = SharedPrefixPlan([-1, -1], [0, 0], [-1, -1], 2, 1, 64, max_suffix=5, device="cpu")
    assert plan.n_items == 0 and plan.parts == 0 and plan.max_slot == -1


@pytest.mark.parametrize("kw", [
    dict(prefix_ids=[]), dict(prefix_ids=[0.5]), dict(prefix_ids=[-2]), dict(prefix_lengths=[1, 2]),
    dict(prefix_lengths=[-1]), dict(prefix_ids=[-1]), dict(suffix_ids=[[0]]), dict(num_q_heads=3),
    dict(num_kv_heads=0), dict(head_dim=60), dict(head_dim=264), dict(max_suffix=-1),
    dict(max_suffix=True), dict(max_suffix=2 ** 31), dict(max_suffix=2 ** 30 + 1),
    dict(prefix_lengths=[2 ** 30 + 1]), dict(suffix_ids=[2 ** 31])])
def test_plan_refusals(kw):
    base = dict(prefix_ids=[0], prefix_lengths=[5], suffix_ids=[1], num_q_heads=4, num_kv_heads=2,
                head_dim=64, max_suffix=8, device="cpu")
    with pytest.raises(ValueError):
        SharedPrefixPlan(**{**base, **kw})


# ------------------------------------------------- refusals without a device
def test_host_tensors_are_refused():
    c = torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16)
    k = torch.zeros(1, 1, 8, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        append_rotary(k, k, c, c, table, i, i, RotaryTable(8, 4, device="cpu"))
    plan = SharedPrefixPlan([0], [1], [0], 1, 1, 8, max_suffix=1, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        shared_prefix_attention(k, c, c, table, i, plan)


def _refused(name, base, change, text):
    args = dict(base, **change)
    lib = _lib.load()
    assert getattr(lib, name)(*args.values()) == _lib.MOBA_ERR_ARG
    assert text in lib.moba_hip_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(N=0), "nonempty"), (dict(D=257), "[1,256]"),
    (dict(rotary_dim=3), "even"), (dict(rotary_dim=66), "even"), (dict(max_pos=0), "even"),
    (dict(pages=0), "pool"), (dict(width=0), "pool"), (dict(hq=1), "go together"),
    (dict(q=64), "go together"), (dict(N=1 << 24, hkv=8), "2^31"), (dict(cos=8), "aligned")])
def test_append_entry_refuses_before_any_device_work(change, text):
    base = dict(q=None, q_ts=0, q_hs=0, k=64, k_ts=64, k_hs=64, v=64, v_ts=64, v_hs=64, dtype=0, N=1,
                hq=0, hkv=1, D=64, cos=64, max_pos=4, rotary_dim=64, inter=0, kc=64, vc=64, pages=1,
                page=16, table=64, B=1, width=1, seq=64, pos=64, offsets=None, q_out=None,
                status=None, stream=None)
    _refused("moba_hip_append_rotary", base, change, text)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "dtype"), (dict(D=12), "multiple of 8"), (dict(D=264), "multiple of 8"),
    (dict(Nq=0), "Nq"), (dict(hq=3), "multiple of Hkv"), (dict(Nq=1 << 30, hq=8), "Nq"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(pages=1 << 28), "pool"), (dict(page=0), "pool"), (dict(width=1 << 28), "pool"),
    (dict(max_length=-1), "max_length"), (dict(max_length=17), "max_length"),
    (dict(max_length=(1 << 30) + 1, width=(1 << 27) - 1), "max_length"), (dict(hq=1 << 24, hkv=1 << 24), "Hkv")])
def test_attention_entry_refuses_before_any_device_work(change, text):
    base = dict(q=64, dtype=0, Nq=1, hq=2, hkv=2, D=64, scale=1.0, kc=64, vc=64, pages=1, page=16,
                table=64, width=1, lengths=64, add=0, max_length=16, items=64, n_items=0,
                rows=64, parts=64, max_parts=1, uneven=0,
                part_o=64, part_ml=64, out=64, lse=64, stream=None)
    _refused("moba_hip_shared_attention", base, change, text)
