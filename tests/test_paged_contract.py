"""CPU tests of what the paged-cache operators, their prepared step and the
Qwen2 session refuse, and of how they leave things when a part of them fails."""
import contextlib
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from moba_hip import PreparedSharedDecode, RotaryTable, SharedPrefixPlan, prepared_decode
from moba_hip.ops import _lib
from moba_hip.shared_prefix import _scale


# ------------------------------------------------------------- rotary tables
REPLACED = {
    "16 bits": lambda t: t.half(),
    "64 bits": lambda t: t.double(),
    "flat": lambda t: t.flatten(1),
    "strided": lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
    "fewer pairs": lambda t: t[:, :2].contiguous(),
    "cos alone": lambda t: t[..., :1].contiguous(),
    "no rows": lambda t: t[:0],
    "no tensor": lambda t: t.tolist(),
    "misaligned": lambda t: torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape),
}


@pytest.mark.parametrize("how", REPLACED)
def test_replaced_rotary_table_is_checked(how):
    """A kernel reads what ``cos_sin`` holds at the call, so that is what a call tests."""
    t = RotaryTable(8, 6, device="cpu")
    t._check(64, torch.device("cpu"))
    t.cos_sin = REPLACED[how](t.cos_sin)
    with pytest.raises(ValueError, match="cos_sin must be"):
        t._check(64, torch.device("cpu"))


def test_rotary_table_length_is_that_of_its_rows():
    t = RotaryTable(8, 6, device="cpu")
    t.cos_sin = t.cos_sin[:4]
    assert t.max_positions == 4
    t._check(8, torch.device("cpu"))
    with pytest.raises(ValueError, match="exceeds head_dim"):
        t._check(6, torch.device("cpu"))
    with pytest.raises(ValueError, match="cache's device"):
        t._check(8, torch.device("cuda", 0))


# ------------------------------------------------------------------ the plan
RECORDS = {
    "64 bits": lambda t: t.long(),
    "cut": lambda t: t[:-1],
    "longer": lambda t: torch.cat((t, t[:1])),
    "2D": lambda t: t[None],
    "strided": lambda t: torch.stack((t, t), 1)[:, 0],
    "no tensor": lambda t: t.tolist(),
    "misaligned": lambda t: torch.cat((t.new_zeros(1), t))[1:],
}


@pytest.mark.parametrize("how", RECORDS)
def test_replaced_records_of_a_plan_are_checked(how):
    plan = SharedPrefixPlan([0, 0, -1], [70, 70, 0], [1, 2, 2], 4, 2, 64, max_suffix=9, device="cpu")
    plan._check()
    plan.meta = RECORDS[how](plan.meta)
    with pytest.raises(ValueError, match="plan.meta must be"):
        plan._check()


# ------------------------------------------------------------------- the scale
SCALES = [0.0, -1.0, 1e-46, 1e-39, 1.1e30, 1e39, float("inf"), float("nan")]


@pytest.mark.parametrize("scale", SCALES)
def test_scales_that_fp32_does_not_hold_are_refused(scale):
    with pytest.raises(ValueError, match="scale must be"):
        _scale(scale)
    lib = _lib.load()
    args = dict(q=64, dtype=0, Nq=1, hq=2, hkv=2, D=64, scale=scale, kc=64, vc=64, pages=1, page=16,
                table=64, width=1, lengths=64, add=0, max_length=16, items=64, n_items=0, rows=64,
                parts=64, max_parts=1, uneven=0, part_o=64, part_ml=64, out=64, lse=64, stream=None)
    assert lib.moba_hip_shared_attention(*args.values()) == _lib.MOBA_ERR_ARG
    assert "scale" in lib.moba_hip_last_error().decode()


def test_scales_at_the_border():
    assert _scale(2.0 ** -126) == 2.0 ** -126 and _scale(1) == 1.0 and _scale(1e30) == 1e30


# ------------------------------------------------------ failures inside a step
class _Stop(BaseException):
    pass


@pytest.mark.parametrize("where", ["upload", "copy", "launch", "replay", "commit"])
@pytest.mark.parametrize("error", [RuntimeError, _lib.MobaHipError, _Stop])
def test_a_step_that_fails_marks_its_lease(monkeypatch, where, error):
    """Between its plan and its commit a step may leave the device ahead of the
    host: such a lease is done with, and its cache when the lease is closed."""
    def fail(*a, **k):
        raise error(where)

    def maybe(name):
        return fail if where == name else (lambda *a, **k: None)

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: SimpleNamespace(cuda_stream=0))
    monkeypatch.setattr(prepared_decode, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(torch.Tensor, "pin_memory", maybe("upload"))
    monkeypatch.setattr(_lib, "call", maybe("launch"))
    plan = PreparedSharedDecode.__new__(PreparedSharedDecode)
    step = SimpleNamespace(positions=(0,), updates=(1,) if where == "upload" else (),
                           delta=np.zeros((2, 1), np.int32))
    plan.cache = SimpleNamespace(_lock=contextlib.nullcontext(), device=torch.device("cpu"), _stream=0,
                                 _lessee=plan, _broken=False)
    plan._lease = SimpleNamespace(plan=lambda: step, commit=maybe("commit"))
    plan._dev, plan._handle, plan.max_length, plan.rotary = 0, None, 4, None
    plan._delta_uploads = 0
    plan._uploaded = plan.closed = plan.failed = plan.check_finite = False
    plan._calls, plan.delta = [("entry", ())], torch.zeros((2, 1), dtype=torch.int32)
    plan._graph = SimpleNamespace(replay=maybe("replay"))
    plan.ids, plan.dense = (0,), True
    plan.output = plan.lse = None
    plan.q, plan.k, plan.v = (torch.zeros(1, 1, 8) for _ in range(3))
    q = SimpleNamespace()
    monkeypatch.setattr(plan, "_bind_all",
                        lambda specs: [(q, SimpleNamespace(copy_=maybe("copy")))], raising=False)
    with pytest.raises(error, match=where):
        plan.step(q, q, q, use_graph=where == "replay")
    assert plan.failed
    with pytest.raises(RuntimeError, match="discard prepared decode"):
        plan.step(q, q, q)
    plan.close()
    assert plan.cache._broken and plan.closed


# -------------------------------------------------------------- Qwen2 session
ROPE = {
    "default": {},
    "linear": dict(factor=2.0),
    "yarn": dict(factor=4.0),
    "llama3": dict(factor=4.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=64),
    "dynamic": dict(factor=2.0),
    "longrope": dict(short_factor=[1.0] * 32, long_factor=[3.0] * 32,
                     original_max_position_embeddings=64),
}


def qwen2_model(rope="default", device="cpu", max_positions=128):
    from transformers import Qwen2Config, Qwen2ForCausalLM
    torch.manual_seed(0)
    cfg = Qwen2Config(vocab_size=256, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=max_positions, attn_implementation="eager",
                      rope_parameters={"rope_type": rope, "rope_theta": 10000.0, **ROPE[rope]})
    m = Qwen2ForCausalLM(cfg).to(device, torch.bfloat16).eval()
    for p in m.parameters():
        p.requires_grad_(False)
    return m


@pytest.mark.parametrize("rope", ROPE)
def test_frequencies_that_depend_on_the_length_are_refused(rope):
    """The session's angles are one table, made when it is: of the rope types
    only those that keep their frequencies past the original length pass."""
    from moba_hip.qwen2 import Qwen2Branches
    model = qwen2_model(rope)
    emb = model.model.rotary_emb
    before = emb.inv_freq.clone()
    emb(torch.zeros(1, 300, 256), torch.arange(300)[None])
    fixed = torch.equal(before, emb.inv_freq)
    assert fixed == (rope not in ("dynamic", "longrope"))
    with pytest.raises(ValueError, match="CUDA model required" if fixed else "rope type"):
        Qwen2Branches(model, 64, 2, 8)


def _branches(monkeypatch, caches, backend="eager"):
    """A session of two branches on stand-ins for its caches."""
    from moba_hip.qwen2 import Qwen2Branches
    monkeypatch.setattr(Qwen2Branches, "_check", lambda self: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: SimpleNamespace(cuda_stream=0))
    s = Qwen2Branches.__new__(Qwen2Branches)
    s.caches, s.branches, s.new_tokens, s.hq, s.rotary = caches, 2, 8, 4, None
    s.device, s.backend, s.tokens = torch.device("cpu"), backend, torch.zeros((2, 1), dtype=torch.long)
    s.plans, s.graph, s.closed, s.failed, s.logits = [], None, False, False, None
    s.model = SimpleNamespace(config=SimpleNamespace(vocab_size=9))
    return s


@pytest.mark.parametrize("error", [RuntimeError, _Stop])
def test_a_session_step_that_fails_marks_every_lease(monkeypatch, error):
    def fail():
        raise error("step")
    s = _branches(monkeypatch, [])
    s.plans = [SimpleNamespace(_plan_step=lambda stream: None, failed=False) for _ in range(3)]
    monkeypatch.setattr(s, "_compute_step", fail, raising=False)
    with pytest.raises(error, match="step"):
        s.step([1, 2])
    assert s.failed and all(p.failed for p in s.plans)


@pytest.mark.parametrize("fails", [0, 2, "capture"])
@pytest.mark.parametrize("error", [ValueError, _Stop])
def test_a_session_that_cannot_be_prepared_keeps_no_lease(monkeypatch, fails, error):
    """A failure at any layer, or in the capture, gives back what was leased
    before it; the session can be prepared again."""
    leased = set()

    def lease(i):
        def make(*a, **k):
            if fails == i:
                raise error("prepare")
            assert i not in leased
            leased.add(i)
            return SimpleNamespace(close=lambda: leased.remove(i))
        return make

    def capture():
        if fails == "capture":
            raise error("prepare")
    s = _branches(monkeypatch, [SimpleNamespace(lengths=(5, 0, 0), prepare_shared_decode=lease(i))
                                for i in range(3)], "model_graph")
    monkeypatch.setattr(s, "_capture", capture, raising=False)
    with pytest.raises(error, match="prepare"):
        s.prepare()
    assert not leased and not s.plans and s.graph is None
    with pytest.raises(ValueError, match="prepare first"):
        s.step([1, 2])
    fails = None
    s.prepare()
    assert leased == {0, 1, 2} and len(s.plans) == 3
    s.close()
    assert not leased


@pytest.mark.parametrize("kw,match", [(dict(page=0), "page_size"), (dict(page=None), "page_size"),
                                      (dict(page=16.0), "page_size"), (dict(branches=0), "branches"),
                                      (dict(new_tokens=True), "new_tokens"), (dict(chunk=-1), "chunk"),
                                      (dict(capacity="9"), "capacity"), (dict(backend="graph"), "backend")])
def test_sizes_of_a_session_are_checked(kw, match):
    """Before anything is divided by them or asked of a device."""
    from moba_hip.qwen2 import Qwen2Branches
    with pytest.raises(ValueError, match=match):
        Qwen2Branches(qwen2_model(), **{"capacity": 64, "branches": 2, "new_tokens": 8, **kw})
