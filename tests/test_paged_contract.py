"""CPU tests of what the paged-cache operators, their prepared step and the
Qwen2 session refuse, and of how they leave things when a part of them fails."""
import pytest
import torch

from moba_hip import RotaryTable, SharedPrefixPlan


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
