"""CPU tests of the 8-bit cache: shapes of a pool, what its operators, cache and session
refuse, and how a lease that fails is left."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from moba_hip import (PreparedQuantizedDecode, QuantizedKVCache, QuantizedPages, prepared_decode,
                      quantized_append, quantized_attention, quantized_read)
from moba_hip.ops import _lib
from moba_hip.qwen2 import Qwen2Session


@pytest.mark.parametrize("fmt,dtype", [("int8", torch.int8), ("fp8", torch.float8_e4m3fn)])
@pytest.mark.parametrize("d,width", [(8, 16), (16, 16), (40, 48), (128, 128), (200, 208), (256, 256)])
def test_pool_shapes(fmt, dtype, d, width):
    p = QuantizedPages.empty(3, 5, 2, d, format=fmt, device="cpu")
    assert p.k.shape == p.v.shape == (3, 2, 5, width) and p.k.dtype == p.v.dtype == dtype
    assert p.k_scale.shape == p.v_scale.shape == (3, 2, 5) and p.k_scale.dtype == torch.float32
    assert p.format == fmt and p.head_dim == d


@pytest.mark.parametrize("kw", [dict(format="int4"), dict(format=None), dict(num_pages=0), dict(page_size=True),
                                dict(num_kv_heads=-1), dict(head_dim=0), dict(head_dim=12),
                                dict(head_dim=264), dict(num_pages=2 ** 27, page_size=16),
                                dict(num_pages=2 ** 22, page_size=16, num_kv_heads=8, head_dim=256)])
def test_pool_refusals(kw):
    with pytest.raises(ValueError):
        QuantizedPages.empty(**{"num_pages": 2, "page_size": 4, "num_kv_heads": 2, "head_dim": 64,
                                "device": "cpu", **kw})


def test_operators_need_a_device():
    p = QuantizedPages.empty(3, 5, 2, 64, device="cpu")
    table, index = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: quantized_append(x, x, p, table, index, index),
                 lambda: quantized_read(p, table, index, index),
                 lambda: quantized_attention(x, p, table, index, index)):
        with pytest.raises(ValueError, match="must be CUDA"):
            call()
    with pytest.raises(ValueError, match="must be QuantizedPages"):
        quantized_read(tuple(p), table, index, index)


# ------------------------------------------------------------------- the C-ABI
POOL = dict(k=64, v=64, ks=64, vs=64, pages=4, page=16)
TABLE = dict(table=64, B=2, width=2)
APPEND = dict(q=None, q_ts=0, q_hs=0, k=64, k_ts=128, k_hs=64, v=64, v_ts=128, v_hs=64, dtype=0, N=1, Hq=0,
              Hkv=2, D=64, cs=None, max_pos=0, rotary=0, inter=0, format=0, kc=64, vc=64, ks=64, vs=64,
              pages=4, page=16, **TABLE, seq=64, pos=64, offsets=None, q_out=None, status=None, stream=None)
READ = dict(format=0, **POOL, Hkv=2, D=64, **TABLE, seq=64, pos=64, N=1, dtype=0, k_out=64, v_out=64,
            status=None, stream=None)
MEANS = dict(format=0, k=64, ks=64, pages=4, page=16, Hkv=2, D=64, **TABLE, seq=64, chunk_or_pos=64, n=1,
             mode=0, chunk=8, dtype=0, means=64, max_chunks=4, stream=None)
ATTEND = dict(q=64, dtype=0, Nq=1, Hq=4, Hkv=2, D=64, scale=1.0, format=0, **POOL, **TABLE, q_seq=64,
              lengths=64, add=0, max_length=32, selected=None, slots=0, chunk=0, work=64, out=64, lse=64,
              stream=None)
BAD_POOL = [dict(format=2), dict(D=60), dict(D=264), dict(D=0), dict(Hkv=0), dict(pages=0), dict(page=0),
            dict(B=0), dict(width=0), dict(pages=2 ** 27), dict(width=2 ** 27),
            dict(pages=2 ** 26, Hkv=64, D=256)]


def _refused(name, base, change, word=""):
    lib = _lib.load()
    args = {**base, **change}
    assert list(args) == list(base)
    assert getattr(lib, name)(*args.values()) == _lib.MOBA_ERR_ARG, change
    assert word in lib.moba_hip_last_error().decode()


@pytest.mark.parametrize("change", BAD_POOL + [
    dict(kc=72), dict(vs=66), dict(dtype=2), dict(N=0), dict(Hq=-1), dict(Hq=2), dict(q=64), dict(q_out=64),
    dict(Hq=2, q=64, q_out=64), dict(cs=64, rotary=0, max_pos=4), dict(cs=64, rotary=66, max_pos=4),
    dict(cs=64, rotary=7, max_pos=4), dict(cs=64, rotary=8, max_pos=0), dict(cs=72, rotary=8, max_pos=4),
    dict(N=2 ** 28)])
def test_append_entry_refusals(change):
    _refused("moba_hip_quantized_append", APPEND, change, "quantized_append")


@pytest.mark.parametrize("change", BAD_POOL + [dict(k=72), dict(dtype=-1), dict(N=0), dict(k_out=72),
                                               dict(v_out=8), dict(N=2 ** 28)])
def test_read_entry_refusals(change):
    _refused("moba_hip_quantized_read", READ, change, "quantized_read")


@pytest.mark.parametrize("change", BAD_POOL + [dict(dtype=3), dict(chunk=0), dict(chunk=1025),
                                               dict(max_chunks=0), dict(max_chunks=2 ** 29), dict(n=2 ** 28)])
def test_means_entry_refusals(change):
    _refused("moba_hip_quantized_means", MEANS, change, "quantized_means")


@pytest.mark.parametrize("change", BAD_POOL + [
    dict(dtype=2), dict(Nq=0), dict(Hq=3), dict(Hq=0), dict(scale=0.0), dict(scale=float("nan")),
    dict(scale=1e31), dict(scale=-1.0), dict(max_length=0), dict(max_length=33), dict(selected=64), dict(slots=3),
    dict(selected=64, slots=17, chunk=8), dict(selected=64, slots=3, chunk=0), dict(q=72), dict(out=72),
    dict(work=None), dict(work=72), dict(Nq=2 ** 26)])
def test_attention_entry_refusals(change):
    _refused("moba_hip_quantized_attention", ATTEND, change, "quantized_attention")


def test_workspace_sizes():
    f = _lib.load().moba_hip_quantized_attention_work
    for bad in ((0, 4, 2, 64, 0, 0, 9), (1, 3, 2, 64, 0, 0, 9), (1, 4, 2, 264, 0, 0, 9), (1, 4, 2, 64, 17, 8, 9),
                (1, 4, 2, 64, 3, 0, 9), (1, 4, 2, 64, 0, 0, 0)):
        assert f(*bad) == -1
    # grows with what it is for
    assert f(1, 4, 2, 64, 0, 0, 128) < f(8, 4, 2, 64, 0, 0, 128) <= f(8, 4, 2, 64, 0, 0, 4096)
    assert f(8, 4, 2, 64, 4, 1024, 4096) > f(8, 4, 2, 64, 0, 0, 4096)   # and the lists of chunks


# --------------------------------------------------------------- cache, session
@pytest.mark.parametrize("kw", [dict(format="bf16"), dict(head_dim=36), dict(head_dim=272), dict(dtype=torch.int8),
                                dict(chunk_size=2048), dict(device="cpu"), dict(page_size=0)])
def test_cache_constructor_refusals(kw):
    with pytest.raises(ValueError):
        QuantizedKVCache(**{"batch_size": 1, "max_seq_len": 8, "num_kv_heads": 1, "head_dim": 64, **kw})


def test_session_format_refusal():
    with pytest.raises(ValueError, match="int8 or fp8"):
        Qwen2Session(None, 8, kv_format="int4")


class _Stop(BaseException):
    pass


@pytest.mark.parametrize("where", ["copy", "launch", "replay"])
@pytest.mark.parametrize("error", [RuntimeError, _lib.MobaHipError, _Stop])
def test_an_attend_that_fails_marks_its_lease(monkeypatch, where, error):
    def fail(*a, **k):
        raise error(where)

    def maybe(name):
        return fail if where == name else (lambda *a, **k: None)

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(prepared_decode, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(_lib, "call", maybe("launch"))
    plan = PreparedQuantizedDecode.__new__(PreparedQuantizedDecode)
    plan.cache = SimpleNamespace(_lock=contextlib.nullcontext(), device=torch.device("cpu"), _stream=0,
                                 _lessee=plan, _broken=False)
    plan._lease = SimpleNamespace(positions=lambda: torch.tensor([3]))
    plan._dev, plan._handle, plan.rotary = 0, None, None
    plan.q = None
    plan._bind_all = lambda specs: [(None, SimpleNamespace(copy_=maybe("copy")))]
    plan._attend_calls = [("entry", ())]
    plan._attend_graph = SimpleNamespace(replay=maybe("replay"))
    plan.closed = plan.failed = False
    plan._result = lambda positions: positions
    with pytest.raises(error):
        plan.attend(None, use_graph=where == "replay")
    assert plan.failed
    with pytest.raises(RuntimeError, match="discard"):
        plan.attend(None)
