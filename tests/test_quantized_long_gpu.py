"""Attention over long 8-bit rows in which a part that is lost, or taken twice, shows."""
import pytest
import torch

from quant_check import attention, cells, check_attention, make_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,n,hq,hkv,d,chunk", [
    ("fp8", 131071, 14, 2, 64, None), ("int8", 131071, 2, 1, 64, None), ("int8", 60001, 8, 1, 128, None),
    ("fp8", 60001, 32, 1, 128, None), ("int8", 30011, 4, 1, 256, None), ("int8", 30011, 3, 1, 192, None),
    ("int8", 40000, 20, 1, 64, 1000), ("fp8", 40000, 4, 1, 128, 512)])
def test_no_part_of_a_long_row_is_lost(fmt, n, hq, hkv, d, chunk):
    """The value of a token is one in the dim that its place in the row belongs to and zero in
    the others: a result is that part's share of the weights, without cancellation, and its
    bound a few thousandths of it, where 32 tokens are a hundredth of a part or more."""
    from moba_hip import QuantizedPages, quantized_append, quantized_attention
    dtype, page = torch.bfloat16, 16
    table, n_pages = make_table([n], page, 1)
    pages = QuantizedPages.empty(n_pages, page, hkv, d, format=fmt)
    seq, pos = cells([n])
    g = torch.Generator().manual_seed(n)
    k = torch.randn(n, hkv, d, generator=g).to("cuda", dtype)
    v = torch.zeros(n, hkv, d, dtype=dtype, device="cuda")
    part = pos.long() * d // n
    v[torch.arange(n, device="cuda"), :, part] = 1.0
    quantized_append(k, v, pages, table, seq, pos)
    q = (torch.randn(1, hq, d, generator=g) * 0.2).to("cuda", dtype)     # nearly flat weights
    dev = dict(dtype=torch.int32, device="cuda")
    rows, lens = torch.zeros(1, **dev), torch.full((1,), n, **dev)
    selected = None
    if chunk:
        count = -(-n // chunk)
        selected = torch.stack([torch.randperm(count, generator=g)[:9] for _ in range(hq)])[None].to("cuda", torch.int32)
    got = quantized_attention(q, pages, table, rows, lens, selected=selected, chunk_size=chunk)
    want = attention(q, pages, table, rows, lens, selected, chunk)
    check_attention(got, want)
    # 32 tokens of nearly equal weights are 32 / 2048 of the largest part: more than the bound
    held = want[0] > 0
    assert (want[2][held] < 0.0075 * want[0][held]).all()
    if chunk is None:
        assert held.all()
