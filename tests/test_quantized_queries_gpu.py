"""Queries of an 8-bit cache that are not finite."""
import pytest
import torch

from quant_check import attention, cells, make_table

pytestmark = pytest.mark.gpu


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to("cuda", dtype)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,d", [(4, 64), (4, 128), (20, 40), (4, 256)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_query_that_is_not_finite_gives_nan(fmt, dtype, hq, d, bad):
    """Keys of one sign in the dim of an infinity: its scores are all +inf or all -inf, and
    the softmax of either is no number.  The other heads and rows are as they were, and a row
    that attends nothing is zeros whatever its query holds."""
    from moba_hip import QuantizedPages, quantized_append, quantized_attention
    n, dim = 70, 3
    table, n_pages = make_table([n], 16, 0)
    pages = QuantizedPages.empty(n_pages, 16, 1, d, format=fmt)
    seq, pos = cells([n])
    k = _rand((n, 1, d), dtype, 1)
    k[..., dim] = -k[..., dim].abs() - 0.5
    quantized_append(k, _rand((n, 1, d), dtype, 2), pages, table, seq, pos)
    q = _rand((3, hq, d), dtype, 3)
    dev = dict(dtype=torch.int32, device="cuda")
    rows, lens = torch.zeros(3, **dev), torch.tensor([n, 33, 0], **dev)
    for selected in (None, torch.tensor([0, 2], **dev).expand(3, hq, 2).contiguous()):
        chunk = None if selected is None else 20
        want = attention(q, pages, table, rows, lens, selected, chunk)
        other = q.clone()
        other[0, 1, dim] = other[2, 0, d - 1] = bad
        out, lse = quantized_attention(other, pages, table, rows, lens, selected=selected, chunk_size=chunk)
        assert torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, 1])
        kept = torch.ones(3, hq, dtype=torch.bool, device="cuda")
        kept[0, 1] = kept[2] = False
        assert ((out.double() - want[0]).abs() <= want[2])[kept].all()
        assert ((lse.double() - want[1]).abs() <= want[3])[kept].all()
        assert (out[2] == 0).all() and (lse[2] == -float("inf")).all()


@pytest.mark.parametrize("fmt,d", [("int8", 64), ("int8", 128), ("fp8", 64)])
@pytest.mark.parametrize("scale", [2.0 ** -126, 1e30 * (1 - 2.0 ** -50), 1e30])
def test_the_ends_of_scale(fmt, d, scale):
    """Queries so small that scores are ordinary ones; with outputs of the caller too, which
    the other host path serves."""
    from quant_check import check_attention
    from moba_hip import QuantizedPages, quantized_append, quantized_attention
    table, n_pages = make_table([50], 16, 0)
    pages = QuantizedPages.empty(n_pages, 16, 1, d, format=fmt)
    seq, pos = cells([50])
    k = _rand((50, 1, d), torch.bfloat16, 1)
    quantized_append(k, k, pages, table, seq, pos)
    q = (_rand((1, 4, d), torch.float32, 3) / max(scale, 1.0)).bfloat16()
    dev = dict(dtype=torch.int32, device="cuda")
    args = q, pages, table, torch.tensor([0], **dev), torch.tensor([50], **dev)
    want = attention(*args, scale=scale)
    check_attention(quantized_attention(*args, scale=scale), want)
    check_attention(quantized_attention(*args, scale=scale, out=torch.empty_like(q)), want)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,large", [(torch.bfloat16, 2.0 ** 13), (torch.bfloat16, 2.0 ** 18),
                                         (torch.bfloat16, 1e9), (torch.float16, 60000.0)])
@pytest.mark.parametrize("hq,d", [(4, 64), (6, 96), (20, 128), (3, 192), (4, 256)])
def test_a_large_value_in_a_query_leaves_the_others_their_digits(fmt, dtype, large, hq, d):
    """One dim of some heads' queries is much larger than the others, and the keys are zero
    there: scores are those of the other dims, which the bound goes by."""
    from quant_check import check_attention
    from moba_hip import QuantizedPages, quantized_append, quantized_attention
    n, dim = 300, 5
    table, n_pages = make_table([n], 16, 0)
    pages = QuantizedPages.empty(n_pages, 16, 1, d, format=fmt)
    seq, pos = cells([n])
    k = _rand((n, 1, d), dtype, 1)
    k[..., dim] = 0.0
    quantized_append(k, _rand((n, 1, d), dtype, 2), pages, table, seq, pos)
    q = _rand((3, hq, d), dtype, 3)
    q[0, :, dim], q[1, ::2, dim] = large, -large / 3
    dev = dict(dtype=torch.int32, device="cuda")
    args = q, pages, table, torch.zeros(3, **dev), torch.tensor([n, 257, n], **dev)
    check_attention(quantized_attention(*args), attention(*args))
    # the large value itself, against a key that has it
    k[7, 0, dim] = 1.0 / large
    quantized_append(k, _rand((n, 1, d), dtype, 2), pages, table, seq, pos)
    check_attention(quantized_attention(*args), attention(*args))
