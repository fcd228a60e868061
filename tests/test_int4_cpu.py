"""Products with weights of 4 bits: the plain form against 64 bits, the quantiser's layout, refusals."""
import pytest
import torch

from llmctl_b200.io.quantize import Int4GroupQuantizer
from llmctl_b200.ops import functional as ops

from int4_oracle import check, matrix, product


@pytest.mark.parametrize("shape,rows", [((3, 128), 5), ((2, 3, 384), 16), ((0, 256), 4), ((1, 128), 1), ((640,), 7)])
@pytest.mark.parametrize("gated", [False, True])
def test_plain_form(shape, rows, gated):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).bfloat16()
    w, scale = matrix(rows * (2 if gated else 1), shape[-1], 2)
    got = (ops.linear_swiglu_int4 if gated else ops.linear_int4)(x, w, scale)
    assert got.dtype == x.dtype and got.shape == (*shape[:-1], rows)
    if x.numel():
        check(got, product(x, w, scale, gated))


def test_takes_what_the_quantiser_writes():
    g = torch.Generator().manual_seed(3)
    sd = Int4GroupQuantizer().quantize({"up": torch.randn(12, 256, generator=g) * 0.02})
    x = torch.randn(4, 256, generator=g)
    back = Int4GroupQuantizer().dequantize(sd, torch.float32)["up"]
    assert torch.equal(ops.dequantize_int4(sd["up"], sd["up.scale"], torch.float32), back)
    torch.testing.assert_close(ops.linear_int4(x, sd["up"], sd["up.scale"]), x @ back.t(), rtol=1e-5, atol=1e-6)


def test_refusals():
    x = torch.randn(2, 256)
    w, scale = matrix(6, 256, 4)
    for bad in [(x[:, :200], w, scale), (x, w[:, :64], scale), (x, w.int(), scale), (x, w, scale.float()), (x, w, scale[:5]), (x, w, scale[:, :1]), (x.long(), w, scale), (x, w.view(-1), scale)]:
        with pytest.raises(ValueError, match="weights of 4 bits"):
            ops.linear_int4(*bad)
    with pytest.raises(ValueError, match="as many"):
        ops.linear_swiglu_int4(x, w[:5], scale[:5])
    with pytest.raises(ValueError, match="no backward"):
        ops.linear_int4(x.requires_grad_(True), w, scale)
    with torch.no_grad():
        assert ops.linear_int4(x, w, scale).shape == (2, 6)
