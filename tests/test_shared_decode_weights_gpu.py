"""Decode attention over shared prefixes: attention's weights keep 16 bits, as where the sequences are read by themselves."""
import math

import pytest
import torch

from llmctl_b200.ops import native, serving as sops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    torch.cuda.synchronize()
    native.check_waits("test")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("count,per_head,shared,own", [(2, 1, 64, 2), (4, 4, 128, 70), (12, 4, 80, 16), (40, 1, 64, 30), (30, 4, 192, 20), (70, 5, 320, 80), (1, 1, 0, 2)])
def test_weights_that_cancel(dim, count, per_head, shared, own):
    """Half of the tokens have a score of 8 units and values of 1, half of them 7 and -1: the result is tanh(unit / 2), and all weights of a half are off by the same.  The unit is
    such that bf16 rounds the smaller weight by nearly half a step, 2^-9: that alone moves the result by 2^-10.  Scores are whole numbers, exact."""
    step, heads, page, n = 250.5 / 256, 2, 16, shared + own
    unit = -math.log(step)
    blocks = (shared + count * (own + page)) // page + 2
    k = torch.zeros(blocks, page, heads, dim, device="cuda", dtype=torch.bfloat16)
    v = torch.ones_like(k)
    k[..., 3] = 8
    k[:, 1::2, :, 3] = 7
    v[:, 1::2] = -1
    per = (own + page - 1) // page
    tables = torch.zeros(count, shared // page + per, dtype=torch.int32)
    for b in range(count):
        tables[b, :shared // page] = torch.arange(shared // page)
        tables[b, shared // page:] = shared // page + b * per + torch.arange(per)
    q = torch.zeros(count, heads * per_head, dim, device="cuda", dtype=torch.bfloat16)
    q[..., 3] = 1
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    with torch.no_grad():
        got = sops.paged_attention_decode_shared(q, k, v, tables.cuda(), ints([n] * count), ints([0, count]), ints([shared]), unit).double()
    want = math.tanh(unit / 2)
    # weights of 16 bits are off by 2^-16, the exponential by 2^-21 and its argument, at most 1, by 2^-22; sums of n numbers by n 2^-23, numerator and divisor alike; the result
    # by half a step of bf16
    bound = 2 * (2.0 ** -16 + 2.0 ** -20 + n * 2.0 ** -23) + want * 2.0 ** -8
    assert bound < 2.0 ** -11
    assert (got - want).abs().max().item() <= bound
