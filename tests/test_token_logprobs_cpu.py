"""Log probabilities of tokens on the CPU: the plain form against 64 bits and differences, and what the operator refuses."""
import pytest
import torch


@pytest.fixture
def ops():
    from llmctl_b200.ops import functional
    return functional


def _logits(*shape, seed=0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 3).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,top", [((1, 1), 1), ((3, 7), 0), ((2, 3, 50), 5), ((5, 300), 64), ((0, 9), 2)])
def test_forward(ops, shape, top, dtype):
    top = min(top, shape[-1])
    x, tokens = _logits(*shape, dtype=dtype), torch.randint(0, shape[-1], shape[:-1], generator=torch.Generator().manual_seed(1))
    got = ops.token_logprobs(x, tokens, top)
    lp = torch.log_softmax(x.double(), -1)
    torch.testing.assert_close(got.logprobs.double(), lp.gather(-1, tokens[..., None])[..., 0], rtol=1e-6, atol=4e-6)
    torch.testing.assert_close(got.entropy.double(), -(lp.exp() * lp).sum(-1), rtol=1e-6, atol=1e-5)
    assert (got.top_ids is None) == (got.top_logprobs is None) == (top == 0)
    if top:
        order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[..., :top]
        assert torch.equal(got.top_ids, order)
        torch.testing.assert_close(got.top_logprobs.double(), lp.gather(-1, order), rtol=1e-6, atol=4e-6)


def test_rows_with_masks(ops):
    inf = float("inf")
    x = torch.tensor([[0.0, -inf, 0.0, -inf], [-inf] * 4, [torch.finfo(torch.float32).min] * 4, [1.0, float("nan"), 0.0, 2.0], [0.0, inf, 1.0, 2.0]])
    got = ops.token_logprobs(x, torch.tensor([0, 0, 3, 0, 1]), 3)
    half, quarter = -torch.log(torch.tensor(2.0)), -torch.log(torch.tensor(4.0))
    assert torch.allclose(got.logprobs[[0, 2]], torch.stack([half, quarter])) and torch.allclose(got.entropy[[0, 2]], -torch.stack([half, quarter]))
    assert got.logprobs[[1, 3, 4]].isnan().all() and got.entropy[[1, 3, 4]].isnan().all() and got.top_logprobs[[1, 3, 4]].isnan().all()
    assert got.top_ids.tolist()[:4] == [[0, 2, 1], [0, 1, 2], [0, 1, 2], [3, 0, 2]]
    assert got.top_logprobs[0, 2] == -inf


def test_tokens_outside_of_the_vocabulary(ops):
    x = _logits(3, 11).requires_grad_(True)
    got = ops.token_logprobs(x, torch.tensor([-100, 4, 11]))
    assert got.logprobs[0] == 0 and got.logprobs[2] == 0 and got.logprobs[1] < 0 and (got.entropy > 0).all()
    dx, = torch.autograd.grad(got.logprobs.sum(), x)
    assert not dx[0].any() and not dx[2].any() and dx[1].any()


def test_gradients_against_differences(ops):
    x = _logits(3, 13).double().requires_grad_(True)
    tokens = torch.tensor([0, 12, 5])
    assert torch.autograd.gradcheck(lambda x: (lambda r: (r.logprobs, r.entropy, r.top_logprobs))(ops.token_logprobs(x, tokens, 4)), (x,))


def test_refusals(ops):
    x, tokens = _logits(2, 9), torch.zeros(2, dtype=torch.int64)
    for bad in ((x, tokens.int(), 0), (x, tokens[:1], 0), (x, tokens[:, None], 0), (x, tokens, 10), (x, tokens, -1), (_logits(2, 100), tokens, 65), (x.long(), tokens, 0)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*bad)
