"""Kernels of csrc/loss/token_logprobs.cu against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(cuda_device):
    from llmctl_b200.ops import functional
    return functional


def _logits(rows, V, dtype, std=3.0, shift=0, pad=0, seed=0):
    """Rows of a wider buffer (``pad`` more numbers to a row) that begins ``shift`` numbers past a 16-byte boundary."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.empty(shift + rows * (V + pad), device="cuda", dtype=torch.float32).normal_(0, std, generator=g).to(dtype)
    return buf[shift:].view(rows, V + pad)[:, :V]


def _tokens(rows, V, seed=1):
    return torch.randint(0, V, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _want(x, tokens, top):
    x = x.detach().double()
    lp = torch.log_softmax(x, -1)
    entropy = -torch.where(lp == float("-inf"), 0.0, lp.exp() * lp).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, lp.gather(1, tokens[:, None])[:, 0], entropy, order


def _slack(lp, V):
    """Errors of 32 bits: a thread adds up to V / 256 + 40 terms one by one (2^-24 each), each exponential is off by its argument's rounding and its
    own (|x - m| 2^-23 + 2^-22 of it, of which x - m weighted by the exponential is at most 1) -> relative error of the sum, which is the logarithm's."""
    return (V / 256 + 40) * 2.0 ** -24 + 2.0 ** -21


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,top,shift,pad", [(1, 1, 1, 0, 0), (3, 7, 7, 1, 0), (5, 50, 20, 0, 14), (2, 511, 64, 3, 0), (33, 1000, 5, 0, 24), (4, 4097, 64, 1, 2), (7, 32000, 20, 0, 0),
                                                  (300, 32001, 1, 0, 127), (2, 50257, 3, 0, 0), (2, 200000, 20, 2, 1), (9, 777, 0, 5, 3), (40, 128000, 64, 0, 0), (150, 8200, 5, 1, 1), (1200, 5000, 20, 0, 0), (1, 131072, 1, 0, 0)])
def test_forward(ops, rows, V, top, shift, pad, dtype):
    x, tokens = _logits(rows, V, dtype, shift=shift, pad=pad), _tokens(rows, V)
    kept = x.clone()
    got = ops.token_logprobs(x, tokens, top)
    lp, chosen, entropy, order = _want(x, tokens, top)
    eps = _slack(lp, V)
    assert ((got.logprobs - chosen).abs() <= eps + 2.0 ** -22 * chosen.abs()).all()
    assert ((got.entropy - entropy).abs() <= eps * (2 + 2 * entropy) + 1e-6).all()
    if top:
        assert torch.equal(got.top_ids, order)
        assert ((got.top_logprobs - lp.gather(1, order)).abs() <= eps + 2.0 ** -22 * lp.gather(1, order).abs()).all()
    assert torch.equal(x, kept)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 100001), (torch.float32, 50001)])
@pytest.mark.parametrize("rows,top", [(60, 20), (120, 1), (200, 20), (296, 5), (297, 64)])
def test_clusters_of_every_size(ops, rows, top, dtype, V):
    """Rows so long that eight, four, two or one CTA go to each by how many of them there are."""
    x, tokens = _logits(rows, V, dtype, pad=3), _tokens(rows, V)
    got = ops.token_logprobs(x, tokens, top)
    lp, chosen, entropy, order = _want(x, tokens, top)
    eps = _slack(lp, V)
    assert ((got.logprobs - chosen).abs() <= eps + 2.0 ** -22 * chosen.abs()).all()
    assert ((got.entropy - entropy).abs() <= eps * (2 + 2 * entropy) + 1e-6).all()
    assert torch.equal(got.top_ids, order)
    assert ((got.top_logprobs - lp.gather(1, order)).abs() <= eps + 2.0 ** -22 * lp.gather(1, order).abs()).all()


@pytest.mark.parametrize("V,top", [(4000, 20), (40, 40), (33000, 64)])
def test_ties_and_order(ops, V, top):
    """Equal logits: the lowest ids; logits that rise or fall along the row, and rows whose largest numbers all stand in one thread's units."""
    tokens = torch.zeros(5, dtype=torch.int64, device="cuda")
    x = torch.zeros(5, V, device="cuda")
    x[1] = torch.arange(V, device="cuda")
    x[2] = -torch.arange(V, device="cuda")
    x[3] = torch.arange(V, device="cuda") % 3
    x[4, ::2] = -0.0
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        got = ops.token_logprobs(y, tokens, top)
        assert torch.equal(got.top_ids, _want(y, tokens, top)[3])


@pytest.mark.parametrize("dtype,unit", [(torch.bfloat16, 8), (torch.float32, 4)])
@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("many", [40, 300])
def test_many_candidates(ops, dtype, unit, rows, many):
    """The units of four neighbouring threads hold all of the row's larger numbers: up to 9600, more than the list of candidates has room for."""
    top, V = 24, 256 * unit * many
    x = torch.full((1, V), -5.0, device="cuda")
    place = (torch.arange(many, device="cuda")[:, None, None] * 256 + torch.arange(4, device="cuda")[None, :, None]) * unit + torch.arange(unit, device="cuda")
    place = place.reshape(-1)[torch.randperm(place.numel(), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))]
    x[:, place] = (torch.arange(place.numel(), device="cuda") % 200).float() * 0.25
    x = x.to(dtype)
    tokens = place[:1].clone()
    want = _want(x, tokens, top)
    got = ops.token_logprobs(x.expand(rows, V), tokens.expand(rows), top)
    assert torch.equal(got.top_ids, want[3].expand(rows, top)) and torch.equal(got.logprobs, got.logprobs[:1].expand(rows))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9, 5003])
def test_masks_and_infinities(ops, V, dtype):
    inf = float("inf")
    x = _logits(7, V, dtype)
    x[0, 1:] = -inf                                        # one token is left
    x[1] = -inf                                            # none
    x[2] = torch.finfo(dtype).min                          # all at the type's lowest number
    x[3, V // 2:] = torch.finfo(dtype).min
    x[4, V // 2] = float("nan")
    x[5, 2] = inf
    x[6, ::2] = -inf
    tokens = torch.tensor([0, 0, 1, 0, 0, 2, 1], device="cuda")
    got = ops.token_logprobs(x, tokens, 3)
    lp, chosen, entropy, order = _want(x, tokens, 3)
    fine, eps = [0, 2, 3, 6], _slack(lp, V)
    assert ((got.logprobs - chosen).abs()[fine] <= eps + 2.0 ** -22 * chosen.abs()[fine]).all()
    assert ((got.entropy - entropy).abs()[fine] <= eps * (2 + 2 * entropy[fine]) + 1e-6).all()
    assert torch.equal(got.top_ids[[0, 1, 2, 3, 5, 6]], order[[0, 1, 2, 3, 5, 6]])
    for bad in (1, 4, 5):
        assert got.logprobs[bad].isnan() and got.entropy[bad].isnan() and got.top_logprobs[bad].isnan().all()
    assert got.top_logprobs[0, 1] == -inf


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9, 5003, 200000])
def test_the_largest_numbers(ops, V, dtype):
    """Finite logits up to the type's largest among ordinary ones have numbers for all results and gradients, of the log probability alone and with the
    entropy's; differences that 32 bits do not hold are -inf."""
    most = torch.finfo(dtype).max
    x = _logits(7, V, dtype)
    x[0, V // 2] = most
    x[1, 0] = x[1, V - 1] = most
    x[2] = most
    x[3, ::2], x[3, 1] = -most, most
    x[4, 3], x[4, 4:] = 2.4e38, float("-inf")
    x[5, 2], x[6, 2] = 1e30, 5e29
    tokens = torch.tensor([V // 2, 1, 0, 0, 3, 2, 0], device="cuda")
    x.requires_grad_(True)
    got = ops.token_logprobs(x, tokens, 3)
    lp, chosen, entropy, order = _want(x, tokens, 3)
    eps = _slack(lp, V)
    assert torch.allclose(got.logprobs, chosen.float(), rtol=2.0 ** -22, atol=eps)
    assert ((got.entropy - entropy).abs() <= eps * (2 + 2 * entropy) + 1e-6).all()
    assert torch.equal(got.top_ids, order) and torch.allclose(got.top_logprobs, lp.gather(1, order).float(), rtol=2.0 ** -22, atol=eps)
    g, gh = torch.randn(7, device="cuda"), torch.randn(7, device="cuda")
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for outs, grads in (((got.logprobs,), (g,)), ((got.logprobs, got.entropy), (g, gh))):
        dx, = torch.autograd.grad(outs, x, grads, retain_graph=True)
        want, size = _gradient(x, tokens, 0, None, g, gh if len(grads) == 2 else torch.zeros_like(gh), None)
        assert ((dx.double() - want).abs() <= rounding * want.abs() + (4 * eps + 2.0 ** -20) * size + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9, 5003])
def test_large_gradients_of_the_entropy_beside_masks(ops, V, dtype):
    """A masked logit has no part in the gradient however large the entropy's is."""
    x = _logits(4, V, dtype)
    x[:, ::3], x[1, 1::3] = float("-inf"), torch.finfo(dtype).min
    x[2, 1] = -1e30
    tokens = torch.tensor([1, 2, 4, 5], device="cuda")
    x.requires_grad_(True)
    got = ops.token_logprobs(x, tokens)
    for much in (1e7, 1e9, 1e20, 1e35):
        gh = torch.tensor([much, -much, much, 1.0], device="cuda")
        dx, = torch.autograd.grad(got.entropy, x, gh, retain_graph=True)
        want, size = _gradient(x, tokens, 0, None, torch.zeros_like(gh), gh, None)
        rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        assert ((dx.double() - want).abs() <= rounding * want.abs() + (4 * _slack(None, V) + 2.0 ** -20) * size + 1e-30).all()
        assert not dx[:, ::3].any()


def _gradient(x, tokens, top, order, g, gh, gt):
    """The formula in 64 bits and the sum of magnitudes of its terms."""
    x = x.detach().double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    safe = torch.where(p == 0, 0.0, lp)
    h = -(p * safe).sum(-1, keepdim=True)
    given = ((tokens >= 0) & (tokens < x.shape[1]))[:, None]
    g = torch.where(given, g.double()[:, None], 0.0)
    total = g + (gt.double().sum(-1, keepdim=True) if top else 0.0)
    dx = -p * (total + gh.double()[:, None] * (safe + h))
    size = p * ((g.abs() + (gt.double().abs().sum(-1, keepdim=True) if top else 0.0)) + gh.double().abs()[:, None] * (safe.abs() + h + 1))
    at = torch.where(given, tokens[:, None], 0)
    dx.scatter_add_(1, at, g)
    size.scatter_add_(1, at, g.abs())
    if top:
        dx.scatter_add_(1, order, gt.double())
        size.scatter_add_(1, order, gt.double().abs())
    return dx, size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,top,shift,pad", [(1, 5, 5, 0, 0), (3, 777, 0, 1, 0), (4, 4000, 3, 0, 96), (130, 32000, 0, 0, 0), (3, 50257, 20, 3, 0), (700, 3000, 2, 0, 8)])
def test_backward(ops, rows, V, top, shift, pad, dtype):
    x, tokens = _logits(rows, V, dtype, shift=shift, pad=pad), _tokens(rows, V)
    x[:, V // 2] = float("-inf")
    tokens[tokens == V // 2] = 0
    if rows > 2:
        tokens[1], tokens[2] = -100, V
    x.requires_grad_(True)
    got = ops.token_logprobs(x, tokens, top)
    g, gh, gt = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda"), torch.randn(rows, max(top, 1), device="cuda")
    if top and rows == 1:
        tokens[0] = got.top_ids[0, 1]                      # the token is among the most probable
        got = ops.token_logprobs(x, tokens, top)
    if top == V:                                           # the masked token's log probability is -inf: no gradient asked of it
        gt[:, -1] = 0
    outs, grads = (got.logprobs, got.entropy) + ((got.top_logprobs,) if top else ()), (g, gh) + ((gt,) if top else ())
    dx, = torch.autograd.grad(outs, x, grads, retain_graph=True)
    order = _want(x, torch.zeros_like(tokens), top)[3]
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    eps = 4 * _slack(None, V) + 2.0 ** -20                 # of a probability: the sums' error, and that of its own argument (up to 30 in 2^-24)
    for outs_, used in ((outs, grads), (outs[:1], (g,)), (outs[1:2], (gh,)), *(((outs[2:], (gt,)),) if top else ())):
        zero = torch.zeros_like
        want, size = _gradient(x, tokens, top, order, *(v if any(v is u for u in used) else zero(v) for v in (g, gh, gt)))
        dx, = torch.autograd.grad(outs_, x, used, retain_graph=True)
        assert dx.dtype == dtype and dx.shape == x.shape
        assert ((dx.double() - want).abs() <= rounding * want.abs() + eps * size + 1e-30).all()


def test_gradient_against_differences(ops):
    x, tokens = _logits(2, 300, torch.float32, std=1.0).requires_grad_(True), _tokens(2, 300)
    direction = torch.randn(2, 300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))

    def loss(out):
        return (out.logprobs * 1.5).sum() + out.entropy.sum() * 0.5 - out.top_logprobs.sum() * 0.25
    dx, = torch.autograd.grad(loss(ops.token_logprobs(x, tokens, 4)), x)
    f = [loss(ops.token_logprobs((x.detach() + e * direction).cpu().double(), tokens.cpu(), 4)) for e in (1e-4, -1e-4)]
    slope = float((f[0] - f[1]) / 2e-4)
    # differences of a smooth function at 1e-4 are off by their third order, about 1e-8 x |direction|^3; the gradient's numbers by 2^-20 of their size
    assert abs(float((dx.double() * direction.double()).sum()) - slope) <= 1e-4 * (1 + abs(slope))


def test_graph_replay_beside_an_eager_call(ops):
    x, tokens = _logits(20, 5000, torch.bfloat16), _tokens(20, 5000)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.token_logprobs(x, tokens, 5)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.token_logprobs(x, tokens, 5)
    y = _logits(20, 5000, torch.bfloat16, seed=9)
    x.copy_(y)
    graph.replay()
    eager = ops.token_logprobs(y, tokens, 5)
    torch.cuda.synchronize()
    for a, b in zip(out, eager):
        assert torch.equal(a, b)


def test_leading_dimensions_and_strides(ops):
    x, tokens = _logits(6, 400, torch.bfloat16), _tokens(6, 400)
    flat = ops.token_logprobs(x, tokens, 2)
    for y in (x.view(2, 3, 400), torch.stack([x, x], -1)[..., 0].view(2, 3, 400), x.t().contiguous().t().unflatten(0, (2, 3))):
        got = ops.token_logprobs(y, tokens.view(2, 3), 2)
        for a, b in zip(got, flat):
            assert torch.equal(a, b.view_as(a)) and a.shape[:2] == (2, 3)
    one = ops.token_logprobs(x[:1].expand(6, 400), tokens[:1].expand(6), 2)
    assert torch.equal(one.top_ids, flat.top_ids[:1].expand(6, 2))


def test_gradients_of_broadcast_and_shared_logits(ops):
    """One row under six tokens, and a row used twice: its gradient is the sum of theirs."""
    x, tokens, g = _logits(1, 500, torch.float32).requires_grad_(True), _tokens(6, 500), torch.randn(6, device="cuda")
    dx, = torch.autograd.grad(ops.token_logprobs(x.expand(6, 500), tokens).logprobs, x, g)
    rows, = torch.autograd.grad(ops.token_logprobs(x.repeat(6, 1), tokens).logprobs, x, g)
    assert torch.allclose(dx, rows, rtol=1e-5, atol=1e-7) and dx.shape == (1, 500)
    y = x * 2
    both, = torch.autograd.grad(ops.token_logprobs(y, tokens[:1]).logprobs.sum() + ops.token_logprobs(y, tokens[:1], 3).entropy.sum(), x)
    want = torch.log_softmax(x.detach().double() * 2, -1)
    p = want.exp()
    h = -(p * want).sum()
    ref = -p * (1 + want + h)
    ref[0, tokens[0]] += 1
    assert (both.double() - 2 * ref).abs().max() <= 1e-5


def test_saved_logits_that_a_hook_changes_are_refused(ops):
    x, tokens = _logits(3, 100, torch.bfloat16).requires_grad_(True), _tokens(3, 100)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float() if t.dtype == torch.bfloat16 else t):
        out = ops.token_logprobs(x, tokens)
        with pytest.raises(RuntimeError):
            out.logprobs.sum().backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = ops.token_logprobs(x, tokens, 2)
        dx, = torch.autograd.grad(out.logprobs.sum(), x)
    assert torch.equal(dx, torch.autograd.grad(ops.token_logprobs(x, tokens, 2).logprobs.sum(), x)[0])


def test_engine_log_probabilities(ops):
    from llmctl_b200.comms import mesh
    from llmctl_b200.models.config import ModelConfig
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    cfg = ModelConfig(name="logprob-test", layers=2, hidden=256, ffn=704, heads=4, vocab_size=4001, max_position_embeddings=256)
    eng = InferenceEngine(cfg, max_batch_size=4, max_batch_tokens=1024, num_kv_blocks=64)
    seqs = [eng.add_request(list(range(3, 3 + n)), 6, temperature=0.0, logprobs=4) for n in (5, 33)]
    while eng.has_work():
        eng.step()
    for s in seqs:
        assert [r["token"] for r in s.token_logprobs] == s.generated
        for i, r in enumerate(s.token_logprobs):
            logits = eng.model(torch.tensor([s.prompt_ids + s.generated[:i]], device="cuda"))[-1, :4001].double()
            lp = torch.log_softmax(logits, -1)
            # the decoding step's logits are rounded to bf16 and come by other kernels than the prompt's
            assert abs(r["logprob"] - float(lp[r["token"]])) < 0.1 and len(r["top"]) == 4 and r["top"][0] == (r["token"], r["logprob"])
            assert abs(r["entropy"] + float((lp.exp() * lp).sum())) < 0.05
