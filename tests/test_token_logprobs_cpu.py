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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("top", [0, 1, 4])
@pytest.mark.parametrize("numbers", [1, 200, 1 << 21])
def test_rows_in_portions_and_as_a_whole(ops, monkeypatch, numbers, top, dtype):
    """With gradients, and under a transform, all rows are computed at once, without some at a time: the same numbers, rows with masks and NaN among them."""
    monkeypatch.setattr(ops, "_PLAIN_NUMBERS", numbers)
    x = _logits(2, 4, 60).round().to(dtype)
    x[0, 0, 1:], x[0, 1], x[0, 2, 7], x[1, 0, ::2], x[1, 1, 5] = float("-inf"), float("-inf"), float("nan"), float("-inf"), float("inf")
    tokens = torch.randint(-1, 61, (2, 4), generator=torch.Generator().manual_seed(3))
    got, kept = ops.token_logprobs(x, tokens, top), x.clone()
    whole = ops.token_logprobs(x.clone().requires_grad_(True), tokens, top)
    each = torch.vmap(lambda x, t: tuple(v for v in ops.token_logprobs(x, t, top) if v is not None))(x, tokens)
    # sums of 60 terms in another order: 60 roundings and an exponential's own, relative to sums of at least 1 and weighted logarithms of at most log 60
    eps = 80 * torch.finfo(torch.float32 if dtype == torch.bfloat16 else dtype).eps / 2 * 5
    for a, b, c in zip(got, whole, each):
        assert a.dtype == b.dtype and a.shape == b.shape
        for other in (b, c):
            assert torch.equal(a, other) if a.dtype == torch.int64 else torch.allclose(a, other.detach(), rtol=eps, atol=eps, equal_nan=True)
    assert len([v for v in got if v is not None]) == len(each) == (4 if top else 2) and torch.equal(x.nan_to_num(), kept.nan_to_num())


def test_the_best_guess_takes_no_sort(ops):
    """What evaluation asks for, over a vocabulary of any size, is a pass for the largest number of a row."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as p:
        ops.token_logprobs(_logits(3, 5000), torch.zeros(3, dtype=torch.int64), 1)
        ops.token_logprobs(_logits(3, 5000).requires_grad_(True), torch.zeros(3, dtype=torch.int64), 1)
    assert not [e.key for e in p.key_averages() if "sort" in e.key or "topk" in e.key]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_numbers(ops, dtype):
    """Finite logits up to the type's largest have numbers for all results and gradients."""
    most, inf = torch.finfo(dtype).max, float("inf")
    x = torch.tensor([[0.0, most, 1.0, 2.0], [most, 1.0, -most, most], [most] * 4, [1.0, 2.5e38, -inf, 0.0]], dtype=dtype).requires_grad_(True)
    got = ops.token_logprobs(x, torch.tensor([1, 0, 2, 0]), 2)
    two, four = torch.log(torch.tensor(2.0)), torch.log(torch.tensor(4.0))
    assert torch.allclose(got.logprobs[:3], torch.stack([torch.tensor(0.0), -two, -four])) and got.logprobs[3] == 1 - x[3, 1].float()
    assert torch.allclose(got.entropy, torch.stack([torch.tensor(0.0), two, four, torch.tensor(0.0)])) and got.top_ids.tolist() == [[1, 3], [0, 3], [0, 1], [1, 0]]
    dx, = torch.autograd.grad(got.logprobs.sum() + 3 * got.entropy.sum(), x)
    want = torch.tensor([[0.0, 0.0, 0.0, 0.0], [0.5, 0.0, 0.0, -0.5], [-0.25, -0.25, 0.75, -0.25], [1.0, -1.0, 0.0, 0.0]])
    assert torch.allclose(dx.float(), want, atol=1e-6)


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


def _engine(**kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    return InferenceEngine("gpt-tiny", device="cpu", kv_block_size=4, num_kv_blocks=64, **kw)


def test_engine_gives_log_probabilities_with_its_tokens():
    eng = _engine(max_batch_size=3, max_batch_tokens=256)
    prompts = [[5, 6, 7], [9, 8], [3]]
    seqs = [eng.add_request(p, 4, temperature=t, logprobs=n) for p, t, n in zip(prompts, (0.0, 1.3, 0.0), (3, 0, None))]
    while eng.has_work():
        eng.step()
    assert seqs[2].token_logprobs == [] and len(seqs[2].generated) == 4
    for s, n in zip(seqs[:2], (3, 0)):
        assert [r["token"] for r in s.token_logprobs] == s.generated
        for i, r in enumerate(s.token_logprobs):
            lp = torch.log_softmax(eng.model(torch.tensor([s.prompt_ids + s.generated[:i]]))[-1, :512].double(), -1)
            best = torch.topk(lp, 3)
            assert abs(r["logprob"] - float(lp[r["token"]])) < 1e-3 and abs(r["entropy"] + float((lp.exp() * lp).sum())) < 1e-3
            assert len(r["top"]) == n
            if n:
                assert [t for t, _ in r["top"]] == best.indices.tolist() and r["top"][0][0] == r["token"]
                assert all(abs(v - float(w)) < 1e-3 for (_, v), w in zip(r["top"], best.values))
    for bad in (-1, 65):
        with pytest.raises(ValueError, match="logprobs"):
            eng.add_request([5], 4, logprobs=bad)


def test_http_log_probabilities():
    import json

    from fastapi.testclient import TestClient
    from llmctl_b200.serve.server import InferenceServer
    srv = InferenceServer("gpt-tiny", engine=_engine(max_batch_size=4, max_batch_tokens=512))
    srv.start_background()
    try:
        c = TestClient(srv.app)
        ask = {"prompt": "hello", "max_tokens": 5, "temperature": 0.0}
        plain, body = c.post("/v1/completions", json=ask).json(), c.post("/v1/completions", json={**ask, "logprobs": 2}).json()
        assert "logprobs" not in plain and body["text"] == plain["text"]
        said = body["logprobs"]
        assert set(said) == {"tokens", "token_ids", "token_logprobs", "entropy", "top_logprobs"} and len({len(v) for v in said.values()}) == 1
        assert all(v <= 0 for v in said["token_logprobs"]) and all(len(t) == 2 and t[0]["token_id"] == i for t, i in zip(said["top_logprobs"], said["token_ids"]))
        with c.stream("POST", "/v1/completions", json={**ask, "logprobs": 0, "stream": True}) as s:
            events = [json.loads(x[6:]) for x in s.iter_lines() if x.startswith("data: {")]
        assert [e["logprobs"]["token_logprobs"] for e in events if "text" in e][:len(said["token_ids"])] == said["token_logprobs"]
        assert c.post("/v1/completions", json={**ask, "logprobs": 21}).status_code == 422
    finally:
        srv.shutdown()


def test_lockstep_engine_passes_log_probabilities_on():
    """The leader's queue carries the number of alternatives to the engine of every rank."""
    import threading

    from llmctl_b200.serve import lockstep
    eng = _engine(max_batch_size=2, max_batch_tokens=256)
    lock = lockstep.LockstepEngine.__new__(lockstep.LockstepEngine)
    lock.engine, lock._lock, lock._pending, lock.on_pending = eng, threading.Lock(), [], None
    got = []
    with pytest.raises(ValueError, match="logprobs"):
        lock.add_request([5, 6], 3, 0.0, logprobs=99)
    assert not lock._pending
    t = threading.Thread(target=lambda: got.append(lock.add_request([5, 6], 3, 0.0, logprobs=1)))
    t.start()
    while not lock._pending:
        pass
    (args, holder), = lock._pending
    lock._apply({"adds": [args], "cancels": []}, [holder])
    t.join(10)
    assert got[0].logprobs == 1 and got[0].max_tokens == 3 and got[0].temperature == 0.0


def test_eval_reads_likelihood_and_best_guess_from_one_call(tmp_path):
    import math

    from llmctl_b200.cli.commands.eval import evaluate_checkpoint
    from llmctl_b200.io.dataset import build_dataset
    from llmctl_b200.serve.engine import load_model_for_inference
    res = evaluate_checkpoint("gpt-tiny", ["perplexity", "accuracy"], batches=2, batch_size=2, seq_len=32, device="cpu")
    model, cfg, _, _ = load_model_for_inference("gpt-tiny", "cpu")
    ds = build_dataset(None, cfg.vocab_size, 32, seed=4242)
    rows = torch.stack([torch.from_numpy(ds[i]) for i in range(4)])
    logits = model(rows[:, :-1].contiguous()).double()[:, :cfg.vocab_size]
    lp = torch.log_softmax(logits, -1).gather(1, rows[:, 1:].reshape(-1, 1))
    task = res["tasks"]["perplexity"]
    assert task["tokens"] == lp.numel() and abs(task["loss"] + float(lp.mean())) < 1e-5 and abs(task["perplexity"] - math.exp(-float(lp.mean()))) < 1e-2
    assert res["tasks"]["accuracy"]["next_token_accuracy"] == float((logits.argmax(-1) == rows[:, 1:].reshape(-1)).double().mean())


def test_eval_refuses_tokens_that_the_model_does_not_know(monkeypatch):
    """A target outside of the vocabulary has no likelihood to be counted."""
    import numpy as np

    from llmctl_b200.cli.commands.eval import evaluate_checkpoint
    from llmctl_b200.io import dataset
    rows = [np.arange(3, 36, dtype=np.int64) for _ in range(4)]
    monkeypatch.setattr(dataset, "build_dataset", lambda *a, **k: rows)
    fine = evaluate_checkpoint("gpt-tiny", ["perplexity"], batches=2, batch_size=2, seq_len=32, device="cpu")
    assert fine["tasks"]["perplexity"]["tokens"] == 4 * 32
    for bad in (512, -1):
        rows[3] = np.concatenate([np.arange(3, 35), [bad]])
        with pytest.raises(ValueError, match="vocabulary"):
            evaluate_checkpoint("gpt-tiny", ["perplexity"], batches=2, batch_size=2, seq_len=32, device="cpu")
