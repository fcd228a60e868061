"""Completions of one prompt that share its blocks, and models whose projections stay in 4 bits: the engine, the block manager, the server, the command."""
import json

import pytest
import torch


def _engine(artifact="gpt-tiny", **kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    return InferenceEngine(artifact, device="cpu", **{"kv_block_size": 4, "num_kv_blocks": 64, "max_batch_size": 6, "max_batch_tokens": 512, **kw})


def _is_greedy(eng, prompt, out, slack=1e-4):
    for i, t in enumerate(out):
        logits = eng.model(torch.tensor([prompt + out[:i]])).float()[-1, :eng.cfg.vocab_size]
        assert logits.max() - logits[t] <= slack


def test_blocks_are_shared_and_given_back():
    from llmctl_b200.serve.native_host import KVBlockManager
    kv = KVBlockManager(16, 4, 0.0)
    assert kv.allocate(1, 10) and kv.allocate(2, 10)
    assert kv.free_blocks == 10
    own = kv.block_table(2)
    kv.share(1, 2, 2)
    a, b = kv.block_table(1), kv.block_table(2)
    assert a[:2] == b[:2] and b[2] == own[2] and kv.free_blocks == 12
    kv.share(1, 2, 2)                          # again: nothing changes
    assert kv.free_blocks == 12 and kv.block_table(2) == b
    assert kv.allocate(2, 13) and kv.block_table(2)[:3] == b
    assert kv.free(1) == 1 and kv.free_blocks == 12          # the shared two stay for the other
    assert kv.allocate(3, 48) and not set(kv.block_table(3)) & set(b)
    assert kv.free(2) == 4 and kv.free(3) == 12 and kv.free_blocks == 16
    for args in ((1, 2, 1), (7, 8, 0)):
        with pytest.raises(RuntimeError, match="share"):
            kv.share(*args)
    kv.allocate(1, 4), kv.allocate(2, 8)
    for args in ((1, 2, 2), (2, 1, 2), (1, 2, -1)):
        with pytest.raises(RuntimeError, match="share"):
            kv.share(*args)


@pytest.mark.parametrize("length", [1, 4, 15, 33])
@pytest.mark.parametrize("cache", ["auto", "fp8"])
def test_completions_of_one_prompt(length, cache, monkeypatch):
    from llmctl_b200.serve import engine
    monkeypatch.setattr(engine, "_SHARED_BYTES", 1)
    eng = _engine(kv_cache_dtype=cache)
    prompt, steps = torch.randint(3, 500, (length,)).tolist(), []
    decode = eng._decode
    monkeypatch.setattr(eng, "_decode", lambda seqs, groups=None: (steps.append(groups), decode(seqs, groups))[1])
    alone = eng.generate([prompt], max_tokens=6, temperature=0.0)[0]
    spent = eng.stats["prefill_tokens"]
    seqs = eng.add_requests(prompt, 4, 6, 0.0) + [eng.add_request([9, 8, 7], 6, 0.0)]
    eng.step()
    whole = length // 4
    tables = [eng.kv.block_table(s.req_id) for s in seqs[:4]]
    assert all(t[:whole] == tables[0][:whole] for t in tables) and len({t[-1] for t in tables}) == 4
    assert eng.stats["prefill_tokens"] - spent == length + 3
    while eng.has_work():
        eng.step()
    for s in seqs[:4]:
        _is_greedy(eng, prompt, s.generated, 1e-4 if cache == "auto" else 0.2)
    if cache == "auto":
        assert all(s.generated == alone for s in seqs[:4])
        assert ([(4, whole * 4)] in steps) == (whole > 0)
    _is_greedy(eng, [9, 8, 7], seqs[4].generated, 1e-4 if cache == "auto" else 0.2)
    assert eng.kv.free_blocks == 64 and all(s.prompt_logits is None for s in seqs)


def test_completions_that_come_and_go(monkeypatch):
    """More completions than seats, too few blocks (preemptions), some that are cancelled: each one's tokens are its own prompt's."""
    from llmctl_b200.serve import engine
    monkeypatch.setattr(engine, "_SHARED_BYTES", 1)
    eng = _engine(num_kv_blocks=24, max_batch_size=4)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(3, 500, (n,), generator=g).tolist() for n in (18, 9)]
    seqs = [(p, s) for p in prompts for s in eng.add_requests(p, 5, 14, 0.0)]
    for i in range(400):
        if not eng.has_work():
            break
        if i == 3:
            seqs[0][1].cancel_requested = True
        eng.step()
    assert not eng.has_work() and eng.kv.free_blocks == 24
    for p, s in seqs[1:]:
        assert len(s.generated) == 14
        _is_greedy(eng, p, s.generated)


def test_more_than_no_completion():
    with pytest.raises(ValueError, match="at least one"):
        _engine().add_requests([1, 2], 0)
    assert len(_engine().generate([[1, 2], [3]], max_tokens=3, n=2)) == 4


def test_server_gives_choices():
    from fastapi.testclient import TestClient
    from llmctl_b200.serve.server import InferenceServer
    server = InferenceServer("gpt-tiny", engine=_engine())
    server.start_background()
    try:
        with TestClient(server.app) as client:
            r = client.post("/v1/completions", json={"prompt": "hello there", "max_tokens": 5, "temperature": 0.0, "n": 3, "logprobs": 1}).json()
            assert [c["index"] for c in r["choices"]] == [0, 1, 2] and len({c["id"] for c in r["choices"]}) == 3
            assert len({c["text"] for c in r["choices"]}) == 1 and all(len(c["logprobs"]["tokens"]) == c["usage"]["completion_tokens"] for c in r["choices"])
            assert r["usage"]["completion_tokens"] == sum(c["usage"]["completion_tokens"] for c in r["choices"])
            one = client.post("/v1/completions", json={"prompt": "hello there", "max_tokens": 5, "temperature": 0.0}).json()
            assert one["text"] == r["choices"][0]["text"] and "choices" not in one
            assert client.post("/v1/completions", json={"prompt": "a", "n": 2, "stream": True}).status_code == 422
            assert client.post("/v1/completions", json={"prompt": "a", "n": 0}).status_code == 422
    finally:
        server.shutdown()


def test_a_server_takes_no_more_completions_than_requests():
    from fastapi.testclient import TestClient
    from llmctl_b200.serve.server import InferenceServer
    server = InferenceServer("gpt-tiny", engine=_engine(), max_concurrent_requests=3)
    server.start_background()
    try:
        with TestClient(server.app) as client:
            ask = lambda n: client.post("/v1/completions", json={"prompt": "a", "max_tokens": 2, "n": n}).status_code  # noqa: E731
            assert [ask(n) for n in (4, 3, 1)] == [503, 200, 200] and not server.active_requests
    finally:
        server.shutdown()


def test_weights_in_4_bits(tmp_path):
    """An int4 artifact's codes are served as they stand; other weights are quantised."""
    from safetensors.torch import save_file
    from llmctl_b200.io.quantize import Int4GroupQuantizer
    from llmctl_b200.models.int4 import Int4Linear
    plain = _engine()
    sd = {k: v.detach().clone() for k, v in plain.model.named_parameters()}
    codes = Int4GroupQuantizer().quantize(sd)
    eng = _engine(weight_dtype="int4")
    layers = [m for m in eng.model.modules() if isinstance(m, Int4Linear)]
    assert len(layers) == 4 * eng.cfg.layers + 1 and eng.dtype == torch.float32
    (tmp_path / "model_config.json").write_text(json.dumps(eng.cfg.to_dict()))
    (tmp_path / "export.json").write_text(json.dumps({"quantization": "int4"}))
    save_file({k: v.contiguous() for k, v in codes.items()}, str(tmp_path / "model.safetensors"))
    served = _engine(str(tmp_path), weight_dtype="int4")
    for a, b, (path, _) in zip(served.model.modules(), eng.model.modules(), eng.model.named_modules()):
        if isinstance(a, Int4Linear):
            assert torch.equal(a.weight, codes[path + ".weight"]) and torch.equal(a.scale, codes[path + ".weight.scale"]) and torch.equal(a.weight, b.weight)
    prompt = [5, 6, 7, 200, 9]
    outs = served.generate([prompt], max_tokens=6, temperature=0.0)
    _is_greedy(served, prompt, outs[0])
    assert outs == eng.generate([prompt], max_tokens=6, temperature=0.0)
    # the same numbers as bf16 weights
    loaded = _engine(str(tmp_path))
    x = torch.tensor([prompt])
    a, b = served.model(x), loaded.model(x)
    assert (a - b).norm() / b.norm() < 0.02


def test_weights_in_4_bits_are_refused_elsewhere():
    from typer.testing import CliRunner
    from llmctl_b200.cli.main import app
    from llmctl_b200.config.schemas import ServeConfig
    with pytest.raises(ValueError, match="weight_dtype"):
        _engine(weight_dtype="int2")
    assert ServeConfig(artifact="x", weight_dtype="int4").weight_dtype == "int4"
    with pytest.raises(ValueError):
        ServeConfig(artifact="x", weight_dtype="int3")
    run = lambda *a: CliRunner().invoke(app, ["serve", "start", "--artifact", "gpt-tiny", "--dry-run", *a])  # noqa: E731
    assert run("--weight-dtype", "int4").exit_code == 0
    assert run("--weight-dtype", "int5").exit_code != 0
    assert run("--weight-dtype", "int4", "--tensor-parallel", "2").exit_code != 0
