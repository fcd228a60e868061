"""The engine on the GPU with projections in 4 bits and completions of one prompt: the operators one after the other, as a decoding step uses them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    return cuda_device


def _engine(cfg, **kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    return InferenceEngine(cfg, **{"max_batch_size": 12, "max_batch_tokens": 8192, "num_kv_blocks": 512, **kw})


def _config(heads=4, hidden=512):
    from llmctl_b200.models.config import ModelConfig
    return ModelConfig(name="completions-test", layers=2, hidden=hidden, ffn=1408, heads=heads, vocab_size=4096, max_position_embeddings=1024)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("weights", ["auto", "int4"])
@pytest.mark.parametrize("heads,hidden", [(4, 512), (4, 256)])
def test_completions(graphs, weights, heads, hidden, monkeypatch):
    """Greedy tokens against a full recomputation: the best one or next to it (bf16 layers differ by 2^-8 of their numbers)."""
    from llmctl_b200.serve import engine
    monkeypatch.setattr(engine, "_SHARED_BYTES", 1)
    eng = _engine(_config(heads, hidden), weight_dtype=weights, cuda_graphs=graphs)
    calls, shared = [], engine.sops.paged_attention_decode_shared
    monkeypatch.setattr(engine.sops, "paged_attention_decode_shared", lambda *a: (calls.append(a[0].shape), shared(*a))[1])
    prompts = [torch.randint(3, 4000, (n,)).tolist() for n in (203, 64)]
    seqs = [(p, s) for p, n in zip(prompts, (5, 3)) for s in eng.add_requests(p, n, 18, 0.0)]
    seqs.append((prompts[1][:9], eng.add_request(prompts[1][:9], 18, 0.0)))
    while eng.has_work():
        eng.step()
    assert calls and eng.kv.free_blocks == 512
    for p, s in seqs:
        assert len(s.generated) == 18
        logits = eng.model(torch.tensor([p + s.generated[:-1]], device="cuda")).float()[len(p) - 1:, :4096]
        chosen = logits.gather(1, torch.tensor(s.generated, device="cuda")[:, None])[:, 0]
        assert (logits.amax(1) - chosen <= 0.1 * logits.std()).all()


def test_a_step_with_shared_prefixes_gives_the_logits_of_one_without(monkeypatch):
    from llmctl_b200.serve import engine
    monkeypatch.setattr(engine, "_SHARED_BYTES", 1)
    eng = _engine(_config(), cuda_graphs=False)
    seqs = eng.add_requests(torch.randint(3, 4000, (600,)).tolist(), 6, 20, 1.0) + [eng.add_request([5, 6, 7], 20, 1.0)]
    for _ in range(3):
        eng.step()
    order, groups = eng._in_groups(seqs)
    assert groups == [(6, 592)] and order == seqs
    with_groups, without = eng._decode(order, groups).float(), eng._decode(order).float()
    assert (with_groups - without).norm() / without.norm() < 0.02


def test_int4_against_the_same_numbers_in_bf16():
    """A model with its projections in 4 bits and the same numbers rounded to bf16 weights: one token, a batch, a prompt."""
    from llmctl_b200.models.int4 import Int4Linear
    from llmctl_b200.ops import functional as ops
    cfg = _config()
    a, b = _engine(cfg, weight_dtype="int4"), _engine(cfg)
    of = dict(a.model.named_modules())
    with torch.no_grad():
        for path, m in b.model.named_modules():
            if isinstance(of.get(path), Int4Linear):
                m.weight.copy_(ops.dequantize_int4(of[path].weight, of[path].scale))
    for n in (1, 7, 20, 100, 300):
        x = torch.randint(3, 4000, (1, n), device="cuda")
        with torch.no_grad():
            y, z = a.model(x).float(), b.model(x).float()
        assert (y - z).norm() / z.norm() < 0.03
