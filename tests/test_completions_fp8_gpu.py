"""Completions of one prompt over a cache of 8 bits on the GPU: a late one has the prompt's last block as it stands alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    return cuda_device


@pytest.mark.parametrize("length", [5, 64, 203])
def test_a_late_completion_has_the_prompt_as_it_stands_alone(length):
    from llmctl_b200.comms import mesh
    from llmctl_b200.models.config import ModelConfig
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    cfg = ModelConfig(name="completions-test", layers=2, hidden=256, ffn=704, heads=4, vocab_size=4096, max_position_embeddings=1024)
    eng = InferenceEngine(cfg, kv_cache_dtype="fp8", max_batch_size=2, max_batch_tokens=8192, num_kv_blocks=128)
    with torch.no_grad():
        for blk in eng.model.blocks:            # tokens whose keys and values are of unlike size
            blk.attn.qkv.weight[:, ::7] *= 40
    prompt, whole, rows = torch.randint(3, 4000, (length,)).tolist(), length // 16, length % 16

    def last_block(seq):
        b = eng.kv.block_table(seq.req_id)[whole]
        return [x for caches, scales in ((eng.k_caches, eng.k_scales), (eng.v_caches, eng.v_scales)) for c, s in zip(caches, scales)
                for x in (c[b, :, :rows].contiguous().view(torch.uint8), s[b].clone())]

    seq = eng.add_request(prompt, 10, 0.0)
    eng.step()
    alone = last_block(seq) if rows else []
    while eng.has_work():
        eng.step()
    eng.add_request([9, 8, 7], 8, 0.0)          # takes the second seat for eight steps
    first, late = eng.add_requests(prompt, 2, 10, 0.0)
    while not late.generated:
        eng.step()
    assert len(first.generated) >= 8 and eng.kv.block_table(first.req_id)[:whole] == eng.kv.block_table(late.req_id)[:whole]
    if rows:
        assert all(torch.equal(a, b) for a, b in zip(last_block(late), alone))
    while eng.has_work():
        eng.step()
    assert eng.kv.free_blocks == 128 and late.group.tail is None and len(late.generated) == 10
