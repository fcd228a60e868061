"""Completions of one prompt over a cache of 8 bits: a block that the prompt does not fill, and completions that come when others have gone on in theirs."""
import pytest
import torch


def _engine(**kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    eng = InferenceEngine("gpt-tiny", device="cpu", kv_cache_dtype="fp8", **{"kv_block_size": 16, "num_kv_blocks": 64, "max_batch_size": 2, "max_batch_tokens": 512, **kw})
    with torch.no_grad():
        for blk in eng.model.blocks:            # tokens whose keys and values are of unlike size
            blk.attn.qkv.weight[:, ::7] *= 40
    return eng


def _last_block(eng, seq, rows):
    """Codes and scales of the prompt's last block, layer by layer."""
    b = eng.kv.block_table(seq.req_id)[len(seq.prompt_ids) // eng.block_size]
    return [(c[b, :, :rows].view(torch.uint8).clone(), s[b].clone()) for caches, scales in ((eng.k_caches, eng.k_scales), (eng.v_caches, eng.v_scales)) for c, s in zip(caches, scales)]


@pytest.mark.parametrize("length", [3, 5, 16, 19, 27])
def test_a_late_completion_has_the_prompt_as_it_stands_alone(length):
    eng, rows = _engine(), length % 16
    prompt = torch.randint(3, 500, (length,), generator=torch.Generator().manual_seed(5)).tolist()
    eng.add_request(prompt, 10, 0.0)
    eng.step()
    alone = _last_block(eng, next(iter(eng.seqs.values())), rows) if rows else []
    while eng.has_work():
        eng.step()
    eng.add_request([9, 8, 7], 8, 0.0)          # takes the second seat for eight steps
    first, late = eng.add_requests(prompt, 2, 10, 0.0)
    while not late.generated:
        eng.step()
    assert len(first.generated) >= 8 and len(late.generated) == 1
    assert eng.kv.block_table(first.req_id)[:length // 16] == eng.kv.block_table(late.req_id)[:length // 16]
    if rows:
        grown = _last_block(eng, first, rows)
        assert any((a[1] != b[1]).any() for a, b in zip(grown, alone)), "the first one's own tokens changed no scale"
        for got, want in zip(_last_block(eng, late, rows), alone):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    while eng.has_work():
        eng.step()
    assert late.group.held == [] and late.group.tail is None
