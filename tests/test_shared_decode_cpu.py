"""Decode attention over shared prefixes: the plain form against 64 bits, refusals."""
import pytest
import torch

import shared_decode_oracle as oracle
from llmctl_b200.ops import serving as sops


@pytest.mark.parametrize("groups,singles", [([(3, 32)], 0), ([(1, 16), (4, 40)], 2), ([], 3), ([(2, 0), (2, 8)], 1)])
def test_plain_form(groups, singles):
    s = oracle.batch(groups, [5, 1, 17], 8, 4, 2, 16, singles=singles)
    oracle.check(sops.paged_attention_decode_shared(**s), oracle.attention(**s))


def test_a_sequence_without_tokens_and_one_shorter_than_its_group():
    s = oracle.batch([(3, 32)], [4], 8, 2, 2, 16)
    s["context_lens"] = torch.tensor([36, 0, 20], dtype=torch.int32)
    got = sops.paged_attention_decode_shared(**s)
    oracle.check(got, oracle.attention(**s))
    assert not got[1].any()


def test_the_shared_tokens_are_those_of_the_first_table():
    s = oracle.batch([(2, 16)], [3], 8, 2, 2, 16)
    want = oracle.attention(**s)
    s["block_tables"][1, :2] = 0
    oracle.check(sops.paged_attention_decode_shared(**s), want)


def test_refusals():
    s = oracle.batch([(2, 16)], [3], 8, 4, 2, 16)
    bad = [dict(q=s["q"][0]), dict(k_cache=s["k_cache"].float()), dict(v_cache=s["v_cache"][:1]), dict(k_cache=s["k_cache"].transpose(1, 2)), dict(q=s["q"][:, :3]),
           dict(block_tables=s["block_tables"].long()), dict(block_tables=s["block_tables"][:1]), dict(context_lens=s["context_lens"][:1]), dict(context_lens=s["context_lens"].long()),
           dict(group_starts=s["group_starts"][:1]), dict(shared_lens=s["shared_lens"].long()), dict(group_starts=s["group_starts"].float()), dict(scale=0.0), dict(scale=-1.0)]
    for change in bad:
        with pytest.raises(ValueError):
            sops.paged_attention_decode_shared(**{**s, **change})
    with pytest.raises(ValueError, match="no backward"):
        sops.paged_attention_decode_shared(**{**s, "q": s["q"].requires_grad_(True)})
