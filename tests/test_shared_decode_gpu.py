"""Decode attention over shared prefixes on the GPU, against 64 bits: groups and heads of every form, odd lengths, bad pages, strides, streams, graphs."""
import pytest
import torch

import shared_decode_oracle as oracle
from llmctl_b200.ops import native, serving as sops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    torch.cuda.synchronize()
    native.check_waits("test")


def run(s):
    with torch.no_grad():
        return sops.paged_attention_decode_shared(**s)


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (3, 3, 128), (8, 2, 128), (12, 2, 64), (5, 1, 64)])
@pytest.mark.parametrize("groups,after,page,singles", [
    ([(2, 16)], [1], 16, 0), ([(4, 300)], [20, 1, 129], 16, 0), ([], [1, 127, 128, 129, 300], 8, 7), ([(1, 64), (33, 128), (2, 264), (0, 40)], [3, 200], 8, 2),
    ([(40, 1000)], [1, 2, 3], 64, 1), ([(3, 256), (2, 2560)], [100], 256, 0), ([(2, 48), (3, 96)], [30, 70], 24, 1)])
def test_against_64_bits(heads, kv_heads, dim, groups, after, page, singles):
    s = oracle.batch(groups, after, page, heads, kv_heads, dim, device="cuda", singles=singles)
    oracle.check(run(s), oracle.attention(**s))


def test_more_rows_than_a_tile_and_more_entries_than_threads():
    s = oracle.batch([(2, 16)] * 120, [9, 1], 16, 2, 2, 64, device="cuda", singles=10)
    oracle.check(run(s), oracle.attention(**s))
    s = oracle.batch([(50, 400)], [40, 300], 16, 32, 4, 128, device="cuda")
    oracle.check(run(s), oracle.attention(**s))


def test_scores_far_apart():
    """References that move from tile to tile, and rows whose largest score comes first, last or in the shared part."""
    s = oracle.batch([(3, 512)], [400, 130, 7], 16, 4, 4, 128, device="cuda", spread=12.0)
    oracle.check(run(s), oracle.attention(**s))
    s["scale"] = 1e-4
    oracle.check(run(s), oracle.attention(**s))


def test_shared_tokens_that_are_no_whole_blocks():
    s = oracle.batch([(4, 320)], [50, 9], 16, 4, 2, 64, device="cuda")
    want = oracle.attention(**s)
    for n in (0, 1, 13, 127, 200, 319, 320):
        s["shared_lens"] = torch.tensor([n], dtype=torch.int32, device="cuda")
        oracle.check(run(s), want)


def test_lengths_that_end_early():
    s = oracle.batch([(4, 320)], [50], 16, 4, 2, 64, device="cuda")
    s["context_lens"] = torch.tensor([370, 0, 33, 320], dtype=torch.int32, device="cuda")
    got = run(s)
    oracle.check(got, oracle.attention(**s))
    assert not got[1].any()
    s["context_lens"] = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert not run(s).any()
    s["context_lens"] = torch.tensor([10 ** 9, -5, 2 ** 31 - 1, 370], dtype=torch.int32, device="cuda")      # beyond the table: left out
    s["block_tables"] = s["block_tables"][:, :20].contiguous()
    s["shared_lens"] = torch.tensor([10 ** 9], dtype=torch.int32, device="cuda")
    assert torch.isfinite(run(s)).all()


def test_bad_pages_and_groups_out_of_order_read_nothing_else():
    s = oracle.batch([(3, 64), (2, 32)], [20], 16, 4, 4, 64, device="cuda")
    good = run(s)
    tables = s["block_tables"].clone()
    s["block_tables"][1, 4] = -7
    s["block_tables"][4, 2] = 2 ** 30
    got = run(s)
    assert torch.isfinite(got).all() and all(torch.equal(got[i], good[i]) for i in (0, 2, 3))
    s["block_tables"] = tables
    for starts in ([0, 3, 3], [3, 0, 5], [5, 5, 5], [-4, 2, 99], [0, 5, 0]):
        s["group_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        assert torch.isfinite(run(s)[:2]).all()


def test_strides_and_no_sequences():
    s = oracle.batch([(3, 64)], [20], 16, 4, 4, 64, device="cuda")
    want = run(s)
    packed = torch.zeros(3, 12 * 64, device="cuda", dtype=torch.bfloat16)
    packed[:, :256] = s["q"].reshape(3, 256)
    assert torch.equal(run({**s, "q": packed[:, :256].view(3, 4, 64)}), want)
    assert torch.equal(run({**s, "q": s["q"].transpose(1, 2).contiguous().transpose(1, 2)}), want)
    odd = torch.zeros(3 * 256 + 1, device="cuda", dtype=torch.bfloat16)
    odd[1:] = s["q"].reshape(-1)
    assert torch.equal(run({**s, "q": odd[1:].view(3, 4, 64)}), want)
    wide = torch.zeros(3, 40, dtype=torch.int32, device="cuda")
    wide[:, :s["block_tables"].shape[1]] = s["block_tables"]
    assert torch.equal(run({**s, "block_tables": wide[:, :s["block_tables"].shape[1]]}), want)
    assert run({**s, "q": s["q"][:0]}).shape == (0, 4, 64)


def test_caches_past_32_bits():
    """Blocks at the end of a cache of more than 2^31 numbers."""
    s = oracle.batch([(5, 320)], [50, 9], 16, 32, 32, 128, device="cuda")
    want, blocks, need = run(s), 40_000, s["k_cache"].shape[0]
    far = {**s, "block_tables": s["block_tables"] + (blocks - need)}
    for name in ("k_cache", "v_cache"):
        far[name] = torch.empty(blocks, 16, 32, 128, dtype=torch.bfloat16, device="cuda")
        far[name][-need:] = s[name]
    assert far["k_cache"].numel() > 2 ** 31 and torch.equal(run(far), want)


def test_refusals_on_the_gpu():
    s = oracle.batch([(2, 16)], [3], 8, 4, 2, 64, device="cuda")
    for change in [dict(q=s["q"].cpu()), dict(q=s["q"].float(), k_cache=s["k_cache"].float(), v_cache=s["v_cache"].float()), dict(context_lens=s["context_lens"].cpu()),
                   dict(shared_lens=s["shared_lens"].cpu()), dict(k_cache=s["k_cache"].half()), dict(scale=0.0)]:
        with pytest.raises(ValueError):
            run({**s, **change})
    for other in (oracle.batch([(2, 16)], [3], 12, 4, 2, 64, device="cuda"), oracle.batch([(2, 16)], [3], 8, 4, 2, 32, device="cuda")):
        with pytest.raises(ValueError, match="multiple of 8|64 or 128"):
            run(other)
    with pytest.raises(ValueError, match="no backward"):
        sops.paged_attention_decode_shared(**{**s, "q": s["q"].requires_grad_(True)})


def test_graphs_follow_the_lengths_and_run_beside_one_another():
    a = oracle.batch([(6, 512)], [200, 3], 16, 8, 8, 128, device="cuda")
    b = oracle.batch([(5, 96), (2, 800)], [33], 16, 8, 2, 128, seed=1, device="cuda")
    graphs, outs = [], []
    for s in (a, b):
        run(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for shorter in (0, 1, 150):
        for s in (a, b):
            s["context_lens"].sub_(shorter).clamp_(min=1)
        want = [oracle.attention(**s) for s in (a, b)]
        torch.cuda.synchronize()
        for g, t in zip(graphs, streams):
            with torch.cuda.stream(t):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = run(a)
        torch.cuda.synchronize()
        for o, w in zip((*outs, eager), (*want, want[0])):
            oracle.check(o, w)
