"""Append with rotation and the paged cache of 8 bits on the CPU: the plain forms against the oracle in 64 bits, and what the operators refuse."""
import pytest
import torch

import fp8_cache_oracle as oracle


@pytest.fixture
def sops():
    from llmctl_b200.ops import serving
    return serving


def _rows(T, H, Hk, D, seed=0, dtype=torch.float32):
    return torch.randn(T, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _tables(D, n=64):
    from llmctl_b200.ops import functional
    return functional.rope_tables(D, n)


def _state(blocks, Hk, size, D, seed=1):
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp2(torch.randint(-6, 1, (blocks, Hk), generator=g).float())
    return (torch.randn(blocks, Hk, size, D, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn), scale


# what the slots of a call look like: (rows to a block, slots)
SLOTS = [
    (16, list(range(40))),                                # a prompt from the first row of a block
    (16, [5]),                                            # one token behind others
    (16, [21, 22, 23, 3, 40, 41]),                        # portions of several sequences
    (8, [7, 8, 15, 16, -1, 31, 64, 10 ** 12]),            # ends of blocks, slots outside of the cache
    (16, [33, 2, 34, 1, 33, 32]),                         # one block's rows apart and out of order, a slot twice, a block begun last
    (5, [4, 5, 6, 7, 8, 9, 10]),                          # blocks of odd size
    (16, [-1, -1]),
]


@pytest.mark.parametrize("size,slots", SLOTS)
@pytest.mark.parametrize("H,Hk,D", [(2, 2, 16), (6, 2, 32)])
def test_append_of_8_bits(sops, size, slots, H, Hk, D):
    T, blocks = len(slots), 4
    qkv, (cos, sin) = _rows(T, H, Hk, D), _tables(D)
    qkv[:, -D:] *= 30
    qkv[0, H * D] = 0.0
    positions = torch.tensor([(7 * i) % 64 for i in range(T)], dtype=torch.int32)
    slots = torch.tensor(slots)
    (k, ks), (v, vs) = _state(blocks, Hk, size, D), _state(blocks, Hk, size, D, seed=2)
    x = qkv.view(T, H + 2 * Hk, D).clone()
    rotated = oracle.rotated32(x[:, :H + Hk], cos[positions.long()], sin[positions.long()], fused=False)
    want_k = oracle.append(rotated[:, H:], k.double(), ks.double(), slots)
    want_v = oracle.append(x[:, H + Hk:], v.double(), vs.double(), slots)
    assert sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D, kv_heads=Hk, k_scale=ks, v_scale=vs) is qkv
    assert torch.equal(qkv.view(T, -1, D)[:, :H + Hk], rotated) and torch.equal(qkv.view(T, -1, D)[:, H + Hk:], x[:, H + Hk:])
    for got, want in (((k, ks), want_k), ((v, vs), want_v)):
        assert torch.equal(got[0].double(), want[0]) and torch.equal(got[1].double(), want[1])


def test_a_block_keeps_its_numbers_as_its_scale_grows(sops):
    """Twelve tokens one by one, each larger than the one before: what the codes stand for is off by at most half a step of e4m3 (2^-4 of the
    number), and among the subnormals by half their step for each doubling that is still to come: together less than one subnormal step of the last scale."""
    H, D, size = 1, 16, 16
    cos, sin = torch.ones(1, D // 2), torch.zeros(1, D // 2)
    (k, ks), (v, vs) = sops.allocate_fp8_cache(1, size, H, D), sops.allocate_fp8_cache(1, size, H, D)
    said = []
    for t in range(12):
        row = _rows(1, H, H, D, seed=t) * 1.9 ** t
        said.append(row[0, D:2 * D].clone())
        sops.rope_kv_append(row, cos, sin, torch.zeros(1, dtype=torch.int32), k, v, torch.tensor([t]), H, D, k_scale=ks, v_scale=vs)
    held, said = k[0, 0, :12].double() * ks[0, 0].double(), torch.stack(said).double()
    assert ((held - said).abs() <= 2.0 ** -4 * said.abs() + 2.0 ** -9 * float(ks[0, 0])).all()
    assert float(ks[0, 0]) == 2.0 ** round(float(torch.log2(ks[0, 0])))


def test_numbers_that_are_not_finite(sops):
    H, D = 1, 16
    cos, sin = torch.ones(1, D // 2), torch.zeros(1, D // 2)
    (k, ks), (v, vs) = sops.allocate_fp8_cache(2, 4, H, D), sops.allocate_fp8_cache(2, 4, H, D)
    row = _rows(1, H, H, D)
    row[0, 2 * D], row[0, 2 * D + 1], row[0, 2 * D + 2] = float("inf"), float("nan"), 3.0e38
    sops.rope_kv_append(row, cos, sin, torch.zeros(1, dtype=torch.int32), k, v, torch.tensor([4]), H, D, k_scale=ks, v_scale=vs)
    assert v[1, 0, 0].float().isnan().tolist() == [True, True] + [False] * (D - 2)
    assert vs[1, 0] == oracle.scale_for(3.0e38) and vs[0, 0] == 0 and k[1, 0, 0].float().isfinite().all()


@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 2)])
def test_append_of_16_bits_is_rotation_and_append(sops, H, Hk):
    from llmctl_b200.ops import functional
    T, D, dtype = 7, 32, torch.bfloat16
    qkv, (cos, sin) = _rows(T, H, Hk, D, dtype=dtype), _tables(D)
    positions, slots = torch.tensor([3, 4, 5, 0, 1, 63, 9], dtype=torch.int32), torch.tensor([3, 4, 5, 8, 9, -1, 99])
    want = functional.rope_packed(qkv.clone(), cos, sin, H + Hk, D, 64, positions)
    k, v = torch.zeros(4, 4, Hk, D, dtype=dtype), torch.zeros(4, 4, Hk, D, dtype=dtype)
    sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D, kv_heads=Hk)
    assert torch.equal(qkv, want)
    kept = slots[:5]
    for c, first in ((k, H), (v, H + Hk)):
        assert torch.equal(c.view(-1, Hk, D)[kept], want.view(T, -1, D)[:5, first:first + Hk])
        c.view(-1, Hk, D)[kept] = 0
        assert not c.any()


@pytest.mark.parametrize("D", [2, 8, 24, 40])
def test_append_of_16_bits_takes_any_even_head(sops, D):
    """Heads of a multiple of 16 are what kernels and caches of 8 bits need; the plain form of the others' does not."""
    from llmctl_b200.ops import functional
    T, H = 5, 3
    qkv, (cos, sin) = _rows(T, 3 * H, 0, D), _tables(D)
    positions, slots = torch.tensor([3, 4, 5, 0, 63], dtype=torch.int32), torch.tensor([3, 4, 5, 8, -1])
    want = functional.rope_packed(qkv.clone(), cos, sin, 2 * H, D, 64, positions)
    k, v = torch.zeros(4, 4, H, D), torch.zeros(4, 4, H, D)
    sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D)
    assert torch.equal(qkv, want)
    for c, first in ((k, H), (v, 2 * H)):
        assert torch.equal(c.view(-1, H, D)[slots[:4]], want.view(T, -1, D)[:4, first:first + H])
    codes, scales = torch.zeros(1, H, 4, D, dtype=torch.float8_e4m3fn), torch.zeros(1, H)
    with pytest.raises(ValueError, match="multiple of 16"):
        sops.rope_kv_append(qkv, cos, sin, positions, codes, codes.clone(), slots, H, D, k_scale=scales, v_scale=scales.clone())
    with pytest.raises(ValueError, match="even"):
        sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D + 1)


@pytest.mark.parametrize("head", [8, 24, 40])
def test_engine_on_the_cpu_serves_any_even_head(head):
    from llmctl_b200.comms import mesh
    from llmctl_b200.models.config import ModelConfig
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    cfg = ModelConfig(name="heads-test", layers=2, hidden=4 * head, ffn=64, heads=4, vocab_size=300, max_position_embeddings=64)
    eng = InferenceEngine(cfg, device="cpu", kv_block_size=4, num_kv_blocks=64, max_batch_size=2, max_batch_tokens=128)
    prompts = [[5, 6, 7, 8, 9], [11]]
    for p, o in zip(prompts, eng.generate(prompts, max_tokens=6, temperature=0.0)):
        assert len(o) == 6
        for i, t in enumerate(o):
            logits = eng.model(torch.tensor([p + o[:i]])).float()[-1, :300]
            assert logits.max() - logits[t] <= 1e-4


@pytest.mark.parametrize("H,Hk,size", [(2, 2, 16), (6, 2, 5)])
def test_attention(sops, H, Hk, size):
    B, D = 4, 64
    lens = torch.tensor([1, 0, 2 * size + 3, 3 * size], dtype=torch.int32)
    tables = torch.tensor([[3, 0, 0], [0, 0, 0], [7, 1, 5], [2, 4, 6]], dtype=torch.int32)
    (k, ks), (v, vs) = _state(8, Hk, size, D), _state(8, Hk, size, D, seed=2)
    k.view(torch.uint8)[5, :, 3:] = v.view(torch.uint8)[5, :, 3:] = 0x7f                # NaN behind the third sequence
    q = torch.randn(B, H, D, generator=torch.Generator().manual_seed(5)) * 0.01
    for most in (3 * size, size + 2):
        got = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, lens, most)
        want, bound = oracle.attend(q, k, ks, v, vs, tables, lens, D ** -0.5, most)
        assert ((got.double() - want).abs() <= oracle.tolerance(want, bound, D)).all()
    assert not got[1].any()


def test_refusals(sops):
    T, H, Hk, D, size = 3, 4, 2, 32, 8
    cos, sin = _tables(D)
    good = {"qkv": _rows(T, H, Hk, D), "cos": cos, "sin": sin, "positions": torch.zeros(T, dtype=torch.int32), "k_cache": None, "v_cache": None,
            "slot_mapping": torch.arange(T), "heads": H, "head_dim": D, "kv_heads": Hk}
    (good["k_cache"], good["k_scale"]), (good["v_cache"], good["v_scale"]) = sops.allocate_fp8_cache(2, size, Hk, D), sops.allocate_fp8_cache(2, size, Hk, D)

    def call(**other):
        return sops.rope_kv_append(**{**good, **other})
    call()
    wide = torch.zeros(2, Hk, size, 2 * D, dtype=torch.float8_e4m3fn)
    for other in ({"qkv": good["qkv"][:, 1:]}, {"heads": 3}, {"head_dim": 8}, {"positions": torch.zeros(T, dtype=torch.int64)}, {"positions": torch.zeros(T + 1, dtype=torch.int32)},
                  {"slot_mapping": torch.zeros(T, dtype=torch.int32)}, {"slot_mapping": torch.arange(T + 1)}, {"cos": cos.double()}, {"sin": sin[:5]}, {"cos": cos[:, :3], "sin": sin[:, :3]},
                  {"k_scale": None}, {"k_scale": good["k_scale"][:1]}, {"v_scale": good["v_scale"].double()}, {"k_cache": wide[..., ::2]}, {"v_cache": wide},
                  {"v_cache": good["v_cache"].to(torch.float8_e5m2)}, {"k_cache": torch.zeros(2, size, Hk, D)}, {"qkv": good["qkv"].clone().requires_grad_(True)},
                  {"k_cache": torch.zeros(2, size, Hk, D), "v_cache": torch.zeros(2, size, Hk, D)},
                  {"k_cache": torch.zeros(2, size, Hk, D).half(), "v_cache": torch.zeros(2, size, Hk, D).half(), "k_scale": None, "v_scale": None}):
        with pytest.raises(ValueError):
            call(**other)
    q = torch.randn(2, H, D)
    fine = (q, good["k_cache"], good["v_cache"], good["k_scale"], good["v_scale"], torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), 16)
    sops.paged_attention_decode_fp8(*fine)
    for i, bad in ((0, torch.randn(2, 3, D)), (0, torch.randn(2, H, D, requires_grad=True)), (1, wide), (2, good["v_cache"].float()), (3, good["k_scale"][:1]), (5, torch.zeros(1, 2, dtype=torch.int32)),
                   (5, torch.zeros(2, 2, dtype=torch.int64)), (6, torch.ones(1, dtype=torch.int32)), (6, torch.ones(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            sops.paged_attention_decode_fp8(*fine[:i], bad, *fine[i + 1:])


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls the entry point with addresses of nothing: it has to end at the missing device")
@pytest.mark.parametrize("block_size", [16, 5])
@pytest.mark.parametrize("batch,heads,kv_heads", [(1, 32, 32), (16, 32, 32), (3, 8, 2)])
def test_a_cache_without_blocks_needs_no_scratch(sops, block_size, batch, heads, kv_heads):
    """What a launch writes to scratch has to fit into what is asked for beforehand, which does not know of the cache's blocks: without blocks it writes nothing,
    so that the entry point takes a null and goes on to the launch (refused arguments are answered with 1)."""
    from llmctl_b200.ops import native
    if not native.available():
        pytest.skip("library not built")
    for limit in (0, 1, 512, 1000, 4096, 100000):
        for splits in (0, 1, 3, 256):
            rc = native.lib().llmctl_paged_attn_decode_fp8(4096, heads * 128, 4096, 4096, 4096, 4096, 4096, limit // block_size + 1, 4096, 4096, None, batch, heads, kv_heads, 128, 0, block_size, limit,
                                                           splits, 1.0, None)
            assert rc not in (0, 1)


def test_attention_over_a_cache_without_blocks(sops):
    (k, ks), (v, vs) = (sops.allocate_fp8_cache(0, 16, 2, 64) for _ in range(2))
    out = sops.paged_attention_decode_fp8(torch.randn(2, 4, 64), k, v, ks, vs, torch.zeros(2, 256, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 4096)
    assert not out.any()


def _engine(**kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    return InferenceEngine("gpt-tiny", device="cpu", kv_block_size=4, num_kv_blocks=64, **kw)


def test_engine_with_a_cache_of_8_bits():
    """Greedy tokens of a served model are its best or next to it: the logits of a full recomputation differ by what e4m3 rounds (half a step of 2^-4 of
    a key or value, in a model whose logits spread by about 1)."""
    eng = _engine(max_batch_size=3, max_batch_tokens=256, kv_cache_dtype="fp8")
    assert all(c.dtype == torch.float8_e4m3fn for c in eng.k_caches + eng.v_caches) and len(eng.k_scales) == len(eng.v_scales) == 2
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(3, 500, (n,), generator=g).tolist() for n in (1, 9, 30)]
    outs = eng.generate(prompts, max_tokens=7, temperature=0.0)
    assert eng.kv.free_blocks == 64 and all(s.any() for s in eng.k_scales + eng.v_scales)
    for p, o in zip(prompts, outs):
        assert len(o) == 7
        for i, t in enumerate(o):
            logits = eng.model(torch.tensor([p + o[:i]])).float()[-1, :512]
            assert logits.max() - logits[t] <= 0.1 * logits.std()
    plain = _engine(max_batch_size=3, max_batch_tokens=256)
    bytes_of = [sum(t.numel() * t.element_size() for t in e.k_caches + getattr(e, "k_scales", [])) for e in (plain, eng)]
    assert bytes_of[1] < 0.3 * bytes_of[0]                     # of 32 bits here


def test_engine_refuses_what_has_no_cache_of_8_bits():
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        _engine(kv_cache_dtype="int3")
    from llmctl_b200.config.schemas import ServeConfig
    assert ServeConfig(artifact="x", kv_cache_dtype="fp8").kv_cache_dtype == "fp8"
    with pytest.raises(ValueError):
        ServeConfig(artifact="x", kv_cache_dtype="fp9")


def test_serve_command_takes_the_cache_type():
    from typer.testing import CliRunner
    from llmctl_b200.cli.main import app
    r = CliRunner().invoke(app, ["serve", "start", "--artifact", "gpt-tiny", "--kv-cache-dtype", "fp8", "--dry-run"])
    assert r.exit_code == 0, r.output
    assert CliRunner().invoke(app, ["serve", "start", "--artifact", "gpt-tiny", "--kv-cache-dtype", "fp4", "--dry-run"]).exit_code != 0
