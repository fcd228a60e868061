"""Append with rotation and decode attention over the paged cache of 8 bits: the kernels against the oracle in 64 bits."""
import pytest
import torch

import fp8_cache_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture
def sops(cuda_device):
    from llmctl_b200.ops import serving
    return serving


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed=0, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=_gen(seed)) * std).bfloat16()


def _tables(D, n=4096):
    from llmctl_b200.ops import functional
    return functional.rope_tables(D, n, device="cuda")


def _state(blocks, Hk, size, D, seed=1):
    g = _gen(seed)
    scale = torch.exp2(torch.randint(-8, 1, (blocks, Hk), device="cuda", generator=g).float())
    return (torch.randn(blocks, Hk, size, D, device="cuda", generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _prompt(n, first=0):
    return list(range(first, first + n))


SLOTS = [
    (16, [5]), (16, _prompt(40)), (16, [21, 22, 23, 3, 40, 41]), (8, [7, 8, 15, 16, -1, 31, 64, 10 ** 12]), (16, [33, 2, 34, 1, 33, 32]), (16, [-1, -1]),
    (64, _prompt(70, 3)), (200, _prompt(333, 150)), (16, _prompt(300, 7)), (16, _prompt(290, 160) + _prompt(20, 25) + [-1] * 9 + [30, 160, 161, 30]), (1, [0, 3, 2, 2]), (24, _prompt(29, 20)),
]


@pytest.mark.parametrize("size,slots", SLOTS)
@pytest.mark.parametrize("H,Hk,D", [(12, 12, 64), (8, 2, 128), (3, 1, 96), (2, 2, 16), (1, 1, 512)])
def test_append_of_8_bits(sops, size, slots, H, Hk, D):
    T, blocks = len(slots), (600 + size - 1) // size if size > 1 else 4
    qkv, (cos, sin) = _randn(T, (H + 2 * Hk) * D), _tables(D)
    qkv[:, -D:] *= 30
    positions = torch.tensor([(37 * i) % 4096 for i in range(T)], dtype=torch.int32, device="cuda")
    slots = torch.tensor(slots, device="cuda")
    (k, ks), (v, vs) = _state(blocks, Hk, size, D), _state(blocks, Hk, size, D, seed=2)
    ks[:, 0] = 0
    k[:, 0] = torch.zeros_like(k[:, 0])
    x = qkv.view(T, H + 2 * Hk, D).clone()
    rotated = oracle.rotated32(x[:, :H + Hk], cos[positions.long()], sin[positions.long()], fused=True)
    want_k = oracle.append(rotated[:, H:].cpu(), k.cpu().double(), ks.cpu().double(), slots.cpu())
    want_v = oracle.append(x[:, H + Hk:].float().cpu(), v.cpu().double(), vs.cpu().double(), slots.cpu())
    assert sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D, kv_heads=Hk, k_scale=ks, v_scale=vs) is qkv
    assert torch.equal(qkv.view(T, -1, D)[:, :H + Hk], rotated.bfloat16()) and torch.equal(qkv.view(T, -1, D)[:, H + Hk:], x[:, H + Hk:])
    for got, want in (((k, ks), want_k), ((v, vs), want_v)):
        assert torch.equal(got[0].cpu().double(), want[0]) and torch.equal(got[1].cpu().double(), want[1])


@pytest.mark.parametrize("order", ["prompts", "any"])
@pytest.mark.parametrize("size", [16, 64, 3])
@pytest.mark.parametrize("T", [200, 512, 513, 2999, 3000, 5001])
def test_append_of_long_calls(sops, T, size, order):
    """Prompts one after the other, and tokens in any order; some without a row, some slots named twice by tokens far from each other."""
    H, Hk, D = 2, 1, 32
    blocks = 6000 // size
    if order == "any":
        slots = torch.randperm(blocks * size, generator=torch.Generator().manual_seed(T + size))[:T]
    else:
        table = torch.randperm(blocks, generator=torch.Generator().manual_seed(T + size))
        at = torch.cat([torch.arange(7, 7 + T // 3), torch.arange((T // 3 // size + 2) * size, (T // 3 // size + 2) * size + T - T // 3)])
        slots = table[at // size] * size + at % size
    slots[T // 5::97] = -1
    slots[T - 40:] = slots[:40]
    slots[T // 2] = slots[3]
    qkv, (cos, sin) = _randn(T, (H + 2 * Hk) * D), _tables(D)
    qkv *= torch.exp2(torch.randint(-3, 4, (T, 1), device="cuda", generator=_gen(9)).float()).bfloat16()
    positions = torch.arange(T, dtype=torch.int32, device="cuda") % 4096
    (k, ks), (v, vs) = _state(blocks, Hk, size, D), _state(blocks, Hk, size, D, seed=2)
    x = qkv.view(T, H + 2 * Hk, D).clone()
    rotated = oracle.rotated32(x[:, :H + Hk], cos[positions.long()], sin[positions.long()], fused=True)
    want_k = oracle.append(rotated[:, H:].cpu(), k.cpu().double(), ks.cpu().double(), slots)
    want_v = oracle.append(x[:, H + Hk:].float().cpu(), v.cpu().double(), vs.cpu().double(), slots)
    sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots.cuda(), H, D, kv_heads=Hk, k_scale=ks, v_scale=vs)
    assert torch.equal(qkv.view(T, -1, D)[:, :H + Hk], rotated.bfloat16()) and torch.equal(qkv.view(T, -1, D)[:, H + Hk:], x[:, H + Hk:])
    for got, want in (((k, ks), want_k), ((v, vs), want_v)):
        assert torch.equal(got[0].cpu().double(), want[0]) and torch.equal(got[1].cpu().double(), want[1])


def test_long_calls_captured_and_without_scratch(sops):
    """A captured long call on other rows and slots, and the C entry without the scratch for its marks: the same bytes as the eager call."""
    from llmctl_b200.ops import native
    T, H, D, size, blocks = 4001, 2, 32, 16, 300
    cos, sin = _tables(D)
    positions = torch.arange(T, dtype=torch.int32, device="cuda") % 4096
    rows = [_randn(T, 3 * H * D, seed=s) for s in (1, 2)]
    slots = [torch.randperm(blocks * size, device="cuda", generator=_gen(s))[:T] for s in (3, 4)]
    state = [_state(blocks, H, size, D, seed=s) for s in (5, 6)]

    def fresh():
        return [x.clone() for pair in state for x in pair]

    def run(qkv, at, c):
        sops.rope_kv_append(qkv, cos, sin, positions, c[0], c[2], at, H, D, k_scale=c[1], v_scale=c[3])

    want = []
    for i in range(2):
        qkv, c = rows[i].clone(), fresh()
        run(qkv, slots[i], c)
        want.append([qkv, *c])
    held, at, c = rows[0].clone(), slots[0].clone(), fresh()
    run(held, at, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(held, at, c)
    for i in (1, 0):
        for x, y in zip((held, at, *c), (rows[i], slots[i], *fresh())):
            x.copy_(y)
        graph.replay()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((held, *c), want[i]))
    qkv, c = rows[0].clone(), fresh()
    native.call("llmctl_rope_kv_append_fp8", qkv.data_ptr(), qkv.stride(0), T, H, H, D, cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), slots[0].data_ptr(),
                c[0].data_ptr(), c[2].data_ptr(), c[1].data_ptr(), c[3].data_ptr(), blocks, size, None, native.stream_ptr())
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((qkv, *c), want[0]))


def test_numbers_that_are_not_finite(sops):
    H, D = 2, 64
    cos, sin = _tables(D)
    (k, ks), (v, vs) = sops.allocate_fp8_cache(2, 8, H, D, "cuda"), sops.allocate_fp8_cache(2, 8, H, D, "cuda")
    row = _randn(2, 3 * H * D)
    row[0, 2 * H * D], row[0, 2 * H * D + 1], row[1, 2 * H * D] = float("inf"), float("nan"), 3.0e38
    row[:, H * D] = float("-inf")
    sops.rope_kv_append(row, cos, sin, torch.tensor([0, 5], dtype=torch.int32, device="cuda"), k, v, torch.tensor([8, 9], device="cuda"), H, D, k_scale=ks, v_scale=vs)
    assert v[1, 0, 0].float().isnan().tolist() == [True, True] + [False] * (D - 2) and not v[1, 1].float().isnan().any()
    assert float(vs[1, 0]) == oracle.scale_for(float(row[1, 2 * H * D])) and not vs[0].any() and not k[0].float().any()
    assert k[1, 0, 0, 0].float().isnan() and ks.isfinite().all()


@pytest.mark.parametrize("H,Hk,D", [(12, 12, 64), (8, 2, 128), (3, 1, 96)])
@pytest.mark.parametrize("T", [1, 33, 1777])
def test_append_of_16_bits_is_rotation_and_append(sops, H, Hk, D, T):
    """The same bits as the rotation in place and the append one after the other."""
    from llmctl_b200.ops import functional
    qkv, (cos, sin) = _randn(T, (H + 2 * Hk) * D), _tables(D)
    positions = torch.randint(0, 4096, (T,), device="cuda", generator=_gen(3)).int()
    slots = torch.randperm(4000, device="cuda", generator=_gen(4))[:T]
    slots[T // 2] = -1
    slots[T // 3] = 16 * 250
    want = functional.rope_packed(qkv.clone(), cos, sin, H + Hk, D, 4096, positions)
    k, v = (torch.zeros(250, 16, Hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D, kv_heads=Hk)
    assert torch.equal(qkv, want)
    kept = (slots >= 0) & (slots < 4000)
    for c, first in ((k, H), (v, H + Hk)):
        plain = torch.zeros_like(c)
        plain.view(-1, Hk, D)[slots[kept]] = want.view(T, -1, D)[kept, first:first + Hk]
        assert torch.equal(c, plain)


@pytest.mark.parametrize("form", ["wide", "odd", "columns"])
@pytest.mark.parametrize("fp8", [False, True])
def test_append_of_other_layouts(sops, form, fp8):
    """Rows of a wider buffer, at odd addresses, and columns: the same as from packed rows, what lies beside them is left."""
    T, H, D = 5, 2, 64
    width = 3 * H * D
    cos, sin = _tables(D)
    positions, slots = torch.arange(T, device="cuda", dtype=torch.int32), torch.arange(3, 3 + T, device="cuda")

    def run(qkv):
        if fp8:
            (k, ks), (v, vs) = (sops.allocate_fp8_cache(2, 8, H, D, "cuda") for _ in range(2))
        else:
            (k, ks), (v, vs) = ((torch.zeros(2, 8, H, D, device="cuda", dtype=torch.bfloat16), None) for _ in range(2))
        out = sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D, k_scale=ks, v_scale=vs)
        return out[:, :width].clone(), k.float(), v.float()
    plain = _randn(T, width)
    buf = _randn(T * (width + 9) + 1, seed=5)
    if form == "wide":
        qkv = buf[:T * (width + 8)].view(T, width + 8)
    elif form == "odd":
        qkv = buf[1:].view(T, width + 9)
    else:
        qkv = _randn(width, T, seed=5).t()
    qkv[:, :width] = plain
    beside = qkv[:, width:].clone()
    for a, b in zip(run(qkv), run(plain)):
        assert torch.equal(a, b)
    assert torch.equal(qkv[:, width:], beside)


def _batch(lens, size, seed=0):
    """Block tables over pages in any order, two of them in nobody's table."""
    pages = [(n + size - 1) // size for n in lens]
    perm = torch.randperm(sum(pages) + 2, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.zeros(len(lens), max(pages + [1]), dtype=torch.int32), 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[at:at + n]
        at += n
    return table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), sum(pages) + 2


LENS = [[1], [300], [1, 0, 17, 128, 129, 500], [127, 128, 256, 255, 257], [2000, 3, 999], [0, 0]]


@pytest.mark.parametrize("H,Hk,D,size", [(12, 12, 64, 16), (4, 4, 128, 16), (8, 2, 128, 64), (24, 4, 64, 8), (8, 1, 128, 32), (16, 1, 64, 16), (32, 1, 128, 16), (2, 2, 128, 5), (2, 1, 64, 24),
                                         (2, 2, 128, 128), (2, 2, 64, 256)])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("splits", [None, 1, 3, 12])
def test_attention(sops, H, Hk, D, size, lens, splits):
    tables, n, blocks = _batch(lens, size)
    (k, ks), (v, vs) = _state(blocks, Hk, size, D), _state(blocks, Hk, size, D, seed=2)
    k[:, :, :, 3] = (k[:, :, :, 3].float() * 4).clamp(-448, 448).to(k.dtype)
    for b, c in enumerate(lens):                           # NaN behind every sequence's last token
        if c % size:
            for t in (k, v):
                t.view(torch.uint8)[int(tables[b, c // size]), :, c % size:] = 0x7f
    qkv = _randn(len(lens), (H + 2 * Hk) * D, seed=5, std=0.1)
    q = qkv[:, :H * D].view(len(lens), H, D)
    got = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, max(lens + [1]), num_splits=splits).cpu().double()
    want, bound = oracle.attend(q.cpu(), k.cpu().float(), ks.cpu(), v.cpu().float(), vs.cpu(), tables.cpu(), n.cpu(), D ** -0.5)
    assert ((got - want).abs() <= oracle.tolerance(want, bound, D)).all()


@pytest.mark.parametrize("H,Hk,D", [(8, 1, 128), (6, 1, 64), (32, 4, 64), (2, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("key_step,value_step", [(0.01, 0.0), (0.2, 0.0), (0.0, 0.15), (0.05, -0.3), (-0.2, 1.0)])
@pytest.mark.parametrize("splits", [None, 1])
def test_attention_of_rising_scores(sops, H, Hk, D, key_step, value_step, splits):
    """Keys along the query whose scores rise (or fall) from block to block, values whose scales do, by little and by much: as far as any weight's reference is left standing, and beyond."""
    size, lens = 16, [1900, 131, 700]
    tables, n, blocks = _batch(lens, size)
    (k, ks), (v, vs) = _state(blocks, Hk, size, D), _state(blocks, Hk, size, D, seed=2)
    q = _randn(len(lens), H, D, seed=5, std=0.02) + 0.1
    for b, c in enumerate(lens):
        for page in range((c + size - 1) // size):
            at = int(tables[b, page])
            k[at] = (k[at].float() * 0.05 + 10 + page * key_step * 10).clamp(-448, 448).to(k.dtype)
            ks[at] = 2.0 ** -4
            vs[at] = 2.0 ** round(page * value_step)
    got = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, max(lens), num_splits=splits).cpu().double()
    want, bound = oracle.attend(q.cpu(), k.cpu().float(), ks.cpu(), v.cpu().float(), vs.cpu(), tables.cpu(), n.cpu(), D ** -0.5)
    assert ((got - want).abs() <= oracle.tolerance(want, bound, D)).all()


@pytest.mark.parametrize("size", [16, 5])
def test_attention_scales(sops, size):
    """Scales of values that differ by 2^60 between pages, a page of zeros, keys that decide alone, and a scale of the softmax."""
    H, D, lens = 2, 128, [5 * size]
    tables, n, blocks = _batch(lens, size)
    (k, ks), (v, vs) = _state(blocks, H, size, D), _state(blocks, H, size, D, seed=2)
    q = _randn(1, H, D, seed=5)
    ks[:] = 2.0 ** -9
    for page, (a, b) in enumerate([(0.0, 0.0), (2.0 ** -3, 2.0 ** -30), (2.0 ** -9, 2.0 ** 30), (2.0 ** -7, 1.0), (2.0 ** -8, 2.0 ** -60)]):
        ks[int(tables[0, page])], vs[int(tables[0, page])] = a, b
    for scale in (D ** -0.5, 0.5, 1e-3):
        got = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, lens[0], scale=scale).cpu().double()
        want, bound = oracle.attend(q.cpu(), k.cpu().float(), ks.cpu(), v.cpu().float(), vs.cpu(), tables.cpu(), n.cpu(), scale)
        # a weight's error is relative to it: what bounds the result's is the sum of the weighted magnitudes, not the largest value
        kk = (k.cpu().double() * ks.cpu().double()[..., None, None])[tables[0].long().cpu()].transpose(0, 1).reshape(H, -1, D)
        vv = (v.cpu().double() * vs.cpu().double()[..., None, None])[tables[0].long().cpu()].transpose(0, 1).reshape(H, -1, D)
        p = torch.softmax(torch.einsum("hd,hnd->hn", q[0].cpu().double(), kk) * scale, -1)
        weighted = torch.einsum("hn,hnd->hd", p, vv.abs())[None]
        score = (D + 16) * 2.0 ** -23 * bound[..., 0:1]
        # weights a 2^-28 part of the largest weighted value (of any dimension) and less may be lost
        lost = 2.0 ** -28 * lens[0] * (p[..., None] * vv.abs()).amax((1, 2))[None, :, None] * 2
        assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2 * score + 2.0 ** -11) * weighted + lost).all()


def test_attention_of_many_small_weights(sops):
    """One key of a large score before 20000 whose weights are 2^-20 of its own: they count together."""
    H, D, size, n = 1, 128, 16, 20001
    tables, lens, blocks = _batch([n], size)
    k, v = (torch.zeros(blocks, H, size, D, device="cuda") for _ in range(2))
    k[int(tables[0, 0]), 0, 0, 0] = 20 * 0.6931471805599453 * D ** 0.5
    v[...] = 1.0
    v[int(tables[0, 0]), 0, 0] = -1.0
    q = torch.zeros(1, H, D, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1
    one = torch.ones(blocks, H, device="cuda")
    k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
    for splits in (1, 7):
        got = sops.paged_attention_decode_fp8(q, k, v, one, one, tables, lens, n, num_splits=splits).cpu().double()
        want, bound = oracle.attend(q.cpu(), k.cpu().float(), one.cpu(), v.cpu().float(), one.cpu(), tables.cpu(), lens.cpu(), D ** -0.5)
        assert ((got - want).abs() <= oracle.tolerance(want, bound, D)).all()


def test_attention_bad_pages_and_limits(sops):
    """A block outside of the cache gives NaN and reads nothing; tokens beyond max_context or the table are left out."""
    H, D, size = 2, 64, 16
    tables, n, blocks = _batch([40, 40, 40], size)
    (k, ks), (v, vs) = _state(blocks, H, size, D), _state(blocks, H, size, D, seed=2)
    q = _randn(3, H, D, std=0.1)
    good = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, 40)
    tables[1, 1], tables[2, 2] = blocks, -7
    bad = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, 40)
    assert torch.equal(bad[0], good[0]) and bad[1:].isnan().all()
    n2 = n.clone()
    n2[0] = 10 ** 9
    want, bound = oracle.attend(q.cpu()[:1], k.cpu().float(), ks.cpu(), v.cpu().float(), vs.cpu(), tables.cpu()[:1], n.cpu()[:1] - 7, D ** -0.5)
    got = sops.paged_attention_decode_fp8(q[:1], k, v, ks, vs, tables, n2, 33)[:1].cpu().double()
    assert ((got - want).abs() <= oracle.tolerance(want, bound, D)).all()
    assert torch.equal(sops.paged_attention_decode_fp8(q[:1], k, v, ks, vs, tables[:, :2].contiguous(), n2, 10 ** 6), sops.paged_attention_decode_fp8(q[:1], k, v, ks, vs, tables, n2, 32))


def _attend64(q, k, ks, v, vs, tables, lens):
    """The oracle's formula and bounds, a sequence at a time on the GPU."""
    B, H, D = q.shape
    Hk, size = k.shape[1], k.shape[2]
    out, bound = torch.zeros(B, H, D, device="cuda", dtype=torch.float64), torch.zeros(B, H, 2, device="cuda", dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = tables[b, :(n + size - 1) // size].long()
        kk, vv = ((c[pages].double() * s[pages].double()[..., None, None]).transpose(0, 1).reshape(Hk, -1, D)[:, :n] for c, s in ((k, ks), (v, vs)))
        qq = q[b].double().view(Hk, H // Hk, D)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", qq, kk) * D ** -0.5, -1)
        out[b] = torch.einsum("hgn,hnd->hgd", p, vv).reshape(H, D)
        bound[b, :, 0] = (torch.einsum("hgd,hnd->hgn", qq.abs(), kk.abs()).amax(-1) * D ** -0.5).reshape(H)
        bound[b, :, 1] = vv.abs().amax((1, 2)).repeat_interleave(H // Hk)
    return out, bound


def _lens(B, most, every=7):
    """Contexts of unlike lengths, some sequences without tokens (the first and the last, and runs of them) among them."""
    return [0 if i % every in (0, 3) or i == B - 1 or 20 <= i < 26 else 1 + (i * 7919 + 13) % most for i in range(B - 1)] + [0]


# What a CTA's run is: (sequences, longest context, ...) of whole items, one or two of them and more, two and three CTAs to an SM; of items of four kinds of groups;
# of tiles that begin and end inside of items, behind the first 32 sequences and the first 64, two and three CTAs to an SM
MANY = [(70, 200, 16, 16, 128, 16), (70, 200, 8, 8, 128, 16), (150, 300, 24, 4, 64, 16), (300, 140, 16, 1, 64, 8), (200, 260, 8, 4, 64, 32), (300, 150, 4, 4, 64, 16), (40, 1000, 8, 8, 128, 16),
        (40, 3000, 4, 4, 128, 16), (100, 2000, 4, 2, 64, 16), (70, 2000, 8, 1, 128, 64), (40, 2500, 16, 1, 64, 16), (64, 5200, 16, 16, 128, 64)]


@pytest.mark.parametrize("B,most,H,Hk,D,size", MANY)
@pytest.mark.parametrize("splits", [None, 1, 40])
def test_attention_of_many_sequences(sops, B, most, H, Hk, D, size, splits):
    lens = _lens(B, most)
    tables, n, blocks = _batch(lens, size)
    (k, ks), (v, vs) = _state(blocks, Hk, size, D), _state(blocks, Hk, size, D, seed=2)
    q = _randn(B, H, D, seed=5, std=0.1)
    got = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, max(lens), num_splits=splits).double()
    want, bound = _attend64(q, k, ks, v, vs, tables, lens)
    assert ((got - want).abs() <= oracle.tolerance(want, bound, D)).all()


def test_a_wait_that_ran_out_is_raised_by_the_next_call(sops):
    """The byte that the decode kernel sets when a wait of its runs out, set by a kernel that does nothing else."""
    from llmctl_b200.ops import native
    tables, n, blocks = _batch([20], 16)
    (k, ks), (v, vs) = (sops.allocate_fp8_cache(blocks, 16, 2, 64, "cuda") for _ in range(2))
    q = _randn(1, 2, 64)
    native.register_signature("llmctl_wait_status_report", [native.c_int, native.c_void_p])
    native.call("llmctl_wait_status_report", 4, native.stream_ptr())
    torch.cuda.synchronize()
    with pytest.raises(native.NativeError, match=native._OTHER_WAITS[0]):
        sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, 20)
    assert sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, 20).isfinite().all()
    native.check_waits()


@pytest.mark.parametrize("size", [16, 5])
@pytest.mark.parametrize("B,H,Hk,D,limit", [(1, 32, 32, 128, 4096), (16, 32, 32, 128, 4096), (3, 8, 2, 64, 20000), (2, 2, 2, 64, 100)])
def test_attention_over_a_cache_without_blocks(sops, B, H, Hk, D, limit, size):
    """Zeros for sequences without tokens, NaN for others (their blocks lie outside of the cache), and what lies behind the results is left."""
    (k, ks), (v, vs) = (sops.allocate_fp8_cache(0, size, Hk, D, "cuda") for _ in range(2))
    tables, n = torch.zeros(B, limit // size + 1, device="cuda", dtype=torch.int32), torch.zeros(B, device="cuda", dtype=torch.int32)
    for splits in (None, 3):
        assert not sops.paged_attention_decode_fp8(_randn(B, H, D), k, v, ks, vs, tables, n, limit, num_splits=splits).any()
        n[0] = 70
        out = sops.paged_attention_decode_fp8(_randn(B, H, D), k, v, ks, vs, tables, n, limit, num_splits=splits)
        assert out[0].isnan().all() and not out[1:].any()
        n[0] = 0


def test_run_together_in_a_graph_beside_another(sops):
    """Prompt, then decoding steps of append and attention over the same cache: captured twice and replayed side by side on two streams, each against the
    oracle's view of the cache."""
    H, Hk, D, size, B = 8, 2, 128, 16, 3
    cos, sin = _tables(D)

    def conversation(seed):
        lens = [37, 16, 200]
        tables, n, blocks = _batch([x + 8 for x in lens], size, seed)
        caches = [*sops.allocate_fp8_cache(blocks, size, Hk, D, "cuda"), *sops.allocate_fp8_cache(blocks, size, Hk, D, "cuda")]
        for b, x in enumerate(lens):
            at = torch.arange(x, device="cuda")
            sops.rope_kv_append(_randn(x, (H + 2 * Hk) * D, seed=seed + b), cos, sin, at.int(), caches[0], caches[2], tables[b].long()[at // size] * size + at % size, H, D, kv_heads=Hk,
                                k_scale=caches[1], v_scale=caches[3])
        qkv, positions, slots = torch.zeros(B, (H + 2 * Hk) * D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, device="cuda", dtype=torch.int32), torch.full((B,), -1, device="cuda")
        ctx = torch.zeros(B, device="cuda", dtype=torch.int32)

        def step():
            sops.rope_kv_append(qkv, cos, sin, positions, caches[0], caches[2], slots, H, D, kv_heads=Hk, k_scale=caches[1], v_scale=caches[3])
            return sops.paged_attention_decode_fp8(qkv[:, :H * D].view(B, H, D), caches[0], caches[2], caches[1], caches[3], tables, ctx, 256)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            out = step()
        return lens, tables, caches, qkv, positions, slots, ctx, graph, out, side
    both = [conversation(10), conversation(20)]
    for i in range(3):
        for j, (lens, tables, caches, qkv, positions, slots, ctx, graph, out, side) in enumerate(both):
            at = torch.tensor([x + i for x in lens], device="cuda")
            qkv.copy_(_randn(*qkv.shape, seed=100 * j + i))
            positions.copy_(at)
            ctx.copy_(at + 1)
            slots.copy_(tables[torch.arange(B, device="cuda"), at // size].long() * size + at % size)
        torch.cuda.synchronize()
        for c in both:
            with torch.cuda.stream(c[-1]):
                c[-3].replay()
        torch.cuda.synchronize()
        for lens, tables, caches, qkv, positions, slots, ctx, graph, out, side in both:
            q = qkv[:, :H * D].view(B, H, D).cpu()
            want, bound = oracle.attend(q, caches[0].cpu().float(), caches[1].cpu(), caches[2].cpu().float(), caches[3].cpu(), tables.cpu(), ctx.cpu(), D ** -0.5)
            assert ((out.cpu().double() - want).abs() <= oracle.tolerance(want, bound, D)).all()


def test_gpu_refusals(sops):
    H, D = 2, 64
    (k, ks), (v, vs) = (sops.allocate_fp8_cache(2, 8, H, D, "cuda") for _ in range(2))
    tables, n = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q = _randn(1, H, D)
    sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, n, 8)
    for args in ((q.float(), k, v, ks, vs, tables, n, 8), (q, k.cpu(), v, ks, vs, tables, n, 8), (q, k, v, ks.cpu(), vs, tables, n, 8), (q, k, v, ks, vs, tables.cpu(), n, 8),
                 (q, k, v, ks, vs, tables, n.cpu(), 8), (_randn(1, H, 32), *(c for _ in range(2) for c in [sops.allocate_fp8_cache(2, 8, H, 32, "cuda")[0]]), ks, vs, tables, n, 8)):
        with pytest.raises(ValueError):
            sops.paged_attention_decode_fp8(*args)
    cos, sin = _tables(D)
    p, s = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    for args in ((_randn(1, 3 * H * D).half(), cos, sin, p, k, v, s), (_randn(1, 3 * H * D), cos.cpu(), sin, p, k, v, s), (_randn(1, 3 * H * D), cos, sin, p.cpu(), k, v, s),
                 (_randn(1, 3 * H * D), cos, sin, p, k, v, s.cpu())):
        with pytest.raises(ValueError):
            sops.rope_kv_append(*args, H, D, k_scale=ks, v_scale=vs)
    from llmctl_b200.ops import native
    assert native.lib().llmctl_paged_attn_decode_fp8(q.data_ptr(), H * D, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), tables.data_ptr(), 2, n.data_ptr(), q.data_ptr(), None, 1, H, H, 32, 2,
                                                     8, 8, 1, 1.0, native.stream_ptr()) == 1


@pytest.mark.parametrize("D", [64, 128])
def test_values_and_keys_that_are_no_numbers(sops, D):
    """A NaN among the values reaches its dimension of its head's output and no other, one among the keys or the queries the whole of its head."""
    H, size, n = 2, 16, 100
    tables, lens, blocks = _batch([n] * 4, size)
    (k, ks), (v, vs) = _state(blocks, H, size, D), _state(blocks, H, size, D, seed=2)
    q = _randn(4, H, D, std=0.1)
    plain = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, lens, n)
    v.view(torch.uint8)[int(tables[0, 2]), 1, 3, 5] = 0x7f
    k.view(torch.uint8)[int(tables[1, 6]), 0, 3, 7] = 0xff
    q[2, 1, 3], q[3, 0, 0] = float("inf"), float("nan")
    for splits in (None, 1, 3):
        out = sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, lens, n, num_splits=splits)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[0, 1, 5], bad[1, 0], bad[2, 1], bad[3, 0] = True, True, True, True
        assert torch.equal(out.isnan(), bad)
        assert torch.allclose(out[~bad].float(), plain[~bad].float(), rtol=2.0 ** -6, atol=1e-3)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("heads,hidden", [(4, 512), (4, 256)])
def test_engine_with_a_cache_of_8_bits(sops, graphs, heads, hidden):
    """Greedy tokens against a full recomputation in bf16: the best one or next to it, prompts and decoding steps past the ends of blocks, graphs or not."""
    from llmctl_b200.comms import mesh
    from llmctl_b200.models.config import ModelConfig
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    cfg = ModelConfig(name="fp8-test", layers=2, hidden=hidden, ffn=704, heads=heads, vocab_size=4096, max_position_embeddings=512)
    eng = InferenceEngine(cfg, max_batch_size=4, max_batch_tokens=2048, num_kv_blocks=256, kv_cache_dtype="fp8", cuda_graphs=graphs)
    prompts = [torch.randint(3, 4000, (n,)).tolist() for n in (17, 64, 5, 130)]
    outs = eng.generate(prompts, max_tokens=20, temperature=0.0)
    for p, o in zip(prompts, outs):
        for i, t in enumerate(o):
            logits = eng.model(torch.tensor([p + o[:i]], device="cuda")).float()[-1, :4096]
            assert logits.max() - logits[t] <= 0.15 * logits.std()
    assert eng.kv.free_blocks == 256


def test_engine_refuses_heads_that_the_kernel_has_not(sops):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    with pytest.raises(ValueError, match="heads of 32"):
        InferenceEngine("gpt-tiny", num_kv_blocks=16, kv_cache_dtype="fp8")


def test_engine_of_16_bits_gives_the_bits_of_rotation_and_append(sops, monkeypatch):
    """The engine's one kernel for rotation and append against the two that it had: the same logits and caches bit for bit."""
    from llmctl_b200.comms import mesh
    from llmctl_b200.models.config import ModelConfig
    from llmctl_b200.ops import functional
    from llmctl_b200.serve.engine import InferenceEngine
    cfg = ModelConfig(name="append-test", layers=2, hidden=256, ffn=704, heads=4, vocab_size=4096, max_position_embeddings=512)
    prompts = [list(range(3, 3 + n)) for n in (17, 40)]

    def run(old):
        mesh.reset_state()
        eng = InferenceEngine(cfg, max_batch_size=2, max_batch_tokens=1024, num_kv_blocks=64, cuda_graphs=False)
        if old:
            def append(i, qkv, positions, slots):
                cos, sin = eng.model.rope_tables(eng.device)
                qkv = functional.rope_packed(qkv, cos, sin, 8, 64, 512, positions)
                sops.kv_append(qkv, eng.k_caches[i], eng.v_caches[i], slots, 4, 64)
                return qkv
            eng._append = append
        return eng.generate(prompts, max_tokens=9, temperature=0.0), eng.k_caches + eng.v_caches
    (a, ca), (b, cb) = run(True), run(False)
    assert a == b and all(torch.equal(x, y) for x, y in zip(ca, cb))
