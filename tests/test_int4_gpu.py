"""Products with weights of 4 bits on the GPU, against 64 bits: every way a call can take, odd sizes, strides, streams, graphs."""
import pytest
import torch

from llmctl_b200.ops import functional as ops, native

from int4_oracle import check, matrix, product

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    torch.cuda.synchronize()
    native.check_waits("test")


def tokens(n, width, seed=1):
    x = torch.randn(n, width, generator=torch.Generator().manual_seed(seed))
    x[:, 5] *= 30                     # a channel of outliers
    return x.bfloat16().cuda()


def run(x, w, scale, gated):
    return (ops.linear_swiglu_int4 if gated else ops.linear_int4)(x, w, scale)


# chunks of 8 tokens with one and two tiles of rows, the tensor cores' kernel with 16, 32 and 64 tokens and several chunks of them, widened weights
@pytest.mark.parametrize("n,width,rows", [(1, 128, 1), (1, 4096, 4096), (2, 256, 33), (7, 1280, 9500), (8, 11008, 130), (9, 128, 16), (16, 4096, 12289), (31, 384, 200), (33, 5120, 9000),
                                          (64, 11008, 4096), (65, 4096, 13001), (128, 4224, 12800), (129, 256, 24), (190, 5120, 9000), (193, 5120, 9000), (200, 4096, 1001)])
@pytest.mark.parametrize("gated", [False, True])
def test_against_64_bits(n, width, rows, gated):
    x = tokens(n, width)
    w, scale = matrix(rows * (2 if gated else 1), width, 2, "cuda")
    check(run(x, w, scale, gated), product(x, w, scale, gated, widened=n > ops._int4_tokens(w)))


@pytest.mark.parametrize("n", [3, 40, 250])
@pytest.mark.parametrize("gated", [False, True])
def test_layouts(n, gated):
    x, (w, scale) = tokens(n, 5120), matrix(9216, 5120, 3, "cuda")
    want = run(x, w, scale, gated)
    wide = torch.zeros(n, 5128, device="cuda", dtype=torch.bfloat16)
    wide[:, :5120] = x
    odd = torch.zeros(n * 5120 + 1, device="cuda", dtype=torch.bfloat16)
    odd[1:] = x.view(-1)
    for other in (wide[:, :5120], x.t().contiguous().t(), odd[1:].view(n, 5120), x.view(1, n, 5120)):
        assert torch.equal(run(other, w, scale, gated).reshape(n, -1), want)
    w2 = torch.zeros(9216, 2576, device="cuda", dtype=torch.uint8)
    w2[:, :2560] = w
    s2 = torch.zeros(9216, 43, device="cuda", dtype=torch.half)
    s2[:, 1:41] = scale
    bytes_ = torch.zeros(w.numel() + 3, device="cuda", dtype=torch.uint8)
    bytes_[3:] = w.view(-1)
    for a, b in ((w2[:, :2560], s2[:, 1:41]), (w.t().contiguous().t(), scale.t().contiguous().t()), (bytes_[3:].view(9216, 2560), scale)):
        assert torch.equal(run(x, a, b, gated), want)


def test_nothing_to_do():
    w, scale = matrix(64, 256, 4, "cuda")
    assert ops.linear_int4(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), w, scale).shape == (0, 64)
    assert ops.linear_int4(torch.empty(3, 256, device="cuda", dtype=torch.bfloat16), w[:0], scale[:0]).shape == (3, 0)


@pytest.mark.parametrize("n", [2, 20, 240])
def test_numbers_that_are_not_finite_stay_with_their_token(n):
    x, (w, scale) = tokens(n, 4096), matrix(13000, 4096, 5, "cuda")
    clean = ops.linear_int4(x, w, scale)
    x[1, 77] = float("inf")
    x[0, 4095] = float("nan")
    got = ops.linear_int4(x, w, scale)
    assert torch.equal(got[2:], clean[2:]) and got[0].isnan().all() and not got[1].isfinite().any()


@pytest.mark.parametrize("n", [4, 48])
def test_other_types_take_the_plain_form(n):
    w, scale = matrix(48, 256, 6, "cuda")
    x = tokens(n, 256).float()
    got = ops.linear_int4(x, w, scale)
    assert got.dtype == torch.float32
    torch.testing.assert_close(got.double(), product(x, w, scale)[0], rtol=1e-4, atol=1e-4)


def test_refusals_on_the_gpu():
    x, (w, scale) = tokens(2, 256), matrix(6, 256, 7, "cuda")
    for bad in [(x, w.cpu(), scale), (x, w, scale.cpu()), (x.cpu(), w, scale), (x, w, scale[:, :1]), (x[:, :128], w, scale)]:
        with pytest.raises(ValueError, match="weights of 4 bits"):
            ops.linear_int4(*bad)
    with pytest.raises(ValueError, match="no backward"):
        ops.linear_swiglu_int4(x.requires_grad_(True), w, scale)


@pytest.mark.parametrize("n", [1, 50, 300])
def test_streams_and_graphs(n):
    """Calls on two streams and two replayed graphs at once, each with partial sums of its own."""
    w, scale = matrix(12800, 4096, 8, "cuda")
    xs = [tokens(n, 4096, s) for s in range(4)]
    want = [ops.linear_int4(x, w, scale) for x in xs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(4)]
    for x in xs[:2]:
        ops.linear_int4(x, w, scale)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([ops.linear_int4(x, w, scale) for _ in range(3)])
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = []
        for x, s in zip(xs[2:], streams[2:]):
            with torch.cuda.stream(s):
                eager.append([ops.linear_int4(x, w, scale) for _ in range(3)])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(o, want[i]) for o in outs[i]) and all(torch.equal(o, want[2 + i]) for o in eager[i])


def test_long_runs_of_many_tokens():
    """Many units to a CTA, several chunks: stages of every ring are handed on many times."""
    w, scale = matrix(40000, 4096, 9, "cuda")
    for n in (16, 32, 64, 130):
        x = tokens(n, 4096)
        want, first = product(x, w, scale), ops.linear_int4(x, w, scale)
        check(first, want)
        for _ in range(30):
            assert torch.equal(ops.linear_int4(x, w, scale), first)


@pytest.mark.parametrize("n", [3, 40, 250, 700])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_of_any_size(n, gated):
    """Tokens and rows of weights whose sizes lie far apart, scales from fp16's least to its largest, rows of zeros."""
    g = torch.Generator().manual_seed(11)
    x = (tokens(n, 1024).float() * torch.exp2(torch.randint(-40, 20, (n, 1), generator=g).float()).cuda()).bfloat16()
    x[n // 2] = 0
    w, scale = matrix(4000, 1024, 12, "cuda")
    scale *= torch.exp2(torch.randint(-14, 14, (4000, 1), generator=g).float()).cuda().half()
    scale[7], scale[8, 0], scale[9, 1], scale[10, 2] = 0, 65504.0, 2.0 ** -24, 2.0 ** -15
    check(run(x, w, scale, gated), product(x, w, scale, gated, widened=n > ops._int4_tokens(w)))


def test_the_largest_numbers_of_a_prompt():
    """Products that pass fp16's range, and fp32's where only a factor does."""
    w, scale = matrix(512, 256, 13, "cuda")
    for size in (2.0 ** 110, 2.0 ** -120):
        x = (tokens(300, 256).float().clamp(-4, 4) * size).bfloat16()
        y, _ = product(x, w, scale, widened=True)
        got = ops.linear_int4(x, w, scale).double()
        assert torch.isfinite(got).all() and ((got - y).norm() / y.norm()).item() < 2.0 ** -8
    scale[3, 1] = float("inf")
    scale[4, 0] = float("nan")
    got = ops.linear_int4(tokens(300, 256), w, scale)
    assert not got[:, 3:5].isfinite().any() and got[:, :3].isfinite().all() and got[:, 5:].isfinite().all()


@pytest.mark.parametrize("n", [2, 12, 300])
def test_offsets_past_32_bits(n):
    """The last rows of a matrix of more than 2^31 bytes are what they are by themselves."""
    rows, width = 1_100_008, 4096
    w = torch.empty(rows, width // 2, dtype=torch.uint8, device="cuda").random_(0, 256)
    scale = torch.empty(rows, width // 128, dtype=torch.half, device="cuda").normal_(0, 0.01)
    x = tokens(n, width)
    got = ops.linear_int4(x, w, scale)
    for part in (slice(0, 8), slice(rows - 72, rows)):
        check(got[:, part], product(x, w[part], scale[part], widened=n > 192))


@pytest.mark.parametrize("n", [1, 20, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_ways_to_call(n, gated):
    x, (w, scale) = tokens(n, 512), matrix(264, 512, 14, "cuda")
    want = run(x, w, scale, gated)
    with torch.inference_mode():
        assert torch.equal(run(x, w, scale, gated), want)
    with torch.no_grad():
        assert torch.equal(run(x.clone().requires_grad_(True), w, scale, gated), want)
    assert torch.equal(run(x.view(n, 1, 1, 512), w, scale, gated), want.view(n, 1, 1, -1))
    assert torch.equal(run(x[0], w, scale, gated), run(x[:1], w, scale, gated)[0])
    assert run(x.expand(2, n, 512), w, scale, gated).shape == (2, n, 132 if gated else 264)
