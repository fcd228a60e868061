"""The C++ host side (csrc/torch/ops.cpp) of append with rotation, decode over a cache of 8 bits and token log probabilities against the Python operators
behind it: the same kernels, so the same bits, launches, gradients and refusals."""
import pytest
import torch

from test_operators_gpu import _both, _randn, python_operators

pytestmark = pytest.mark.gpu


@pytest.fixture
def sops(cuda_device):
    from llmctl_b200.ops import native, serving
    native.lib()
    assert not isinstance(native.fast, native._NoOps)
    return serving


@pytest.fixture
def ops(sops):
    from llmctl_b200.ops import functional
    return functional


def _taken(name, *args):
    """Whether the C++ side takes the call itself."""
    from llmctl_b200.ops import native
    return getattr(native.fast, name)(*args) is not None


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form", ["plain", "wide", "odd", "transposed", "sliced"])
def test_append(sops, ops, fp8, form):
    T, H, Hk, D = 6, 4, 2, 64
    width = (H + 2 * Hk) * D
    cos, sin = ops.rope_tables(D, 64, device="cuda")

    def state():
        qkv = {"plain": _randn(T, width), "wide": _randn(T, width + 8), "odd": _randn(T, width, shift=1), "transposed": _randn(width, T).t(), "sliced": _randn(T, width)}[form]
        positions, slots = torch.arange(2 * T, device="cuda", dtype=torch.int32)[::2], torch.arange(3, 3 + T, device="cuda")
        if form != "sliced":
            positions = positions.contiguous()
        if fp8:
            (k, ks), (v, vs) = (sops.allocate_fp8_cache(2, 8, Hk, D, "cuda") for _ in range(2))
        else:
            k, v, ks, vs = *(torch.zeros(2, 8, Hk, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)), None, None
        return qkv, cos, sin, positions, k, v, slots, ks, vs

    def run():
        qkv, cos, sin, positions, k, v, slots, ks, vs = state()
        version = qkv._version
        out = sops.rope_kv_append(qkv, cos, sin, positions, k, v, slots, H, D, kv_heads=Hk, k_scale=ks, v_scale=vs)
        assert out is qkv and qkv._version > version
        return [qkv.clone(), k.float(), v.float()] + ([ks, vs] if fp8 else [])
    _both(run)
    qkv, cos, sin, positions, k, v, slots, ks, vs = state()
    assert _taken("rope_kv_append", qkv, cos, sin, positions, k, v, slots, H, Hk, D, ks, vs) == (form in ("plain", "wide"))


@pytest.mark.parametrize("form", ["plain", "packed", "odd", "tables"])
@pytest.mark.parametrize("splits", [None, 1, 5])
@pytest.mark.parametrize("context", [40, 3000])
def test_decode(sops, form, splits, context):
    B, H, Hk, D, size = 3, 4, 2, 128, 16
    pages = (context + size - 1) // size

    def run():
        q = _randn(B, H, D, shift=1 if form == "odd" else 0)
        if form == "packed":
            q = _randn(B, (H + 2 * Hk) * D)[:, :H * D].view(B, H, D)
        k, v = (_randn(B * pages, Hk, size, D, seed=s).to(torch.float8_e4m3fn) for s in (1, 2))
        ks, vs = (_randn(B * pages, Hk, seed=s).float().abs() for s in (3, 4))
        tables = torch.arange(B * pages, device="cuda", dtype=torch.int32).view(B, pages)
        if form == "tables":
            tables = torch.stack([tables, tables], -1)[..., 0]
        lens = torch.tensor([context, 7, context // 2], device="cuda", dtype=torch.int32)
        return sops.paged_attention_decode_fp8(q, k, v, ks, vs, tables, lens, context, num_splits=splits)
    _both(run)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("form", ["plain", "sliced", "odd", "three", "one", "columns"])
@pytest.mark.parametrize("grad", [False, True])
def test_logprobs(ops, dtype, top, form, grad):
    V = 777

    def run():
        x = _randn(6, V, shift=1 if form == "odd" else 0).to(dtype) * 3
        x = {"sliced": lambda: torch.cat([x, x], -1)[:, 5:5 + V], "three": lambda: x.view(2, 3, V), "one": lambda: x[0], "columns": lambda: x.t().contiguous().t()}.get(form, lambda: x)()
        x = x.detach().requires_grad_(grad)
        tokens = torch.randint(0, V, x.shape[:-1], device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
        out = ops.token_logprobs(x, tokens, top)
        values = [t.detach() for t in out if t is not None]
        assert len(values) == (4 if top else 2) and all(t.requires_grad == (grad and t.is_floating_point()) for t in out if t is not None)
        if grad:
            outs = [out.logprobs, out.entropy] + ([out.top_logprobs] if top else [])
            grads = [_randn(t.numel(), seed=9 + i).float().view(t.shape) for i, t in enumerate(outs)]
            values += [torch.autograd.grad(outs, x, grads, retain_graph=True)[0]]
            values += [torch.autograd.grad(o, x, g, retain_graph=True)[0] for o, g in zip(outs, grads)]
        return tuple(values)
    _both(run)


def test_gradients_of_gradients_are_refused(ops):
    x, tokens = _randn(4, 100).requires_grad_(True), torch.zeros(4, device="cuda", dtype=torch.int64)

    def run():
        out = ops.token_logprobs(x, tokens)
        dx, = torch.autograd.grad(out.logprobs.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.float().square().sum().backward()
        return dx.detach()
    _both(run)


def test_logits_that_change_before_the_backward_are_noticed(ops):
    x, tokens = (_randn(4, 100) * 1).requires_grad_(True), torch.zeros(4, device="cuda", dtype=torch.int64)
    for _ in range(2):
        y = x * 1
        out = ops.token_logprobs(y, tokens)
        y.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.entropy.sum().backward()
        with python_operators():
            out = ops.token_logprobs(x * 1, tokens)


def test_refusals_are_the_python_operators(sops, ops):
    """What the checks refuse raises ValueError whether the C++ side is there or not."""
    H, D = 2, 64
    (k, ks), (v, vs) = (sops.allocate_fp8_cache(2, 8, H, D, "cuda") for _ in range(2))
    cos, sin = ops.rope_tables(D, 64, device="cuda")
    row, p, s = _randn(1, 3 * H * D), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    bad = [lambda: sops.rope_kv_append(row, cos, sin, p.long(), k, v, s, H, D, k_scale=ks, v_scale=vs), lambda: sops.rope_kv_append(row, cos, sin, p, k, v, s, H, D),
           lambda: sops.rope_kv_append(row, cos, sin, p, k, v, s, 3, D, kv_heads=2, k_scale=ks, v_scale=vs),
           lambda: sops.rope_kv_append(row.clone().requires_grad_(True), cos, sin, p, k, v, s, H, D, k_scale=ks, v_scale=vs),
           lambda: sops.paged_attention_decode_fp8(_randn(1, H, D), k, v, ks, vs, torch.zeros(1, 2, dtype=torch.int64, device="cuda"), p, 8),
           lambda: sops.paged_attention_decode_fp8(_randn(1, H, D), k, v, ks, vs, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), p, 8, num_splits=0),
           lambda: ops.token_logprobs(_randn(2, 50), torch.zeros(3, dtype=torch.int64, device="cuda")), lambda: ops.token_logprobs(_randn(2, 50), torch.zeros(2, dtype=torch.int64, device="cuda"), 51),
           lambda: ops.token_logprobs(_randn(2, 50), torch.zeros(2, dtype=torch.int32, device="cuda"))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
        with python_operators(), pytest.raises(ValueError):
            call()


def test_calls_on_threads_and_streams(sops, ops):
    """Four threads on streams of their own, each with its own cache, against one."""
    import threading
    H, D, size = 4, 64, 16
    cos, sin = ops.rope_tables(D, 2048, device="cuda")

    def work(i):
        (k, ks), (v, vs) = (sops.allocate_fp8_cache(80, size, H, D, "cuda") for _ in range(2))
        n = 1000 + i
        at = torch.arange(n, device="cuda")
        qkv = _randn(n, 3 * H * D, seed=i)
        sops.rope_kv_append(qkv, cos, sin, at.int(), k, v, at, H, D, k_scale=ks, v_scale=vs)
        o = sops.paged_attention_decode_fp8(qkv[-1:, :H * D].view(1, H, D), k, v, ks, vs, torch.arange(80, device="cuda", dtype=torch.int32).view(1, 80),
                                            torch.tensor([n], device="cuda", dtype=torch.int32), n)
        lp = ops.token_logprobs(qkv, at % 7, 3)
        return o, lp.logprobs, lp.top_ids
    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    got = [None] * 4

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = work(i)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
