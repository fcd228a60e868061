"""Timed operators of a decoding step's two readings, its weights and its contexts, through the framework's public entry points or in plain form.

* ``linear``: products with weights of 4 bits as the ``int4`` quantiser writes them (two to a byte, a scale for each 128 input channels);
* ``gated``: the same of a gated MLP's first half, silu(x Wg^T) * (x Wu^T);
* ``shared``: one query token per sequence against a paged cache in which groups of sequences begin with the same blocks (completions of one
  prompt), which are read once for a group.

``listed()`` names twelve cases, ``draw(rng)`` makes one more of the same ranges, ``prepare`` builds what a program has in hand, ``run`` is one
pass (``own``: by the framework's kernels, else in elementary operations), ``work`` what a pass cannot do without, ``exact`` the same
outputs in 64 bits.  Widths and heads are those of the model presets (``llmctl_b200.models.config.PRESETS``) or generic.
"""
import math

import torch

own = False

GROUP = 128                     # input channels to a scale
# (hidden, ffn) of the presets gpt-125m, gpt-1b, gpt-7b and gpt-13b
_WIDTHS = [(768, 2048), (2048, 5632), (4096, 11008), (5120, 13824)]
# (query heads, heads of keys and values, head size): the presets gpt-125m, gpt-7b and gpt-13b, and two with shared keys and values
_SMALL, _LARGE, _XL, _GROUPED, _GROUPED_SMALL = (12, 12, 64), (32, 32, 128), (40, 40, 128), (32, 8, 128), (24, 4, 64)
_MOST_FLOPS = 2 * 4096 * 4096 * 2 * 11008
_MOST_CACHE = 50000 * 32 * 128 + 16 * 2000 * 32 * 128


def listed():
    return [
        # one decoding conversation of the 7B preset, attention's output projection: latency
        {"name": "linear_one", "kind": "linear", "tokens": 1, "width": 4096, "rows": 4096},
        # a decoding step of a batch of 16, the MLP's second half
        {"name": "linear_step", "kind": "linear", "tokens": 16, "width": 11008, "rows": 4096},
        # more sequences than a tile of tokens, the 13B preset's packed q | k | v
        {"name": "linear_batch", "kind": "linear", "tokens": 61, "width": 5120, "rows": 15360},
        # a prompt of any length, packed q | k | v of the 7B preset
        {"name": "linear_prompt", "kind": "linear", "tokens": 1777, "width": 4096, "rows": 12288},
        # the gated half of an MLP: one conversation; a full batch of the 1B preset; several prompts at once
        {"name": "gated_one", "kind": "gated", "tokens": 1, "width": 4096, "rows": 11008},
        {"name": "gated_step", "kind": "gated", "tokens": 32, "width": 2048, "rows": 5632},
        {"name": "gated_prompt", "kind": "gated", "tokens": 4096, "width": 4096, "rows": 11008},
        # four completions of one short prompt, the smallest preset: latency
        {"name": "shared_one", "kind": "shared", "batch": 4, "groups": 1, "prefix": 288, "own": 20, "page": 16, "heads": 12, "kv_heads": 12, "dim": 64},
        # 32 completions of one long prompt
        {"name": "shared_batch", "kind": "shared", "batch": 32, "groups": 1, "prefix": 4096, "own": 256, "page": 16, "heads": 32, "kv_heads": 32, "dim": 128},
        # eight prompts of unlike numbers of completions, keys and values shared by heads, larger pages
        {"name": "shared_groups", "kind": "shared", "batch": 67, "groups": 8, "prefix": 8000, "own": 1001, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128},
        # completions that have grown longer than their prompt
        {"name": "shared_short", "kind": "shared", "batch": 48, "groups": 3, "prefix": 400, "own": 777, "page": 16, "heads": 40, "kv_heads": 40, "dim": 128},
        # a very long document that 16 sequences ask about
        {"name": "shared_long", "kind": "shared", "batch": 16, "groups": 1, "prefix": 50000, "own": 2000, "page": 16, "heads": 32, "kv_heads": 32, "dim": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "gated", "gated", "shared", "shared", "shared"])
    if kind == "shared":
        heads, kv_heads, dim = rng.choice([_SMALL, _LARGE, _LARGE, _XL, _GROUPED, _GROUPED_SMALL])
        page = rng.choice([8, 16, 16, 16, 32, 64])
        batch = _log(rng, 2, 128)
        groups = min(batch, _log(rng, 1, 16))
        room = _MOST_CACHE // (kv_heads * dim)                   # tokens in the cache
        after = min(_log(rng, 1, 2000), max(1, room // (2 * batch)))
        prefix = min(_log(rng, page, 50000), max(page, room // (2 * groups)))
        return {"kind": kind, "batch": batch, "groups": groups, "prefix": prefix, "own": after, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim}
    hidden, ffn = rng.choice(_WIDTHS)
    if kind == "gated":
        width, rows = hidden, ffn
    else:
        width, rows = rng.choice([(hidden, 3 * hidden), (hidden, hidden), (ffn, hidden), (hidden, 32000), (GROUP * _log(rng, 1, 100), _log(rng, 100, 20000))])
    tokens = _log(rng, 1, 64) if rng.random() < 0.6 else _log(rng, 64, 4096)
    most = _MOST_FLOPS // (2 * width * rows * (2 if kind == "gated" else 1))
    return {"kind": kind, "tokens": max(1, min(tokens, most)), "width": width, "rows": rows}


# ---------------------------------------------------------------------------------------------------------------------
# inputs: made from the seed alone
# ---------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)


def _weight4(g, rows, width):
    """A matrix rounded to 4 bits as the ``int4`` quantiser does it: codes of value + 8, the even column in the low half of a byte; scales
    fp16, the largest of a group over 7."""
    x = _randn(g, rows, width // GROUP, GROUP, std=0.02, dtype=torch.float32)
    x *= torch.exp2(torch.randint(-2, 3, (rows, 1, 1), device="cuda", generator=g).float())     # output channels of unlike size
    scale = x.abs().amax(2, keepdim=True).clamp_min(1e-8) / 7.0
    q = ((x / scale).round_().clamp_(-7, 7) + 8).to(torch.uint8).view(rows, width)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scale.squeeze(2).to(torch.float16)


def _lengths(n, longest):
    """Lengths of a batch: the longest first, the others spread down to a quarter of it."""
    return [max(1, longest - (3 * longest * i) // (4 * max(n, 2))) for i in range(n)]


def _layout(case):
    """Of a ``shared`` case, for each group the rows' first and last + 1 and how many tokens they share, for each row how many of its own."""
    B, G, page = case["batch"], case["groups"], case["page"]
    sizes = [B // G + (i < B % G) for i in range(G)]
    for i in range(0, G - 1, 2):                # of two neighbours one has three times the completions
        moved = sizes[i + 1] // 2
        sizes[i], sizes[i + 1] = sizes[i] + moved, sizes[i + 1] - moved
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    shared = [max(page, n // page * page) for n in _lengths(G, case["prefix"])]     # whole pages
    return starts, shared, _lengths(B, case["own"])


def _shared_inputs(case, g):
    starts, shared, after = _layout(case)
    B, page = case["batch"], case["page"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    of = [i for i in range(len(shared)) for _ in range(starts[i], starts[i + 1])]
    first = [n // page for n in shared]
    behind = [(n + page - 1) // page for n in after]
    pages = sum(first) + sum(behind)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()     # pages scattered over the pool
    table, at, heads_of = torch.zeros(B, max(first[of[b]] + behind[b] for b in range(B)), dtype=torch.int32), 0, []
    for n in first:
        heads_of.append(perm[at:at + n])
        at += n
    for b in range(B):
        n = first[of[b]]
        table[b, :n] = heads_of[of[b]]
        table[b, n:n + behind[b]] = perm[at:at + behind[b]]
        at += behind[b]
    k, v = _randn(g, pages, page, Hk, D), _randn(g, pages, page, Hk, D)
    k[..., 3] *= 4                              # some channels of keys are larger than the rest
    qkv = _randn(g, B, (H + 2 * Hk) * D)        # queries as they stand in the packed projection
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"q": qkv[:, :H * D].view(B, H, D), "k": k, "v": v, "tables": table.cuda(), "lens": ints([shared[of[b]] + after[b] for b in range(B)]),
            "group_starts": ints(starts), "shared_lens": ints(shared)}


def _inputs(case, seed):
    g = _generator(seed)
    if case["kind"] == "shared":
        return _shared_inputs(case, g)
    x = _randn(g, case["tokens"], case["width"])
    x[:, 5] *= 8                                # a channel of outliers
    w, scale = _weight4(g, case["rows"] * (2 if case["kind"] == "gated" else 1), case["width"])
    return {"x": x, "w": w, "scale": scale}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return {"linear": _linear, "gated": _gated, "shared": _shared}[s["case"]["kind"]](s)


def _product(s):
    """x W^T in 32 bits."""
    w = s["w"]
    codes = torch.stack([w & 15, w >> 4], 2).view(w.shape[0], -1, GROUP).float() - 8.0
    return s["x"].float() @ (codes * s["scale"].float()[..., None]).view(w.shape[0], -1).t()


def _linear(s):
    if own:
        from llmctl_b200.ops import functional
        return functional.linear_int4(s["x"], s["w"], s["scale"])
    return _product(s).to(s["x"].dtype)


def _gated(s):
    if own:
        from llmctl_b200.ops import functional
        return functional.linear_swiglu_int4(s["x"], s["w"], s["scale"])
    gate, up = _product(s).chunk(2, -1)
    return (gate / (1 + torch.exp(-gate)) * up).to(s["x"].dtype)


def _shared(s):
    if own:
        from llmctl_b200.ops import serving
        return serving.paged_attention_decode_shared(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["group_starts"], s["shared_lens"])
    c = s["case"]
    B, G, page = c["batch"], c["groups"], c["page"]
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    starts, shared, after = _layout(c)
    M, S, A = max(b - a for a, b in zip(starts, starts[1:])), max(shared), max(after)
    dev, table = s["q"].device, s["tables"].long()
    row = torch.arange(B, device=dev)
    group = torch.searchsorted(s["group_starts"][1:], row, right=True)
    member = row - s["group_starts"][group]
    q = s["q"].float().view(B, Hk, H // Hk, D) / math.sqrt(D)
    # the shared tokens once for each group, its sequences as further rows of a product
    blocks = table[s["group_starts"][:-1].long(), :S // page]
    ks, vs = (x[blocks].view(G, S, Hk, D).permute(0, 2, 1, 3).float() for x in (s["k"], s["v"]))
    padded = torch.zeros(G, M, Hk, H // Hk, D, device=dev)
    padded[group, member] = q
    scores = padded.transpose(1, 2).reshape(G, Hk, -1, D) @ ks.transpose(2, 3)
    scores = scores.view(G, Hk, M, H // Hk, S).transpose(1, 2)[group, member]
    seen = torch.arange(S, device=dev) < s["shared_lens"][group][:, None]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    # each sequence's own
    at = s["shared_lens"][group][:, None] + torch.arange(A, device=dev)
    block = table.gather(1, (at // page).clamp(max=table.shape[1] - 1))
    ko, vo = (x[block, at % page].permute(0, 2, 1, 3).float() for x in (s["k"], s["v"]))
    mine = (q @ ko.transpose(2, 3)).masked_fill(~(at < s["lens"][:, None])[:, None, None], float("-inf"))
    p = torch.cat([scores, mine], -1)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    weights = torch.zeros(G, M, Hk, H // Hk, S, device=dev)
    weights[group, member] = p[..., :S]
    o = weights.transpose(1, 2).reshape(G, Hk, -1, S) @ vs
    o = o.view(G, Hk, M, H // Hk, D).transpose(1, 2)[group, member] + p[..., S:] @ vo
    return (o / total).reshape(B, H, D).to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "shared":
        starts, shared, after = _layout(case)
        B, H, Hk, D, page = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "page"))
        once = sum(shared) + sum(after)
        seen = sum((b - a) * n for a, b, n in zip(starts, starts[1:], shared)) + sum(after)
        return {"bytes": 4 * once * Hk * D + 4 * (once // page) + 4 * B * H * D, "flops": 4 * seen * H * D}
    T, K, N = case["tokens"], case["width"], case["rows"]
    matrix = N * (2 if case["kind"] == "gated" else 1)
    return {"bytes": matrix * K // 2 + matrix * (K // GROUP) * 2 + 2 * T * K + 2 * T * N, "flops": 2 * T * matrix * K}


# ---------------------------------------------------------------------------------------------------------------------
# the same outputs in 64 bits, written apart from the plain form
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(case, s)
    x, parts = s["x"].double(), []
    for i in range(0, s["w"].shape[0], 4096):   # a block of weight rows at a time
        w = s["w"][i:i + 4096]
        full = torch.empty(w.shape[0], case["width"], dtype=torch.float64, device=w.device)
        full[:, 0::2] = torch.bitwise_and(w, 0x0F).double()
        full[:, 1::2] = torch.div(w, 16, rounding_mode="floor").double()
        full = (full - 8) * torch.repeat_interleave(s["scale"][i:i + 4096].double(), GROUP, dim=1)
        parts.append(torch.einsum("tk,nk->tn", x, full))
    y = torch.cat(parts, 1)
    if case["kind"] == "linear":
        return y
    return torch.nn.functional.silu(y[:, :case["rows"]]) * y[:, case["rows"]:]


def _exact_shared(case, s):
    H, Hk, D, page = (case[n] for n in ("heads", "kv_heads", "dim", "page"))
    starts, shared, after = _layout(case)
    out = torch.zeros(case["batch"], H, D, dtype=torch.float64, device="cuda")
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        for i in range(a, b):
            n = shared[g] + after[i]
            pages = s["tables"][i, :(n + page - 1) // page].long()
            q = s["q"][i].double().view(Hk, H // Hk, D)
            for h in range(0, Hk, 8):           # eight heads of the cache at a time
                k, v = (x[pages, :, h:h + 8].reshape(-1, min(8, Hk - h), D)[:n].double() for x in (s["k"], s["v"]))
                p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[h:h + 8], k) / math.sqrt(D), -1)
                out[i, h * (H // Hk):(h + 8) * (H // Hk)] = torch.einsum("hgn,nhd->hgd", p, v).reshape(-1, D)
    return out
