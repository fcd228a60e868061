"""Timed operators of serving and of training on log probabilities, through the framework's public entry points or in plain form.

Three operators that one decoding step uses one after the other:

* ``append``: the packed q | k | v rows of new tokens are rotated to their positions and their keys and values written to a paged cache,
  of 16 bits or of 8 bits (e4m3) with a scale for each page and head;
* ``attend``: one query token per sequence against such a cache of 8 bits;
* ``logprobs``: log probabilities of given tokens, the entropy and the most probable alternatives from rows of logits; with gradients where a
  model is trained on them.

``listed()`` names twelve cases, ``draw(rng)`` makes one more of the same ranges, ``prepare`` builds what a program has in hand, ``run`` is one
pass (``own``: by the framework's kernels, else in elementary operations), ``work`` what a pass cannot do without, ``exact`` the same
outputs in 64 bits.  Heads, widths and vocabularies are those of the model presets (``llmctl_b200.models.config.PRESETS``) or generic.
"""
import math

import torch

own = False

# (query heads, heads of keys and values, head size): the presets gpt-125m, gpt-7b and gpt-13b, and two with shared keys and values
_SMALL, _LARGE, _XL, _GROUPED, _GROUPED_SMALL = (12, 12, 64), (32, 32, 128), (40, 40, 128), (32, 8, 128), (24, 4, 64)
_POSITIONS = 4096               # rows of the rotation tables
_E4M3_MAX = 448.0


def listed():
    return [
        # one decoding conversation of the smallest preset: latency
        {"name": "append_one", "kind": "append", "bits": 8, "tokens": 1, "prompt": False, "context": 300, "page": 16, "heads": 12, "kv_heads": 12, "dim": 64},
        # a decoding step of a full batch of the 7B preset
        {"name": "append_decode", "kind": "append", "bits": 8, "tokens": 64, "prompt": False, "context": 4096, "page": 16, "heads": 32, "kv_heads": 32, "dim": 128},
        # a prompt of any length into a cache of 16 bits
        {"name": "append_prompt", "kind": "append", "bits": 16, "tokens": 1777, "prompt": True, "context": 1777, "page": 16, "heads": 32, "kv_heads": 32, "dim": 128},
        # two long prompts of the 13B preset into a cache of 8 bits
        {"name": "append_prompt_long", "kind": "append", "bits": 8, "tokens": 8000, "prompt": True, "context": 4000, "page": 16, "heads": 40, "kv_heads": 40, "dim": 128},
        # one short conversation; a full batch; a full batch with shared keys and values in larger pages; a few very long contexts
        {"name": "attend_one", "kind": "attend", "batch": 1, "context": 300, "page": 16, "heads": 12, "kv_heads": 12, "dim": 64},
        {"name": "attend_batch", "kind": "attend", "batch": 16, "context": 4096, "page": 16, "heads": 32, "kv_heads": 32, "dim": 128},
        {"name": "attend_grouped", "kind": "attend", "batch": 64, "context": 4096, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128},
        {"name": "attend_long", "kind": "attend", "batch": 4, "context": 50001, "page": 16, "heads": 32, "kv_heads": 32, "dim": 128},
        # the sampled token of one conversation with twenty alternatives; of a full batch with five
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 32000, "top": 20, "bits": 16, "grad": False},
        {"name": "logprobs_step", "kind": "logprobs", "rows": 64, "vocab": 32000, "top": 5, "bits": 16, "grad": False},
        # evaluation of a prompt over a vocabulary of odd size, logits in 32 bits: likelihood and best guess
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2000, "vocab": 50257, "top": 1, "bits": 32, "grad": False},
        # training on log probabilities with an entropy bonus: 8 sequences of 512 tokens, forward and backward
        {"name": "logprobs_train", "kind": "logprobs", "rows": 4096, "vocab": 32000, "top": 0, "bits": 16, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    if kind == "logprobs":
        grad = rng.random() < 0.5
        rows, vocab = _log(rng, 1, 4096), _log(rng, 500, 130000)
        rows = max(1, min(rows, 4096 * 32000 // vocab))
        return {"kind": kind, "rows": rows, "vocab": vocab, "top": 0 if grad and rng.random() < 0.5 else rng.choice([0, 1, 3, 5, 20]), "bits": rng.choice([16, 16, 32]), "grad": grad}
    heads, kv_heads, dim = rng.choice([_SMALL, _LARGE, _LARGE, _XL, _GROUPED, _GROUPED_SMALL])
    page = rng.choice([8, 16, 16, 16, 32, 64])
    if kind == "attend":
        batch, context = _log(rng, 1, 128), _log(rng, 1, 60000)
        context = max(1, min(context, 4 * 50001 * 32 * 128 // (batch * kv_heads * dim)))
        return {"kind": kind, "batch": batch, "context": context, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if rng.random() < 0.5:
        return {"kind": kind, "bits": rng.choice([8, 8, 16]), "tokens": _log(rng, 1, 128), "prompt": False, "context": _log(rng, 20, 4096), "page": page, "heads": heads,
                "kv_heads": kv_heads, "dim": dim}
    tokens = _log(rng, 2, 8000)
    return {"kind": kind, "bits": rng.choice([8, 8, 16]), "tokens": tokens, "prompt": True, "context": min(tokens, _log(rng, 100, 4096)), "page": page, "heads": heads,
            "kv_heads": kv_heads, "dim": dim}


# ---------------------------------------------------------------------------------------------------------------------
# inputs: made from the seed alone
# ---------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)


def _lengths(n, longest):
    """Context lengths of a batch: the longest first, the others spread down to a quarter of it."""
    return [max(1, longest - (3 * longest * i) // (4 * max(n, 2))) for i in range(n)]


def _tables(g, lens, page):
    """Block tables [sequences, most pages] over pages scattered over the pool, and how many pages there are."""
    pages = [(n + page - 1) // page for n in lens]
    perm = torch.randperm(sum(pages), generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.zeros(len(lens), max(pages), dtype=torch.int32), 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[at:at + n]
        at += n
    return table.cuda(), sum(pages)


def _cache8(g, pages, heads, page, dim):
    """Keys or values as they stand in a cache of 8 bits: pages of different magnitude, some channels larger than the rest."""
    x = _randn(g, pages, heads, page, dim)
    x *= torch.exp2(torch.randint(0, 3, (pages, heads, 1, 1), device="cuda", generator=g)).to(x.dtype)
    x[..., 3] *= 4
    most = x.abs().amax((2, 3)).float()
    scale = torch.exp2(torch.ceil(torch.log2(most / _E4M3_MAX)))
    return x.div_(scale.to(x.dtype)[..., None, None]).to(torch.float8_e4m3fn), scale


def _rotation(dim):
    """cos and sin [positions, dim / 2] of the usual frequencies, angles in 64 bits."""
    angle = torch.outer(torch.arange(_POSITIONS, device="cuda", dtype=torch.float64), 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
    return angle.cos().float(), angle.sin().float()


def _inputs(case, seed):
    g, k = _generator(seed), case["kind"]
    if k == "logprobs":
        R, V = case["rows"], case["vocab"]
        wide = (V + 127) // 128 * 128           # rows of the output head's padded vocabulary
        logits = _randn(g, R, wide, std=2.5, dtype=torch.float32)
        tokens = torch.randint(0, V, (R,), device="cuda", generator=g)
        logits[torch.arange(R, device="cuda"), tokens] += 6.0       # the tokens that follow are likely ones
        logits = logits.to(torch.bfloat16 if case["bits"] == 16 else torch.float32)[:, :V]
        s = {"logits": logits, "tokens": tokens}
        if case["grad"]:
            s["d_logprobs"], s["d_entropy"] = _randn(g, R, dtype=torch.float32), _randn(g, R, std=0.01, dtype=torch.float32)
            if case["top"]:
                s["d_top"] = _randn(g, R, case["top"], std=0.1, dtype=torch.float32)
        return s
    H, Hk, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if k == "attend":
        lens = _lengths(case["batch"], case["context"])
        tables, pages = _tables(g, lens, page)
        kc, ks = _cache8(g, pages, Hk, page, D)
        vc, vs = _cache8(g, pages, Hk, page, D)
        qkv = _randn(g, len(lens), (H + 2 * Hk) * D, std=0.5)       # queries as they stand in the packed projection
        return {"q": qkv[:, :H * D].view(len(lens), H, D), "k": kc, "v": vc, "ks": ks, "vs": vs, "tables": tables,
                "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "most": max(lens)}
    T = case["tokens"]
    if case["prompt"]:                          # whole prompts one behind the other
        lens = [case["context"]] * (T // case["context"]) + ([T % case["context"]] if T % case["context"] else [])
        tables, pages = _tables(g, lens, page)
        of = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        positions = torch.cat([torch.arange(n) for n in lens])
    else:
        lens = _lengths(T, case["context"])
        tables, pages = _tables(g, lens, page)
        of, positions = torch.arange(T), torch.tensor(lens) - 1
    of, positions = of.cuda(), positions.cuda()
    slots = tables[of, positions // page].long() * page + positions % page
    s = {"qkv": _randn(g, T, (H + 2 * Hk) * D), "positions": positions.to(torch.int32), "slots": slots}
    s["cos"], s["sin"] = _rotation(D)
    if case["bits"] == 16:
        s["k"], s["v"] = (torch.zeros(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    elif case["prompt"]:                        # pages that nothing has been written to
        s["k"], s["v"] = (torch.zeros(pages, Hk, page, D, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
        s["ks"], s["vs"] = (torch.zeros(pages, Hk, device="cuda") for _ in range(2))
    else:
        (s["k"], s["ks"]), (s["v"], s["vs"]) = (_cache8(g, pages, Hk, page, D) for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "logprobs" and case["grad"]:
        s["logits"].requires_grad_(True)
    return {"case": case, **s}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return {"append": _append, "attend": _attend, "logprobs": _logprobs}[s["case"]["kind"]](s)


def _append(s):
    c = s["case"]
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    if own:
        from llmctl_b200.ops import serving
        serving.rope_kv_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["k"], s["v"], s["slots"], H, D, kv_heads=Hk, k_scale=s.get("ks"), v_scale=s.get("vs"))
    else:
        x = s["qkv"].view(-1, H + 2 * Hk, D)
        at = s["positions"].long()
        # a rotated key may stand next to a border between two numbers of 8 bits: products in 64 bits, one rounding to 32
        cos, sin = s["cos"][at][:, None].double(), s["sin"][at][:, None].double()
        a, b = x[:, :H + Hk, :D // 2].double(), x[:, :H + Hk, D // 2:].double()
        rotated = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float()
        x[:, :H + Hk] = rotated.to(x.dtype)
        if c["bits"] == 16:
            s["k"].view(-1, Hk, D)[s["slots"]] = x[:, H:H + Hk]
            s["v"].view(-1, Hk, D)[s["slots"]] = x[:, H + Hk:]
        else:
            _quantise(rotated[:, H:], s["k"], s["ks"], s["slots"])
            _quantise(x[:, H + Hk:].float(), s["v"], s["vs"], s["slots"])
    return {n: s[n] for n in ("qkv", "k", "v", "ks", "vs") if n in s}


def _quantise(x, cache, scale, slots):
    """Rows of 32 bits into their pages.  A page's scale is the smallest power of two under which its largest number fits; rows that are there
    already keep what they stand for when it grows, unless the page is begun anew by its first row."""
    size = cache.shape[2]
    page, row = slots // size, slots % size
    most = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
    begun = torch.zeros(scale.shape[0], dtype=torch.bool, device=x.device)
    begun[page[row == 0]] = True
    mantissa, exponent = torch.frexp(most)
    need = torch.where(most > 0, torch.ldexp(torch.ones_like(most), (exponent - 9 + (mantissa > _E4M3_MAX / 512).to(exponent.dtype)).clamp(min=-126)), 0.0)
    new = torch.where(begun[:, None], need, torch.maximum(scale, need))
    factor = torch.where(begun[:, None] | (new == scale) | (new == 0), 1.0, scale / new)
    cache[page] = (cache[page].float() * factor[page][..., None, None]).to(cache.dtype)
    cache.permute(0, 2, 1, 3)[page, row] = (x / torch.where(new > 0, new, 1.0)[page][..., None]).to(cache.dtype)
    scale[page] = new[page]


def _attend(s):
    c = s["case"]
    H, Hk, D, size = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if own:
        from llmctl_b200.ops import serving
        return serving.paged_attention_decode_fp8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"], s["most"])
    B, G = c["batch"], H // Hk
    q = s["q"].float().view(B, Hk, G, D)

    def rows(cache, scale):                     # [sequences, heads, tokens, dim] in 32 bits
        x = cache[s["tables"].long()].float() * scale[s["tables"].long()][..., None, None]
        return x.transpose(1, 2).reshape(B, Hk, -1, D)

    scores = torch.matmul(q, rows(s["k"], s["ks"]).transpose(2, 3)) / math.sqrt(D)
    seen = torch.arange(scores.shape[-1], device=q.device) < s["lens"][:, None, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.matmul(p, rows(s["v"], s["vs"])) / p.sum(-1, keepdim=True)
    return o.reshape(B, H, D).to(s["q"].dtype)


def _logprobs(s):
    c = s["case"]
    logits, tokens, top = s["logits"], s["tokens"], c["top"]
    if own:
        from llmctl_b200.ops import functional
        out = functional.token_logprobs(logits, tokens, top=top)
        if not c["grad"]:
            return {n: v for n, v in out._asdict().items() if v is not None}
        # the logits are a leaf here; a program's come from its output head
        outs, grads = [out.logprobs, out.entropy], [s["d_logprobs"], s["d_entropy"]]
        if top:
            outs, grads = outs + [out.top_logprobs], grads + [s["d_top"]]
        dx, = torch.autograd.grad(outs, logits, grads)
        return {**{n: v.detach() for n, v in out._asdict().items() if v is not None}, "d_logits": dx}
    x = logits.detach().float()
    lp = x - x.amax(-1, keepdim=True)
    lp = lp - lp.exp().sum(-1, keepdim=True).log()
    p = lp.exp()
    entropy = -(p * lp).sum(-1)
    out = {"logprobs": lp.gather(1, tokens[:, None])[:, 0], "entropy": entropy}
    if top:
        # of equal logits the one with the lowest index: a stable order of the largest
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
        out |= {"top_ids": order, "top_logprobs": lp.gather(1, order)}
    if c["grad"]:
        g, e = s["d_logprobs"][:, None], s["d_entropy"][:, None]
        total = g + s["d_top"].sum(-1, keepdim=True) if top else g
        dx = -p * (total + e * (lp + entropy[:, None]))
        dx.scatter_add_(1, tokens[:, None], g)
        if top:
            dx.scatter_add_(1, out["top_ids"], s["d_top"])
        out["d_logits"] = dx.to(logits.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * case["bits"] // 8 * (2 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top"]), "flops": n * (9 if case["grad"] else 5)}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attend":
        lens = _lengths(case["batch"], case["context"])
        pages = sum((n + case["page"] - 1) // case["page"] for n in lens)
        return {"bytes": 2 * sum(lens) * Hk * D + pages * (8 * Hk + 4) + 4 * len(lens) * H * D, "flops": 4 * sum(lens) * H * D}
    T = case["tokens"]
    rows = T * D * (2 * (H + 2 * Hk) + 2 * (H + Hk) + 2 * Hk * case["bits"] // 8)
    return {"bytes": rows + min(T, case["context"]) * 4 * D + 12 * T, "flops": 3 * T * (H + Hk) * D + (4 * T * Hk * D if case["bits"] == 8 else 0)}


# ---------------------------------------------------------------------------------------------------------------------
# the same outputs in 64 bits, written apart from the plain form
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(case, s)
    return _exact_attend(case, s) if case["kind"] == "attend" else _exact_append(case, s)


def _exact_logprobs(case, s):
    out = {"logprobs": [], "entropy": [], "top_logprobs": [], "d_logits": []}
    for i in range(0, case["rows"], 256):       # a block of rows at a time
        x = s["logits"][i:i + 256].detach().double().requires_grad_(case["grad"])
        lp = torch.log_softmax(x, -1)
        p = torch.softmax(x, -1)
        chosen, entropy = lp[torch.arange(x.shape[0]), s["tokens"][i:i + 256]], -torch.special.xlogy(p, p).sum(-1)
        outs = [chosen, entropy]
        out["logprobs"].append(chosen.detach())
        out["entropy"].append(entropy.detach())
        if case["top"]:
            best = torch.topk(lp, case["top"]).values
            out["top_logprobs"].append(best.detach())
            outs.append(best)
        if case["grad"]:
            # among equal logits of 16 bits either may be the one that topk names: the sum of their gradients is what is defined
            given = [s["d_logprobs"][i:i + 256].double(), s["d_entropy"][i:i + 256].double()] + ([s["d_top"][i:i + 256].double()] if case["top"] else [])
            out["d_logits"].append(torch.autograd.grad(outs, x, given)[0])
    got = {n: torch.cat(v) for n, v in out.items() if v}
    if case["top"]:
        got["top_ids"] = None
        if case["grad"] and case["bits"] == 16:
            got["d_logits"] = None
    return got


def _exact_attend(case, s):
    H, Hk, D, size = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(case["batch"], H, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case["batch"], case["context"])):
        pages = s["tables"][b, :(n + size - 1) // size].long()
        for h in range(Hk):
            k = (s["k"][pages, h].double() * s["ks"][pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s["v"][pages, h].double() * s["vs"][pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            for i in range(h * H // Hk, (h + 1) * H // Hk):
                out[b, i] = torch.softmax(k @ s["q"][b, i].double() / math.sqrt(D), 0) @ v
    return out


def _exact_append(case, s):
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    T, size = case["tokens"], case["page"]
    x = s["qkv"].double().view(T, H + 2 * Hk, D)
    at = s["positions"].long()
    z = torch.complex(x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:]) * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, H + Hk:]], 1)
    got = {"qkv": x.reshape(T, -1)}
    if case["bits"] == 16:
        for name, part in (("k", x[:, H:H + Hk]), ("v", x[:, H + Hk:])):
            got[name] = s[name].double()
            got[name].view(-1, Hk, D)[s["slots"]] = part
        return got
    # the numbers that the codes of 8 bits round: what stands in a page over its new scale
    for name, part in (("k", x[:, H:H + Hk]), ("v", x[:, H + Hk:])):
        page, row = s["slots"] // size, s["slots"] % size
        scale, codes = s[name + "s"].double(), s[name].double()
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=x.device)
        touched[page] = True
        begun = torch.zeros_like(touched)
        begun[page[row == 0]] = True
        most = torch.full_like(scale, 0.0).scatter_reduce_(0, page[:, None].expand(-1, Hk), part.abs().amax(-1), "amax")
        need = torch.where(most > 0, torch.pow(2.0, torch.ceil(torch.log2(most / _E4M3_MAX))), 0.0)
        new = torch.where(begun[:, None], need, torch.maximum(scale, need))
        new = torch.where(touched[:, None], new, scale)
        keep = ~begun[:, None] & (new > 0)
        codes = torch.where(keep[..., None, None], codes * (scale / torch.where(new > 0, new, 1.0))[..., None, None], codes)
        codes.transpose(1, 2)[page, row] = part / new[page][..., None]
        got[name], got[name + "s"] = codes, new
    return got
