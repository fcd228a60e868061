"""Decode attention over shared prefixes in 64 bits, with a bound for the kernel's roundings, and batches to try it on."""
import math

import torch


def batch(groups, after, page, heads, kv_heads, dim, seed=0, device="cpu", singles=0, spread=1.0):
    """groups: (sequences, shared tokens); after: tokens of each sequence behind them, in turn; singles: sequences in no group behind the groups'.  Pages are scattered, what
    they hold behind a sequence's last token is no number."""
    g = torch.Generator().manual_seed(seed)
    starts, shared, lens, own = [0], [n for _, n in groups], [], []
    for count, n in groups:
        starts.append(starts[-1] + count)
        for _ in range(count):
            own.append(after[len(own) % len(after)])
            lens.append(n + own[-1])
    for _ in range(singles):
        own.append(after[len(own) % len(after)])
        lens.append(own[-1])
    B = len(lens)
    need = sum((n + page - 1) // page for n in lens) + 1
    perm, at = torch.randperm(need, generator=g).to(torch.int32), 0
    tables = torch.zeros(B, max(1, max((n + page - 1) // page for n in lens)), dtype=torch.int32)
    k, v = (torch.full((need, page, kv_heads, dim), float("nan")) for _ in range(2))
    group = [i for i, (count, _) in enumerate(groups) for _ in range(count)] + [-1] * singles
    common = {}
    for b in range(B):
        whole = shared[group[b]] // page if group[b] >= 0 else 0
        if group[b] >= 0 and group[b] not in common:
            common[group[b]] = perm[at:at + whole]
            at += whole
        rest = (lens[b] + page - 1) // page - whole
        if whole:
            tables[b, :whole] = common[group[b]]
        tables[b, whole:whole + rest] = perm[at:at + rest]
        at += rest
    shared = [n // page * page for n in shared]
    for b in range(B):
        for t in range(0, lens[b]):
            block, row = int(tables[b, t // page]), t % page
            if torch.isnan(k[block, row]).any():
                k[block, row] = torch.randn(kv_heads, dim, generator=g) * spread
                v[block, row] = torch.randn(kv_heads, dim, generator=g)
    q = torch.randn(B, heads, dim, generator=g)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=q.bfloat16().to(device), k_cache=k.bfloat16().to(device), v_cache=v.bfloat16().to(device), block_tables=tables.to(device), context_lens=ints(lens),
                group_starts=ints(starts), shared_lens=ints(shared))


def attention(q, k_cache, v_cache, block_tables, context_lens, group_starts=None, shared_lens=None, scale=None):
    """(value, bound): every sequence over its own table, in 64 bits.  A weight rounded to bf16 is off by 2^-8 of itself at most (half a step), and so may the weighted sum be of
    sum p |v|, as may the sum that it is divided by; scores in 32 bits are off by dim 2^-23 of their products' sizes, which the exponential takes as a relative error,
    exponentials by 2^-21; the output's own rounding is 2^-8 of it."""
    B, H, D = q.shape
    page, Hk = k_cache.shape[1:3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    q, k_cache, v_cache, block_tables = q.cpu(), k_cache.cpu(), v_cache.cpu(), block_tables.cpu()
    for b in range(B):
        n = min(int(context_lens[b]), block_tables.shape[1] * page)
        if n <= 0:
            continue
        idx = torch.arange(n)
        at = block_tables[b, idx // page].long()
        k, v = (c[at, idx % page].double().repeat_interleave(H // Hk, 1) for c in (k_cache, v_cache))       # [n, H, D]
        x = q[b].double()
        p = torch.softmax(torch.einsum("hd,nhd->hn", x, k) * scale, -1)
        size = torch.einsum("hd,nhd->hn", x.abs(), k.abs()).amax(-1) * scale
        out[b] = torch.einsum("hn,nhd->hd", p, v)
        most = torch.einsum("hn,nhd->hd", p, v.abs())
        off = 2.0 ** -8 + 2.0 ** -20 + (D * 2.0 ** -22) * size[:, None]
        bound[b] = most * off + out[b].abs() * off
        bound[b] += (out[b].abs() + bound[b]) * 2.0 ** -8 + 1e-30
    return out, bound


def check(got, want):
    y, bound = want
    got = got.double().cpu()
    assert got.shape == y.shape and torch.isfinite(got).all()
    over = (got - y).abs() - bound
    assert over.max() <= 0, f"off by {over.max().item():.3g} more than the bound"
