"""Serving ops: paged KV append (K13) with or without the rotation, paged decode attention (K12) over caches of 16 or 8 bits, batched sampling (K14).
CUDA/bf16 runs the native kernels; CPU tensors run a plain PyTorch restatement (used by the CPU tests and as the oracle).

A cache of 8 bits is [blocks, kv_heads, block_size, head_dim] of ``torch.float8_e4m3fn`` with scales, fp32 [blocks, kv_heads]: a number is its code times
its block's scale (``allocate_fp8_cache``)."""
from __future__ import annotations

import contextlib
import math
from functools import lru_cache
from typing import Optional

import torch

from . import native

c_void_p, c_int, c_ll, c_float = native.c_void_p, native.c_int, native.c_ll, native.c_float
native.register_signature("llmctl_kv_append", [c_void_p, c_ll, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p])
native.register_signature("llmctl_paged_attn_decode",
                          [c_void_p, c_ll, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_ll, c_void_p,
                           c_int, c_int, c_int, c_int, c_int, c_int, c_float, c_void_p])
native.register_signature("llmctl_paged_attn_scratch_elems", [c_int, c_int, c_int, c_int], restype=c_ll)
native.register_signature("llmctl_rope_kv_append", [c_void_p, c_ll] + [c_int] * 4 + [c_void_p, c_void_p, c_int] + [c_void_p] * 4 + [c_ll, c_void_p])
native.register_signature("llmctl_rope_kv_append_fp8", [c_void_p, c_ll] + [c_int] * 4 + [c_void_p, c_void_p, c_int] + [c_void_p] * 6 + [c_int, c_int, c_void_p, c_void_p])
native.register_signature("llmctl_rope_kv_append_fp8_scratch_elems", [c_int], restype=c_ll)
native.register_signature("llmctl_paged_attn_fp8_scratch_elems", [c_int] * 8, restype=c_ll)
native.register_signature("llmctl_paged_attn_decode_fp8", [c_void_p, c_ll] + [c_void_p] * 5 + [c_int] + [c_void_p] * 3 + [c_int] * 8 + [c_float, c_void_p])
native.register_signature("llmctl_sample", [c_void_p, c_int, c_ll, c_int, c_int] + [c_void_p] * 6 + [c_void_p])

native.register_signature("llmctl_paged_attn_shared_scratch_elems", [c_int] * 4, restype=c_ll)
native.register_signature("llmctl_paged_attn_decode_shared", [c_void_p, c_ll, c_void_p, c_void_p, c_void_p, c_int] + [c_void_p] * 5 + [c_int] * 7 + [c_float, c_void_p])


def _check(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _check_cache(cache: torch.Tensor, like: torch.Tensor, row: int) -> None:
    _check(cache.is_cuda and cache.dtype == like.dtype and cache.is_contiguous() and cache.data_ptr() % 16 == 0 and cache.numel() % row == 0,
           f"a cache is contiguous rows of {row} {like.dtype} numbers on the GPU, from a 16-byte boundary")


def kv_append(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
              heads: int, head_dim: int) -> None:
    """qkv: [T, 3*heads*head_dim] (post-RoPE); caches: [blocks, block_size, heads, head_dim];
    slot_mapping: int64 [T] (negative = skip)."""
    hd = heads * head_dim
    if qkv.is_cuda:
        if native.fast.kv_append(qkv, k_cache, v_cache, slot_mapping, heads, head_dim) is not None:
            return
        _check(qkv.dim() == 2 and qkv.dtype.itemsize == 2 and qkv.shape[1] >= 3 * hd > 0, f"qkv: 16-bit rows of at least {3 * hd} numbers")
        _check_cache(k_cache, qkv, hd)
        _check_cache(v_cache, qkv, hd)
        _check(slot_mapping.is_cuda and slot_mapping.dtype == torch.int64 and slot_mapping.numel() >= qkv.shape[0], "slot_mapping: int64 on the GPU, one per row")
        slot_mapping = slot_mapping.contiguous()
        if qkv.stride(1) != 1 or qkv.data_ptr() % 16:
            qkv = qkv.clone(memory_format=torch.contiguous_format)
        native.call("llmctl_kv_append", qkv.data_ptr(), qkv.stride(0), hd, 2 * hd, k_cache.data_ptr(),
                    v_cache.data_ptr(), slot_mapping.data_ptr(), qkv.shape[0], heads, head_dim, native.stream_ptr())
        return
    ok = slot_mapping >= 0
    kc, vc = k_cache.view(-1, hd), v_cache.view(-1, hd)
    kc[slot_mapping[ok]] = qkv[ok, hd:2 * hd]
    vc[slot_mapping[ok]] = qkv[ok, 2 * hd:3 * hd]


def choose_splits(batch: int, heads: int, max_context: int, block_size: int, sms: int = 148) -> int:
    # Each CTA walks block table -> K/V rows -> online softmax in a dependent chain, so HBM fills up with a few CTAs per SM and many more
    # to follow.  Splits are whole KV blocks of >= 64 tokens; the merge pass costs (head_dim + 2) floats per split, ~3 % of the K/V bytes at
    # 64 tokens per split.
    # Up to 512 (head, sequence) pairs a CTA walks at most 512 tokens where 8 splits allow it; more pairs fill the waves by themselves, and
    # what each split adds is lost.  Around the line the splits differ by 2% either way (us by splits, contexts from a quarter of the stated
    # one: 16 sequences of up to 4096, 32 heads of 128 2: 109.0, 8: 110.8, 16: 118.0; 32 of them 2: 200.1, 8: 203.3; 64 1: 374.6, 4: 383.5; 256 of up
    # to 1500 1: 551.7, 4: 575.2; 64 of up to 2304, 12 heads of 64 1: 55.3, 2: 53.9, 8: 54.3); it was drawn for a kernel that took a quarter
    # longer, whose full batches of unlike contexts gained 10% by 8 splits.
    want = max(1, (8 * sms + batch * heads - 1) // (batch * heads), min(8, (max_context + 511) // 512) if batch * heads <= 512 else 1)
    per_split = max(block_size, (64 // block_size) * block_size) if block_size <= 64 else block_size
    return int(max(1, min(want, max(1, max_context // per_split), 256)))


@lru_cache(maxsize=4096)
def _launch_splits(batch: int, heads: int, head_dim: int, max_context: int, block_size: int, sms: int = 148) -> int:
    # One launch, merged inside clusters of up to 8 splits, while all CTAs (three per SM) are resident together and none walks
    # more than 768 tokens (us in one launch / in the splits of choose_splits with a merge kernel: one context of 4096, 32 heads of 128
    # 14.5 in 8 / 16.8 in 16; 8 of up to 2304, 4 heads 13.5 / 13.8; 64 of 500, 4 heads 12.6 / 12.3).  Beyond one
    # wave a single split without a merge kernel pays for the shortest walks only (64 of 500, 12 heads of 64: 13.5 / 14.8; 32 heads of
    # 128: 65.1 / 62.8); larger batches and longer contexts take choose_splits.
    resident = min(8, 3 * sms // (batch * heads))
    if max_context <= 768 * resident:
        return max(1, min(resident, max_context // 64))
    if resident == 0 and max_context * head_dim <= 512 * 64:
        return 1
    return choose_splits(batch, heads, max_context, block_size, sms)


def paged_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_tables: torch.Tensor, context_lens: torch.Tensor, max_context: int,
                           scale: Optional[float] = None, num_splits: Optional[int] = None,
                           scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q: [B, heads, head_dim]; block_tables: int32 [B, max_blocks]; context_lens: int32 [B] -> [B, heads, head_dim]."""
    B, H, D = q.shape
    block_size = k_cache.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if q.is_cuda:
        ns = num_splits or _launch_splits(B, H, D, max_context, block_size)
        if scratch is None:
            out = native.fast.paged_decode(q, k_cache, v_cache, block_tables, context_lens, max_context, ns, scale)
            if out is not None:
                return out
        _check(q.dtype == torch.bfloat16, "q: bfloat16")
        _check_cache(k_cache, q, H * D)
        _check_cache(v_cache, q, H * D)
        _check(k_cache.shape == v_cache.shape, "k_cache and v_cache: of one shape")
        _check(block_tables.is_cuda and block_tables.dtype == torch.int32 and block_tables.dim() == 2 and block_tables.shape[0] >= B,
               "block_tables: int32 on the GPU, a row per sequence")
        _check(context_lens.is_cuda and context_lens.dtype == torch.int32 and context_lens.numel() >= B, "context_lens: int32 on the GPU, one per sequence")
        block_tables, context_lens = block_tables.contiguous(), context_lens.contiguous()
        if q.stride(2) != 1 or q.stride(1) != D or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
        need = native.lib().llmctl_paged_attn_scratch_elems(B, H, D, ns)
        if need and (scratch is None or scratch.numel() < need or scratch.dtype != torch.float32 or not scratch.is_contiguous()):
            scratch = torch.empty(need, dtype=torch.float32, device=q.device)
        out = torch.empty(B, H, D, dtype=q.dtype, device=q.device)
        native.call("llmctl_paged_attn_decode", q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
                    block_tables.data_ptr(), block_tables.shape[1], context_lens.data_ptr(), out.data_ptr(),
                    out.stride(0), native.ptr(scratch), B, H, D, block_size, int(max_context), ns, float(scale),
                    native.stream_ptr())
        if need:
            native.count_launches(1)        # the merge kernel
        return out
    out = torch.zeros(B, H, D, dtype=q.dtype)
    for b in range(B):
        n = int(context_lens[b])
        if n == 0:
            continue
        idx = torch.arange(n)
        slots = block_tables[b, idx // block_size].long() * block_size + idx % block_size
        k = k_cache.view(-1, H, D)[slots].float()
        v = v_cache.view(-1, H, D)[slots].float()
        s = torch.einsum("hd,nhd->hn", q[b].float(), k) * scale
        out[b] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), v).to(q.dtype)
    return out


# ---- rotation and append in one pass; caches of 8 bits ---------------------------------------------------------------------------------------------
FP8 = torch.float8_e4m3fn
_FP8_MAX = 448.0


def allocate_fp8_cache(num_blocks: int, block_size: int, kv_heads: int, head_dim: int, device=None):
    """``(codes, scales)`` of an empty cache of 8 bits for keys or for values."""
    return (torch.zeros(num_blocks, kv_heads, block_size, head_dim, dtype=FP8, device=device), torch.zeros(num_blocks, kv_heads, dtype=torch.float32, device=device))


def _on_device(t: torch.Tensor):
    """Launches go to the current device's stream: a context in which that is the tensor's device."""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _check_fp8_caches(k_cache, v_cache, k_scale, v_scale, head_dim: int, device) -> None:
    for c, s in ((k_cache, k_scale), (v_cache, v_scale)):
        _check(c.dim() == 4 and c.dtype == FP8 and c.is_contiguous() and c.device == device and c.shape[3] == head_dim and c.data_ptr() % 16 == 0,
               f"a cache of 8 bits is contiguous [blocks, kv_heads, block_size, {head_dim}] of {FP8} beside the rows, from a 16-byte boundary")
        _check(s is not None and s.dtype == torch.float32 and s.is_contiguous() and s.device == device and s.shape == c.shape[:2],
               "scales of a cache of 8 bits: contiguous float32 [blocks, kv_heads] beside it")
    _check(k_cache.shape == v_cache.shape, "k_cache and v_cache: of one shape")


def _quantise_rows(x: torch.Tensor, cache: torch.Tensor, scale: torch.Tensor, slots: torch.Tensor) -> None:
    """x: fp32 [T, kv_heads, head_dim] to the rows ``slots`` of a cache of 8 bits, as the kernel does it (csrc/serve/rope_kv_append.cu)."""
    size = cache.shape[2]
    last = {int(s): i for i, s in enumerate(slots.tolist()) if 0 <= s < cache.shape[0] * size}      # of a slot's tokens the last
    for block in sorted({s // size for s in last}):
        rows = [r for r in range(size) if block * size + r in last]
        new = x[[last[block * size + r] for r in rows]].transpose(0, 1)                              # [kv_heads, rows, head_dim]
        most = torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 2))
        mantissa, exponent = torch.frexp(most)
        need = torch.where(most > 0, torch.ldexp(torch.ones_like(most), (exponent - 9 + (mantissa > _FP8_MAX / 512).int()).clamp(min=-126)), 0.0)
        old = torch.zeros_like(need) if rows[0] == 0 else scale[block].clamp(min=0.0)
        to = torch.maximum(need, old)
        if rows[0] != 0:
            grown = (to > old).nonzero().reshape(-1)
            others = torch.tensor([r for r in range(size) if block * size + r not in last], dtype=torch.int64)
            for h in grown.tolist():
                cache[block, h, others] = (cache[block, h, others].float() * (old[h] / to[h])).to(FP8)
        inv = torch.where(to > 0, 1.0 / to, 0.0)[:, None, None]
        cache[block][:, torch.tensor(rows)] = torch.where(new.isfinite(), new * inv, float("nan")).to(FP8)
        scale[block] = to


def rope_kv_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slot_mapping: torch.Tensor, heads: int, head_dim: int, *, kv_heads: Optional[int] = None, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates q and k of the packed rows ``qkv`` [T, (heads + 2 kv_heads) * head_dim] in place to their ``positions`` (int32 [T], rows of the tables ``cos`` /
    ``sin``, fp32 [positions, head_dim / 2]; one outside of them reads the nearest) and writes k and v to the rows ``slot_mapping`` (int64 [T]; outside of the
    cache = skip) of the caches: [blocks, block_size, kv_heads, head_dim] of the rows' type, or caches of 8 bits with their scales.  head_dim is a multiple of 16 on a GPU and for
    caches of 8 bits, else even.  Returns ``qkv``.

    In a cache of 16 bits a row that the call names more than once is left with numbers of any of those tokens, of several perhaps: name it once, as with
    ``kv_append``.  In a cache of 8 bits the last is kept.  There a block's scale is the smallest power of two under which the largest number
    written to it fits, and the tokens of a block may stand anywhere in the call.  A block whose first row is written begins anew; in any other
    the rows that the call does not write keep what they stand for, in codes of the larger scale where it grows.  NaN and infinities become NaN."""
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.is_cuda and native.fast.rope_kv_append(qkv, cos, sin, positions, k_cache, v_cache, slot_mapping, heads, kv_heads, head_dim, k_scale, v_scale) is not None:
        return qkv
    fp8 = k_cache.dtype == FP8
    T, width = qkv.shape[0], (heads + 2 * kv_heads) * head_dim
    _check(heads > 0 and kv_heads > 0 and heads % kv_heads == 0, "heads: a multiple of kv_heads")
    _check(head_dim > 0 and head_dim % (16 if qkv.is_cuda or fp8 else 2) == 0, "head_dim: a multiple of 16 on a GPU and in a cache of 8 bits, else even")
    _check(qkv.dim() == 2 and qkv.shape[1] >= width, f"qkv: rows of at least {width} numbers")
    _check(not (torch.is_grad_enabled() and qkv.requires_grad), "rope_kv_append has no backward: call it under no_grad")
    for t in (cos, sin):
        _check(t.dim() == 2 and t.shape == cos.shape and t.shape[0] > 0 and t.shape[1] == head_dim // 2 and t.dtype == torch.float32 and t.device == qkv.device,
               f"cos and sin: float32 [positions, {head_dim // 2}] beside the rows")
    _check(positions.shape == (T,) and positions.dtype == torch.int32 and positions.device == qkv.device, "positions: int32 beside the rows, one per row")
    _check(slot_mapping.shape == (T,) and slot_mapping.dtype == torch.int64 and slot_mapping.device == qkv.device, "slot_mapping: int64 beside the rows, one per row")
    if fp8:
        _check_fp8_caches(k_cache, v_cache, k_scale, v_scale, head_dim, qkv.device)
        _check(k_cache.shape[1] == kv_heads and 1 <= k_cache.shape[2] <= 4096 and head_dim <= 512 and kv_heads <= 512,
               f"a cache of 8 bits of {kv_heads} heads, at most 512 of them and of at most 512 numbers, in blocks of at most 4096 rows")
    else:
        _check(k_scale is None and v_scale is None, "scales belong to caches of 8 bits")
        for c in (k_cache, v_cache):
            _check(c.dtype == qkv.dtype and c.device == qkv.device and c.is_contiguous() and c.dim() == 4 and c.shape[2:] == (kv_heads, head_dim) and c.data_ptr() % 16 == 0,
                   f"a cache is contiguous [blocks, block_size, {kv_heads}, {head_dim}] of the rows' type beside them, from a 16-byte boundary")
        _check(k_cache.shape == v_cache.shape, "k_cache and v_cache: of one shape")
    if qkv.is_cuda:
        _check(qkv.dtype == torch.bfloat16, "qkv: bfloat16")
        cos, sin, positions, slot_mapping = (t.contiguous() for t in (cos, sin, positions, slot_mapping))
        cos, sin = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (cos, sin))
        rows = qkv if qkv.stride(1) == 1 and qkv.stride(0) % 8 == 0 and qkv.stride(0) >= width and qkv.data_ptr() % 16 == 0 else _aligned_rows(qkv, width)
        args = (rows.data_ptr(), rows.stride(0), T, heads, kv_heads, head_dim, cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
                slot_mapping.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr())
        with _on_device(qkv):
            if fp8:
                need = native.lib().llmctl_rope_kv_append_fp8_scratch_elems(T)
                scratch = torch.empty(need, dtype=torch.int32, device=qkv.device) if need else None
                native.call("llmctl_rope_kv_append_fp8", *args, k_scale.data_ptr(), v_scale.data_ptr(), k_cache.shape[0], k_cache.shape[2], native.ptr(scratch),
                            native.stream_ptr())
                if need:
                    native.count_launches(1)        # which windows of tokens write to which blocks
            else:
                native.call("llmctl_rope_kv_append", *args, k_cache.shape[0] * k_cache.shape[1], native.stream_ptr())
            if rows is not qkv:
                qkv[:, :width].copy_(rows)
            elif not qkv.is_inference():
                torch.autograd.graph.increment_version(qkv)
        return qkv
    x = qkv[:, :width].view(T, heads + 2 * kv_heads, head_dim)
    half = head_dim // 2
    at = positions.long().clamp(0, cos.shape[0] - 1)
    c, s = cos[at].unsqueeze(1), sin[at].unsqueeze(1)
    a, b = x[:, :heads + kv_heads, :half].float(), x[:, :heads + kv_heads, half:].float()
    rotated = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    x[:, :heads + kv_heads] = rotated.to(x.dtype)
    if fp8:
        _quantise_rows(rotated[:, heads:], k_cache, k_scale, slot_mapping)
        _quantise_rows(x[:, heads + kv_heads:].float(), v_cache, v_scale, slot_mapping)
        return qkv
    ok = (slot_mapping >= 0) & (slot_mapping < k_cache.shape[0] * k_cache.shape[1])
    k_cache.view(-1, kv_heads, head_dim)[slot_mapping[ok]] = x[ok, heads:heads + kv_heads]
    v_cache.view(-1, kv_heads, head_dim)[slot_mapping[ok]] = x[ok, heads + kv_heads:]
    return qkv


def _aligned_rows(x: torch.Tensor, width: int) -> torch.Tensor:
    """A copy of the first ``width`` columns in rows that begin at 16-byte boundaries."""
    return x[:, :width].clone(memory_format=torch.contiguous_format)


def paged_attention_decode_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                               block_tables: torch.Tensor, context_lens: torch.Tensor, max_context: int, scale: Optional[float] = None,
                               num_splits: Optional[int] = None) -> torch.Tensor:
    """``paged_attention_decode`` over caches of 8 bits: q [B, heads, head_dim], a token per sequence; block_tables: int32 [B, max_blocks]; context_lens: int32
    [B], at most ``max_context`` (tokens beyond it, or beyond the table, are left out) -> [B, heads, head_dim].  heads may be a multiple of the cache's heads:
    query head h reads head h // (heads / kv_heads).  A sequence without tokens gets zeros.  What the cache holds behind a sequence's last token does not matter.  On a GPU
    blocks of a multiple of 8 tokens are read at six times the speed of others."""
    B, H, D = q.shape
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if q.is_cuda and num_splits != 0:
        out = native.fast.paged_decode_fp8(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, max_context, num_splits or 0, scale)
        if out is not None:
            return out
    blocks, kv_heads, block_size = k_cache.shape[:3]
    _check(not (torch.is_grad_enabled() and q.requires_grad), "paged_attention_decode_fp8 has no backward: call it under no_grad")
    _check_fp8_caches(k_cache, v_cache, k_scale, v_scale, D, q.device)
    _check(H % kv_heads == 0, "heads: a multiple of the cache's")
    _check(block_tables.dim() == 2 and block_tables.shape[0] >= B and block_tables.dtype == torch.int32 and block_tables.device == q.device, "block_tables: int32 beside the queries, a row per sequence")
    _check(context_lens.dim() == 1 and context_lens.numel() >= B and context_lens.dtype == torch.int32 and context_lens.device == q.device, "context_lens: int32 beside the queries, one per sequence")
    max_context = max(0, min(int(max_context), block_tables.shape[1] * block_size))
    if q.is_cuda:
        _check(q.dtype == torch.bfloat16 and D in (64, 128), "q: bfloat16, heads of 64 or 128")
        _check(num_splits is None or 1 <= num_splits <= 256, "num_splits: 1 to 256")
        out = torch.empty(B, H, D, dtype=q.dtype, device=q.device)
        if B == 0:
            return out
        ns = num_splits or 0
        block_tables, context_lens = block_tables.contiguous(), context_lens.contiguous()
        if q.stride(2) != 1 or q.stride(1) != D or q.data_ptr() % 16 or q.stride(0) % 8:
            q = q.clone(memory_format=torch.contiguous_format)
        need = native.lib().llmctl_paged_attn_fp8_scratch_elems(B, H, kv_heads, D, block_tables.shape[1], block_size, max_context, ns)
        scratch = torch.empty(need, dtype=torch.float32, device=q.device) if need else None
        with _on_device(q):
            native.call("llmctl_paged_attn_decode_fp8", q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                        v_scale.data_ptr(), block_tables.data_ptr(), block_tables.shape[1], context_lens.data_ptr(), out.data_ptr(), native.ptr(scratch), B, H,
                        kv_heads, D, blocks, block_size, max_context, ns, float(scale), native.stream_ptr())
        if need:
            native.count_launches(1)        # the merge kernel
        return out
    out = torch.zeros(B, H, D, dtype=q.dtype)
    for b in range(B):
        n = min(int(context_lens[b]), max_context)
        if n <= 0:
            continue
        pages = block_tables[b, :(n + block_size - 1) // block_size].long()
        k, v = ((c[pages].float() * s[pages][..., None, None]).transpose(0, 1).reshape(kv_heads, -1, D)[:, :n] for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        s = torch.einsum("kgd,knd->kgn", q[b].float().view(kv_heads, H // kv_heads, D), k) * scale
        out[b] = torch.einsum("kgn,knd->kgd", torch.softmax(s, -1), v).reshape(H, D).to(q.dtype)
    return out


def paged_attention_decode_shared(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                                  group_starts: torch.Tensor, shared_lens: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """``paged_attention_decode`` of groups of sequences whose contexts begin with the same blocks, completions of one prompt for instance, which are read once
    for a group.  q: [B, heads, head_dim], a token per sequence; caches [blocks, block_size, kv_heads, head_dim] of q's type; block_tables: int32 [B, max_blocks];
    context_lens: int32 [B] (tokens beyond the table are left out).  group_starts: int32 [G + 1], ascending: the sequences group_starts[g] up to group_starts[g + 1] are
    one group, whose tables name the same blocks for their first shared_lens[g] (int32 [G]) tokens; a number that is not of whole blocks is taken too.  Sequences in no
    group, and a group of one, share nothing.  All stand beside q, and what they hold is read when the kernel runs, so that a captured call follows them.
    -> [B, heads, head_dim].

    heads may be a multiple of the cache's heads: query head h reads head h // (heads / kv_heads).  A sequence without tokens gets zeros, one that is
    shorter than what its group shares its own tokens of them.  What the cache holds behind a sequence's last token does not matter (but for what its group shares,
    which has to be numbers).  On a GPU: bfloat16, heads of 64 or 128, blocks of a multiple of 8 tokens."""
    _check(q.dim() == 3, "q: [sequences, heads, head_dim]")
    B, H, D = q.shape
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if q.is_cuda:
        out = native.fast.paged_decode_shared(q, k_cache, v_cache, block_tables, context_lens, group_starts, shared_lens, scale)
        if out is not None:
            return out
    _check(not (torch.is_grad_enabled() and q.requires_grad), "paged_attention_decode_shared has no backward: call it under no_grad")
    _check(scale > 0, "scale: positive")
    for c in (k_cache, v_cache):
        _check(c.dim() == 4 and c.dtype == q.dtype and c.is_contiguous() and c.device == q.device and c.shape[3] == D and c.data_ptr() % 16 == 0,
               f"a cache is contiguous [blocks, block_size, kv_heads, {D}] of q's type beside it, from a 16-byte boundary")
    _check(k_cache.shape == v_cache.shape, "k_cache and v_cache: of one shape")
    blocks, block_size, kv_heads = k_cache.shape[:3]
    _check(kv_heads > 0 and H % kv_heads == 0, "heads: a multiple of the cache's")
    _check(block_tables.dim() == 2 and block_tables.shape[0] >= B and block_tables.dtype == torch.int32 and block_tables.device == q.device, "block_tables: int32 beside the queries, a row per sequence")
    _check(context_lens.dim() == 1 and context_lens.numel() >= B and context_lens.dtype == torch.int32 and context_lens.device == q.device, "context_lens: int32 beside the queries, one per sequence")
    G = shared_lens.numel()
    _check(shared_lens.dim() == 1 and shared_lens.dtype == torch.int32 and shared_lens.device == q.device, "shared_lens: int32 beside the queries, one per group")
    _check(group_starts.dim() == 1 and group_starts.numel() == G + 1 and group_starts.dtype == torch.int32 and group_starts.device == q.device,
           "group_starts: int32 beside the queries, one more than groups")
    if q.is_cuda:
        _check(q.dtype == torch.bfloat16 and D in (64, 128), "q: bfloat16, heads of 64 or 128")
        _check(block_size % 8 == 0 and block_size > 0, "blocks of a multiple of 8 tokens")
        out = torch.empty(B, H, D, dtype=q.dtype, device=q.device)
        if out.numel() == 0:
            return out
        if blocks == 0:
            return out.zero_()
        block_tables, context_lens, group_starts, shared_lens = (t.contiguous() for t in (block_tables, context_lens, group_starts, shared_lens))
        if q.stride(2) != 1 or q.stride(1) != D or q.data_ptr() % 16 or q.stride(0) % 8:
            q = q.clone(memory_format=torch.contiguous_format)
        scratch = torch.empty(native.lib().llmctl_paged_attn_shared_scratch_elems(B, G, H, D), dtype=torch.float32, device=q.device)
        with _on_device(q):
            native.call("llmctl_paged_attn_decode_shared", q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), block_tables.shape[1],
                        context_lens.data_ptr(), group_starts.data_ptr(), shared_lens.data_ptr(), out.data_ptr(), scratch.data_ptr(), B, G, H, kv_heads, D, blocks, block_size,
                        float(scale), native.stream_ptr())
        return out
    out = torch.zeros(B, H, D, dtype=q.dtype)
    first, starts = list(range(B)), group_starts.tolist()          # whose table holds a sequence's shared tokens
    shared = [0] * B
    limit = block_tables.shape[1] * block_size
    for g, n in enumerate(shared_lens.tolist()):
        a, b = (max(0, min(s, B)) for s in starts[g:g + 2])
        for i in range(a, b):
            first[i], shared[i] = a, max(0, min(n, int(context_lens[a]), limit)) if b - a > 1 else 0
    for b in range(B):
        n = min(int(context_lens[b]), limit)
        if n <= 0:
            continue
        idx = torch.arange(n)
        table = torch.where(idx < shared[b], block_tables[first[b]][idx // block_size], block_tables[b][idx // block_size]).long()
        k, v = (c[table, idx % block_size].float().transpose(0, 1) for c in (k_cache, v_cache))
        s = torch.einsum("kgd,knd->kgn", q[b].float().view(kv_heads, H // kv_heads, D), k) * scale
        out[b] = torch.einsum("kgn,knd->kgd", torch.softmax(s, -1), v).reshape(H, D).to(q.dtype)
    return out


def sample_reference(logits: torch.Tensor, temperature: float, top_k: int, top_p: float,
                     generator: Optional[torch.Generator] = None) -> int:
    """The reference's sampling pipeline for one row (reference llmctl/serve/server.py:209-235), restated."""
    x = logits.float().clone()      # never edit the caller's logits
    if temperature <= 0:
        return int(x.argmax())
    if temperature != 1.0:
        x = x / temperature
    if top_k and top_k > 0:
        kth = torch.topk(x, min(top_k, x.numel())).values[-1]
        x = torch.where(x < kth, torch.full_like(x, float("-inf")), x)
    if top_p < 1.0:
        sx, si = torch.sort(x, descending=True)
        cp = torch.softmax(sx, -1).cumsum(-1)
        remove = cp > top_p
        remove[1:] = remove[:-1].clone()
        remove[0] = False
        x[si[remove]] = float("-inf")
    return int(torch.multinomial(torch.softmax(x, -1), 1, generator=generator))


def sample(logits: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor,
           uniform: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Batched sampling.  logits [B, V] bf16/fp32; per-row parameter tensors; returns int64 [B]."""
    B, V = logits.shape
    if logits.is_cuda:
        if uniform is None:
            uniform = torch.rand(B, device=logits.device)
        out = torch.empty(B, dtype=torch.int64, device=logits.device)
        native.call("llmctl_sample", logits.data_ptr(), int(logits.dtype == torch.float32), logits.stride(0), B, V,
                    temperature.data_ptr(), top_k.data_ptr(), top_p.data_ptr(), uniform.data_ptr(), out.data_ptr(),
                    None, native.stream_ptr())
        return out
    return torch.tensor([sample_reference(logits[i], float(temperature[i]), int(top_k[i]), float(top_p[i]))
                         for i in range(B)], dtype=torch.int64)
