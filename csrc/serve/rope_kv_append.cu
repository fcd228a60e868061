// Rotation of new tokens' packed q | k | v rows and the write of their keys and values into a paged cache, in one pass over the rows.
//
//   q', k' = rotation of q, k to the token's position (rotate-half pairs d, d + D/2; the products are rounded as rope.cu rounds them)
//   cache[slot] = k', v
//
// in place for q and k.  Two forms of the cache:
//   16 bits  [blocks, block_size, kv_heads, head_dim] bf16, as kv_append in paged_attention.cu writes it
//   8 bits   [blocks, kv_heads, block_size, head_dim] e4m3 with a scale (fp32) for each (block, head): the number that a code c stands for is
//            c * scale.  What shares a scale stands together in memory.
//
// A block's scale is a power of two: the smallest under which the largest number that was written to it fits (448 is e4m3's largest).  When a later token does
// not fit, the scale grows and the codes that stand in the block are divided by the power of two that it grew by: exact but where a number
// comes to lie among e4m3's subnormals (2^-10 of the scale off at most), so that what a number loses does not add up over a block's tokens.
// The first row of a block begins it anew.  Keys are rounded once, from the rotated value in 32 bits.
//
// Reference: none — the reference keeps no cache (reference llmctl/serve/server.py:199-204).
#include "../common/dependent.cuh"
#include "../common/fast_div.h"
#include "../common/fp8.cuh"
#include "../common/ptx.cuh"
#include "../common/util.cuh"

namespace llmctl {

// (a0, a1) = (a0, a1) * (b0, b1) + (c0, c1)
__device__ __forceinline__ void fma2vv(float& a0, float& a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 ra, rb, rc;\n\t"
      "mov.b64 ra, {%0, %1};\n\tmov.b64 rb, {%2, %3};\n\tmov.b64 rc, {%4, %5};\n\t"
      "fma.rn.f32x2 ra, ra, rb, rc;\n\t"
      "mov.b64 {%0, %1}, ra;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// Eight pairs (a: from the first half, b: from the second) of one row, rotated.
__device__ __forceinline__ void rotate8(float (&a)[8], float (&b)[8], const float* __restrict__ cos_row, const float* __restrict__ sin_row) {
  float c[8], s[8];
  *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cos_row);
  *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(cos_row + 4);
  *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sin_row);
  *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(sin_row + 4);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {            // a c - b s and b c + a s, the products with s rounded by themselves
    float t0, t1, u0, u1;
    ptx::mul2v(t0, t1, b[j], b[j + 1], s[j], s[j + 1]);
    ptx::mul2v(u0, u1, a[j], a[j + 1], s[j], s[j + 1]);
    fma2vv(a[j], a[j + 1], c[j], c[j + 1], -t0, -t1);
    fma2vv(b[j], b[j + 1], c[j], c[j + 1], u0, u1);
  }
}

struct RopeRows {
  __nv_bfloat16* qkv;
  long long row_stride;
  int tokens, heads, kv_heads, head_dim;
  const float *cos_t, *sin_t;
  int table_rows;
  const int* positions;
};

// Row of the rotation tables for a token; a position outside of them reads their nearest row instead of other memory.
__device__ __forceinline__ long long table_row(const RopeRows& r, const int* positions, int tok) {
  return static_cast<long long>(min(max(positions[tok], 0), r.table_rows - 1)) * (r.head_dim >> 1);
}

// ---------------------------------------------------------------------------------------------
// 16 bits: a thread takes 16 numbers of a head, eight pairs of q and k or 16 neighbours of v.  Bound by the pass over the rows.
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
rope_kv_append_kernel(RopeRows r, uint32_t total, FastDiv per_token, FastDiv per_head, const long long* __restrict__ slots,
                      __nv_bfloat16* __restrict__ k_cache, __nv_bfloat16* __restrict__ v_cache, long long cache_rows, int tok0) {
  __nv_bfloat16* qkv = r.qkv;
  const float *cos_t = r.cos_t, *sin_t = r.sin_t;
  const int* positions = r.positions;
  wait_for_previous(qkv, cos_t, sin_t, positions, slots, k_cache, v_cache);
  release_dependents();
  const int half = r.head_dim >> 1;
  for (uint32_t idx = blockIdx.x * blockDim.x + threadIdx.x; idx < total; idx += gridDim.x * blockDim.x) {
    uint32_t unit, at;
    const int tok = tok0 + static_cast<int>(per_token.divide(idx, unit)), head = static_cast<int>(per_head.divide(unit, at));
    __nv_bfloat16* p = qkv + tok * r.row_stride + static_cast<long long>(head) * r.head_dim;
    const long long slot = head >= r.heads ? slots[tok] : -1;
    const bool kept = slot >= 0 && slot < cache_rows;
    if (head < r.heads + r.kv_heads) {
      p += at * 8;
      float a[8], b[8];
      unpack8(load8(p), a);
      unpack8(load8(p + half), b);
      const long long row = table_row(r, positions, tok) + at * 8;
      rotate8(a, b, cos_t + row, sin_t + row);
      const bf16x8 x = pack8(a), y = pack8(b);
      store8(p, x);
      store8(p + half, y);
      if (kept) {
        __nv_bfloat16* dst = k_cache + (slot * r.kv_heads + (head - r.heads)) * r.head_dim + at * 8;
        store8(dst, x);
        store8(dst + half, y);
      }
    } else if (kept) {
      p += at * 16;
      const bf16x8 x = load8(p), y = load8(p + 8);
      __nv_bfloat16* dst = v_cache + (slot * r.kv_heads + (head - r.heads - r.kv_heads)) * r.head_dim + at * 16;
      store8(dst, x);
      store8(dst + 8, y);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// 8 bits.  A block of the cache is written by one CTA alone (for its share of the heads), which finds all tokens of the call that go to it, wherever they
// stand and however often a slot is named (the last token of a slot is the one that is kept): no atomics on results, and the same bytes every
// time.
//
// CTAs 0 .. windows * parts - 1: of the tokens of a window, one that is the first of the call in its block takes the block.  A scan over the slots tells,
// which is left out where the token before goes to the same block (in a prompt, 15 of 16).  A warp then writes a head's block: the rows as they
// are into registers (again, where a block is longer than they hold), the largest rotated number, the scale, the codes.  The others rotate q, four
// units to a thread.
// ---------------------------------------------------------------------------------------------
namespace append8 {
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 4;                     // rows that a lane holds of its place in them
constexpr int kUnits = 4;                    // of q, to a thread
constexpr int kMaxBlock = 4096;
constexpr int kParts = 1000;                 // CTAs of a call that write blocks, or as many as have work

// |x| as an integer that grows with it: kInfinite and more for what is no finite number
constexpr uint32_t kInfinite = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_magnitude(float x) { return magnitude(x) < kInfinite ? magnitude(x) : 0u; }
// The largest |x| of eight, NaN if there is one.
__device__ __forceinline__ float most_of(const bf16x8& v) {
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(v.v[0]), __habs2(v.v[1])), __hmax2_nan(__habs2(v.v[2]), __habs2(v.v[3])));
  const float2 f = __bfloat1622float2(m);
  return f.x != f.x ? f.x : f.y != f.y ? f.y : fmaxf(f.x, f.y);
}
// The smallest power of two (of 2^-126 and up) under which a number of this magnitude is at most 448; 0 for zero.
__device__ __forceinline__ float scale_for(uint32_t most) {
  if (most == 0u) return 0.f;
  const int e = static_cast<int>(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}
}  // namespace append8

__global__ void __launch_bounds__(append8::kThreads, 3)
rope_kv_append_fp8_kernel(RopeRows r, const long long* __restrict__ slots, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
                          float* __restrict__ k_scale, float* __restrict__ v_scale, int blocks, int block_size, int window, int windows, int parts,
                          uint32_t q_units, FastDiv per_token, FastDiv per_head) {
  using namespace append8;
  extern __shared__ int2 row_of[];            // [block_size]: the token that a row of the block at hand is written from, or -1, and its row in the tables
  __shared__ int first_token, twice;
  __nv_bfloat16* qkv = r.qkv;
  const float *cos_t = r.cos_t, *sin_t = r.sin_t;
  const int* positions = r.positions;
  wait_for_previous(qkv, cos_t, sin_t, positions, slots, k_cache, v_cache, k_scale, v_scale);
  release_dependents();
  const int half = r.head_dim >> 1, per_row = r.head_dim >> 4;      // lanes to a row: eight pairs, or 16 neighbours, each
  const int work = static_cast<int>(blockIdx.x);

  if (work >= windows * parts) {              // q
    const uint32_t first = static_cast<uint32_t>(work - windows * parts) * (kThreads * kUnits) + threadIdx.x;
    bf16x8 x[kUnits], y[kUnits];
    __nv_bfloat16* at[kUnits];
    long long row[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const uint32_t idx = first + i * kThreads;
      at[i] = nullptr;
      if (idx < q_units) {
        uint32_t unit, pair;
        const int tok = static_cast<int>(per_token.divide(idx, unit)), head = static_cast<int>(per_head.divide(unit, pair));
        at[i] = qkv + tok * r.row_stride + head * r.head_dim + pair * 8;
        row[i] = table_row(r, positions, tok) + pair * 8;
        x[i] = load8(at[i]);
        y[i] = load8(at[i] + half);
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      if (at[i] != nullptr) {
        float a[8], b[8];
        unpack8(x[i], a);
        unpack8(y[i], b);
        rotate8(a, b, cos_t + row[i], sin_t + row[i]);
        store8(at[i], pack8(a));
        store8(at[i] + half, pack8(b));
      }
    return;
  }

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = work / windows, t0 = (work - part * windows) * window, t1 = min(r.tokens, t0 + window);
  const long long rows = static_cast<long long>(blocks) * block_size;
  // heads of keys that no block's writer rotates: all of a token's, this part's share
  auto rotate_keys = [&](int tok) {
    for (int i = threadIdx.x; i < r.kv_heads * per_row; i += kThreads)
      if ((i / per_row) % parts == part) {
        const int at = i % per_row;
        __nv_bfloat16* p = qkv + tok * r.row_stride + static_cast<long long>(r.heads + i / per_row) * r.head_dim + at * 8;
        float a[8], b[8];
        unpack8(load8(p), a);
        unpack8(load8(p + half), b);
        const long long row = table_row(r, positions, tok) + at * 8;
        rotate8(a, b, cos_t + row, sin_t + row);
        store8(p, pack8(a));
        store8(p + half, pack8(b));
      }
  };

  const int sub = lane / per_row, at = lane - sub * per_row, step = 32 / per_row;      // rows of a warp at a time; lanes past them idle
  // Of the window's tokens (16 at most, a lane each): those without a row, and those that may be the first in their block.
  long long slot = -1, before = -1;
  if (t0 + lane < t1) {
    slot = slots[t0 + lane];
    if (t0 + lane > 0) before = slots[t0 + lane - 1];
  }
  const bool padded = slot < 0 || slot >= rows, behind = !padded && before >= 0 && before < rows && before / block_size == slot / block_size;
  const unsigned window_mask = t1 - t0 >= 32 ? ~0u : (1u << (t1 - t0)) - 1u;
  for (unsigned left = __ballot_sync(0xffffffffu, padded) & window_mask; left != 0u; left &= left - 1u) rotate_keys(t0 + __ffs(left) - 1);
  for (unsigned left = __ballot_sync(0xffffffffu, !padded && !behind) & window_mask; left != 0u; left &= left - 1u) {
    const int t = t0 + __ffs(left) - 1, block = static_cast<int>(__shfl_sync(0xffffffffu, slot, t - t0) / block_size);
    const long long lo = static_cast<long long>(block) * block_size, hi = lo + block_size;
    __syncthreads();                          // the rows of the block before have been read
    for (int i = threadIdx.x; i < block_size; i += kThreads) row_of[i].x = -1;
    if (threadIdx.x == 0) {
      first_token = t;
      twice = 0;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < r.tokens; i += kThreads) {
      const long long s = slots[i];
      if (s >= lo && s < hi) {
        if (i < t) atomicMin(&first_token, i);
        if (atomicMax(&row_of[s - lo].x, i) >= 0) twice = 1;
      }
    }
    __syncthreads();
    if (first_token != t) continue;
    for (int i = threadIdx.x; i < block_size; i += kThreads)
      if (row_of[i].x >= 0) row_of[i].y = min(max(positions[row_of[i].x], 0), r.table_rows - 1);
    if (twice)
      for (int i = 0; i < r.tokens; ++i) {
        const long long s = slots[i];
        if (s >= lo && s < hi && row_of[s - lo].x != i) rotate_keys(i);
      }
    __syncthreads();
    const bool begun = row_of[0].x >= 0;

    for (int task = part + warp * parts; task < 2 * r.kv_heads; task += kWarps * parts) {
      const bool key = task < r.kv_heads;
      const int head = key ? task : task - r.kv_heads;
      uint8_t* codes = (key ? k_cache : v_cache) + (static_cast<long long>(block) * r.kv_heads + head) * block_size * r.head_dim;
      float* scale_at = (key ? k_scale : v_scale) + static_cast<long long>(block) * r.kv_heads + head;
      __nv_bfloat16* src = qkv + static_cast<long long>(r.heads + task) * r.head_dim + (key ? at * 8 : at * 16);
      const int second = key ? half : 8;
      bf16x8 x[kRows], y[kRows];              // as they stand: rotated again for the codes, which costs less than the registers
      auto row_at = [&](int row0, int i) {
        const int row = row0 + i * step + sub;
        return sub < step && row < block_size ? row : -1;
      };
      auto load = [&](int row0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int row = row_at(row0, i), tok = row >= 0 ? row_of[row].x : -1;
          if (tok >= 0) {
            x[i] = load8(src + tok * r.row_stride);
            y[i] = load8(src + tok * r.row_stride + second);
          }
        }
      };
      // f(row, its token, the numbers in 32 bits) for each row that is written
      auto each = [&](int row0, auto&& f) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int row = row_at(row0, i);
          if (row < 0) continue;
          const int2 of = row_of[row];
          if (of.x < 0) continue;
          float a[8], b[8];
          unpack8(x[i], a);
          unpack8(y[i], b);
          if (key) {
            const long long table = static_cast<long long>(of.y) * half + at * 8;
            rotate8(a, b, cos_t + table, sin_t + table);
          }
          f(row, of.x, a, b);
        }
      };
      const bool once = block_size <= kRows * step;
      const float old = begun ? 0.f : fmaxf(*scale_at, 0.f);
      uint32_t most = 0u;
      for (int row0 = 0; row0 < block_size; row0 += kRows * step) {
        load(row0);
        if (key)
          each(row0, [&](int, int, const float (&a)[8], const float (&b)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, max(magnitude(a[j]), magnitude(b[j])));
          });
        else
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            const int row = row_at(row0, i);
            if (row >= 0 && row_of[row].x >= 0) most = max(most, max(magnitude(most_of(x[i])), magnitude(most_of(y[i]))));
          }
      }
      most = __reduce_max_sync(0xffffffffu, most);
      const bool finite = most < kInfinite;
      if (!finite) {                          // rare: once more without them
        most = 0u;
        for (int row0 = 0; row0 < block_size; row0 += kRows * step) {
          if (!once) load(row0);
          each(row0, [&](int, int, const float (&a)[8], const float (&b)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, max(finite_magnitude(a[j]), finite_magnitude(b[j])));
          });
        }
        most = __reduce_max_sync(0xffffffffu, most);
      }
      const float need = scale_for(most), scale = fmaxf(need, old);
      if (!begun && scale > old) {            // what stands in the block, in the new scale
        const float factor = old / scale;
        for (int i = lane * 8; i < block_size * r.head_dim; i += 256) {
          if (row_of[i / r.head_dim].x >= 0) continue;
          uint2 c = *reinterpret_cast<const uint2*>(codes + i);
          float f[8];
          unpack_e4m3x8(c, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] *= factor;
          *reinterpret_cast<uint2*>(codes + i) = pack_e4m3x8(f);
        }
      }
      const float inv = scale > 0.f ? 1.f / scale : 0.f;
      for (int row0 = 0; row0 < block_size; row0 += kRows * step) {
        if (!once) load(row0);
        each(row0, [&](int row, int tok, float (&a)[8], float (&b)[8]) {
          if (key) {
            __nv_bfloat16* dst = src + tok * r.row_stride;
            store8(dst, pack8(a));
            store8(dst + half, pack8(b));
          }
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            ptx::mul2(a[j], a[j + 1], a[j], a[j + 1], inv);
            ptx::mul2(b[j], b[j + 1], b[j], b[j + 1], inv);
          }
          if (!finite)                        // an infinity has no code, and no other number becomes one: inv is at most 2^126, and 0 beside zeros alone
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (!isfinite(a[j])) a[j] = NAN;
              if (!isfinite(b[j])) b[j] = NAN;
            }
          uint8_t* dst = codes + row * r.head_dim + (key ? at * 8 : at * 16);
          const uint2 c = pack_e4m3x8(a), d = pack_e4m3x8(b);
          if (key) {
            *reinterpret_cast<uint2*>(dst) = c;
            *reinterpret_cast<uint2*>(dst + half) = d;
          } else {
            *reinterpret_cast<uint4*>(dst) = make_uint4(c.x, c.y, d.x, d.y);
          }
        });
      }
      if (lane == 0) *scale_at = scale;
      __syncwarp();
    }
  }
}

static bool rope_rows_ok(const RopeRows& r) {
  return r.heads > 0 && r.kv_heads > 0 && r.tokens >= 0 && r.head_dim > 0 && r.head_dim % 16 == 0 && r.table_rows > 0 && r.row_stride % 8 == 0 &&
         r.row_stride >= static_cast<long long>(r.heads + 2 * r.kv_heads) * r.head_dim && aligned16(r.qkv, r.cos_t, r.sin_t);
}

}  // namespace llmctl

using namespace llmctl;

// Rotates q and k of `tokens` rows [heads | kv_heads | kv_heads] x head_dim (bf16) in place and writes k and v to the rows `slots` (int64; outside of
// the cache: not written) of caches [cache_rows, kv_heads, head_dim].  cos / sin: fp32 [table_rows, head_dim / 2]; positions: int32.
LLMCTL_API int llmctl_rope_kv_append(void* qkv, long long row_stride, int tokens, int heads, int kv_heads, int head_dim, const float* cos_t,
                                     const float* sin_t, int table_rows, const int* positions, const long long* slots, void* k_cache, void* v_cache,
                                     long long cache_rows, void* stream) {
  LLMCTL_BEGIN();
  const RopeRows r{static_cast<__nv_bfloat16*>(qkv), row_stride, tokens, heads, kv_heads, head_dim, cos_t, sin_t, table_rows, positions};
  LLMCTL_REQUIRE(rope_rows_ok(r) && cache_rows >= 0 && aligned16(k_cache, v_cache));
  if (tokens == 0) return 0;
  const long long per_token = static_cast<long long>(heads + 2 * kv_heads) * (head_dim / 16);
  LLMCTL_REQUIRE(per_token < (1 << 30));
  const long long most = (1 << 30) / per_token;              // tokens of a launch: its units are counted in 31 bits
  for (long long tok0 = 0; tok0 < tokens; tok0 += most) {
    const long long n = tokens - tok0 < most ? tokens - tok0 : most, total = n * per_token;
    long long ctas = (total + 255) / 256;
    if (ctas > kNumSMs * 16) ctas = kNumSMs * 16;
    LLMCTL_CHECK(launch_dependent(rope_kv_append_kernel, static_cast<int>(ctas), 256, 0, (cudaStream_t)stream, r, static_cast<uint32_t>(total),
                                  FastDiv(static_cast<uint32_t>(per_token)), FastDiv(head_dim / 16), slots, (__nv_bfloat16*)k_cache,
                                  (__nv_bfloat16*)v_cache, cache_rows, static_cast<int>(tok0)));
  }
  LLMCTL_RETURN_LAST();
}

// The same into caches [blocks, kv_heads, block_size, head_dim] of e4m3 codes with scales [blocks, kv_heads] (fp32): see the top of this file.
LLMCTL_API int llmctl_rope_kv_append_fp8(void* qkv, long long row_stride, int tokens, int heads, int kv_heads, int head_dim, const float* cos_t,
                                         const float* sin_t, int table_rows, const int* positions, const long long* slots, void* k_cache, void* v_cache,
                                         float* k_scale, float* v_scale, int blocks, int block_size, void* stream) {
  LLMCTL_BEGIN();
  using namespace append8;
  const RopeRows r{static_cast<__nv_bfloat16*>(qkv), row_stride, tokens, heads, kv_heads, head_dim, cos_t, sin_t, table_rows, positions};
  LLMCTL_REQUIRE(rope_rows_ok(r) && head_dim <= 512 && blocks >= 0 && block_size >= 1 && block_size <= kMaxBlock && aligned16(k_cache, v_cache));
  if (tokens == 0) return 0;
  const int window = tokens > 256 ? 16 : 1, windows = (tokens + window - 1) / window, most = (2 * kv_heads + kWarps - 1) / kWarps;
  int parts = (kParts + windows - 1) / windows;
  if (parts > most) parts = most;
  const long long per_token = static_cast<long long>(heads) * (head_dim / 16), units = per_token * tokens;
  LLMCTL_REQUIRE(units < (1LL << 30));
  const int q_ctas = static_cast<int>((units + kThreads * kUnits - 1) / (kThreads * kUnits));
  LLMCTL_CHECK(launch_dependent(rope_kv_append_fp8_kernel, windows * parts + q_ctas, kThreads, block_size * sizeof(int2), (cudaStream_t)stream, r, slots,
                                (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, blocks, block_size, window, windows, parts,
                                static_cast<uint32_t>(units), FastDiv(static_cast<uint32_t>(per_token)), FastDiv(head_dim / 16)));
  LLMCTL_RETURN_LAST();
}
