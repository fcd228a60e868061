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
#include <type_traits>

#include "../common/dependent.cuh"
#include "../common/fast_div.h"
#include "../common/fp8.cuh"
#include "../common/mma_sync.cuh"
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

// The angles of eight pairs.
__device__ __forceinline__ void load_angles(float (&c)[8], float (&s)[8], const float* __restrict__ cos_row, const float* __restrict__ sin_row) {
  *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cos_row);
  *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(cos_row + 4);
  *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sin_row);
  *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(sin_row + 4);
}
// Eight pairs (a: from the first half, b: from the second) of one row, rotated.
__device__ __forceinline__ void rotate8(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {            // a c - b s and b c + a s, the products with s rounded by themselves
    float t0, t1, u0, u1;
    ptx::mul2v(t0, t1, b[j], b[j + 1], s[j], s[j + 1]);
    ptx::mul2v(u0, u1, a[j], a[j + 1], s[j], s[j + 1]);
    fma2vv(a[j], a[j + 1], c[j], c[j + 1], -t0, -t1);
    fma2vv(b[j], b[j + 1], c[j], c[j + 1], u0, u1);
  }
}
__device__ __forceinline__ void rotate8(float (&a)[8], float (&b)[8], const float* __restrict__ cos_row, const float* __restrict__ sin_row) {
  float c[8], s[8];
  load_angles(c, s, cos_row, sin_row);
  rotate8(a, b, c, s);
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
// 16 bits: a thread takes 16 numbers of a head, eight pairs of q and k or 16 neighbours of v.  Bound by the pass over the rows:
// 1777 tokens, 32 heads of 128 19.0 us, 5.4 TB/s.  (Two such pieces to a thread: more registers, fewer threads on the chip, slower.)
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
// which is left out where the token before goes to the same block (in a prompt, 15 of 16).  Windows of one token share their blocks' heads instead (a prompt
// of 200 tokens, 32 heads of 128 6.3 us, 19.2 where the first token's CTAs write alone; over 8 heads in blocks of 64 7.5 / 22.5).  Then a lane has one place in one row of the block for
// all heads, and keeps its token's angles; as many warps as the block's rows need write a head after the other: the largest rotated number, by
// all of them, the scale, the codes.  The next head's numbers are asked for beside that.  (A warp to a head's block had to read the angles anew for each
// row and head and rotate twice, for want of registers: 8000 tokens, 40 heads of 128 130 us, so 112.)  Blocks of more than twice the rows
// that 8 warps hold are read twice, by a warp to a head (8000 tokens, 40 heads of 128 in blocks of 64 104 us, of 128 175, of 256 207).  The other CTAs rotate q, four units to a thread.
//
// Prompts: 8000 tokens, 40 heads of 128 99 us, 5.0 TB/s (floor 75), 60000 of 32 heads 560 (5.3).  No unit is at its limit (DRAM 54% of its peak, 2.2 instructions a
// clock and SM, warps 36%).  A CTA's heads of keys
// take 3.3 thousand clocks each (10 KB read and written), those of values 2.0 (6 KB), and q the rest of the time at the same 18.5 bytes a clock and SM; finding a block's
// tokens and the first rows take 9 of a CTA's 60 thousand.  Decoded tokens by the chain slots - block's codes - maximum - codes: one 3.6 us, 64 with 32 heads 6.9.
// ---------------------------------------------------------------------------------------------
namespace append8 {
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnits = 4;                    // of q, to a thread
// Calls of so many tokens may be of as many sequences: CTAs to each token, of which those whose tokens go to one block share its heads.  us with windows of 16
// tokens / so: 400 decoded tokens, 32 heads of 128 45 / 16, over 8 42 / 8.6; a prompt of 400 8.8 / 11.1, over 8 5.5 / 6.9; 1000 decoded 68 / 36, a prompt 13.8 / 25.4.
constexpr int kFew = 512;
constexpr int kMaxBlock = 4096;
constexpr int kStages = 4;                   // heads under way (1: 8000 tokens, 40 heads of 128 142 us)
constexpr uint32_t kInfinite = 0x7f800000u;
// CTAs that write blocks: one wave of them, else two to a block, or one where that is several waves or little work for each.  us by CTAs to a block: 64 decoded
// tokens, 32 heads of 128 5: 6.6, 8: 8.1; 1000 tokens 6: 13.7, 8: 16.6, 4: 15.5; 4000 1: 49.6, 2: 46.5, 3: 46.6; 60000 1: 561, 2: 592; 12 heads of 64 4000 1:
// 13.4, 2: 14.8; 8000 1: 22.7, 2: 25.0; 60000 1: 139, 2: 177; 8000, 40 heads 1: 104, 2: 98.7, 3: 104.
constexpr int resident(int held) { return (held == 2 ? 2 : 3) * kNumSMs; }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The smallest power of two (of 2^-126 and up) under which a number of this magnitude is at most 448; 0 for zero.
__device__ __forceinline__ float scale_for(uint32_t most) {
  if (most == 0u) return 0.f;
  const int e = static_cast<int>(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}
// Of long prompts a kernel before this one marks which blocks each window of kMarked tokens writes to, in a table of 1024 bits by a hash of the
// block: who looks for a block's tokens then looks through the few windows that have its bit.  (All of the call's slots for each of its blocks
// are work in the square of its length.)  us without / with marks: 2100 tokens, 32 heads of
// 128 25.5 / 26.3, 4000 51.5 / 46.6, 8000 89.5 / 82.4, 60000 1350 / 575; 12 heads of 64 8.9 / 9.4, 19.2 / 14.8, 31.9 / 25.2, 624 / 177.
constexpr int kMarked = 256, kMarkWords = 32, kMarkedFrom = 3000;
__device__ __forceinline__ uint32_t mark_of(uint32_t block) { return block * 2654435761u >> 22; }
// 1 / scale, 0 for 0: exact for the powers of two that this file writes
__device__ __forceinline__ float inverse(float scale) {
  const uint32_t u = __float_as_uint(scale);
  if ((u & 0x7fffffu) == 0u && u >= 1u << 23 && u < 253u << 23) return __uint_as_float((254u << 23) - u);
  return scale > 0.f ? 1.f / scale : 0.f;
}
// Warps that write a block together: as many as the rows that are written need, a power of two.
__device__ __forceinline__ int warps_together(int rows, int step) {
  int w = 1;
  while (w < kWarps && w * step < rows) w *= 2;
  return w;
}
}  // namespace append8

namespace append8 {
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// A block of the cache and what is written to it.
struct Block {
  const RopeRows& r;
  const float *cos_t, *sin_t;
  const int* positions;
  uint8_t *k, *v;                             // codes and scales of its heads
  float *ks, *vs;
  const int *row_token, *row_list;            // as in the kernel
  int n, block_size;
  bool begun;
  // tasks: heads of keys, then of values
  __device__ __forceinline__ uint8_t* codes_of(int task) const {
    const int size = block_size * r.head_dim;
    return task < r.kv_heads ? k + task * size : v + (task - r.kv_heads) * size;
  }
  __device__ __forceinline__ float* scale_of(int task) const { return task < r.kv_heads ? ks + task : vs + (task - r.kv_heads); }
};
__device__ __forceinline__ void write_codes(uint8_t* dst, bool key, int at, int half, float (&a)[8], float (&b)[8], float inv) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    ptx::mul2(a[j], a[j + 1], a[j], a[j + 1], inv);
    ptx::mul2(b[j], b[j + 1], b[j], b[j + 1], inv);
  }
  const uint2 u = pack_e4m3x8(a), v = pack_e4m3x8(b);
  if (key) {
    *reinterpret_cast<uint2*>(dst + at * 8) = u;
    *reinterpret_cast<uint2*>(dst + at * 8 + half) = v;
  } else {
    *reinterpret_cast<uint4*>(dst + at * 16) = make_uint4(u.x, u.y, v.x, v.y);
  }
}
// What stands in the block, in its larger scale; by `threads` threads.
__device__ __forceinline__ void grow(const Block& b, uint8_t* codes, float factor, int thread, int threads) {
  for (int i = thread * 8; i < b.block_size * b.r.head_dim; i += threads * 8) {
    if (b.row_token[i / b.r.head_dim] >= 0) continue;
    float f[8];
    unpack_e4m3x8(*reinterpret_cast<const uint2*>(codes + i), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= factor;
    *reinterpret_cast<uint2*>(codes + i) = pack_e4m3x8(f);
  }
}
// A head's block by one warp, in two passes over its rows, of any number of them; what is not finite has no code but NaN.
__device__ __forceinline__ void write_alone(const Block& bk, int task) {
  const RopeRows& r = bk.r;
  const int lane = threadIdx.x & 31, per_row = r.head_dim >> 4, step = 32 / per_row, sub = lane / per_row, at = lane - sub * per_row, half = r.head_dim >> 1;
  const bool key = task < r.kv_heads;
  float* const scale_at = bk.scale_of(task);
  uint8_t* const codes = bk.codes_of(task);
  const float old = bk.begun ? 0.f : fmaxf(*scale_at, 0.f);
  auto each = [&](auto&& f) {                 // f(row, where the token's numbers stand, the numbers)
#pragma unroll 2
    for (int i = sub; i < bk.n; i += step) {
      if (sub >= step) break;
      const int row = bk.row_list[i], tok = bk.row_token[row];
      __nv_bfloat16* p = r.qkv + tok * r.row_stride + static_cast<long long>(r.heads + task) * r.head_dim + (key ? at * 8 : at * 16);
      float a[8], b[8];
      unpack8(load8(p), a);
      unpack8(load8(p + (key ? half : 8)), b);
      if (key) {
        const long long table = table_row(r, bk.positions, tok) + at * 8;
        rotate8(a, b, bk.cos_t + table, bk.sin_t + table);
      }
      f(row, p, a, b);
    }
  };
  uint32_t most = 0u;
  each([&](int, __nv_bfloat16*, float (&a)[8], float (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (isfinite(a[j])) most = max(most, __float_as_uint(fabsf(a[j])));
      if (isfinite(b[j])) most = max(most, __float_as_uint(fabsf(b[j])));
    }
  });
  const float scale = fmaxf(scale_for(__reduce_max_sync(0xffffffffu, most)), old), inv = inverse(scale);
  if (!bk.begun && scale > old) grow(bk, codes, old / scale, lane, 32);
  each([&](int row, __nv_bfloat16* p, float (&a)[8], float (&b)[8]) {
    if (key) {
      store8(p, pack8(a));
      store8(p + half, pack8(b));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {             // (no finite number becomes an infinity: inv is at most 2^126, and 0 beside zeros alone)
      if (!isfinite(a[j])) a[j] = NAN;
      if (!isfinite(b[j])) b[j] = NAN;
    }
    write_codes(codes + row * r.head_dim, key, at, half, a, b, inv);
  });
  if (lane == 0) *scale_at = scale;
  __syncwarp();
}
}  // namespace append8

__global__ void __launch_bounds__(append8::kMarked)
rope_kv_append_marks_kernel(const long long* __restrict__ slots, int tokens, long long rows, int block_size, uint32_t* __restrict__ marks) {
  using namespace append8;
  __shared__ uint32_t words[kMarkWords];
  wait_for_previous(slots, marks);
  release_dependents();
  if (threadIdx.x < kMarkWords) words[threadIdx.x] = 0u;
  __syncthreads();
  const long long i = static_cast<long long>(blockIdx.x) * kMarked + threadIdx.x, slot = i < tokens ? slots[i] : -1;
  if (slot >= 0 && slot < rows) {
    const uint32_t mark = mark_of(static_cast<uint32_t>(slot / block_size));
    atomicOr(&words[mark >> 5], 1u << (mark & 31u));
  }
  __syncthreads();
  if (threadIdx.x < kMarkWords) marks[static_cast<long long>(blockIdx.x) * kMarkWords + threadIdx.x] = words[threadIdx.x];
}

// kHeld: rows of a block that a lane has a place in (so many of 8 warps' are a block's at most), or 0: blocks of more.
template <int kHeld>
__global__ void __launch_bounds__(append8::kThreads, kHeld == 2 ? 2 : 3)
rope_kv_append_fp8_kernel(RopeRows r, const long long* __restrict__ slots, const uint32_t* __restrict__ marks, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
                          float* __restrict__ k_scale, float* __restrict__ v_scale, int blocks, int block_size, int window, int windows, int parts,
                          uint32_t q_units, FastDiv per_token, FastDiv per_head) {
  using namespace append8;
  extern __shared__ __align__(16) int row_token[];          // [block_size]: the token that a row of the block at hand is written from, or -1; then those rows
  __shared__ int ahead, others, twice, written;             // tokens of the block: before this one; but this one
  int* const row_list = row_token + (block_size + 3) / 4 * 4;          // (what follows both lies on a 16-byte boundary)
  __shared__ uint32_t warp_most[2][kWarps];
  __nv_bfloat16* qkv = r.qkv;
  const float *cos_t = r.cos_t, *sin_t = r.sin_t;
  const int* positions = r.positions;
  wait_for_previous(qkv, cos_t, sin_t, positions, slots, marks, k_cache, v_cache, k_scale, v_scale);
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
  const bool few = window == 1;               // one token, whatever its place in its block
  const int part0 = work / windows, parts0 = parts, t0 = (work - part0 * windows) * window, t1 = min(r.tokens, t0 + window);
  const long long rows = static_cast<long long>(blocks) * block_size;
  // heads of keys that no block's writer rotates: all of a token's, this part's share
  int part = part0;
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

  const int sub = lane / per_row, at = lane - sub * per_row, step = 32 / per_row;      // rows of a warp; lanes past them idle
  // Of the window's tokens (16 at most, a lane each): those without a row, and those that may be the first in their block.
  long long slot = -1, before = -1;
  if (t0 + lane < t1) {
    slot = slots[t0 + lane];
    if (t0 + lane > 0) before = slots[t0 + lane - 1];
  }
  const bool padded = slot < 0 || slot >= rows, behind = !padded && before >= 0 && before < rows && before / block_size == slot / block_size;
  const unsigned window_mask = t1 - t0 >= 32 ? ~0u : (1u << (t1 - t0)) - 1u;
  for (unsigned left = __ballot_sync(0xffffffffu, padded) & window_mask; left != 0u; left &= left - 1u) rotate_keys(t0 + __ffs(left) - 1);
  for (unsigned left = __ballot_sync(0xffffffffu, !padded && (few || !behind)) & window_mask; left != 0u; left &= left - 1u) {
    const int t = t0 + __ffs(left) - 1, block = static_cast<int>(__shfl_sync(0xffffffffu, slot, t - t0) / block_size);
    const long long lo = static_cast<long long>(block) * block_size, hi = lo + block_size;
    __syncthreads();                          // the rows of the block before have been read
    for (int i = threadIdx.x; i < block_size; i += kThreads) row_token[i] = -1;
    if (threadIdx.x == 0) {
      ahead = others = twice = written = 0;
    }
    __syncthreads();
    auto meet = [&](int i, long long s) {
      if (s >= lo && s < hi) {
        if (few && i != t) atomicAdd(&others, 1);
        if (i < t) atomicAdd(&ahead, 1);
        if (atomicMax(&row_token[s - lo], i) >= 0) twice = 1;
      }
    };
    const uint32_t mark = mark_of(static_cast<uint32_t>(block));
    const int groups_marked = (r.tokens - 1) / kMarked + 1;
    auto marked = [&](int g) { return (marks[static_cast<long long>(g) * kMarkWords + (mark >> 5)] >> (mark & 31u) & 1u) != 0u; };
    if (marks != nullptr) {
      for (int g0 = 0; g0 < groups_marked; g0 += kThreads) {
        const int g = g0 + lane * kWarps + warp;
        for (unsigned hit = __ballot_sync(0xffffffffu, g < groups_marked && marked(g)); hit != 0u; hit &= hit - 1u) {
          const int from = (g0 + (__ffs(hit) - 1) * kWarps + warp) * kMarked + lane;
          long long s[kMarked / 32];
#pragma unroll
          for (int k = 0; k < kMarked / 32; ++k) s[k] = from + k * 32 < r.tokens ? slots[from + k * 32] : -1;
#pragma unroll
          for (int k = 0; k < kMarked / 32; ++k) meet(from + k * 32, s[k]);
        }
      }
    } else {
      const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(slots) >> 3 & 1u);      // a slot before the first 16-byte boundary
      if (threadIdx.x == 0 && odd != 0) meet(0, slots[0]);
      const longlong2* two = reinterpret_cast<const longlong2*>(slots + odd);
      const int pairs = (r.tokens - odd) >> 1;
#pragma unroll 8
      for (int i = threadIdx.x; i < pairs; i += kThreads) {
        const longlong2 s = two[i];
        meet(odd + 2 * i, s.x);
        meet(odd + 2 * i + 1, s.y);
      }
      if (threadIdx.x == 0 && (r.tokens - odd) % 2 != 0) meet(r.tokens - 1, slots[r.tokens - 1]);
    }
    __syncthreads();
    if (few && others > 0) {                 // as many CTAs for each token: those of a block's tokens share its heads, as far as they go round
      const int members = others + 1, groups = kWarps / warps_together(members, step), most = min(parts0 * members, max((2 * r.kv_heads + groups - 1) / groups, parts0));
      part = ahead * parts0 + part0;
      parts = min(most, r.kv_heads);
      if (part >= parts) return;
    } else if (!few && ahead != 0) {
      continue;
    }
    for (int i = threadIdx.x; i < block_size; i += kThreads)
      if (row_token[i] >= 0) row_list[atomicAdd(&written, 1)] = i;          // in whatever order: rows do not depend on each other
    if (twice)
      for (int g = 0; g < groups_marked; ++g) {
        if (marks != nullptr && !marked(g)) continue;
        for (int i = g * kMarked; i < min(r.tokens, (g + 1) * kMarked); ++i) {
          const long long s = slots[i];
          if (s >= lo && s < hi && row_token[s - lo] != i) rotate_keys(i);
        }
      }
    __syncthreads();
    const int n = written, together = warps_together(n, step), groups = kWarps / together, group = warp / together, mine = warp - group * together;
    const bool begun = row_token[0] >= 0;

    const long long at_block = static_cast<long long>(block) * r.kv_heads;
    Block bk{r, cos_t, sin_t, positions, k_cache + at_block * block_size * r.head_dim, v_cache + at_block * block_size * r.head_dim, k_scale + at_block,
             v_scale + at_block, row_token, row_list, n, block_size, begun};
    const int tasks = 2 * r.kv_heads;
    if constexpr (kHeld == 0) {
      for (int task = part + warp * parts; task < tasks; task += kWarps * parts) write_alone(bk, task);
      continue;
    }

    // the lane's places: of the rows that are written one, or one of each half, and the tokens that they are written from, or -1
    constexpr int R = kHeld > 0 ? kHeld : 1;
    int row[R], tok[R];
    __nv_bfloat16* base[R];
    float c[R][8] = {}, s[R][8] = {};
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int i = (k * together + mine) * step + sub;
      row[k] = sub < step && i < n ? row_list[i] : 0;
      tok[k] = sub < step && i < n ? row_token[row[k]] : -1;
      base[k] = qkv + max(tok[k], 0) * r.row_stride + static_cast<long long>(r.heads) * r.head_dim;
      if (tok[k] >= 0) {
        const long long table = table_row(r, positions, tok[k]) + at * 8;
        load_angles(c[k], s[k], cos_t + table, sin_t + table);
      }
    }
    // The numbers of the heads to come, kStages - 1 of them, on their way into places that only the lane itself reads.
    uint8_t* const ring = reinterpret_cast<uint8_t*>(row_list + (block_size + 3) / 4 * 4) + warp * (kStages * R * 1024) + lane * 16;
    auto ask = [&](int task, int stage) {
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (task < tasks && tok[k] >= 0) {
          const __nv_bfloat16* p = base[k] + task * r.head_dim + (task < r.kv_heads ? at * 8 : at * 16);
          cp_async_16(ring + (stage * R + k) * 1024, p);
          cp_async_16(ring + (stage * R + k) * 1024 + 512, p + (task < r.kv_heads ? half : 8));
        }
      cp_async_commit();
    };
    const int first = part + group * parts, by = groups * parts;
    int turn = 0, turns = 0;
    uint32_t later = 0u;                      // a bit for each of the turns, 32 to a lane
    auto largest = [&](uint32_t most) {       // over the warps that write the block together
      most = __reduce_max_sync(0xffffffffu, most);
      if (together > 1) {
        uint32_t* const of = warp_most[turn++ & 1] + group * together;
        if (lane == 0) of[mine] = most;
        ptx::named_bar_sync(1 + group, together * 32);
        most = __reduce_max_sync(0xffffffffu, of[lane & (together - 1)]);
      }
      return most;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) ask(first + i * by, i);
    int stage = 0;
    auto one = [&](int task, auto of_keys) {
      constexpr bool key = of_keys.value;     // (known at compile time: what only keys need would be stepped over one by one for values)
      float* const scale_at = bk.scale_of(task);
      const float old = begun ? 0.f : fmaxf(*scale_at, 0.f);
      float a[R][8] = {}, b[R][8] = {}, x8 = 0.f;          // rows that are not there hold zeros
      ask(task + (kStages - 1) * by, (stage + kStages - 1) % kStages);
      cp_async_wait<kStages - 1>();
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (tok[k] >= 0) {
          unpack8(*reinterpret_cast<const bf16x8*>(ring + (stage * R + k) * 1024), a[k]);
          unpack8(*reinterpret_cast<const bf16x8*>(ring + (stage * R + k) * 1024 + 512), b[k]);
        }
        if (key) rotate8(a[k], b[k], c[k], s[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j) x8 = max_nan(x8, max_nan(fabsf(a[k][j]), fabsf(b[k][j])));
      }
      stage = (stage + 1) % kStages;
      const uint32_t most = largest(__float_as_uint(x8) & 0x7fffffffu);
      if (most >= kInfinite) {                // rare, and written behind the others
        if (lane == turns >> 5) later |= 1u << (turns & 31);
        return;
      }
      const float need = scale_for(most), scale = fmaxf(need, old), inv = inverse(scale);
      uint8_t* const codes = bk.codes_of(task);
      if (!begun && scale > old) grow(bk, codes, old / scale, mine * 32 + lane, together * 32);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (tok[k] < 0) continue;
        if (key) {
          __nv_bfloat16* dst = base[k] + task * r.head_dim + at * 8;
          store8(dst, pack8(a[k]));
          store8(dst + half, pack8(b[k]));
        }
        write_codes(codes + row[k] * r.head_dim, key, at, half, a[k], b[k], inv);
      }
      if (together == 1) __syncwarp();        // else they have met since they read it
      if (lane == 0 && mine == 0) *scale_at = scale;
    };
    int task = first;
    for (; task < r.kv_heads; task += by, ++turns) one(task, std::true_type());
    for (; task < tasks; task += by, ++turns) one(task, std::false_type());
    cp_async_wait<0>();
    if (mine == 0 && __any_sync(0xffffffffu, later != 0u))                 // heads with a number that is not finite
      for (int i = 0; i < turns; ++i)
        if (__shfl_sync(0xffffffffu, later, i >> 5) >> (i & 31) & 1u) write_alone(bk, first + i * by);
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

// Scratch of the call below in 32-bit words; 0: none.
LLMCTL_API long long llmctl_rope_kv_append_fp8_scratch_elems(int tokens) {
  using namespace append8;
  return tokens < kMarkedFrom ? 0 : static_cast<long long>((tokens - 1) / kMarked + 1) * kMarkWords;
}

// The same into caches [blocks, kv_heads, block_size, head_dim] of e4m3 codes with scales [blocks, kv_heads] (fp32): see the top of this file.  Without
// scratch (null) it does the same, in the square of the time.
LLMCTL_API int llmctl_rope_kv_append_fp8(void* qkv, long long row_stride, int tokens, int heads, int kv_heads, int head_dim, const float* cos_t,
                                         const float* sin_t, int table_rows, const int* positions, const long long* slots, void* k_cache, void* v_cache,
                                         float* k_scale, float* v_scale, int blocks, int block_size, void* scratch, void* stream) {
  LLMCTL_BEGIN();
  using namespace append8;
  const RopeRows r{static_cast<__nv_bfloat16*>(qkv), row_stride, tokens, heads, kv_heads, head_dim, cos_t, sin_t, table_rows, positions};
  LLMCTL_REQUIRE(rope_rows_ok(r) && head_dim <= 512 && kv_heads <= 512 && blocks >= 0 && block_size >= 1 && block_size <= kMaxBlock && aligned16(k_cache, v_cache));
  LLMCTL_REQUIRE(static_cast<long long>(blocks) * kv_heads < (1LL << 31) && static_cast<long long>(kv_heads) * block_size * head_dim < (1LL << 31));
  if (tokens == 0) return 0;
  const bool few = tokens <= kFew;
  const int window = few ? 1 : 16, windows = (tokens + window - 1) / window;
  // A block to each token where they may all be of other sequences, else to each block_size of them.
  const int writers = few ? tokens : (tokens + block_size - 1) / block_size, most = few ? (2 * kv_heads + kWarps - 1) / kWarps : kv_heads;
  const int held = (block_size - 1) / (kWarps * (32 / (head_dim / 16))) + 1;          // rows to a lane
  int parts = writers <= resident(held) / 2 ? resident(held) / writers : writers >= 4 * resident(held) || kv_heads <= 2 * kWarps ? 1 : 2;
  if (parts > most) parts = most;
  const long long per_token = static_cast<long long>(heads) * (head_dim / 16), units = per_token * tokens;
  LLMCTL_REQUIRE(units < (1LL << 30));
  const int q_ctas = static_cast<int>((units + kThreads * kUnits - 1) / (kThreads * kUnits));
  const int smem = (block_size + 3) / 4 * 4 * 2 * static_cast<int>(sizeof(int)) + (held <= 2 ? kWarps * kStages * held * 1024 : 0);
  auto kern = held == 1 ? rope_kv_append_fp8_kernel<1> : held == 2 ? rope_kv_append_fp8_kernel<2> : rope_kv_append_fp8_kernel<0>;
  const cudaError_t e = allow_smem(kern, smem);
  if (e != cudaSuccess) LLMCTL_FAIL(e, "shared memory");
  const uint32_t* marks = tokens < kMarkedFrom ? nullptr : static_cast<const uint32_t*>(scratch);
  if (marks != nullptr)
    LLMCTL_CHECK(launch_dependent(rope_kv_append_marks_kernel, (tokens - 1) / kMarked + 1, kMarked, 0, (cudaStream_t)stream, slots, tokens,
                                  static_cast<long long>(blocks) * block_size, block_size, static_cast<uint32_t*>(scratch)));
  LLMCTL_CHECK(launch_dependent(kern, windows * parts + q_ctas, kThreads, smem, (cudaStream_t)stream, r, slots, marks,
                                (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, blocks, block_size, window, windows, parts,
                                static_cast<uint32_t>(units), FastDiv(static_cast<uint32_t>(per_token)), FastDiv(head_dim / 16)));
  LLMCTL_RETURN_LAST();
}
