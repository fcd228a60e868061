// Products of a few token rows with weights of 4 bits and group scales, as the `int4` quantiser writes them:
//     y[t, n] = sum_g s[n, g] sum_{k in g} x[t, k] (q[n, k] - 8)        g: 128 columns of K
// W is [N, K / 2] bytes, column 2i in the low half of byte i and 2i + 1 in the high one; s is fp16 [N, K / 128].  GATED: N = 2F rows, gate rows first, and
// the output is silu(gate) * up, [T, F].
//
// Bound by the pass over the weights, half a byte each, and next to it by the instructions that widen them.  They go from memory to the registers of
// the lane that multiplies them: weight rows are the M side of mma.m16n8k16, and since the order of K within a group is free (the same for both
// operands), a lane's four 8-column words of a row serve as its fragments without any exchange: a quad reads the 64 bytes of a row's group, 16 to a lane.
// (0x4300 | q is 128 + q in bf16, and two columns four apart of a word stand in the halves of a register as they come; one packed subtraction of 136
// leaves q - 8, exactly.)  Products and sums of a group are those of the whole numbers q - 8 with x, in 32 bits; the scale multiplies a group's sum in 32
// bits, so nothing is rounded before the output.
//
// A CTA has one or two tiles of 16 rows and 8 tokens, each of its 8 warps every eighth group of them; they add up through shared memory.  Further chunks of
// 8 tokens are CTAs of their own, which find the weights in L2 (16 tokens as two chunks, 4096 x 4096: 8.0 us; as 16 columns of the products 9.5).  us, weights not in
// L2 (a kernel that only reads them / this one, 1 and 8 tokens): 4096 x 4096 3.1 / 5.0, 5.6; 4096 rows of 11008 5.4 / 10.4, 11.7; 12288 x 4096 5.7 / 11.2, 12.2;
// 32000 x 4096 11.3 / 22.5, 24.3.
// Reference: none.
#include "../common/dependent.cuh"
#include "../common/mma_sync.cuh"
#include "../common/ptx.cuh"
#include "../common/util.cuh"
#include "gemm_int4.h"

#include <cuda_fp16.h>

namespace llmctl {
using namespace ptx;

namespace {
constexpr int kWarps = 8, kTokens = 8;

// Eight columns of a row as four pairs (k, k + 4) of whole numbers in bf16.
__device__ __forceinline__ void widen(uint32_t word, uint32_t (&pair)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = ((word >> 4 * i) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __floats2bfloat162_rn(136.f, 136.f));
    pair[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

struct Int4Args {
  const __nv_bfloat16* x;
  const uint8_t* w;
  const __half* scale;
  __nv_bfloat16* out;
  long long ldx, ldw, lds, ldo;
  int tokens, rows, groups;        // rows: of the output (F where gated)
};
}  // namespace

// Grid: row tiles x chunks of 8 tokens.
template <int MT, bool GATED>
__global__ void __launch_bounds__(32 * kWarps, 2) gemm_int4_rows_kernel(Int4Args a) {
  constexpr int kTileRows = 16 * MT, kOutRows = GATED ? kTileRows / 2 : kTileRows, kPitch = kTileRows + 4, kSums = kPitch * kTokens;
  __shared__ float red[kWarps * kSums];      // [warp][token][row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * kOutRows, token0 = blockIdx.y * kTokens, step = kWarps, first = warp;

  // Row i of the tile: a gated tile of 16 rows has 8 gate rows and the 8 up rows that go with them.  Rows past the last read the last one's weights; what
  // they give is not written.
  const uint8_t* at[MT][2];
  const __half* sc[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long row = min(row0 + (GATED ? m * 8 : m * 16 + h * 8) + g, a.rows - 1) + (GATED && h ? a.rows : 0);
      at[m][h] = a.w + row * a.ldw + first * 64LL + t * 16;
      sc[m][h] = a.scale + row * a.lds + first;
      if (first < a.groups) asm volatile("prefetch.global.L2 [%0];" ::"l"(at[m][h]));
    }
  const bool there = token0 + g < a.tokens;
  const __nv_bfloat16* xp = a.x + (token0 + g) * a.ldx + first * 128 + t * 32;
  wait_for_previous(a.out);
  release_dependents();

  float total[MT][4] = {};
  uint4 next[MT][2], xn[4];
  __half next_s[MT][2];
  auto fetch = [&] {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        next[m][h] = ld_nc_v4(at[m][h]);
        next_s[m][h] = *sc[m][h];
        at[m][h] += step * 64;
        sc[m][h] += step;
      }
  };
  auto fetch_x = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i) xn[i] = there ? *reinterpret_cast<const uint4*>(xp + i * 8) : make_uint4(0, 0, 0, 0);
    xp += step * 128;
  };
  if (first < a.groups) {
    fetch();
    fetch_x();
  }
  for (int group = first; group < a.groups; group += step) {
    uint4 words[MT][2], xs[4];
    float s[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        words[m][h] = next[m][h];
        s[m][h] = __half2float(next_s[m][h]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) xs[i] = xn[i];
    if (group + step < a.groups) {
      fetch();
      fetch_x();
    }
    float part[2][MT][4] = {};           // two sums: half the chain of products that wait for one another
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = xs[i];                 // the columns, put into the pairs in which the weights come
      const uint32_t b[4] = {__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632)};
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t lo[4], hi[4];
        widen(reinterpret_cast<const uint32_t*>(&words[m][0])[i], lo);
        widen(reinterpret_cast<const uint32_t*>(&words[m][1])[i], hi);
        const uint32_t f0[4] = {lo[0], hi[0], lo[1], hi[1]}, f1[4] = {lo[2], hi[2], lo[3], hi[3]};
        mma_bf16_16816(part[0][m], f0, b[0], b[1]);
        mma_bf16_16816(part[1][m], f1, b[2], b[3]);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) total[m][c] = fmaf(s[m][c >> 1], part[0][m][c] + part[1][m][c], total[m][c]);
  }

#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < 4; ++c) red[warp * kSums + (2 * t + (c & 1)) * kPitch + m * 16 + (c >> 1) * 8 + g] = total[m][c];
  __syncthreads();
  auto joined = [&](int i) {                 // of the warps, in their order
    float v = red[i];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v += red[w * kSums + i];
    return v;
  };
  for (int i = threadIdx.x; i < kOutRows * min(a.tokens - token0, kTokens); i += 32 * kWarps) {
    const int token = i / kOutRows, row = i % kOutRows, at_sum = token * kPitch + (GATED ? (row >> 3) * 16 + (row & 7) : row);
    if (row0 + row >= a.rows) continue;
    float v = joined(at_sum);
    if constexpr (GATED) v = v * __fdividef(1.f, 1.f + __expf(-v)) * joined(at_sum + 8);
    a.out[(token0 + token) * a.ldo + row0 + row] = __float2bfloat16(v);
  }
}

cudaError_t gemm_int4_rows(const void* x, long long ldx, const void* w, long long ldw, const void* scale, long long lds, void* out, long long ldo, int tokens, int rows,
                           int groups, bool gated, cudaStream_t s) {
  const Int4Args a = {static_cast<const __nv_bfloat16*>(x), static_cast<const uint8_t*>(w), static_cast<const __half*>(scale), static_cast<__nv_bfloat16*>(out),
                      ldx, ldw, lds, ldo, tokens, rows, groups};
  const int chunks = (tokens + kTokens - 1) / kTokens;
  auto tiles = [&](int mt) { return static_cast<unsigned>((rows + (gated ? 8 : 16) * mt - 1) / ((gated ? 8 : 16) * mt)); };
  // Two tiles to a CTA, for which a token's columns are put in order once, as soon as that leaves no SM without a CTA.  us, one / two tiles, 8 tokens: 2304 rows of 768
  // 2.0 / 2.3 (72 CTAs of two), 4096 x 4096 5.6 / 6.3 (128), 6144 rows of 2048 5.7 / 5.1 (192), 12288 x 4096 14.1 / 12.2 (384); 16 and 24 tokens, 2048 x 2048 3.6 / 3.9
  // (128), 5.3 / 5.1 (192).
  const bool two = static_cast<long long>(tiles(2)) * chunks > kNumSMs;
  const auto kernel = gated ? (two ? gemm_int4_rows_kernel<2, true> : gemm_int4_rows_kernel<1, true>) : (two ? gemm_int4_rows_kernel<2, false> : gemm_int4_rows_kernel<1, false>);
  return launch_dependent(kernel, dim3(tiles(two ? 2 : 1), chunks), 32 * kWarps, 0, s, a);
}

}  // namespace llmctl
