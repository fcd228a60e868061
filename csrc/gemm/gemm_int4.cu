// Entry points of the products with weights of 4 bits; which kernel a call takes; weights widened to bf16 for prompts.
// Reference: none (quantisation is an option of a stub command, llmctl/cli/commands/export.py:17).
#include "../common/dependent.cuh"
#include "../common/fast_div.h"
#include "../common/util.cuh"
#include "gemm_int4.h"

#include <cuda_fp16.h>

namespace llmctl {

// Operands of a prompt's product: x and the numbers (q - 8) s in fp16, each row brought to one range by a power of two, which the product's epilogue takes back.  bf16 would round
// (q - 8) s to 8 bits, as far off as the output's own rounding (1.4 times the error, 1.7 gated); in fp16 it is off by 2^-11 of itself at most and x, of 8 bits, is exact, both down to 2^-25 of what
// the row's largest is brought to, 2^14: 2^-39 of it, below the products' fp32.  Infinities and NaN stay what they are and have no part in the range.  A warp has a row of x, or up to
// 2048 columns of a row of weights (whose range it finds for itself, in the scales); 8 columns in a lane at a time, which a warp stores as 512 whole bytes.  Bound by what it writes: 12288 x 4096 and 1777 tokens 30.5 us (its 155 MB at the copy rate: 24), 22528 x 4096 and
// 4096 tokens 52 (45).  With the product behind it 146 and 518 (122 and 474 alone) with the chip's full clocks, 172 and 610 with what the power limit leaves to passes back to back; as bf16, without x, 146 and 544, under
// the power limit 6% less.
constexpr int kPiece = 256;          // words of 8 columns
__global__ void __launch_bounds__(256) int4_prepare_kernel(const __nv_bfloat16* x, long long ldx, int tokens, const uint8_t* w, long long ldw, const __half* scale, long long lds, int rows,
                                                           int padded, int K, FastDiv by_pieces, int all, __half* x_out, float* x_by, __half* w_out, float* w_by, long long w_by_half) {
  wait_for_previous(x_out, x_by, w_out, w_by);
  release_dependents();
  const int lane = threadIdx.x & 31, words = K / 8;
  auto largest = [](uint32_t bits, uint32_t none, uint32_t most) { return bits < none ? max(bits, most) : most; };
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += gridDim.x * 8) {
    if (i < tokens) {
      const uint4* from = reinterpret_cast<const uint4*>(x + i * ldx);
      uint32_t most = 0;
#pragma unroll 8
      for (int c = lane; c < words; c += 32) {
        const uint4 v = from[c];
        const uint32_t two[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) most = largest(two[k] & 0x7fffu, 0x7f80u, largest((two[k] >> 16) & 0x7fffu, 0x7f80u, most));
      }
      const int e = max(static_cast<int>(__reduce_max_sync(0xffffffffu, most) >> 7), 15);          // exponents of both factors stay within fp32's
      const float up = __uint_as_float(static_cast<uint32_t>(268 - e) << 23);
      if (lane == 0) x_by[i] = __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
      uint4* to = reinterpret_cast<uint4*>(x_out + static_cast<long long>(i) * K);
#pragma unroll 8
      for (int c = lane; c < words; c += 32) {
        const uint4 v = from[c];
        const uint32_t two[4] = {v.x, v.y, v.z, v.w};
        __half2 h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = __floats2half2_rn(__uint_as_float(two[k] << 16) * up, __uint_as_float(two[k] & 0xffff0000u) * up);
        to[c] = *reinterpret_cast<const uint4*>(h);
      }
      continue;
    }
    uint32_t piece;
    const int row = static_cast<int>(by_pieces.divide(i - tokens, piece)), half = row >= padded ? 1 : 0, in = row - half * padded, c0 = static_cast<int>(piece) * kPiece + lane, end = min(words, c0 - lane + kPiece);
    uint4* to = reinterpret_cast<uint4*>(w_out + static_cast<long long>(row) * K);
    float* by = w_by + half * w_by_half + in;
    if (in >= rows) {
      for (int c = c0; c < end; c += 32) to[c] = make_uint4(0u, 0u, 0u, 0u);
      if (c0 == 0) *by = 1.f;
      continue;
    }
    const long long at = static_cast<long long>(half) * rows + in;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(w + at * ldw);
    const __half* s = scale + at * lds;
    uint32_t now[kPiece / 32], most = 0;
    __half sc[kPiece / 32];
#pragma unroll
    for (int k = 0; k < kPiece / 32; ++k) {
      const int c = c0 + 32 * k;
      now[k] = c < end ? from[c] : 0u;
      sc[k] = c < end ? s[c >> 4] : __ushort_as_half(0);
    }
    for (int g = lane; g < words / 16; g += 32) most = largest(__half_as_ushort(s[g]) & 0x7fffu, 0x7c00u, most);
    const int e = max(static_cast<int>(__reduce_max_sync(0xffffffffu, most) >> 10), 1);
    const float up = __uint_as_float(static_cast<uint32_t>(153 - e) << 23);                         // the largest scale to 2^11, times 8
    if (c0 == 0) *by = __uint_as_float(static_cast<uint32_t>(e + 101) << 23);
#pragma unroll
    for (int k = 0; k < kPiece / 32; ++k) {
      const int c = c0 + 32 * k;
      if (c >= end) break;
      const __half2 one = __float2half2_rn(__half2float(sc[k]) * up);
      const uint32_t even = now[k] & 0x0f0f0f0fu, odd = (now[k] >> 4) & 0x0f0f0f0fu;
      const uint32_t lo = __byte_perm(even, odd, 0x5140), hi = __byte_perm(even, odd, 0x7362);       // columns 0 .. 3, 4 .. 7
      const uint32_t pair[4] = {__byte_perm(lo, 0x64646464u, 0x4140), __byte_perm(lo, 0x64646464u, 0x4342), __byte_perm(hi, 0x64646464u, 0x4140), __byte_perm(hi, 0x64646464u, 0x4342)};
      __half2 h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)                                                                   // 1024 + q less 1032, exact; one rounding
        h[j] = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&pair[j]), __floats2half2_rn(1032.f, 1032.f)), one);
      to[c] = *reinterpret_cast<const uint4*>(h);
    }
  }
}

namespace {
// Chunks of 8 tokens read the weights again, from L2; the tensor cores' kernel reads them once for 64 tokens but has some 5 us of start and merge.  us, chunks / tensor cores:
// 4096 x 4096 (8.4 MB) 16 tokens 8.0 / 8.0, 24 11.8 / 9.8; gated 2048 -> 5632 (11.5 MB) 12 tokens 11.2 / 10.9; 6144 rows of 2048 (6.3 MB) 24 tokens 9.3 / 11.0, 32 12.6 /
// 11.0; 2048 rows of 5632 (5.8 MB) 32 tokens 9.9 / 12.3, 48 14.5 / 14.7; 2048 x 2048 64 tokens 8.9 / 10.8; 12288 x 4096 (25 MB) 9 tokens 18 / 14.0.
bool in_chunks(int tokens, long long matrix_rows, int K) { return tokens <= 8 || (tokens + 7) / 8 * (matrix_rows * (K / 2)) <= (23LL << 20); }

// Tokens up to which the weights are read in 4 bits, once for 64 of them.  For more they are widened to fp16, and the time of the GEMM that follows hardly depends on the number
// of tokens up to 256.  us, in 4 bits / widened: many bytes or a long K, 32000 x 4096 190 tokens 95 / 116, 256 128 / 117; 2048 x 5632 190 26 / 30, 256 35 / 31; fewer, 12288 x 4096
// 100 36 / 45, 190 53 / 50; 4096 x 4096 100 19 / 23, 190 27 / 25; 5120 x 5120 100 27 / 31, 190 37 / 36; neither, 6144 x 2048 60 13 / 16, 65 22 / 16; gated 2048 -> 5632 65
// 29 / 21, 1024 -> 4096 65 19 / 14.  So few bytes that chunks of 8 tokens read them, 2048 x 2048 65 9 / 13, 96 16 / 13; gated 768 -> 2048 65 10.1 / 10.3, 96 13 / 10; 2304 x 768 65
// 6.5 / 7.8, 100 8.6 / 8.0.
int most_tokens(long long matrix_rows, int K) {
  const long long bytes = matrix_rows * (K / 2);
  return bytes >= (32LL << 20) || K > 5120 ? 192 : bytes >= (16LL << 20) || K >= 4096 ? 128 : bytes <= (2LL << 20) ? 72 : 64;
}
}  // namespace
}  // namespace llmctl

using namespace llmctl;

LLMCTL_API int llmctl_gemm_int4_tokens(long long matrix_rows, int K) { return most_tokens(matrix_rows, K); }

LLMCTL_API long long llmctl_gemm_int4_scratch_elems(int tokens, int rows, int K, int gated, int* tickets) {
  *tickets = 0;
  if (tokens <= 0 || rows <= 0 || K <= 0 || in_chunks(tokens, gated ? 2LL * rows : rows, K)) return 0;
  return gemm_int4_t5_scratch(tokens, rows, K / 128, gated != 0, tickets);
}

LLMCTL_API int llmctl_gemm_int4(const void* x, long long ldx, const void* w, long long ldw, const void* scale, long long lds, void* out, long long ldo, int tokens,
                                int rows, int K, int gated, float* partial, long long partial_elems, unsigned int* tickets, int n_tickets, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE(tokens >= 0 && tokens <= 512 && rows >= 0 && rows <= (1 << 28) && K > 0 && K % 128 == 0 && K <= (1 << 28));
  LLMCTL_REQUIRE(aligned16(x, w) && ldx >= K && ldx % 8 == 0 && ldw >= K / 2 && ldw % 16 == 0 && lds >= K / 128 && ldo >= rows);
  if (tokens == 0 || rows == 0) return 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (in_chunks(tokens, gated ? 2LL * rows : rows, K)) {
    LLMCTL_CHECK(gemm_int4_rows(x, ldx, w, ldw, scale, lds, out, ldo, tokens, rows, K / 128, gated != 0, s));
    return 0;
  }
  int want = 0;
  LLMCTL_REQUIRE(partial_elems >= gemm_int4_t5_scratch(tokens, rows, K / 128, gated != 0, &want) && n_tickets >= want);
  LLMCTL_REQUIRE(partial != nullptr && tickets != nullptr);
  LLMCTL_CHECK(gemm_int4_t5(x, ldx, w, ldw, scale, lds, out, ldo, tokens, rows, K / 128, gated != 0, partial, tickets, s));
  return 0;
}

LLMCTL_API int llmctl_int4_prepare(const void* x, long long ldx, int tokens, const void* w, long long ldw, const void* scale, long long lds, int rows, int padded, int halves, int K,
                                   void* x_out, float* x_by, void* w_out, float* w_by, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE(tokens > 0 && rows > 0 && padded >= rows && (halves == 1 || halves == 2) && K > 0 && K % 128 == 0 && static_cast<long long>(padded) * halves * ((K / 8 + kPiece - 1) / kPiece) + tokens < (1LL << 30));
  LLMCTL_REQUIRE(aligned16(x, w, x_out, w_out) && ldx >= K && ldx % 8 == 0 && ldw >= K / 2 && ldw % 16 == 0 && lds >= K / 128);
  const int pieces = (K / 8 + kPiece - 1) / kPiece, all = padded * halves * pieces + tokens;
  LLMCTL_CHECK(launch_dependent(int4_prepare_kernel, min((all + 7) / 8, 8 * kNumSMs), 256, 0, static_cast<cudaStream_t>(stream), static_cast<const __nv_bfloat16*>(x), ldx, tokens,
                                static_cast<const uint8_t*>(w), ldw, static_cast<const __half*>(scale), lds, rows, padded, K, FastDiv(pieces), all, static_cast<__half*>(x_out), x_by,
                                static_cast<__half*>(w_out), w_by, (padded + 63LL) / 64 * 64));
  return 0;
}
