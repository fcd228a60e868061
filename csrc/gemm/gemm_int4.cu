// Entry points of the products with weights of 4 bits; which kernel a call takes; weights widened to bf16 for prompts.
// Reference: none (quantisation is an option of a stub command, llmctl/cli/commands/export.py:17).
#include "../common/dependent.cuh"
#include "../common/fast_div.h"
#include "../common/util.cuh"
#include "gemm_int4.h"

#include <cuda_fp16.h>

namespace llmctl {

// bf16 [halves * padded, K] of W [halves * rows, K / 2]: each number (q - 8) s rounded once, rows past the last of a half zeros.  A thread has 8 columns of a row at a time, 4
// bytes in and 16 out.  The whole number n = q - 8 is exact in bf16 (128 + q less 136), and s = s1 + s0 with 8 and at most 3 significant bits, so that n s0 is exact and
// fma(n, s1, n s0) the product rounded once.  Bound by what it writes.
__global__ void __launch_bounds__(256) int4_widen_kernel(const uint8_t* w, long long ldw, const __half* scale, long long lds, __nv_bfloat16* out, int rows, int padded, FastDiv by_words,
                                                         int all) {
  wait_for_previous(w, scale, out);
  release_dependents();
  const int stride = gridDim.x * 256;
  for (long long i0 = blockIdx.x * 256 + threadIdx.x; i0 < all; i0 += 4LL * stride) {
    uint32_t words[4];
    float s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long i = i0 + static_cast<long long>(k) * stride;
      words[k] = 0x88888888u;
      s[k] = 0.f;
      if (i >= all) continue;
      uint32_t word;
      const int row = static_cast<int>(by_words.divide(static_cast<uint32_t>(i), word)), half = row >= padded ? 1 : 0, in = row - half * padded;
      if (in >= rows) continue;
      const long long from = static_cast<long long>(half) * rows + in;
      words[k] = *reinterpret_cast<const uint32_t*>(w + from * ldw + word * 4);
      s[k] = __half2float(scale[from * lds + (word >> 4)]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long i = i0 + static_cast<long long>(k) * stride;
      if (i >= all) continue;
      const __nv_bfloat16 high = __float2bfloat16(s[k]);
      const float rest = s[k] - __bfloat162float(high);
      const __nv_bfloat162 s1 = __bfloat162bfloat162(high), s0 = __bfloat162bfloat162(__float2bfloat16(fabsf(s[k]) < INFINITY ? rest : 0.f));
      const uint32_t even = words[k] & 0x0f0f0f0fu, odd = (words[k] >> 4) & 0x0f0f0f0fu;
      const uint32_t lo = __byte_perm(even, odd, 0x5140), hi = __byte_perm(even, odd, 0x7362);             // columns 0 .. 3, 4 .. 7
      const uint32_t pair[4] = {__byte_perm(lo, 0x43434343u, 0x4140), __byte_perm(lo, 0x43434343u, 0x4342), __byte_perm(hi, 0x43434343u, 0x4140), __byte_perm(hi, 0x43434343u, 0x4342)};
      bf16x8 r;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const __nv_bfloat162 n = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair[c]), __floats2bfloat162_rn(136.f, 136.f));
        r.v[c] = __hfma2(n, s1, __hmul2(n, s0));
      }
      store8(out + i * 8, r);
    }
  }
}

namespace {
// Chunks of 8 tokens read the weights again, from L2; the tensor cores' kernel reads them once for 64 tokens but has some 5 us of start and merge.  us, chunks / tensor cores:
// 4096 x 4096 (8.4 MB) 16 tokens 8.0 / 8.0, 24 11.8 / 9.8; gated 2048 -> 5632 (11.5 MB) 12 tokens 11.2 / 10.9; 6144 rows of 2048 (6.3 MB) 24 tokens 9.3 / 11.0, 32 12.6 /
// 11.0; 2048 rows of 5632 (5.8 MB) 32 tokens 9.9 / 12.3, 48 14.5 / 14.7; 2048 x 2048 64 tokens 8.9 / 10.8; 12288 x 4096 (25 MB) 9 tokens 18 / 14.0.
bool in_chunks(int tokens, long long matrix_rows, int K) { return tokens <= 8 || (tokens + 7) / 8 * (matrix_rows * (K / 2)) <= (23LL << 20); }
}  // namespace
}  // namespace llmctl

using namespace llmctl;

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

LLMCTL_API int llmctl_int4_widen(const void* w, long long ldw, const void* scale, long long lds, void* out, int rows, int padded, int halves, int K, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE(rows > 0 && padded >= rows && (halves == 1 || halves == 2) && K > 0 && K % 128 == 0 && static_cast<long long>(padded) * halves < (1LL << 31));
  LLMCTL_REQUIRE(aligned16(w, out) && ldw >= K / 2 && ldw % 16 == 0 && lds >= K / 128);
  const long long all = static_cast<long long>(padded) * halves * (K / 8);
  LLMCTL_REQUIRE(all < (1LL << 31));
  const int grid = static_cast<int>(min((all + 1023) / 1024, 8LL * kNumSMs));
  LLMCTL_CHECK(launch_dependent(int4_widen_kernel, grid, 256, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(w), ldw, static_cast<const __half*>(scale), lds,
                                static_cast<__nv_bfloat16*>(out), rows, padded, FastDiv(K / 8), static_cast<int>(all)));
  return 0;
}
