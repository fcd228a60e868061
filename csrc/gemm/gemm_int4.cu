// Entry points of the products with weights of 4 bits; which kernel a call takes; weights widened to bf16 for prompts.
// Reference: none (quantisation is an option of a stub command, llmctl/cli/commands/export.py:17).
#include "../common/dependent.cuh"
#include "../common/util.cuh"
#include "gemm_int4.h"

#include <cuda_fp16.h>

namespace llmctl {

// bf16 [halves * padded, K] of W [halves * rows, K / 2]: each number (q - 8) s rounded once, rows past the last of a half zeros.  A thread has 32 columns: 16 bytes in,
// 64 out.  Bound by what it writes: 22016 x 4096 38 us (5.9 TB/s).
__global__ void __launch_bounds__(256) int4_widen_kernel(const uint8_t* __restrict__ w, long long ldw, const __half* __restrict__ scale, long long lds, __nv_bfloat16* __restrict__ out,
                                                         int rows, int padded, int pieces, long long all) {
  wait_for_previous(w, scale, out);
  release_dependents();
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const int row = static_cast<int>(i / pieces), piece = static_cast<int>(i - static_cast<long long>(row) * pieces), half = row / padded, in = row - half * padded;
    uint4 words = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
    float s = 0.f;
    if (in < rows) {
      const long long from = static_cast<long long>(half) * rows + in;
      words = *reinterpret_cast<const uint4*>(w + from * ldw + piece * 16);
      s = __half2float(scale[from * lds + (piece >> 2)]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t v = reinterpret_cast<const uint32_t*>(&words)[j];
      float f[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) f[c] = static_cast<float>(static_cast<int>((v >> 4 * c) & 15u) - 8) * s;
      store8(out + i * 32 + j * 8, pack8(f));
    }
  }
}

namespace {
// Chunks of 8 tokens read the weights again, from L2; the tensor cores' kernel reads them once but has 6 us of start and merge.  us, chunks / tensor cores: 4096 x 4096 (8.4 MB)
// 16 tokens 8.0 / 9.4, 24 11.8 / 12.5, 32 14.1 / 12.8; gated 2048 -> 5632 (11.5 MB) 16 tokens 11.5 / 12.0, 24 16.8 / 15.0; 6144 rows of 2048 (6.3 MB) 24 tokens 9.3 / 11.4, 32
// 12.6 / 11.8; 2048 x 2048 64 tokens 8.9 / 16.0; 12288 x 4096 (25 MB) 9 tokens 18 / 15.6.
bool in_chunks(int tokens, long long matrix_rows, int K) { return tokens <= 8 || (tokens + 7) / 8 * (matrix_rows * (K / 2)) <= (24LL << 20); }
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
  const long long all = static_cast<long long>(padded) * halves * (K / 32);
  const int grid = static_cast<int>(min((all + 255) / 256, 8LL * kNumSMs));
  LLMCTL_CHECK(launch_dependent(int4_widen_kernel, grid, 256, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(w), ldw, static_cast<const __half*>(scale), lds,
                                static_cast<__nv_bfloat16*>(out), rows, padded, K / 32, all));
  return 0;
}
