// Products with weights of 4 bits: what the files of the operator share.  rows: of the output, half of W's where gated.
#pragma once
#include <cuda_runtime.h>

namespace llmctl {

// A few tokens (gemm_int4_rows.cu).
cudaError_t gemm_int4_rows(const void* x, long long ldx, const void* w, long long ldw, const void* scale, long long lds, void* out, long long ldo, int tokens, int rows,
                           int groups, bool gated, cudaStream_t s);
// More of them (gemm_int4_t5.cu).  partial: floats, and tickets: zero and left so, as many as gemm_int4_t5_scratch says.
long long gemm_int4_t5_scratch(int tokens, int rows, int groups, bool gated, int* tickets);
cudaError_t gemm_int4_t5(const void* x, long long ldx, const void* w, long long ldw, const void* scale, long long lds, void* out, long long ldo, int tokens, int rows,
                         int groups, bool gated, float* partial, unsigned int* tickets, cudaStream_t s);

}  // namespace llmctl
