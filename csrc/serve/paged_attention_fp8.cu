// Decode attention over a paged cache of 8 bits: one query token per sequence against e4m3 keys and values with a scale for each block and head, as
// rope_kv_append.cu writes them.
//
//   out[b, h, :] = sum_j p_j v_j / sum_j p_j,    p_j = exp(scale * q[b, h, :] . k_j),    k_j = sk[block(j)] * ck_j,   v_j = sv[block(j)] * cv_j
//
// over the tokens j < context_lens[b] of the blocks in the sequence's table; query head h reads head h / (heads / kv_heads) of the cache.  A sequence
// without tokens gets zeros.
//
// Blocks of a multiple of 8 tokens go to the tensor cores (paged_attention_fp8_t5.cu).  Of any other size: a warp takes every fourth token, a lane D / 32 dimensions of it; fp32 throughout
// (16 contexts of up to 4096, 32 heads of 128 in blocks of 12 tokens 380 us; there in blocks of 8 62).  Splits of the context are in both merged by a second kernel.
//
// Reference: none — the reference re-runs the model over the whole sequence (reference llmctl/serve/server.py:199-204).
#include "../common/dependent.cuh"
#include "../common/fp8.cuh"
#include "../common/util.cuh"

namespace llmctl {

// paged_attention_fp8_t5.cu
bool paged_attn_fp8_t5_ok(int head_dim, int block_size);
long long paged_attn_fp8_t5_scratch(int batch, int heads, int kv_heads, int head_dim, int limit, int runs);
int launch_paged_attn_fp8_t5(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                             const int* block_tables, int max_blocks, const int* context_lens, void* out, float* partial, int batch, int heads, int kv_heads,
                             int head_dim, int blocks, int block_size, int limit, int runs, float scale, cudaStream_t s);

namespace decode8 {
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
__device__ __forceinline__ void load_codes(const uint8_t* p, float (&f)[D / 32]) {
  if constexpr (D == 128) unpack_e4m3x4(*reinterpret_cast<const uint32_t*>(p), f);
  else {
    const float2 v = unpack_e4m3x2(*reinterpret_cast<const uint16_t*>(p));
    f[0] = v.x, f[1] = v.y;
  }
}
}  // namespace decode8

// Grid: (heads, splits, batch).  partial: [batch, heads, splits, D + 2] = {sum of p v, reference (log2), sum of p}.
template <int D>
__global__ void __launch_bounds__(128)
paged_attn_decode_fp8_kernel(const __nv_bfloat16* __restrict__ q, long long q_stride, const uint8_t* __restrict__ k_cache,
                             const uint8_t* __restrict__ v_cache, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                             const int* __restrict__ block_tables, int max_blocks, const int* __restrict__ context_lens,
                             float* __restrict__ partial, __nv_bfloat16* __restrict__ out, int blocks, int block_size, int group, int limit,
                             int tokens_per_split, float scale_log2) {
  using namespace decode8;
  constexpr int kDims = D / 32;
  __shared__ float s_acc[4][D], s_m[4], s_l[4];
  wait_for_previous(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, partial, out);
  release_dependents();
  const int head = blockIdx.x, split = blockIdx.y, b = blockIdx.z, heads = gridDim.x, nsplit = gridDim.y;
  const int kv_heads = heads / group, kv_head = head / group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ctx = min(context_lens[b], limit);
  const int t0 = split * tokens_per_split, t1 = min(ctx, t0 + tokens_per_split);
  const int* bt = block_tables + static_cast<long long>(b) * max_blocks;

  float qf[kDims], acc[kDims], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kDims; ++i) {
    qf[i] = __bfloat162float(q[b * q_stride + head * D + lane * kDims + i]);
    acc[i] = 0.f;
  }
  for (int t = t0 + warp; t < t1; t += 4) {
    const int block = bt[t / block_size];
    float s = NAN, k[kDims], v[kDims], sv = NAN;        // a block outside of the cache: no number instead of other memory
#pragma unroll
    for (int i = 0; i < kDims; ++i) k[i] = v[i] = 0.f;
    if (block >= 0 && block < blocks) {
      const long long at = static_cast<long long>(block) * kv_heads + kv_head;
      const long long row = (at * block_size + t % block_size) * D + lane * kDims;
      load_codes<D>(k_cache + row, k);
      load_codes<D>(v_cache + row, v);
      sv = v_scale[at];
      s = 0.f;
#pragma unroll
      for (int i = 0; i < kDims; ++i) s += qf[i] * k[i];
      s = warp_sum(s) * (k_scale[at] * scale_log2);
    }
    const float m_new = fmaxf(m, s), ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - ref), p = exp2f(s - ref);
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < kDims; ++i) acc[i] = acc[i] * alpha + p * (sv * v[i]);
    m = m_new;
  }
#pragma unroll
  for (int i = 0; i < kDims; ++i) s_acc[warp][lane * kDims + i] = acc[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float gm = -INFINITY, gl = 0.f, ga = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) gm = fmaxf(gm, s_m[i]);
    const float ref = gm == -INFINITY ? 0.f : gm;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = exp2f(s_m[i] - ref);
      gl += s_l[i] * w;
      ga += s_acc[i][threadIdx.x] * w;
    }
    const long long row = static_cast<long long>(b) * heads + head;
    if (nsplit == 1) {
      out[row * D + threadIdx.x] = __float2bfloat16(t1 > t0 ? ga / gl : 0.f);
    } else {
      float* dst = partial + (row * nsplit + split) * (D + 2);
      dst[threadIdx.x] = ga;
      if (threadIdx.x == 0) {
        dst[D] = gm;
        dst[D + 1] = gl;
      }
    }
  }
}

// One CTA per (head, sequence).  A split without tokens has a sum of 0 and no part in the reference.
template <int D>
__global__ void __launch_bounds__(D)
paged_attn_merge_fp8_kernel(const float* __restrict__ partial, __nv_bfloat16* __restrict__ out, int nsplit) {
  wait_for_previous(partial, out);
  release_dependents();
  const long long row = static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x;
  const float* p = partial + row * nsplit * (D + 2);
  float gm = -INFINITY, gl = 0.f, ga = 0.f;
  for (int s = 0; s < nsplit; ++s) gm = fmaxf(gm, p[s * (D + 2) + D]);
  const float ref = gm == -INFINITY ? 0.f : gm;
  for (int s = 0; s < nsplit; ++s) {
    const float w = exp2f(p[s * (D + 2) + D] - ref);
    gl += p[s * (D + 2) + D + 1] * w;
    ga += p[s * (D + 2) + threadIdx.x] * w;
  }
  out[row * D + threadIdx.x] = __float2bfloat16(gl == 0.f ? 0.f : ga / gl);
}

}  // namespace llmctl

using namespace llmctl;

static int decode8_limit(int max_blocks, int block_size, int max_context) {
  const long long room = static_cast<long long>(max_blocks) * block_size;
  return max_context < room ? max_context : static_cast<int>(room);
}
// Splits of a context where a block is not of whole boxes: some 8 CTAs to an SM, of 64 tokens and more.
static int decode8_splits(int batch, int heads, int limit, int splits) {
  if (splits > 0) return splits;
  const long long want = (8LL * kNumSMs + static_cast<long long>(batch) * heads - 1) / (static_cast<long long>(batch) * heads);
  const int most = limit / 64 < 256 ? limit / 64 : 256;
  return want < most ? static_cast<int>(want) : most > 1 ? most : 1;
}

// Number of fp32 scratch elements llmctl_paged_attn_decode_fp8 needs for a given launch.
LLMCTL_API long long llmctl_paged_attn_fp8_scratch_elems(int batch, int heads, int kv_heads, int head_dim, int max_blocks, int block_size, int max_context,
                                                         int num_splits) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || block_size <= 0) return 0;
  const int limit = decode8_limit(max_blocks, block_size, max_context);
  if (paged_attn_fp8_t5_ok(head_dim, block_size)) return paged_attn_fp8_t5_scratch(batch, heads, kv_heads, head_dim, limit, num_splits);
  const int splits = decode8_splits(batch, heads, limit, num_splits);
  return splits == 1 ? 0 : static_cast<long long>(batch) * heads * splits * (head_dim + 2);
}

// q: bf16 [batch, heads, head_dim], rows q_stride apart; caches [blocks, kv_heads, block_size, head_dim] e4m3, scales fp32 [blocks, kv_heads]; out: bf16
// [batch, heads, head_dim].  scratch: fp32 [llmctl_paged_attn_fp8_scratch_elems(...)] (may be null when that is 0).  num_splits: parts of a context, or (blocks
// of whole boxes) of the batch; 0: as many as fill the chip; 1: none is merged.
LLMCTL_API int llmctl_paged_attn_decode_fp8(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const float* k_scale,
                                            const float* v_scale, const int* block_tables, int max_blocks, const int* context_lens, void* out,
                                            float* scratch, int batch, int heads, int kv_heads, int head_dim, int blocks, int block_size,
                                            int max_context, int num_splits, float scale, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE((head_dim == 128 || head_dim == 64) && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && batch >= 0 && batch < 65536);
  LLMCTL_REQUIRE(num_splits >= 0 && num_splits < 65536 && block_size >= 1 && blocks >= 0 && max_blocks >= 0 && max_context >= 0);
  if (batch == 0) return 0;
  LLMCTL_REQUIRE(aligned16(k_cache, v_cache));
  cudaStream_t s = (cudaStream_t)stream;
  const int limit = decode8_limit(max_blocks, block_size, max_context);
  if (paged_attn_fp8_t5_ok(head_dim, block_size) && blocks > 0) {
    const int rc = launch_paged_attn_fp8_t5(q, q_stride, k_cache, v_cache, k_scale, v_scale, block_tables, max_blocks, context_lens, out, scratch, batch,
                                            heads, kv_heads, head_dim, blocks, block_size, limit, num_splits, scale, s);
    if (rc) LLMCTL_FAIL(rc, "decode over 8 bits");
    LLMCTL_RETURN_LAST();
  }
  // A cache without blocks, of whatever size they would have, has nothing to split: one part, which needs none of the scratch that the function above answers
  // for the kernel that this call does not take.
  const int splits = blocks == 0 ? 1 : decode8_splits(batch, heads, limit, num_splits), per = limit > 0 ? (limit - 1) / splits + 1 : 1;
  LLMCTL_REQUIRE(splits == 1 || scratch != nullptr);
  auto launch = [&](auto kern) {
    return launch_dependent(kern, dim3(heads, splits, batch), 128, 0, s, (const __nv_bfloat16*)q, q_stride, (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                            k_scale, v_scale, block_tables, max_blocks, context_lens, scratch, (__nv_bfloat16*)out, blocks, block_size, heads / kv_heads,
                            limit, per, scale * decode8::kLog2e);
  };
  LLMCTL_CHECK(head_dim == 128 ? launch(paged_attn_decode_fp8_kernel<128>) : launch(paged_attn_decode_fp8_kernel<64>));
  if (splits > 1) {
    if (head_dim == 128)
      LLMCTL_CHECK(launch_dependent(paged_attn_merge_fp8_kernel<128>, dim3(heads, batch), 128, 0, s, scratch, (__nv_bfloat16*)out, splits));
    else
      LLMCTL_CHECK(launch_dependent(paged_attn_merge_fp8_kernel<64>, dim3(heads, batch), 64, 0, s, scratch, (__nv_bfloat16*)out, splits));
  }
  LLMCTL_RETURN_LAST();
}
