// The decode attention of paged_attention_fp8.cu on the 5th-generation tensor cores, for blocks of a multiple of 8 tokens.
//
// A sequence's one token has only the query heads of a group to offer as rows, so the CACHE ROWS are the M side of both products, as they stand in the
// cache, in 8 bits:
//     S^T = K Q^T         128 tokens x N columns, over D                 (A: the key tile as it was loaded, K-major)
//     O^T = V^T P^T       D dimensions x N columns, over 128 tokens      (A: the value tile as it was loaded, M-major)
// kind::f8f6f4 wants 8-bit columns too.  A query head, and a row of weights, is therefore FOUR columns: the number rounded to e4m3 (4 significant
// bits), the rest times 16 rounded, its rest times 16, and so on: 16 bits of what they have, where bf16 has 8, over a range of 2^29.  The products of two
// e4m3 numbers are exact and the four columns are added in 32 bits.  N = 16 columns are four heads, 32 eight, 64 sixteen.
//
// The scales of keys multiply the scores.  Those of values are added to the exponent of a token's weight, w = 2^(s + log2 sv), which has a running reference of
// its own: M over s + log2 sv beside m over s, so that neither a block of tiny values nor one of large ones takes the bits of the others.
//     O = 2^(M - m) sum_j w_j cv_j / l,    w_j = 2^(s_j + log2 sv_j - M),    l = sum_j 2^(s_j - m)
// O of a tile is read from tensor memory and added up in registers, where the reference of the tiles before is caught up with.
//
//   warp 0      TMA producer: 128 tokens of keys and of values, a box for each block that they stand in, a ring of stages
//   warp 1      MMA issuer
//   warps 2-5   the columns of Q, then a token per thread: S^T -> P^T; a dimension per thread: O^T
//
// Every wait is bounded, as in latent_attention_t5.cu.
// Reference: none.
#include "../common/dependent.cuh"
#include "../common/fast_div.h"
#include "../common/fp8.cuh"
#include "../common/ptx.cuh"
#include "../common/tma_host.h"
#include "../common/util.cuh"
#include "../common/wait_status.h"

namespace llmctl {
using namespace ptx;

namespace dec8 {
constexpr int kTile = 128;                   // tokens
constexpr int kThreads = 192;
constexpr int kPieces = 4, kMaxStages = 8;
constexpr float kStep = 16.f;                // between the columns of a number
constexpr float kLog2e = 1.4426950408889634f;
constexpr int stage_bytes(int D) { return 2 * kTile * D; }
constexpr int fixed_smem(int D, int N) { return N * D + 2 * kTile * N + 1024; }       // Q, two of P, alignment

// Two numbers of at most 448 as columns: codes[i] holds piece i of both (the first in the low byte).
__device__ __forceinline__ void split2(float a, float b, uint32_t (&codes)[kPieces]) {
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    codes[i] = pack_e4m3x2(a, b);
    const float2 f = unpack_e4m3x2(codes[i]);
    a = (a - f.x) * kStep;
    b = (b - f.y) * kStep;
  }
}
// The columns of GP numbers, piece after piece, put together.
template <int GP>
__device__ __forceinline__ float joined(const uint32_t* c, int g) {
  float x = __uint_as_float(c[3 * GP + g]);
  x = fmaf(x, 1.f / kStep, __uint_as_float(c[2 * GP + g]));
  x = fmaf(x, 1.f / kStep, __uint_as_float(c[GP + g]));
  return fmaf(x, 1.f / kStep, __uint_as_float(c[g]));
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t* r) {
  if constexpr (N == 16) tmem_ld_x16(at, r);
  else if constexpr (N == 32) tmem_ld_x32(at, r);
  else {
    tmem_ld_x32(at, r);
    tmem_ld_x32(at + 32, r + 32);
  }
}
}  // namespace dec8

// Grid: (heads of the cache x groups of N / 4 query heads, splits, batch).  partial: as in paged_attention_fp8.cu.
template <int D, int N>
__global__ void __launch_bounds__(dec8::kThreads)
paged_attn_decode_fp8_t5_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* __restrict__ q,
                                long long q_stride, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                                const int* __restrict__ block_tables, int max_blocks, const int* __restrict__ context_lens, float* __restrict__ partial,
                                __nv_bfloat16* __restrict__ out, int blocks, int block_size, FastDiv by_block, int box_rows, int kv_heads, int group,
                                int limit, int tokens_per_split, int stages, float scale_log2, unsigned char* wait_byte) {
  using namespace dec8;
  constexpr int GP = N / kPieces, kStage = stage_bytes(D), kHalf = kTile * D;
  constexpr uint32_t kSwizzle = D == 128 ? 2 : 4, kEight = 8 * D;          // layout of the tiles, bytes of eight rows
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_q, bar_full[kMaxStages], bar_empty[kMaxStages], bar_s[2], bar_p[2], bar_o[2];
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;
  __shared__ float top[2][4][2 * GP];                                      // per softmax warp: the tile's largest s and s + log2 sv

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int q_at = stages * kStage, p_at = q_at + N * D;

  if (threadIdx.x == 0) {
    mbar_init(&bar_q, 4);
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], 4);
      mbar_init(&bar_o[i], 1);
    }
    abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 1) tmem_alloc<1>(&tmem_base_smem, 4 * N);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_smem, tO = tmem_base + 2 * N;
  wait_for_previous(q, k_scale, v_scale, block_tables, context_lens, partial, out);
  release_dependents();
  volatile int* abort = &abort_flag;

  const int b = blockIdx.z, split = blockIdx.y, nsplit = gridDim.y;
  const int kv_head = blockIdx.x % kv_heads, g0 = blockIdx.x / kv_heads * GP, ng = min(GP, group - g0), heads = kv_heads * group;
  const int head0 = kv_head * group + g0;
  const int ctx = min(context_lens[b], limit);
  const int t0 = split * tokens_per_split, t1 = min(ctx, t0 + tokens_per_split);
  const int nt = t1 > t0 ? (t1 - t0 + kTile - 1) / kTile : 0;
  const int* bt = block_tables + static_cast<long long>(b) * max_blocks;
  auto block_of = [&](int token, int& row) {
    uint32_t r;
    const uint32_t i = by_block.divide(static_cast<uint32_t>(token), r);
    row = static_cast<int>(r);
    return bt[i];
  };

  if (warp == 0) {
    // ------------------------------------ TMA producer: a lane per box ------------------------------------
    const int boxes = kTile / box_rows, all_rows = blocks * kv_heads * block_size;
    auto row_of = [&](int n) {                            // cache row of the lane's box, -1: none.  A block outside of the cache is filled with zeros
      const int token = t0 + n * kTile + lane * box_rows;
      if (lane >= boxes || n >= nt || token >= t1) return -1;
      int row;
      const int block = block_of(token, row);
      return block >= 0 && block < blocks ? (block * kv_heads + kv_head) * block_size + row : all_rows;
    };
    int row = row_of(0), loaded = 0;
    for (int n = 0; n < nt; ++n) {
      const int st = n % stages, next = row_of(n + 1);
      const bool given = n < stages || mbar_wait_bounded(&bar_empty[st], ((n / stages) & 1u) ^ 1u, abort);
      if (!__all_sync(0xffffffffu, given)) break;
      const int count = __popc(__ballot_sync(0xffffffffu, row >= 0));
      if (lane == 0) mbar_expect_tx(&bar_full[st], count * box_rows * D * 2);
      ++loaded;
      __syncwarp();
      if (row >= 0) {
        uint8_t* dst = smem + st * kStage + lane * box_rows * D;
        tma_load_2d(dst, &tmK, &bar_full[st], 0, row);
        tma_load_2d(dst + kHalf, &tmV, &bar_full[st], 0, row);
      }
      row = next;
    }
    // Copies still in flight when a wait ran out land before the CTA's shared memory is given back.
    if (*abort && lane == 0)
      for (int i = loaded > stages ? loaded - stages : 0; i < loaded; ++i) {
        int none = 0;
        mbar_wait_bounded(&bar_full[i % stages], (i / stages) & 1u, &none);
      }
  } else if (warp == 1) {
    // ------------------------------------ MMA issuer: whichever is there first, the next tile or the weights of this one ------------------------------------
    constexpr uint32_t id_s = make_idesc_e4m3(kTile, N, 0u, 0u);       // A, B K-major
    constexpr uint32_t id_o = make_idesc_e4m3(D, N, 1u, 1u);           // A, B MN-major
    if (nt > 0) mbar_wait_or_abort(&bar_q, 0u, abort);
    const long long since = clock64();
    for (int ns = 0, np = 0; np < nt;) {
      const int st = ns % stages, sp = np % stages;
      const bool tile = ns < nt && ns <= np + 1 && __any_sync(0xffffffffu, mbar_test(&bar_full[st], (ns / stages) & 1u));
      const bool weights = !tile && np < ns && __any_sync(0xffffffffu, mbar_test(&bar_p[np & 1], (np >> 1) & 1u));
      if (tile) {
        mbar_wait_or_abort(&bar_full[st], (ns / stages) & 1u, abort);
        __syncwarp();
        tc_fence_after();
        const uint64_t a = make_smem_desc(smem_base + st * kStage, 16, kEight, kSwizzle), bq = make_smem_desc(smem_base + q_at, 16, kEight, kSwizzle);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma_f8_ss(tmem_base + (ns & 1) * N, a + (k * 32 >> 4), bq + (k * 32 >> 4), id_s, k != 0 ? 1u : 0u);
          umma_commit<1>(&bar_s[ns & 1]);
        }
        ++ns;
      } else if (weights) {
        mbar_wait_or_abort(&bar_p[np & 1], (np >> 1) & 1u, abort);
        __syncwarp();
        tc_fence_after();
        const uint64_t a = make_smem_desc(smem_base + sp * kStage + kHalf, 16, kEight, kSwizzle);
        const uint64_t bp = make_smem_desc(smem_base + p_at + (np & 1) * kTile * N, 128, kTile * 16, 0);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kTile / 32; ++k) umma_f8_ss(tO + (np & 1) * N, a + (k * 32 * D >> 4), bp + (k * 512 >> 4), id_o, k != 0 ? 1u : 0u);
          umma_commit<1>(&bar_empty[sp]);
          umma_commit<1>(&bar_o[np & 1]);
        }
        ++np;
      } else {
        const bool late = clock64() - since > kBoundedWaitCycles;
        if (late) *abort = 1;
        if (__any_sync(0xffffffffu, late || *abort)) break;
      }
    }
  } else {
    // ------------------------------------ softmax warps ------------------------------------
    const int w = warp - 2, quad = warp & 3, t = quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int dim = D == 128 ? t : quad * 16 + lane;      // of O^T: 64 rows stand in 16 lanes of each quadrant
    const bool has_dim = D == 128 || lane < 16;
    const long long row0 = static_cast<long long>(b) * heads + head0;

    // scales of this thread's token, two tiles ahead in the block table
    auto block_at = [&](int n) {
      const int token = t0 + n * kTile + t;
      int row;
      return n < nt && token < t1 ? block_of(token, row) : 0;
    };
    auto scale_at = [&](const float* s, int block) { return block >= 0 && block < blocks ? s[static_cast<long long>(block) * kv_heads + kv_head] : NAN; };
    int block1 = block_at(1);
    float sk = 0.f, sv = 0.f;
    if (nt > 0) {
      const int block0 = block_at(0);
      sk = scale_at(k_scale, block0);
      sv = scale_at(v_scale, block0);
    }

    // Q: a row's largest number comes to stand in 128 .. 255, its four columns K-major, swizzled as TMA swizzles the tiles
    float factor[GP];
    {
      float x[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        x[g] = nt > 0 && t < D && g < ng ? __bfloat162float(q[b * q_stride + static_cast<long long>(head0 + g) * D + t]) : 0.f;
        if (!isfinite(x[g])) x[g] = NAN;                  // an infinity has no columns, and no scores that are numbers
      }
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float m = warp_max_all(fabsf(x[g]));
        if (lane == 0) top[0][w][g] = m;
      }
      named_bar_sync(1, 128);
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float m = fmaxf(fmaxf(top[0][0][g], top[0][1][g]), fmaxf(top[0][2][g], top[0][3][g]));
        const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23), 16), 254);           // biased; what is smaller than 2^-111 is 0 here
        x[g] *= __uint_as_float(static_cast<uint32_t>(max(261 - e, 1)) << 23);                  // 2^(7 - (e - 127))
        factor[g] = __uint_as_float(static_cast<uint32_t>(e - 7) << 23) * scale_log2;
      }
      named_bar_sync(1, 128);                             // top[0] is written again by the first tile
      uint8_t* qs = smem + q_at;
      if (t < D) {
        auto at = [&](int n) {                            // byte t of row n
          return D == 128 ? n * 128 + (((t >> 4) ^ (n & 7)) << 4) + (t & 15) : n * 64 + (((t >> 4) ^ ((n >> 1) & 3)) << 4) + (t & 15);
        };
#pragma unroll
        for (int g = 0; g < GP; g += 2) {
          uint32_t codes[kPieces];
          split2(x[g], x[g + 1], codes);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            qs[at(i * GP + g)] = static_cast<uint8_t>(codes[i]);
            qs[at(i * GP + g + 1)] = static_cast<uint8_t>(codes[i] >> 8);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q);
    }

    float m[GP], M[GP], l[GP], acc[GP], catch_up[GP];     // catch_up: from the reference of the tile before last to that of the last
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      m[g] = M[g] = -INFINITY;
      l[g] = acc[g] = 0.f;
    }
    auto add_tile = [&](int n) {
      mbar_wait_or_abort(&bar_o[n & 1], (n >> 1) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      uint32_t o[N];
      tmem_ld<N>(tO + (n & 1) * N + lane_off, o);
      tmem_ld_wait();
#pragma unroll
      for (int g = 0; g < GP; ++g) acc[g] = fmaf(acc[g], catch_up[g], joined<GP>(o, g));
    };
    for (int n = 0; n < nt; ++n) {
      const int block2 = block_at(n + 2);
      const float next_sk = n + 1 < nt ? scale_at(k_scale, block1) : 0.f, next_sv = n + 1 < nt ? scale_at(v_scale, block1) : 0.f;
      const int j = t0 + n * kTile + t;
      const bool seen = j < t1;
      const float lv = seen ? __log2f(sv) : 0.f;
      mbar_wait_or_abort(&bar_s[n & 1], (n >> 1) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      float s[GP];
      {
        uint32_t c[N];
        tmem_ld<N>(tmem_base + (n & 1) * N + lane_off, c);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < GP; ++g) s[g] = seen ? joined<GP>(c, g) * (sk * factor[g]) : -INFINITY;
      }
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float a = warp_max_all(s[g]), c = warp_max_all(s[g] + lv);
        if (lane == 0) {
          top[n & 1][w][g] = a;
          top[n & 1][w][GP + g] = c;
        }
      }
      named_bar_sync(1, 128);
      uint32_t codes[N / 4];                              // this token's row of P: N bytes, piece after piece
      float from[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        auto over = [&](int i) { return fmaxf(fmaxf(top[n & 1][0][i], top[n & 1][1][i]), fmaxf(top[n & 1][2][i], top[n & 1][3][i])); };
        const float m1 = fmaxf(m[g], over(g)), M1 = fmaxf(M[g], over(GP + g));
        const float ref = m1 == -INFINITY ? 0.f : m1, Ref = M1 == -INFINITY ? 0.f : M1;
        l[g] = fmaf(l[g], ex2_approx(m[g] - ref), ex2_approx(s[g] - ref));
        from[g] = ex2_approx(M[g] - Ref);
        m[g] = m1;
        M[g] = M1;
        s[g] = ex2_approx(s[g] + lv - Ref) * 256.f;
      }
#pragma unroll
      for (int i = 0; i < N / 4; ++i) codes[i] = 0u;
#pragma unroll
      for (int g = 0; g < GP; g += 2) {
        uint32_t two[kPieces];
        split2(s[g], s[g + 1], two);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) codes[(i * GP + g) / 4] |= two[i] << ((i * GP + g) % 4 * 8);
      }
      uint8_t* dst = smem + p_at + (n & 1) * kTile * N + t * 16;
#pragma unroll
      for (int i = 0; i < N / 16; ++i) *reinterpret_cast<uint4*>(dst + i * kTile * 16) = make_uint4(codes[4 * i], codes[4 * i + 1], codes[4 * i + 2], codes[4 * i + 3]);
      // Values past the last token: nothing that the cache holds there may meet a weight of zero.
      if (n == nt - 1 && !seen) {
        mbar_wait_or_abort(&bar_full[n % stages], (n / stages) & 1u, abort);
        uint8_t* row = smem + (n % stages) * kStage + kHalf + t * D;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *reinterpret_cast<uint4*>(row + i * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[n & 1]);
      if (n > 0) add_tile(n - 1);
#pragma unroll
      for (int g = 0; g < GP; ++g) catch_up[g] = from[g];
      sk = next_sk;
      sv = next_sv;
      block1 = block2;
    }
    if (nt > 0) add_tile(nt - 1);

    // ---- sums over the tokens, read-out ----
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      const float x = warp_sum(l[g]);
      if (lane == 0) top[nt & 1][w][g] = x;
    }
    named_bar_sync(1, 128);
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      if (g >= ng || !has_dim) continue;
      const float total = (top[nt & 1][0][g] + top[nt & 1][1][g]) + (top[nt & 1][2][g] + top[nt & 1][3][g]);
      const float o = acc[g] * (M[g] == -INFINITY ? 1.f / 256.f : exp2f(M[g] - m[g]) * (1.f / 256.f));
      if (nsplit > 1) {
        float* dst = partial + ((row0 + g) * nsplit + split) * (D + 2);
        dst[dim] = o;
        if (t == 0) {
          dst[D] = m[g];
          dst[D + 1] = total;
        }
      } else {
        out[(row0 + g) * D + dim] = __float2bfloat16(nt > 0 ? o / total : 0.f);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag) report_wait(wait_byte);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, 4 * N);
  }
}

bool paged_attn_fp8_t5_ok(int head_dim, int block_size) { return (head_dim == 64 || head_dim == 128) && block_size % 8 == 0; }

int launch_paged_attn_fp8_t5(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                             const int* block_tables, int max_blocks, const int* context_lens, void* out, float* partial, int batch, int heads, int kv_heads,
                             int head_dim, int blocks, int block_size, int limit, int tokens_per_split, int splits, float scale, cudaStream_t s) {
  using namespace dec8;
  int box_rows = 8;
  while (box_rows < kTile && block_size % (2 * box_rows) == 0) box_rows *= 2;
  const long long rows = static_cast<long long>(blocks) * kv_heads * block_size;
  if (rows == 0 || rows >= (1LL << 31) - kTile) return static_cast<int>(cudaErrorInvalidValue);
  CUtensorMap tmK, tmV;
  int rc = get_tmap_2d_bytes(&tmK, k_cache, rows, head_dim, head_dim, box_rows, head_dim);
  if (!rc) rc = get_tmap_2d_bytes(&tmV, v_cache, rows, head_dim, head_dim, box_rows, head_dim);
  if (rc) return rc;
  unsigned char* const wait_byte = wait_report(kWaitPagedFp8);
  if (wait_byte == nullptr) return static_cast<int>(cudaErrorMemoryAllocation);
  const int group = heads / kv_heads;
  auto launch = [&](auto kern, int N) {
    const int room = 110 * 1024, fit = (room - fixed_smem(head_dim, N)) / stage_bytes(head_dim), stages = fit < kMaxStages ? fit : kMaxStages;
    const int smem = fixed_smem(head_dim, N) + stages * stage_bytes(head_dim);
    const cudaError_t e = allow_smem(kern, smem);
    if (e != cudaSuccess) return e;
    const int parts = (group + N / kPieces - 1) / (N / kPieces);
    return launch_dependent(kern, dim3(kv_heads * parts, splits, batch), kThreads, smem, s, tmK, tmV, (const __nv_bfloat16*)q, q_stride, k_scale, v_scale,
                            block_tables, max_blocks, context_lens, splits > 1 ? partial : nullptr, (__nv_bfloat16*)out, blocks, block_size,
                            FastDiv(static_cast<uint32_t>(block_size)), box_rows, kv_heads, group, limit, tokens_per_split, stages,
                            scale * kLog2e, wait_byte);
  };
  if (head_dim == 128)
    return static_cast<int>(group <= 4 ? launch(paged_attn_decode_fp8_t5_kernel<128, 16>, 16)
                                       : group <= 8 ? launch(paged_attn_decode_fp8_t5_kernel<128, 32>, 32) : launch(paged_attn_decode_fp8_t5_kernel<128, 64>, 64));
  return static_cast<int>(group <= 4 ? launch(paged_attn_decode_fp8_t5_kernel<64, 16>, 16)
                                     : group <= 8 ? launch(paged_attn_decode_fp8_t5_kernel<64, 32>, 32) : launch(paged_attn_decode_fp8_t5_kernel<64, 64>, 64));
}

}  // namespace llmctl
