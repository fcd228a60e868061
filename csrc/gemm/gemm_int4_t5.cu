// Products of tokens with weights of 4 bits and group scales on the 5th-generation tensor cores:
//     y[t, n] = sum_g s[n, g] sum_{k in g} x[t, k] (q[n, k] - 8)        g: 128 columns of K
// W is [N, K / 2] bytes, column 2i in the low half of byte i and 2i + 1 in the high one; s is fp16 [N, K / 128].  GATED: N = 2F rows, gate rows first, and
// the output is silu(gate) * up, [T, F].
//
// Weight rows are the M side: a unit of work is 128 of them over two groups, 16 KB of weights (rows of 64 bytes, of one group, came at three quarters of the
// rate), against a chunk of P tokens.
//   D_g = A_g X_g^T       128 rows x P tokens, over 128 columns       (A: the whole numbers q - 8, exact in bf16, in tensor memory; B: x as it is, K-major)
// D_g leaves tensor memory after each group, and its rows are multiplied by their scales and added up in 32 bits, so that nothing is rounded before the
// output.  For that the whole numbers need no scale of their own: 0x4300 | q is 128 + q in bf16, less 136: 13 instructions for 8 columns.
//
//   1 warp      TMA producer of weights and of tokens, a ring of stages each
//   2 warps     MMA issuers, of a unit's first and of its second group: 8 products each (one warp's issuing took 400 clocks for a group)
//   8           a row and up to 32 tokens per thread: D_g times its scale into the row's sums; outputs.  Up to 32 tokens the first four look at a unit's first group and the
//               others at its second, above that each at half of the tokens
//   12          a row and a group per thread: from shared memory, widened, to tensor memory; four warps to every third group
//
// The work is one row of units, tile after tile, and the CTAs take equal runs of it, whatever the sizes (4096 rows are 32 tiles, for 148 SMs).  A tile that
// more than one CTA has a part of is put together by the last of them to come, which finds the others' sums in memory and adds all up in the order of the
// CTAs: the result does not depend on which that is, and nobody waits.
//
// us, weights not in L2 (a kernel that only reads them / this one): 4096 rows of 11008, 16 tokens 5.4 / 13.5, 32 16.5; 12288 x 4096, 16 tokens 5.7 / 14.0; 15360 x 5120, 61 tokens
// 7.6 / 23.3; 32000 x 4096, 16 tokens 11.3 / 24.8; gated 2048 -> 5632, 32 tokens 3.4 / 13.3 (14.8 with
// IEEE quotients, whose code, run once by each warp, comes from memory).  Bound by what a unit passes through between the barriers (bytes, whole numbers, products, scaled sums, 1 us
// each way in) and by its ends: 3 us until the first products, 2 to 3 for the tiles in parts.  The tensor cores have 6% (16 tokens) to 21% (64) to do.
// Reference: none.
#include "../common/dependent.cuh"
#include "../common/ptx.cuh"
#include "../common/tma_host.h"
#include "../common/util.cuh"
#include "../common/wait_status.h"
#include "gemm_int4.h"

#include <cuda_fp16.h>

namespace llmctl {
using namespace ptx;

namespace int4t5 {
constexpr int kRows = 128, kUnitBytes = kRows * 128;
// A barrier's phases are told by their parity, so that whoever waits at a stage has to wait for each of its phases: a stage of A belongs to one set of widening warps
// and to one issuer, one of D to one issuer, one of W to the same sets each time around.  The rings are multiples of those.
constexpr int kRingW = 6, kRingA = 6;
constexpr int ring_d(int P) { return P <= 32 ? 4 : 2; }
constexpr int ring_x(int P) { return P <= 32 ? 6 : 3; }
constexpr int kSumAt = 3, kSumWarps = 8, kWidenAt = kSumAt + kSumWarps, kSets = 3, kThreads = 32 * (kWidenAt + 4 * kSets);
constexpr bool by_group(int P) { return P <= 32; }              // the sums' warps share a unit's groups, not the tokens
// Shared memory behind the rings: the second group's sums, and the up rows'.
constexpr int sums_bytes(int P) { return by_group(P) ? P * kRows * 4 : 0; }
constexpr int up_bytes(int P, bool gated) { return gated ? P * (kRows / 2) * 4 : 0; }

struct Args {
  const __half* scale;
  __nv_bfloat16* out;
  float* partial;                  // [chunk][2 CTAs][token of the chunk][128 rows]
  unsigned int* tickets;           // [chunk][tile], zero
  unsigned char* wait_byte;
  long long lds, ldo;
  int tokens, rows, groups, tiles; // rows: of the output (F where gated)
  int run;                         // units of a CTA (of the last one fewer)
};
}  // namespace int4t5

template <int P, bool GATED>
__global__ void __launch_bounds__(int4t5::kThreads, 1)
gemm_int4_t5_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, int4t5::Args a) {
  using namespace int4t5;
  constexpr int kOutRows = GATED ? kRows / 2 : kRows, kPanel = P * 128, kStageX = 4 * kPanel, kRingX = ring_x(P), kRingD = ring_d(P);
  constexpr int kA = kRingD * P;              // of tensor memory: the ring of D, then that of A
  constexpr bool kByGroup = by_group(P);
  static_assert(kRingD * P + kRingA * 64 <= 512 && kRingA % kSets == 0 && kRingA % 2 == 0 && kRingW % kSets == 0 && kRingD % 2 == 0);
  constexpr int kColumns = 512, kOutThreads = kByGroup ? 128 : 256, kMine = kByGroup ? P : P / 2;           // tokens of a thread
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t w_full[kRingW], w_empty[kRingW], x_full[kRingX], x_empty[kRingX], a_full[kRingA], a_empty[kRingA], d_full[kRingD], d_empty[kRingD];
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag, last_one;
  __shared__ uint4 kept_scales[32 * kSumWarps];

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  constexpr int kXAt = kRingW * kUnitBytes, kSumsAt = kXAt + kRingX * kStageX, kUpAt = kSumsAt + sums_bytes(P);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRingW; ++i) mbar_init(&w_full[i], 1), mbar_init(&w_empty[i], 8);
    for (int i = 0; i < kRingX; ++i) mbar_init(&x_full[i], 1), mbar_init(&x_empty[i], 2);
    for (int i = 0; i < kRingA; ++i) mbar_init(&a_full[i], 4), mbar_init(&a_empty[i], 1);
    for (int i = 0; i < kRingD; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], kByGroup ? 4 : 8);
    abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
  }
  if (warp == 1) tmem_alloc<1>(&tmem_base_smem, kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_smem;
  volatile int* abort = &abort_flag;

  // This CTA's run of units.
  const int ctas = gridDim.x, cta = blockIdx.x, G = (a.groups + 1) / 2;       // pairs of groups; of an odd number the last one's second is zeros
  const int u0 = cta * a.run, units = min(a.run, a.tiles * G - u0), tile0 = u0 / G, g0 = u0 - tile0 * G;
  const int token0 = blockIdx.y * P;

  auto load_w = [&](int tile, int g, auto&& load) {
    if constexpr (GATED) {
      load(0, tile * kOutRows, g * 128);
      load(kUnitBytes / 2, a.rows + tile * kOutRows, g * 128);
    } else {
      load(0, tile * kRows, g * 128);
    }
  };
  if (warp == 0 && elect_one()) {             // into L2 only: returns nothing, so it may run beside the kernels before
    int tile = tile0, g = g0;
    for (int i = 0; i < min(units, kRingW); ++i) {
      load_w(tile, g, [&](int, int row, int byte) { tma_prefetch_2d(&tmW, byte, row); });
      if (++g == G) g = 0, ++tile;
    }
  }
  wait_for_previous(a.scale, a.out, a.partial, a.tickets);
  release_dependents();

  if (warp == 0) {
    // ------------------------------------ TMA producer ------------------------------------
    if (elect_one()) {
      int tile = tile0, g = g0, ws = 0, xs = 0;
      uint32_t wp = 1, xp = 1;                // an empty ring's waits return at once
      int xi = 0, xg = g0;
      // The tokens stay fewer units ahead than the weights: both are asked for in the order of their use.
      auto next_x = [&] {
        mbar_wait_or_abort(&x_empty[xs], xp, abort);
        mbar_expect_tx(&x_full[xs], kStageX);
#pragma unroll
        for (int h = 0; h < 4; ++h) tma_load_2d(smem + kXAt + xs * kStageX + h * kPanel, &tmX, &x_full[xs], xg * 256 + h * 64, token0);
        if (++xs == kRingX) xs = 0, xp ^= 1u;
        if (++xg == G) xg = 0;
        ++xi;
      };
      for (int i = 0; i < units; ++i) {
        mbar_wait_or_abort(&w_empty[ws], wp, abort);
        mbar_expect_tx(&w_full[ws], kUnitBytes);
        load_w(tile, g, [&](int at, int row, int byte) { tma_load_2d(smem + ws * kUnitBytes + at, &tmW, &w_full[ws], byte, row); });
        if (++ws == kRingW) ws = 0, wp ^= 1u;
        if (++g == G) g = 0, ++tile;
        if (i >= kRingW - kRingX && xi < units) next_x();
        else if (i < kRingX) next_x();
      }
      while (xi < units) next_x();
      if (*abort) {                           // copies still in flight land before the shared memory is given back
        int none = 0;
        for (int i = units > kRingW ? units - kRingW : 0; i < units; ++i) mbar_wait_bounded(&w_full[i % kRingW], (i / kRingW) & 1u, &none);
        for (int i = units > kRingX ? units - kRingX : 0; i < units; ++i) mbar_wait_bounded(&x_full[i % kRingX], (i / kRingX) & 1u, &none);
      }
    }
  } else if (warp < kSumAt) {
    // ------------------------------------ MMA issuers: the units' first groups, their second ones ------------------------------------
    constexpr uint32_t id = make_idesc_bf16(kRows, P, 0u, 0u);
    const int second = warp - 1;
    const uint64_t b0 = make_smem_desc(smem_base + kXAt + second * 2 * kPanel, 16, 1024, 2);
    int xs = 0;
    uint32_t xp = 0;
    for (int i = second; i < 2 * units; i += 2) {
      const int as = i % kRingA, ds = i % kRingD;
      if (i >= kRingD) mbar_wait_or_abort(&d_empty[ds], ((i / kRingD) & 1u) ^ 1u, abort);
      mbar_wait_or_abort(&x_full[xs], xp, abort);
      mbar_wait_or_abort(&a_full[as], (i / kRingA) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      if (elect_one()) {
        const uint64_t b = b0 + (xs * kStageX >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ts<1>(tmem_base + ds * P, tmem_base + kA + as * 64 + k * 8, b + (((k >> 2) * kPanel + (k & 3) * 32) >> 4), id, k != 0 ? 1u : 0u);
        umma_commit<1>(&d_full[ds]);
        umma_commit<1>(&a_empty[as]);
        umma_commit<1>(&x_empty[xs]);
      }
      if (++xs == kRingX) xs = 0, xp ^= 1u;
    }
  } else if (warp >= kWidenAt) {
    // ------------------------------------ widening: a row of every third group per thread ------------------------------------
    const int first = (warp - kWidenAt) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t to = tmem_base + kA + (static_cast<uint32_t>(quad * 32) << 16);
    const uint8_t* from = smem + row * 128;
    const int swz = row & 7;                  // of the 16-byte pieces of a row, as TMA lays them
    for (int i = first; i < 2 * units; i += kSets) {
      const int u = i >> 1, ws = u % kRingW, as = i % kRingA;
      mbar_wait_or_abort(&w_full[ws], (u / kRingW) & 1u, abort);
      uint4 words[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) words[j] = *reinterpret_cast<const uint4*>(from + ws * kUnitBytes + ((((i & 1) * 4 + j) ^ swz) << 4));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t r[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t v = reinterpret_cast<const uint32_t*>(words)[half * 8 + j];
          const uint32_t even = v & 0x0f0f0f0fu, odd = (v >> 4) & 0x0f0f0f0fu;
          const uint32_t lo = __byte_perm(even, odd, 0x5140), hi = __byte_perm(even, odd, 0x7362);         // columns 0 .. 3, 4 .. 7
          const uint32_t pair[4] = {__byte_perm(lo, 0x43434343u, 0x4140), __byte_perm(lo, 0x43434343u, 0x4342), __byte_perm(hi, 0x43434343u, 0x4140),
                                    __byte_perm(hi, 0x43434343u, 0x4342)};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair[c]), __floats2bfloat162_rn(136.f, 136.f));
            r[j * 4 + c] = *reinterpret_cast<const uint32_t*>(&d);
          }
        }
        if (half == 0) {
          if (i >= kRingA) mbar_wait_or_abort(&a_empty[as], ((i / kRingA) & 1u) ^ 1u, abort);
          __syncwarp();
          tc_fence_after();
        }
        tmem_st_x32(to + as * 64 + half * 32, r);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&a_full[as]);
        mbar_arrive(&w_empty[ws]);
      }
    }
  } else {
    // ------------------------------------ sums: a row per thread ------------------------------------
    const int quad = warp & 3, row = quad * 32 + lane, part = (warp - kSumAt) >> 2, n0 = kByGroup ? 0 : part * kMine;
    const uint32_t from = tmem_base + n0 + (static_cast<uint32_t>(quad * 32) << 16);
    const int tokens = min(a.tokens - token0 - n0, kMine);
    float* second_sums = reinterpret_cast<float*>(smem + kSumsAt);        // [token][row]
    float* up_sums = reinterpret_cast<float*>(smem + kUpAt);              // gated: [token][up row]
    constexpr int kGroups = kByGroup ? 1 : 2;                             // of a unit, that a thread looks at
    int tile = tile0, g = g0;
    auto scale_at = [&](int tile, int group) {
      if (group >= a.groups) return __half();
      const int out = tile * kOutRows + (GATED ? row & 63 : row);
      return a.scale[static_cast<long long>(min(out, a.rows - 1) + (GATED && row >= 64 ? a.rows : 0)) * a.lds + group];
    };
    // Scales are asked for four units at a time, and four ahead: a row's come from memory, a microsecond away.  They are kept where only their thread looks.
    __half* kept = reinterpret_cast<__half*>(&kept_scales[threadIdx.x - 32 * kSumAt]);
    __half next[4 * kGroups];
    int next_tile = tile, next_g = g, next_u = 0;
    auto fetch_scales = [&] {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int h = 0; h < kGroups; ++h) next[kGroups * j + h] = next_u < units ? scale_at(next_tile, 2 * next_g + (kByGroup ? part : h)) : __half();
        ++next_u;
        if (++next_g == G) next_g = 0, ++next_tile;
      }
    };
    fetch_scales();
    float total[kMine];
#pragma unroll
    for (int n = 0; n < kMine; ++n) total[n] = 0.f;
    bool whole = g == 0;                      // this CTA has the tile's first unit
    for (int u = 0; u < units; ++u) {
      if ((u & 3) == 0) {
#pragma unroll
        for (int j = 0; j < 4 * kGroups; ++j) kept[j] = next[j];
        fetch_scales();
      }
      const bool ends = g + 1 == G;
#pragma unroll
      for (int h = 0; h < kGroups; ++h) {
        const int i = 2 * u + (kByGroup ? part : h);
        const float s = __half2float(kept[kGroups * (u & 3) + h]);
        mbar_wait_or_abort(&d_full[i % kRingD], (i / kRingD) & 1u, abort);
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int n = 0; n < kMine; n += 16) {
          uint32_t d[16];
          tmem_ld_x16(from + i % kRingD * P + n, d);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 16; ++c) total[n + c] = fmaf(s, __uint_as_float(d[c]), total[n + c]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_empty[i % kRingD]);
      }
      if (!ends && u + 1 < units) {
        ++g;
        continue;
      }
      // The tile, or this CTA's part of it, is done.
      if constexpr (kByGroup) {
        if (part == 1) {
#pragma unroll
          for (int n = 0; n < kMine; ++n) second_sums[n * kRows + row] = total[n];
        }
        named_bar_sync(2, 256);
        if (part == 0) {
#pragma unroll
          for (int n = 0; n < kMine; ++n) total[n] += second_sums[n * kRows + row];
        }
        named_bar_sync(3, 256);
      }
      if (!kByGroup || part == 0) {
        bool write = true;
        if (!whole || !ends) {
          const int t0 = tile * G, c0 = t0 / a.run, c1 = (t0 + G - 1) / a.run;      // the first and the last CTA with a part
          float* slots = a.partial + static_cast<long long>(blockIdx.y) * 2 * ctas * P * kRows + n0 * kRows + row;
          const long long pitch = P * kRows;
          float* mine = slots + (2 * cta + (cta == c0 ? 1 : 0)) * pitch;
#pragma unroll
          for (int n = 0; n < kMine; ++n) __stcg(mine + n * kRows, total[n]);
          __threadfence();
          named_bar_sync(1, kOutThreads);
          if (threadIdx.x == 32 * kSumAt) {
            unsigned int* ticket = a.tickets + static_cast<long long>(blockIdx.y) * a.tiles + tile;
            last_one = atomicAdd(ticket, 1u) == static_cast<unsigned int>(c1 - c0);
            if (last_one) *ticket = 0;
            __threadfence();
          }
          named_bar_sync(1, kOutThreads);
          write = last_one;
          if (write) {
#pragma unroll
            for (int n = 0; n < kMine; ++n) total[n] = 0.f;
            // (two parts under way at once; behind the last one its neighbour is read again and not used)
            for (int c = c0; c <= c1; c += 2) {
              const float* one = slots + (2 * c + (c == c0 ? 1 : 0)) * pitch;
              const float* other = slots + 2 * min(c + 1, c1) * pitch;
              const float use = c + 1 <= c1 ? 1.f : 0.f;
#pragma unroll
              for (int n = 0; n < kMine; n += 16) {
                float v[16], z[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = __ldcg(one + (n + k) * kRows), z[k] = __ldcg(other + (n + k) * kRows);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  total[n + k] += v[k];
                  if (use != 0.f) total[n + k] += z[k];
                }
              }
            }
          }
        }
        if (write) {
          const int out = tile * kOutRows + (GATED ? row & 63 : row);
          __nv_bfloat16* to = a.out + static_cast<long long>(token0 + n0) * a.ldo + out;
          if constexpr (GATED) {
            if (row >= 64) {
#pragma unroll
              for (int n = 0; n < kMine; ++n) up_sums[(n0 + n) * 64 + row - 64] = total[n];
            }
            named_bar_sync(1, kOutThreads);
            if (row < 64 && out < a.rows) {
#pragma unroll
              for (int n = 0; n < kMine; ++n)
                if (n < tokens) to[n * a.ldo] = __float2bfloat16(total[n] * __fdividef(1.f, 1.f + __expf(-total[n])) * up_sums[(n0 + n) * 64 + row]);
            }
          } else if (out < a.rows) {
#pragma unroll
            for (int n = 0; n < kMine; ++n)
              if (n < tokens) to[n * a.ldo] = __float2bfloat16(total[n]);
          }
        }
        if (GATED || !whole || !ends) named_bar_sync(1, kOutThreads);           // the flag and the up rows have been read
      }
#pragma unroll
      for (int n = 0; n < kMine; ++n) total[n] = 0.f;
      ++tile;
      g = 0;
      whole = true;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<1>(tmem_base, kColumns);
  if (threadIdx.x == 0 && abort_flag) report_wait(a.wait_byte);
}

namespace {
// Runs of one length, as short as one CTA to an SM allows.
int run_of(long long units) { return static_cast<int>((units + kNumSMs - 1) / kNumSMs); }
int ctas_of(int tiles, int groups) {
  const long long units = static_cast<long long>(tiles) * ((groups + 1) / 2);
  return static_cast<int>((units + run_of(units) - 1) / run_of(units));
}
int padded(int tokens) { return tokens <= 16 ? 16 : tokens <= 32 ? 32 : 64; }

template <int P, bool GATED>
cudaError_t launch(const CUtensorMap& w, const CUtensorMap& x, const int4t5::Args& a, int chunks, cudaStream_t s) {
  using namespace int4t5;
  constexpr int smem = kRingW * kUnitBytes + ring_x(P) * 4 * P * 128 + sums_bytes(P) + up_bytes(P, GATED) + 1024;
  const auto kernel = gemm_int4_t5_kernel<P, GATED>;
  if (const cudaError_t e = allow_smem(kernel, smem); e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3(ctas_of(a.tiles, a.groups), chunks), kThreads, smem, s, w, x, a);
}
template <bool GATED>
cudaError_t dispatch(const CUtensorMap& w, const CUtensorMap& x, const int4t5::Args& a, int p, int chunks, cudaStream_t s) {
  return p == 16 ? launch<16, GATED>(w, x, a, chunks, s) : p == 32 ? launch<32, GATED>(w, x, a, chunks, s) : launch<64, GATED>(w, x, a, chunks, s);
}
}  // namespace

long long gemm_int4_t5_scratch(int tokens, int rows, int groups, bool gated, int* tickets) {
  const int p = padded(tokens), chunks = (tokens + p - 1) / p, out = gated ? 64 : 128, tiles = (rows + out - 1) / out;
  *tickets = tiles * chunks;
  return static_cast<long long>(chunks) * 2 * ctas_of(tiles, groups) * p * int4t5::kRows;
}

cudaError_t gemm_int4_t5(const void* x, long long ldx, const void* w, long long ldw, const void* scale, long long lds, void* out, long long ldo, int tokens, int rows,
                         int groups, bool gated, float* partial, unsigned int* tickets, cudaStream_t s) {
  const int p = padded(tokens), chunks = (tokens + p - 1) / p, tile_rows = gated ? 64 : 128;
  const long long matrix = gated ? 2LL * rows : rows;
  if (static_cast<long long>((rows + tile_rows - 1) / tile_rows) * ((groups + 1) / 2) >= (1LL << 31)) return cudaErrorInvalidValue;
  CUtensorMap tw, tx;
  if (const int e = get_tmap_2d_bytes(&tw, w, matrix, groups * 64LL, ldw, tile_rows, 128); e != 0) return static_cast<cudaError_t>(e);
  if (const int e = get_tmap_2d_bf16(&tx, x, tokens, groups * 128LL, ldx, p, 64, 1); e != 0) return static_cast<cudaError_t>(e);
  unsigned char* const byte = wait_report(kWaitInt4);
  if (byte == nullptr) return cudaErrorMemoryAllocation;
  const int tiles = (rows + tile_rows - 1) / tile_rows;
  const int4t5::Args a = {static_cast<const __half*>(scale), static_cast<__nv_bfloat16*>(out), partial, tickets, byte, lds, ldo, tokens, rows, groups, tiles, run_of(static_cast<long long>(tiles) * ((groups + 1) / 2))};
  return gated ? dispatch<true>(tw, tx, a, p, chunks, s) : dispatch<false>(tw, tx, a, p, chunks, s);
}

}  // namespace llmctl
