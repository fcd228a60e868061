// The decode attention of paged_attention_fp8.cu on the 5th-generation tensor cores, for blocks of a multiple of 8 tokens.
//
// A sequence's one token has only the query heads of a group to offer as rows, so the CACHE ROWS are the M side of both products, as they stand in the
// cache, in 8 bits:
//     S^T = K Q^T         128 tokens x N columns, over D                 (A: the key tile as it was loaded, K-major)
//     O^T = V^T P^T       D dimensions x N columns, over 128 tokens      (A: the value tile as it was loaded, M-major)
// kind::f8f6f4 wants 8-bit columns too.  A query head, and a row of weights, is therefore FOUR columns: the number rounded to e4m3 (4 significant
// bits), the rest times 16 rounded, its rest times 16, and so on: 16 bits of what they have, where bf16 has 8, over a range of 2^28.  The products of two
// e4m3 numbers are exact and the four columns are added in 32 bits.  N = 16 columns are four heads, 32 eight, 64 sixteen.
//
// The scales of keys multiply the scores.  Those of values are added to the exponent of a token's weight, w = 2^(s + log2 sv), which has a running reference of
// its own: M over s + log2 sv beside m over s, so that neither a block of tiny values nor one of large ones takes the bits of the others.
//     O = 2^(M - m) sum_j w_j cv_j / l,    w_j = 2^(s_j + log2 sv_j - M),    l = sum_j 2^(s_j - m)
// O of a tile is read from tensor memory and added up in registers, where the reference of the tiles before is caught up with.
//
//   warps 0, 7  TMA producers of keys and of values: 128 tokens, a box for each block that they stand in, a ring of stages; their scales beside them
//   warps 1, 6  MMA issuers, of scores and of values
//   warps 2-5   the columns of Q, then a token per thread: S^T -> P^T; a dimension per thread: O^T
//
// The work is one row of tiles: those of every sequence and head behind one another.  As many CTAs as fit on the chip take equal runs of it, so that
// batches of unlike contexts end together; a sequence and head that more than one CTA has a part of is merged by a second kernel.
// Where contexts are of a few tiles only the runs are cut between heads, and nothing is merged.
//
// Bound by the pass over the cache, 6.5 - 6.9 TB/s of it once all CTAs are under way, and by 6 - 8 us of start, last tiles and merge.  us: 4 contexts of up to
// 50001, 32 heads of 128 180 (6.6 TB/s), 16 of up to 4096, 32 heads 60.6 (5.8), 64 of 1000 to 4000, 32 over 8 63.7 (5.3), one of 300 5.7.
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
constexpr int kThreads = 256;
constexpr int kPieces = 4, kMaxStages = 8, kMaxBoxes = 16;
constexpr int kWholeTokens = 768, kLeast = 2;
constexpr float kStep = 16.f;                // between the columns of a number
// Eight query heads: the references stay where they are while no score is beyond them by more than kSlack, and no weight by kSlackV (log2; a weight of 1 is then
// 128, and none above 430), and no maxima are taken.  us, maxima in each tile / so: 70 contexts of up to 31760, 24 heads of 64 over 4 215 / 188, 8 of 8000, 64 heads of 128
// over 8 31.6 / 31.2; one head 60.9 / 61.2, four 64.5 / 64.6, sixteen 30.9 / 32.9 (floors 110, 14; 53, 52, 7).
constexpr float kSlack = 32.f, kSlackV = 1.75f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int columns(int GP) { return GP < 4 ? 16 : kPieces * GP; }     // of a product: 16 at least, of which those past 4 GP are nobody's
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
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t* r) {
  if constexpr (C == 4) tmem_ld_x4(at, r);
  else if constexpr (C == 8) tmem_ld_x8(at, r);
  else if constexpr (C == 16) tmem_ld_x16(at, r);
  else if constexpr (C == 32) tmem_ld_x32(at, r);
  else {
    tmem_ld_x32(at, r);
    tmem_ld_x32(at + 32, r + 32);
  }
}

// Place in the ring of stages.  (A quotient and a remainder by a number known at launch are 200 clocks in the issuing warp's way, three of them in
// each turn of its loop: 2600 clocks a tile, 16 contexts up to 4096, 32 heads 66.1 us, so 62.2.)
struct Place {
  int st = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++st == stages) {
      st = 0;
      phase ^= 1u;
    }
  }
};

// The row of tiles.  Item: a sequence and up to 16 query heads of one head of the cache, b * per_sequence + x.
struct Work {
  const int* context_lens;
  int batch, per_sequence, limit, least;                 // least: tiles of the shortest run
  int whole, items, items_rest;                          // != 0: runs are of `items` items, the first `items_rest` of one more
  FastDiv by_sequence;
  __device__ __forceinline__ int tokens(int b) const { return b < batch ? max(min(context_lens[b], limit), 0) : 0; }
  __device__ __forceinline__ int tiles(int b) const { return (tokens(b) + kTile - 1) / kTile; }
};
struct Run {
  int b, x, t, left;                                     // first tile, tiles left
  int last_b;                                            // of the last item (runs of whole items)
};
// Tiles of all sequences before `b` and, in `all`, of the whole batch, for one head; by one warp.
__device__ __forceinline__ int tiles_before(const Work& w, int b, int& all) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  all = 0;
  for (int i = lane; i < w.batch; i += 32) {
    const int n = w.tiles(i);
    all += n;
    if (i < b) before += n;
  }
  all = __reduce_add_sync(0xffffffffu, all);
  return __reduce_add_sync(0xffffffffu, before);
}
__device__ __forceinline__ int run_length(const Work& w, int all, int ctas) { return max((all * w.per_sequence + ctas - 1) / ctas, w.least); }

// The run of a CTA, by one warp.
__device__ __forceinline__ Run run_of(const Work& w, int cta, int ctas) {
  const int lane = threadIdx.x & 31;
  Run r = {0, 0, 0, 0, 0};
  uint32_t x;
  if (w.whole) {
    const int first = cta * w.items + min(cta, w.items_rest), last = first + w.items + (cta < w.items_rest ? 1 : 0);
    r.last_b = static_cast<int>(w.by_sequence.divide(last - 1, x));
    r.b = static_cast<int>(w.by_sequence.divide(first, x));
    r.x = static_cast<int>(x);
    int n = 0;
    for (int i = first + lane; i < last; i += 32) n += w.tiles(static_cast<int>(w.by_sequence.divide(i, x)));
    r.left = __reduce_add_sync(0xffffffffu, n);
    return r;
  }
  int all;
  tiles_before(w, 0, all);
  const int length = run_length(w, all, ctas);
  const long long start = static_cast<long long>(length) * cta;
  const int total = all * w.per_sequence;
  if (start >= total) return r;
  const int first = static_cast<int>(start);
  r.left = min(total - first, length);
  int before = 0;                                        // tiles of the items in front of the chunk of 32 sequences
  for (int b0 = 0; b0 < w.batch; b0 += 32) {
    const int n = w.tiles(b0 + lane);
    int end = n;                                         // of the sequences up to this lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += other;
    }
    const int upto = before + end * w.per_sequence;
    const unsigned here = __ballot_sync(0xffffffffu, upto > first);
    if (here != 0u) {
      const int at = __ffs(here) - 1, nb = __shfl_sync(0xffffffffu, n, at), in = first - __shfl_sync(0xffffffffu, upto, at) + nb * w.per_sequence;
      r.b = b0 + at;
      r.x = in / nb;
      r.t = in - r.x * nb;
      return r;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return r;
}
// A run item by item: tiles t .. t + n of the nt of (b, x), whose sequence has `tokens`.
struct Items {
  Run r;
  int nt, n, tokens;
  __device__ __forceinline__ Items(const Run& run, const Work& w) : r(run), nt(0), n(0), tokens(0) {
    if (r.left > 0) skip(w);
  }
  __device__ __forceinline__ void skip(const Work& w) {          // sequences without tokens
    while (r.b < w.batch && (tokens = w.tokens(r.b)) == 0) ++r.b, r.x = 0;
    if (r.b >= w.batch) r.left = 0;                      // (lengths that change meanwhile)
    nt = (tokens + kTile - 1) / kTile;
    n = min(nt - r.t, r.left);
  }
  __device__ __forceinline__ bool more() const { return r.left > 0; }
  __device__ __forceinline__ void next(const Work& w) {
    r.left -= n;
    r.t = 0;
    n = 0;
    if (r.left == 0) return;
    if (++r.x == w.per_sequence) {
      r.x = 0;
      ++r.b;
      skip(w);
    } else {
      n = min(nt, r.left);
    }
  }
};
}  // namespace dec8

// Grid: as many CTAs as there are runs.  GP: query heads of an item.  partial: two rows of items [2 ctas, GP, D + 2] = {sum of w cv at the reference m, m (log2), sum of p}: of the
// item that the run begins inside of, and of the one that it ends inside of.
template <int D, int GP>
__global__ void __launch_bounds__(dec8::kThreads, GP == 16 ? 1 : GP == 1 || (D == 64 && GP == 2) ? 3 : 2)
paged_attn_decode_fp8_t5_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* __restrict__ q,
                                long long q_stride, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                                const int* __restrict__ block_tables, int max_blocks, dec8::Work work, float* __restrict__ partial,
                                __nv_bfloat16* __restrict__ out, int blocks, int block_size, FastDiv by_block, int box_rows, int kv_heads, int group,
                                int stages, float scale_log2, unsigned char* wait_byte) {
  using namespace dec8;
  constexpr int C = kPieces * GP, N = columns(GP), kStage = stage_bytes(D), kHalf = kTile * D;
  constexpr bool kMayStay = GP == 8;
  constexpr float kUnit = kMayStay ? 128.f : 256.f;                        // a weight of 1
  constexpr uint32_t kSwizzle = D == 128 ? 2 : 4, kEight = 8 * D;          // layout of the tiles, bytes of eight rows
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_q, bar_full[kMaxStages], bar_empty[kMaxStages], bar_s[2], bar_p[2], bar_o[2];
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;
  __shared__ __align__(16) float top[2][4][2 * GP];                                      // per softmax warp: the tile's largest s and s + log2 sv
  __shared__ float box_scale[kMaxStages][2][kMaxBoxes];                    // of a stage's boxes: sk, log2 sv

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int q_at = stages * kStage, p_at = q_at + N * D;

  if (threadIdx.x == 0) {
    mbar_init(&bar_q, 4);
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bar_full[i], 4);                         // copies and scales of keys and of values
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
  wait_for_previous(q, k_scale, v_scale, block_tables, work.context_lens, partial, out);
  release_dependents();
  volatile int* abort = &abort_flag;
  const int heads = kv_heads * group;
  const Run run = run_of(work, blockIdx.x, gridDim.x);                     // every warp finds it for itself

  if (warp == 0 || warp == 7) {
    // ------------------------------------ TMA producers, of keys and of values: a lane per box ------------------------------------
    const int boxes = kTile / box_rows, all_rows = blocks * kv_heads * block_size;
    // Three tiles are under way: the block of the one after next is asked for, the scales of the next, and this one is copied: the producer waits for
    // no load that it has just asked for.  A block outside of the cache is filled with zeros, its scales are no numbers.
    struct Box {
      int block, row, head;                               // row: of the block; < 0: no box
    };
    auto find = [&](const Items& it, int tile) {
      const int token = (it.r.t + tile) * kTile + lane * box_rows;
      Box box = {0, -1, 0};
      if (!it.more() || lane >= boxes || token >= it.tokens) return box;
      uint32_t row;
      box.block = block_tables[static_cast<long long>(it.r.b) * max_blocks + by_block.divide(static_cast<uint32_t>(token), row)];
      box.row = static_cast<int>(row);
      box.head = it.r.x < kv_heads ? it.r.x : it.r.x % kv_heads;
      return box;
    };
    auto scale_of = [&](const float* s, const Box& box) {
      return box.row < 0 ? 0.f : box.block >= 0 && box.block < blocks ? s[static_cast<long long>(box.block) * kv_heads + box.head] : NAN;
    };
    const bool keys = warp == 0;
    const CUtensorMap* tm = keys ? &tmK : &tmV;
    const float* scales = keys ? k_scale : v_scale;
    Items it(run, work);
    int tile = 0, loaded = 0;                             // within the item's part; so far
    auto advance = [&] {
      if (it.more() && ++tile == it.n) {
        it.next(work);
        tile = 0;
      }
    };
    Box box = find(it, 0);
    advance();
    Box next = find(it, tile);
    float scale = scale_of(scales, box);
    Place at;
    for (; loaded < run.left; ++loaded, at.next(stages)) {
      const int st = at.st;
      advance();
      const Box after = find(it, tile);
      const float next_scale = scale_of(scales, next);
      const bool given = loaded < stages || mbar_wait_bounded(&bar_empty[st], at.phase ^ 1u, abort);
      if (!__all_sync(0xffffffffu, given)) break;
      const int count = __popc(__ballot_sync(0xffffffffu, box.row >= 0));
      if (lane == 0) mbar_expect_tx(&bar_full[st], count * box_rows * D);
      __syncwarp();
      if (box.row >= 0) {
        const int row = box.block >= 0 && box.block < blocks ? (box.block * kv_heads + box.head) * block_size + box.row : all_rows;
        tma_load_2d(smem + st * kStage + (keys ? 0 : kHalf) + lane * box_rows * D, tm, &bar_full[st], 0, row);
      }
      if (lane < kMaxBoxes) box_scale[st][keys ? 0 : 1][lane] = keys ? scale : __log2f(scale);       // (the first copies do not wait for them)
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_full[st]);
      box = next;
      next = after;
      scale = next_scale;
    }
    // Copies still in flight when a wait ran out land before the CTA's shared memory is given back.
    if (*abort && lane == 0)
      for (int i = loaded > stages ? loaded - stages : 0; i < loaded; ++i) {
        int none = 0;
        mbar_wait_bounded(&bar_full[i % stages], (i / stages) & 1u, &none);
      }
  } else if (warp == 1) {
    // ------------------------------------ scores ------------------------------------
    constexpr uint32_t id = make_idesc_e4m3(kTile, N, 0u, 0u);          // A, B K-major
    const uint64_t a0 = make_smem_desc(smem_base, 16, kEight, kSwizzle), b0 = make_smem_desc(smem_base + q_at, 16, kEight, kSwizzle);
    Place at;
    int n = 0, item = 0;
    for (Items it(run, work); it.more(); it.next(work), ++item) {
      mbar_wait_or_abort(&bar_q, item & 1u, abort);
      for (int i = 0; i < it.n; ++i, ++n, at.next(stages)) {
        if (n >= 2) mbar_wait_or_abort(&bar_p[n & 1], ((n >> 1) & 1u) ^ 1u, abort);       // the scores before last have been read
        mbar_wait_or_abort(&bar_full[at.st], at.phase, abort);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = a0 + (at.st * kStage >> 4);
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma_f8_ss(tmem_base + (n & 1) * N, a + (k * 32 >> 4), b0 + (k * 32 >> 4), id, k != 0 ? 1u : 0u);
          umma_commit<1>(&bar_s[n & 1]);
        }
      }
      if (__any_sync(0xffffffffu, *abort)) break;
    }
  } else if (warp == 6) {
    // ------------------------------------ values, by a warp of their own: each issuer then waits for one thing after the other and never polls ------------------------------------
    constexpr uint32_t id = make_idesc_e4m3(D, N, 1u, 1u);              // A, B MN-major
    const uint64_t a0 = make_smem_desc(smem_base + kHalf, 16, kEight, kSwizzle), b0 = make_smem_desc(smem_base + p_at, 128, kTile * 16, 0);
    Place at;
    for (int n = 0; n < run.left; ++n, at.next(stages)) {
      mbar_wait_or_abort(&bar_p[n & 1], (n >> 1) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = a0 + (at.st * kStage >> 4), b = b0 + ((n & 1) * kTile * N >> 4);
#pragma unroll
        for (int k = 0; k < kTile / 32; ++k) umma_f8_ss(tO + (n & 1) * N, a + (k * 32 * D >> 4), b + (k * 512 >> 4), id, k != 0 ? 1u : 0u);
        umma_commit<1>(&bar_empty[at.st]);
        umma_commit<1>(&bar_o[n & 1]);
      }
      if (__any_sync(0xffffffffu, *abort)) break;
    }
  } else {
    // ------------------------------------ softmax warps ------------------------------------
    const int w = warp - 2, quad = warp & 3, t = quad * 32 + lane, box = t / box_rows;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int dim = D == 128 ? t : quad * 16 + lane;      // of O^T: 64 rows stand in 16 lanes of each quadrant
    const bool has_dim = D == 128 || lane < 16;

    // A row of Q whose largest number comes to stand in 128 .. 255, as four columns K-major, swizzled as TMA swizzles the tiles
    auto load_q = [&](const Items& it, float (&x)[GP]) {
      const int g0 = it.r.x / kv_heads * GP;
      const __nv_bfloat16* src = q + it.r.b * q_stride + static_cast<long long>(it.r.x % kv_heads * group + g0) * D + t;
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        x[g] = it.more() && t < D && g < group - g0 ? __bfloat162float(src[g * D]) : 0.f;
        if (!isfinite(x[g])) x[g] = NAN;                  // an infinity has no columns, and no scores that are numbers
      }
    };
    auto write_q = [&](float (&x)[GP], float (&factor)[GP], int buf) {
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float m = warp_max_all(fabsf(x[g]));
        if (lane == 0) top[buf][w][g] = m;
      }
      named_bar_sync(1, 128);
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float m = fmaxf(fmaxf(top[buf][0][g], top[buf][1][g]), fmaxf(top[buf][2][g], top[buf][3][g]));
        const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23), 16), 254);           // biased
        x[g] *= __uint_as_float(static_cast<uint32_t>(261 - e) << 23);                          // 2^(7 - (e - 127))
        factor[g] = __uint_as_float(static_cast<uint32_t>(e - 7) << 23) * scale_log2;
      }
      uint8_t* qs = smem + q_at;
      if (t < D) {
        auto at = [&](int n) {                            // byte t of row n
          return D == 128 ? n * 128 + (((t >> 4) ^ (n & 7)) << 4) + (t & 15) : n * 64 + (((t >> 4) ^ ((n >> 1) & 3)) << 4) + (t & 15);
        };
#pragma unroll
        for (int g = 0; g < GP; g += 2) {
          uint32_t codes[kPieces];
          split2(x[g], GP > 1 ? x[g + 1] : 0.f, codes);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            qs[at(i * GP + g)] = static_cast<uint8_t>(codes[i]);
            if (GP > 1) qs[at(i * GP + g + 1)] = static_cast<uint8_t>(codes[i] >> 8);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q);
    };

    float m[GP], M[GP], l[GP], acc[GP], catch_up[GP], factor[GP];     // catch_up: from the reference of the tile before last to that of the last
    auto add_tile = [&](int n) {
      mbar_wait_or_abort(&bar_o[n & 1], (n >> 1) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      uint32_t o[C];
      tmem_ld<C>(tO + (n & 1) * N + lane_off, o);
      tmem_ld_wait();
#pragma unroll
      for (int g = 0; g < GP; ++g) acc[g] = fmaf(acc[g], catch_up[g], joined<GP>(o, g));
    };
    Items it(run, work);
    float x[GP];
    load_q(it, x);
    if (work.whole)                                       // sequences without tokens are in nobody's run (of runs with parts: paged_attn_merge_fp8_t5_kernel)
      for (int b = run.b; b <= run.last_b; ++b)
        if (work.tokens(b) == 0)
          for (int i = t; i < heads * D; i += 128) out[static_cast<long long>(b) * heads * D + i] = __float2bfloat16(0.f);
    Place at;
    int n = 0, part = 0;                                  // tiles so far; use of top: items and tiles so far
    if (it.more()) write_q(x, factor, part++ & 1);
    while (it.more()) {
      const int first = n, end = n + it.n, b = it.r.b, g0 = it.r.x / kv_heads * GP, kv_head = it.r.x % kv_heads;
      const int t0 = it.r.t * kTile, t1 = it.tokens;
      const bool whole_item = it.n == it.nt, begins_inside = it.r.t > 0;
      it.next(work);
      load_q(it, x);                                      // of the next item, while this one's tiles come in
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        m[g] = M[g] = -INFINITY;
        l[g] = acc[g] = catch_up[g] = 0.f;
      }
      for (; n < end; ++n, ++part, at.next(stages)) {
        const bool seen = t0 + (n - first) * kTile + t < t1;
        const int st = at.st;
        float (&most)[4][2 * GP] = top[part & 1];
        mbar_wait_or_abort(&bar_s[n & 1], (n >> 1) & 1u, abort);
        mbar_wait_or_abort(&bar_full[st], at.phase, abort);                // it is: the scales, and values that are written below
        __syncwarp();
        tc_fence_after();
        const float sk = box_scale[st][0][box], lv = seen ? box_scale[st][1][box] : 0.f;
        float s[GP];
        {
          uint32_t c[C];
          tmem_ld<C>(tmem_base + (n & 1) * N + lane_off, c);
          tmem_ld_wait();
#pragma unroll
          for (int g = 0; g < GP; ++g) s[g] = seen ? joined<GP>(c, g) * (sk * factor[g]) : -INFINITY;
        }
        bool beyond = !kMayStay;
        if constexpr (kMayStay) {
#pragma unroll
          for (int g = 0; g < GP; ++g) beyond |= !(s[g] - m[g] <= kSlack && s[g] + lv - M[g] <= kSlackV);
        }
        uint32_t codes[C / 4];                            // this token's row of P: C bytes, piece after piece
        float from[GP];
        if (!kMayStay || n == first || named_bar_any(1, 128, beyond)) {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float a = warp_max_all(s[g]), c = warp_max_all(s[g] + lv);
            if (lane == 0) {
              most[w][g] = a;
              most[w][GP + g] = c;
            }
          }
          named_bar_sync(1, 128);
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            auto over = [&](int i) { return fmaxf(fmaxf(most[0][i], most[1][i]), fmaxf(most[2][i], most[3][i])); };
            const float m1 = fmaxf(m[g], over(g)), M1 = fmaxf(M[g], over(GP + g));
            const float ref = m1 == -INFINITY ? 0.f : m1, Ref = M1 == -INFINITY ? 0.f : M1;
            l[g] = fmaf(l[g], ex2_approx(m[g] - ref), ex2_approx(s[g] - ref));
            from[g] = ex2_approx(M[g] - Ref);
            m[g] = m1;
            M[g] = M1;
            s[g] = ex2_approx(s[g] + lv - Ref) * kUnit;
          }
        } else {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            l[g] += ex2_approx(s[g] - m[g]);
            from[g] = 1.f;
            s[g] = ex2_approx(s[g] + lv - M[g]) * kUnit;
          }
        }
#pragma unroll
        for (int i = 0; i < C / 4; ++i) codes[i] = 0u;
#pragma unroll
        for (int g = 0; g < GP; g += 2) {
          uint32_t two[kPieces];
          split2(s[g], GP > 1 ? s[g + 1] : 0.f, two);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) codes[(i * GP + g) / 4] |= two[i] << ((i * GP + g) % 4 * 8);
        }
        uint8_t* dst = smem + p_at + (n & 1) * kTile * N + t * 16;
        if constexpr (C == 4) *reinterpret_cast<uint32_t*>(dst) = codes[0];
        else if constexpr (C == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
        else {
#pragma unroll
          for (int i = 0; i < C / 16; ++i) *reinterpret_cast<uint4*>(dst + i * kTile * 16) = make_uint4(codes[4 * i], codes[4 * i + 1], codes[4 * i + 2], codes[4 * i + 3]);
        }
        // Values past the last token: nothing that the cache holds there may meet a weight of zero.  A row to eight lanes (a lane to its row has all in
        // the same banks: 900 clocks in the way of every short context).
        for (int i = max(t1 - t0 - (n - first) * kTile - quad * 32, 0) + lane / (D / 16); i < 32; i += 512 / D)
          *reinterpret_cast<uint4*>(smem + st * kStage + kHalf + (quad * 32 + i) * D + lane % (D / 16) * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_p[n & 1]);
        if (n == end - 1 && it.more()) write_q(x, factor, ++part & 1);      // of the next item: its first scores run beside what is left of this one
        if (n > first) add_tile(n - 1);
#pragma unroll
        for (int g = 0; g < GP; ++g) catch_up[g] = from[g];
      }
      add_tile(n - 1);

      // ---- sums over the tokens, read-out ----
      float (&sums)[4][2 * GP] = top[part++ & 1];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float v = warp_sum(l[g]);
        if (lane == 0) sums[w][g] = v;
      }
      named_bar_sync(1, 128);
      const long long row0 = static_cast<long long>(b) * heads + kv_head * group + g0;
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        if (g >= group - g0 || !has_dim) continue;
        const float total = (sums[0][g] + sums[1][g]) + (sums[2][g] + sums[3][g]);
        const float o = acc[g] * (M[g] == -INFINITY ? 1.f / kUnit : exp2f(M[g] - m[g]) * (1.f / kUnit));
        if (whole_item) {
          out[(row0 + g) * D + dim] = __float2bfloat16(o / total);
        } else {
          float* dst = partial + ((2LL * blockIdx.x + (begins_inside ? 0 : 1)) * GP + g) * (D + 2);
          dst[dim] = o;
          if (t == 0) {
            dst[D] = m[g];
            dst[D + 1] = total;
          }
        }
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

// Items of more than one run.  Grid: (items of a sequence x GP, batch), a thread per dimension.
template <int D, int GP>
__global__ void __launch_bounds__(D)
paged_attn_merge_fp8_t5_kernel(const float* __restrict__ partial, __nv_bfloat16* __restrict__ out, dec8::Work work, int ctas, int kv_heads, int group) {
  using namespace dec8;
  wait_for_previous(partial, out, work.context_lens);
  release_dependents();
  const int b = blockIdx.y, x = blockIdx.x / GP, g = blockIdx.x % GP, nt = work.tiles(b), g0 = x / kv_heads * GP;
  if (g >= group - g0) return;
  const long long row = (static_cast<long long>(b) * kv_heads + x % kv_heads) * group + g0 + g;
  if (nt == 0) {
    out[row * D + threadIdx.x] = __float2bfloat16(0.f);
    return;
  }
  int all;
  const int before = tiles_before(work, b, all);                          // every warp for itself
  const int length = run_length(work, all, ctas), start = before * work.per_sequence + x * nt;
  const int c0 = start / length, c1 = (start + nt - 1) / length;
  if (c0 == c1) return;
  float m = -INFINITY, l = 0.f, o = 0.f;
  constexpr int kAhead = 8;                               // parts that are asked for before the first is there
  for (int c = c0; c <= c1; c += kAhead) {
    float pm[kAhead], pl[kAhead], po[kAhead], to = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float* p = partial + ((2LL * (c + i) + ((c + i) * length > start ? 0 : 1)) * GP + g) * (D + 2);
      const bool there = c + i <= c1;
      pm[i] = there ? p[D] : -INFINITY;
      pl[i] = there ? p[D + 1] : 0.f;
      po[i] = there ? p[threadIdx.x] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) to = fmaxf(to, pm[i]);
    const float ref = to == -INFINITY ? 0.f : to, u = exp2f(m - ref);
    l *= u;
    o *= u;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float w = exp2f(pm[i] - ref);
      l += pl[i] * w;
      o += po[i] * w;
    }
    m = to;
  }
  out[row * D + threadIdx.x] = __float2bfloat16(o / l);
}

bool paged_attn_fp8_t5_ok(int head_dim, int block_size) { return (head_dim == 64 || head_dim == 128) && block_size % 8 == 0; }

namespace dec8 {
struct Plan {
  int GP, parts, ctas, per_sm, whole;
  long long items, partial;
};
static Plan plan_of(int batch, int heads, int kv_heads, int head_dim, int limit, int runs) {
  Plan p;
  const int group = heads / kv_heads;
  for (p.GP = 1; p.GP < group && p.GP < 16;) p.GP *= 2;
  p.parts = (group + p.GP - 1) / p.GP;
  p.items = static_cast<long long>(batch) * kv_heads * p.parts;
  const long long tiles = p.items * ((limit + kTile - 1) / kTile);
  // Nothing is split where contexts are short: the second kernel is 2 to 3 us, a tile of a longer chain 0.65.  us, whole / split: 16 contexts of up to 600,
  // 32 heads of 128 15.4 / 18.3, of 1000 21.1 / 21.8, 32 heads over 8 10.5 / 13.7; one of 1000, 32 heads 9.3 / 7.6, 64 of 1000 64.7 / 61.3; 16 of 2000
  // 35.5 / 33.8.
  p.whole = runs == 1 || limit <= kWholeTokens || (limit <= 1024 && p.items >= 128 && p.items <= 1024);
  // CTAs to an SM: registers; stages of 192 KB an SM in all.  Three for one head of 128, of two stages each, where each has many items or tiles.  us, two / three: 94
  // contexts of 1, 32 heads 20.9 / 16.2, 64 of 200 23.5 / 20.2, 83 of 425, 40 heads 56.0 / 51.3, 64 of 2000 112 / 109; 16 of 600 15.5 / 17.4, 16 of 4096 61.1 / 61.6.
  const bool many = p.whole ? p.items >= 2 * 3 * kNumSMs : tiles >= 50 * 3 * kNumSMs;
  p.per_sm = p.GP == 16 ? 1 : (head_dim == 64 && p.GP <= 2) || (p.GP == 1 && many) ? 3 : 2;
  const long long most = p.whole ? p.items : runs > 1 ? runs : (tiles + kLeast - 1) / kLeast;
  p.ctas = static_cast<int>(most < p.per_sm * kNumSMs ? (most > 1 ? most : 1) : p.per_sm * kNumSMs);
  p.partial = p.whole ? 0 : 2LL * p.ctas * p.GP * (head_dim + 2);
  return p;
}
}  // namespace dec8

long long paged_attn_fp8_t5_scratch(int batch, int heads, int kv_heads, int head_dim, int limit, int runs) {
  return dec8::plan_of(batch, heads, kv_heads, head_dim, limit, runs).partial;
}

int launch_paged_attn_fp8_t5(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                             const int* block_tables, int max_blocks, const int* context_lens, void* out, float* partial, int batch, int heads, int kv_heads,
                             int head_dim, int blocks, int block_size, int limit, int runs, float scale, cudaStream_t s) {
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
  const Plan p = plan_of(batch, heads, kv_heads, head_dim, limit, runs);
  if (p.partial > 0 && partial == nullptr) return static_cast<int>(cudaErrorInvalidValue);
  if (p.items * ((limit + kTile - 1) / kTile) >= (1LL << 30)) return static_cast<int>(cudaErrorInvalidValue);      // tiles are counted in 31 bits
  const int items = static_cast<int>(p.items);
  const Work work{context_lens, batch, kv_heads * p.parts, limit, kLeast, p.whole, items / p.ctas, items % p.ctas, FastDiv(static_cast<uint32_t>(kv_heads * p.parts))};
  auto launch = [&](auto kern, auto merge) {
    const int room = (p.per_sm == 1 ? 225 : p.per_sm == 2 ? 110 : 72) * 1024, fit = (room - fixed_smem(head_dim, columns(p.GP))) / stage_bytes(head_dim);
    const int stages = fit < kMaxStages ? fit : kMaxStages, smem = fixed_smem(head_dim, columns(p.GP)) + stages * stage_bytes(head_dim);
    cudaError_t e = allow_smem(kern, smem);
    if (e == cudaSuccess)
      e = launch_dependent(kern, p.ctas, kThreads, smem, s, tmK, tmV, (const __nv_bfloat16*)q, q_stride, k_scale, v_scale, block_tables, max_blocks, work,
                           partial, (__nv_bfloat16*)out, blocks, block_size, FastDiv(static_cast<uint32_t>(block_size)), box_rows, kv_heads, group, stages,
                           scale * kLog2e, wait_byte);
    if (e == cudaSuccess && !p.whole)
      e = launch_dependent(merge, dim3(work.per_sequence * p.GP, batch), head_dim, 0, s, partial, (__nv_bfloat16*)out, work, p.ctas, kv_heads, group);
    return static_cast<int>(e);
  };
#define LLMCTL_DECODE8(D, GP) launch(paged_attn_decode_fp8_t5_kernel<D, GP>, paged_attn_merge_fp8_t5_kernel<D, GP>)
#define LLMCTL_DECODE8_OF(D) \
  (p.GP == 1 ? LLMCTL_DECODE8(D, 1) : p.GP == 2 ? LLMCTL_DECODE8(D, 2) : p.GP == 4 ? LLMCTL_DECODE8(D, 4) : p.GP == 8 ? LLMCTL_DECODE8(D, 8) : LLMCTL_DECODE8(D, 16))
  return head_dim == 128 ? LLMCTL_DECODE8_OF(128) : LLMCTL_DECODE8_OF(64);
#undef LLMCTL_DECODE8_OF
#undef LLMCTL_DECODE8
}

}  // namespace llmctl
