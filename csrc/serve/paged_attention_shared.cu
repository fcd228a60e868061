// Decode attention over a paged cache of 16 bits in which groups of sequences begin with the same blocks (completions of one prompt): those tokens are read once
// for a group, each sequence's own after them.
//     o_b = sum_j 2^(s_bj - m) v_j / sum_j 2^(s_bj - m),      s_bj = scale log2(e) q_b k_j,      j over the shared tokens and over b's own
//
// A group's part of a head of the cache has (sequences x query heads of that head) rows of queries, a sequence's own part its query heads alone: both are items of
// the same form, 128 rows of queries against a range of tokens, and one kernel walks over all of them:
//     S = Q K^T       128 rows x 128 tokens, over D         (A: Q, B: the key tile as it was loaded, both K-major)
//     O += P V        128 rows x D, over 128 tokens         (A: P in tensor memory over S, B: the value tile as it was loaded, N-major)
// A row is a thread's: maxima and sums need no exchange.  Weights are rounded to bf16 (2^-9 of each, beside the output's 2^-9) and summed as they were
// rounded; the reference of a row moves when a score is beyond it by 8 (log2), and O is multiplied then.
//
//   warp 0      TMA producer: a box for each cache block and 64 columns, one stage of keys and one of values
//   warp 1      MMA issuer
//   warps 2-5   queries into shared memory, scores to weights, O to memory
//
// Items with few rows leave most of the products' rows to nobody; the tensor cores have room for that: a tile's two products are 1024 clocks, its 64 KB take 2700
// to come.  Two CTAs to an SM, so that one's tiles are on their way while the other one's are looked at.
//
// The tiles of all items stand in one row, and the CTAs take equal runs of it.  What a CTA finds for an item, O at its reference and the reference and the sum of each row,
// goes to memory at 128 c + (rows of the items before), c the CTA: a place of its own, since from each part to the next at least one of the two grows by the part's rows.  A
// second kernel puts the parts together.
//
// Every wait is bounded, as in latent_attention_t5.cu.
// Reference: none.
#include "../common/dependent.cuh"
#include "../common/ptx.cuh"
#include "../common/tma_host.h"
#include "../common/util.cuh"
#include "../common/wait_status.h"

namespace llmctl {
using namespace ptx;

namespace decs {
constexpr int kTile = 128, kRows = 128, kThreads = 192, kCtas = 2 * kNumSMs;
constexpr float kLog2e = 1.4426950408889634f, kSlack = 8.f;

struct Work {
  const int* lens;
  const int* starts;               // [groups + 1]
  const int* shared;               // [groups]
  int batch, groups, per_head, kv_heads, limit, box;       // query heads of a cache head; tokens that the tables hold; rows of a copy
  int* before;                     // [groups + batch + 1][2]: tiles and rows of the items before an entry
  float* parts;                    // [capacity][D + 4]
  long long capacity;

  __device__ __forceinline__ int tokens(int b) const { return max(min(lens[b], limit), 0); }
  __device__ __forceinline__ int start(int g) const { return max(min(starts[g], batch), 0); }
  // Tokens that a group's sequences share: none of a group of one.
  __device__ __forceinline__ int shared_of(int g, int first, int end) const { return end - first < 2 ? 0 : max(min(shared[g], tokens(first)), 0); }
  // The group that b belongs to, the last one that does not begin behind it; -1: none.
  __device__ __forceinline__ int group_of(int b) const {
    int lo = 0, hi = groups;       // starts[lo] <= b < starts[hi], as far as they are in order
    if (groups == 0 || starts[0] > b) return -1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= b) lo = mid;
      else hi = mid;
    }
    return b < starts[lo + 1] ? lo : -1;
  }
};
// The items of one range of tokens: a group's shared ones (e < groups), or those that sequence e - groups has behind them.
struct Entry {
  int first, count;                // sequences; the first one's table is read
  int t0, t1, from, tiles;         // tokens; the first tile's first
  int rows, row_tiles;             // of queries, for a head of the cache
  __device__ __forceinline__ int items(const Work& w) const { return w.kv_heads * row_tiles; }
};
__device__ __forceinline__ Entry entry_of(const Work& w, int e) {
  Entry r;
  if (e < w.groups) {
    r.first = w.start(e);
    const int end = w.start(e + 1);
    r.count = max(end - r.first, 0);
    r.t0 = 0;
    r.t1 = r.count > 0 ? w.shared_of(e, r.first, end) : 0;
  } else {
    r.first = e - w.groups;
    r.count = 1;
    const int g = w.group_of(r.first);
    r.t0 = 0;
    if (g >= 0) r.t0 = w.shared_of(g, w.start(g), w.start(g + 1));
    r.t1 = w.tokens(r.first);
  }
  r.from = r.t0 - r.t0 % w.box;
  r.tiles = r.t1 > r.t0 ? (r.t1 - r.from + kTile - 1) / kTile : 0;
  r.rows = r.count * w.per_head;
  r.row_tiles = (r.rows + kRows - 1) / kRows;
  return r;
}
// Equal runs of `all` tiles.
struct Runs {
  int run, longer;
  __device__ __forceinline__ Runs(int all, int ctas) : run(all / ctas), longer(all % ctas) {}
  __device__ __forceinline__ int begin(int c) const { return c * run + min(c, longer); }
  __device__ __forceinline__ int owner(int tile) const {
    const int cut = longer * (run + 1);
    return tile < cut ? tile / (run + 1) : longer + (tile - cut) / max(run, 1);
  }
};
// A CTA's run, part by part: tiles t .. t + n of item x of entry e.
struct Parts {
  Entry entry;
  int e, x, t, n, left;
  int rows_before;                 // of the items before this one
  __device__ __forceinline__ Parts(const Work& w, int e_, int tiles_in, int left_, int rows_before_) : e(e_), x(0), t(0), n(0), left(left_), rows_before(rows_before_) {
    if (left == 0) return;
    entry = entry_of(w, e);
    if (entry.tiles == 0) {        // (lengths that change meanwhile)
      left = 0;
      return;
    }
    x = tiles_in / entry.tiles;
    t = tiles_in - x * entry.tiles;
    rows_before += x / entry.row_tiles * entry.rows + x % entry.row_tiles * kRows;
    n = min(entry.tiles - t, left);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ int head() const { return x / entry.row_tiles; }
  __device__ __forceinline__ int row0() const { return x % entry.row_tiles * kRows; }
  __device__ __forceinline__ int rows() const { return min(entry.rows - row0(), kRows); }
  __device__ __forceinline__ void next(const Work& w) {
    left -= n;
    if (left == 0) return;
    rows_before += rows();
    t = 0;
    if (++x == entry.items(w)) {
      x = 0;
      do {
        if (++e >= w.groups + w.batch) {
          left = 0;
          return;
        }
        entry = entry_of(w, e);
      } while (entry.tiles == 0);
    }
    n = min(entry.tiles, left);
  }
};
constexpr int stage_bytes(int D) { return kTile * D * 2; }
constexpr int stages(int D) { return D == 64 ? 2 : 1; }
constexpr int smem_bytes(int D) { return kRows * D * 2 + 2 * stages(D) * stage_bytes(D) + 1024; }
}  // namespace decs

template <int D>
__global__ void __launch_bounds__(decs::kThreads, 2)
paged_attn_shared_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* q, long long q_stride,
                         const int* tables, int max_blocks, decs::Work w, int blocks, int block_size, float scale_log2, unsigned char* wait_byte) {
  using namespace decs;
  constexpr int kPanels = D / 64, kPanel = kTile * 128, kStage = stage_bytes(D), kStages = stages(D), kQ = kRows * D * 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], q_full, s_full, p_full, o_full;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag, scan[2][kThreads / 32], found[4];

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  constexpr int kKAt = kQ, kVAt = kQ + kStages * kStage;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1), mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    mbar_init(&q_full, 4);
    mbar_init(&s_full, 1);
    mbar_init(&p_full, 4);
    mbar_init(&o_full, 1);
    abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 1) tmem_alloc<1>(&tmem_base_smem, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tS = tmem_base_smem, tO = tS + kTile;
  wait_for_previous(q, tables, w.lens, w.starts, w.shared, w.before, w.parts);
  release_dependents();
  volatile int* abort = &abort_flag;

  // The run: tiles and rows before each entry, by all threads, an entry each; CTA 0 leaves them for the merge.
  const int entries = w.groups + w.batch, ctas = gridDim.x, cta = blockIdx.x;
  auto sums_before = [&](int e0, int& tiles, int& rows) {       // of the entries e0 .. e0 + this thread's, itself left out; returns through the last thread's those of all
    int t = 0, r = 0;
    if (e0 + static_cast<int>(threadIdx.x) < entries) {
      const Entry x = entry_of(w, e0 + threadIdx.x);
      t = x.items(w) * x.tiles;
      r = x.tiles > 0 ? w.kv_heads * x.rows : 0;
    }
    const int own_t = t, own_r = r;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, t, o), b = __shfl_up_sync(0xffffffffu, r, o);
      if (lane >= o) t += a, r += b;
    }
    if (lane == 31) scan[0][warp] = t, scan[1][warp] = r;
    __syncthreads();
    int all_t = 0, all_r = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i == warp) tiles = all_t + t - own_t, rows = all_r + r - own_r;
      all_t += scan[0][i], all_r += scan[1][i];
    }
    __syncthreads();
    return make_int3(own_t, all_t, all_r);
  };
  int all = 0;
  int3 sums;
  int tiles, rows;
  for (int e0 = 0; e0 < entries; e0 += kThreads) {
    sums = sums_before(e0, tiles, rows);
    all += sums.y;
  }
  const Runs runs(all, ctas);
  const int begin = runs.begin(cta), mine = runs.begin(cta + 1) - begin;
  if (threadIdx.x == 0) found[0] = 0, found[1] = 0, found[2] = 0;
  __syncthreads();
  int tiles0 = 0, rows0 = 0;
  for (int e0 = 0; e0 < entries; e0 += kThreads) {
    if (entries > kThreads) sums = sums_before(e0, tiles, rows);           // (else they are at hand)
    const int at = tiles0 + tiles;
    if (e0 + static_cast<int>(threadIdx.x) < entries) {
      if (begin >= at && begin < at + sums.x) found[0] = e0 + threadIdx.x, found[1] = begin - at, found[2] = rows0 + rows;
      if (cta == 0) {
        w.before[2 * (e0 + threadIdx.x)] = at;
        w.before[2 * (e0 + threadIdx.x) + 1] = rows0 + rows;
      }
    }
    tiles0 += sums.y;
    rows0 += sums.z;
  }
  if (cta == 0 && threadIdx.x == 0) w.before[2 * entries] = all;
  __syncthreads();
  Parts part(w, found[0], found[1], mine, found[2]);

  if (warp == 0) {
    // ------------------------------------ TMA producer: a lane per box ------------------------------------
    const int boxes = kTile / w.box, box = lane & 15, panel = lane >> 4;
    int n = 0;
    for (; part.more(); part.next(w)) {
      const int head = part.head();
      const int* table = tables + static_cast<long long>(part.entry.first) * max_blocks;
      for (int i = 0; i < part.n; ++i, ++n) {
        const int st = n % kStages, token = part.entry.from + (part.t + i) * kTile + box * w.box;
        const uint32_t empty = ((n / kStages) & 1u) ^ 1u;
        const bool has = panel < kPanels && box < boxes && token < part.entry.t1;
        int block = -1, row = 0;
        if (has) {
          block = table[token / block_size];
          row = token % block_size;
          if (block < 0 || block >= blocks) block = blocks;     // outside of the cache: zeros
        }
        const int count = __popc(__ballot_sync(0xffffffffu, has));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t* full = kv == 0 ? &k_full[st] : &v_full[st];
          if (n >= kStages) mbar_wait_or_abort(kv == 0 ? &k_empty[st] : &v_empty[st], empty, abort);
          __syncwarp();
          if (lane == 0) mbar_expect_tx(full, count * w.box * 128);
          __syncwarp();
          if (has) tma_load_4d(smem + (kv == 0 ? kKAt : kVAt) + st * kStage + panel * kPanel + box * w.box * 128, kv == 0 ? &tmK : &tmV, full, panel * 64, head, row, block);
        }
      }
      if (__any_sync(0xffffffffu, *abort)) break;
    }
    if (__any_sync(0xffffffffu, *abort))      // copies still in flight land before the shared memory is given back
      for (int i = n > kStages ? n - kStages : 0; i < n; ++i) {
        int none = 0;
        mbar_wait_bounded(&k_full[i % kStages], (i / kStages) & 1u, &none);
        mbar_wait_bounded(&v_full[i % kStages], (i / kStages) & 1u, &none);
      }
  } else if (warp == 1) {
    // ------------------------------------ MMA issuer ------------------------------------
    constexpr uint32_t id_s = make_idesc_bf16(kRows, kTile, 0u, 0u), id_o = make_idesc_bf16(kRows, D, 0u, 1u);
    const uint64_t q0 = make_smem_desc(smem_base, 16, 1024, 2), k0 = make_smem_desc(smem_base + kKAt, 16, 1024, 2), v0 = make_smem_desc(smem_base + kVAt, kPanel, 1024, 2);
    int n = 0, item = 0;
    for (; part.more(); part.next(w), ++item) {
      mbar_wait_or_abort(&q_full, item & 1u, abort);
      for (int i = 0; i < part.n; ++i, ++n) {
        const int st = n % kStages;
        const uint32_t phase = (n / kStages) & 1u;
        mbar_wait_or_abort(&k_full[st], phase, abort);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint64_t k = k0 + (st * kStage >> 4);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const uint32_t at = ((c >> 2) * kPanel + (c & 3) * 32) >> 4;
            umma_ss<1>(tS, q0 + at, k + at, id_s, c != 0 ? 1u : 0u);
          }
          umma_commit<1>(&k_empty[st]);
          umma_commit<1>(&s_full);
        }
        mbar_wait_or_abort(&v_full[st], phase, abort);
        mbar_wait_or_abort(&p_full, n & 1u, abort);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = v0 + (st * kStage >> 4);
#pragma unroll
          for (int c = 0; c < kTile / 16; ++c) umma_ts<1>(tO, tS + c * 8, v + (c * 2048 >> 4), id_o, (i | c) != 0 ? 1u : 0u);
          umma_commit<1>(&v_empty[st]);
          if (i + 1 == part.n) umma_commit<1>(&o_full);
        }
      }
      if (__any_sync(0xffffffffu, *abort)) break;
    }
  } else {
    // ------------------------------------ a row of queries per thread ------------------------------------
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    int n = 0, item = 0;
    for (; part.more(); part.next(w), ++item) {
      const int rows = part.rows(), r = part.row0() + row, b = part.entry.first + r / w.per_head;
      const bool mine = row < rows, any = quad * 32 < rows;
      int limit = part.entry.t1;
      if (any) {
        const uint4* src = reinterpret_cast<const uint4*>(q + static_cast<long long>(b) * q_stride + (part.head() * w.per_head + r % w.per_head) * D);
        uint8_t* dst = smem + row * 128;
        if (mine) limit = min(w.tokens(b), part.entry.t1);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (mine) x = src[c];
          *reinterpret_cast<uint4*>(dst + (c >> 3) * kPanel + (((c & 7) ^ (row & 7)) << 4)) = x;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < part.n; ++i, ++n) {
        const int st = n % kStages, from = part.entry.from + (part.t + i) * kTile;
        mbar_wait_or_abort(&s_full, n & 1u, abort);
        __syncwarp();
        tc_fence_after();
        if (any) {
          const int lo = part.entry.t0 - from, hi = limit - from;          // columns lo .. hi - 1 count
          const bool cut = __any_sync(0xffffffffu, lo > 0 || hi < kTile);
          // Scores are read twice, 64 columns at a time: all 128 and the weights would not fit a thread's registers.
          auto scores = [&](int at, uint32_t (&s)[64]) {
            tmem_ld_x32(tS + lane_off + at, s);
            tmem_ld_x32(tS + lane_off + at + 32, s + 32);
            tmem_ld_wait();
            if (cut) {
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (at + c < lo || at + c >= hi) s[c] = 0xff800000u;
            }
          };
          float top = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t s[64];
            scores(h * 64, s);
#pragma unroll
            for (int c = 0; c < 64; c += 2) top = max3(top, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
          }
          top *= scale_log2;
          const bool moves = top > m + kSlack || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, moves)) {
            const float to = moves ? top : m, factor = moves ? ex2_approx(m - top) : 1.f;
            if (i != 0) {
#pragma unroll
              for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld_x32(tO + lane_off + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                tmem_st_x32(tO + lane_off + c, o);
              }
            }
            l *= factor;
            m = to;
          }
          const float ref = m == -INFINITY ? 0.f : m;
          float l2 = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t s[64], p[32];
            scores(h * 64, s);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float a = ex2_approx(fmaf(__uint_as_float(s[2 * c]), scale_log2, -ref)), z = ex2_approx(fmaf(__uint_as_float(s[2 * c + 1]), scale_log2, -ref));
              p[c] = pack_bf16x2(a, z);
              add2(l, l2, __uint_as_float(p[c] << 16), __uint_as_float(p[c] & 0xffff0000u));
            }
            tmem_st_x32(tS + lane_off + h * 32, p);            // over scores that have been read
          }
          l += l2;
          tmem_st_wait();
        }
        if (from + kTile > part.entry.t1) {   // what stands behind the last token may be anything
          mbar_wait_or_abort(&v_full[st], (n / kStages) & 1u, abort);
          if (from + row >= part.entry.t1) {
            uint8_t* dst = smem + kVAt + st * kStage + row * 128;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(dst + (c >> 3) * kPanel + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full);
      }
      mbar_wait_or_abort(&o_full, item & 1u, abort);
      __syncwarp();
      tc_fence_after();
      if (any) {
        const long long at = static_cast<long long>(kRows) * cta + part.rows_before + row;
        float* to = w.parts + at * (D + 4);
        const bool fits = mine && at < w.capacity;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld_x32(tO + lane_off + c, o);
          tmem_ld_wait();
          if (fits) {
#pragma unroll
            for (int k = 0; k < 32; k += 4) st_v4(to + c + k, make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]));
          }
        }
        if (fits) st_v4(to + D, make_uint4(__float_as_uint(m), __float_as_uint(l), 0u, 0u));
      }
      tc_fence_before();
      if (__any_sync(0xffffffffu, *abort)) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<1>(tS, 256);
  if (threadIdx.x == 0 && abort_flag) report_wait(wait_byte);
}

// A warp per sequence and query head: the parts of its group's shared tokens and of its own.
template <int D>
__global__ void __launch_bounds__(128) paged_attn_shared_merge_kernel(decs::Work w, __nv_bfloat16* out, int ctas) {
  using namespace decs;
  constexpr int kPer = D / 32;
  wait_for_previous(w.lens, w.starts, w.shared, w.before, w.parts, out);
  release_dependents();
  const int lane = threadIdx.x & 31, heads = w.kv_heads * w.per_head, at = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (at >= w.batch * heads) return;
  const int b = at / heads, h = at - b * heads, head = h / w.per_head;
  const Runs runs(w.before[2 * (w.groups + w.batch)], ctas);
  float o[kPer] = {}, m = -INFINITY, l = 0.f;
  auto add = [&](int e) {
    const Entry x = entry_of(w, e);
    if (x.tiles == 0) return;
    const int r = (b - x.first) * w.per_head + h % w.per_head, row_tile = r / kRows;
    const int tile0 = w.before[2 * e] + (head * x.row_tiles + row_tile) * x.tiles, c1 = runs.owner(tile0 + x.tiles - 1);
    const long long rows = static_cast<long long>(w.before[2 * e + 1]) + head * x.rows + r;
    for (int c = runs.owner(tile0); c <= c1; ++c) {
      const long long place = static_cast<long long>(kRows) * c + rows;
      if (place >= w.capacity) return;
      const float* part = w.parts + place * (D + 4);
      const float2 ml = *reinterpret_cast<const float2*>(part + D);
      float v[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) v[k] = part[lane * kPer + k];
      if (ml.y == 0.f) continue;           // no token that counts
      const float to = fmaxf(m, ml.x), a = m == to ? 1.f : ex2_approx(m - to), z = ml.x == to ? 1.f : ex2_approx(ml.x - to);
      l = l * a + ml.y * z;
#pragma unroll
      for (int k = 0; k < kPer; ++k) o[k] = o[k] * a + v[k] * z;
      m = to;
    }
  };
  const int g = w.group_of(b);
  if (g >= 0) add(g);
  add(w.groups + b);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* to = out + static_cast<long long>(at) * D + lane * kPer;
#pragma unroll
  for (int k = 0; k < kPer; k += 2) *reinterpret_cast<__nv_bfloat162*>(to + k) = __floats2bfloat162_rn(o[k] * inv, o[k + 1] * inv);
}

namespace {
// Floats of scratch: the sums before each entry, then the parts.
long long parts_at(int batch, int groups) { return (2LL * (groups + batch + 1) + 3) / 4 * 4; }
long long capacity_of(int batch, int heads) { return static_cast<long long>(decs::kRows) * decs::kCtas + 2LL * batch * heads; }
int box_rows(int block_size) {
  int box = 1;
  while (box < 128 && block_size % (2 * box) == 0) box *= 2;
  return box;
}

template <int D>
cudaError_t launch(const CUtensorMap& k, const CUtensorMap& v, const __nv_bfloat16* q, long long q_stride, const int* tables, int max_blocks, const decs::Work& w, __nv_bfloat16* out,
                   int blocks, int block_size, float scale, unsigned char* byte, cudaStream_t s) {
  using namespace decs;
  const auto kernel = paged_attn_shared_kernel<D>;
  if (const cudaError_t e = allow_smem(kernel, smem_bytes(D)); e != cudaSuccess) return e;
  if (const cudaError_t e = launch_dependent(kernel, kCtas, kThreads, smem_bytes(D), s, k, v, q, q_stride, tables, max_blocks, w, blocks, block_size, scale * kLog2e, byte); e != cudaSuccess)
    return e;
  const int all = w.batch * w.kv_heads * w.per_head;
  return launch_dependent(paged_attn_shared_merge_kernel<D>, (all + 3) / 4, 128, 0, s, w, out, static_cast<int>(kCtas));
}
}  // namespace
}  // namespace llmctl

using namespace llmctl;

LLMCTL_API long long llmctl_paged_attn_shared_scratch_elems(int batch, int groups, int heads, int head_dim) {
  if (batch <= 0 || groups < 0 || heads <= 0 || head_dim <= 0) return 0;
  return parts_at(batch, groups) + capacity_of(batch, heads) * (head_dim + 4);
}

LLMCTL_API int llmctl_paged_attn_decode_shared(const void* q, long long q_stride, const void* k_cache, const void* v_cache, const int* block_tables, int max_blocks,
                                               const int* context_lens, const int* group_starts, const int* shared_lens, void* out, float* scratch, int batch, int groups, int heads,
                                               int kv_heads, int head_dim, int blocks, int block_size, float scale, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE(batch > 0 && batch < 65536 && groups >= 0 && groups <= 65536 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 4096 && blocks > 0);
  LLMCTL_REQUIRE((head_dim == 64 || head_dim == 128) && block_size > 0 && block_size % 8 == 0 && max_blocks >= 0);
  LLMCTL_REQUIRE(aligned16(q, k_cache, v_cache, out, scratch) && scratch != nullptr && q_stride % 8 == 0);
  const long long limit = static_cast<long long>(max_blocks) * block_size;
  LLMCTL_REQUIRE(limit < (1LL << 31) - 256);
  // tiles of all items, and rows, count in 32 bits
  LLMCTL_REQUIRE(2LL * batch * heads * ((limit >> 7) + 2) < (1LL << 31) && 2LL * batch * heads < (1LL << 30));
  const int box = box_rows(block_size);
  CUtensorMap k, v;
  const uint64_t D = head_dim, Hk = kv_heads, row = D * Hk;
  for (int i = 0; i < 2; ++i)
    if (const int e = get_tmap_4d_bf16(i ? &v : &k, i ? v_cache : k_cache, D, Hk, block_size, blocks, D, row, row * block_size, 64, 1, box, 1, 1); e != 0) LLMCTL_FAIL(e, "tensor map");
  unsigned char* const byte = wait_report(kWaitPagedShared);
  LLMCTL_REQUIRE(byte != nullptr);
  decs::Work w = {context_lens, group_starts, shared_lens, batch, groups, heads / kv_heads, kv_heads, static_cast<int>(limit), box, reinterpret_cast<int*>(scratch),
                  scratch + parts_at(batch, groups), capacity_of(batch, heads)};
  const auto* qs = static_cast<const __nv_bfloat16*>(q);
  auto* o = static_cast<__nv_bfloat16*>(out);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  LLMCTL_CHECK(head_dim == 64 ? launch<64>(k, v, qs, q_stride, block_tables, max_blocks, w, o, blocks, block_size, scale, byte, s)
                              : launch<128>(k, v, qs, q_stride, block_tables, max_blocks, w, o, blocks, block_size, scale, byte, s));
  return 0;
}
