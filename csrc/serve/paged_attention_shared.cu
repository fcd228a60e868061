// Decode attention over a paged cache of 16 bits in which groups of sequences begin with the same blocks (completions of one prompt): those tokens are read once
// for a group, each sequence's own after them.
//     o_b = sum_j 2^(s_bj - m) v_j / sum_j 2^(s_bj - m),      s_bj = scale log2(e) q_b k_j,      j over the shared tokens and over b's own
//
// A group's part of a head of the cache has (sequences x query heads of that head) rows of queries, a sequence's own part its query heads alone: both are items of
// the same form, 128 rows of queries against a range of tokens, and one kernel walks over all of them:
//     S = Q K^T       128 rows x 64 tokens, over D          (A: Q, B: the key tile as it was loaded, both K-major)
//     O += P V        128 rows x D, over 64 tokens          (A: P in tensor memory, B: the value tile as it was loaded, N-major)
// A row is a thread's: maxima and sums need no exchange.  A weight is two numbers of bf16, itself and what that leaves of it (2^-16 of it is lost at most), each multiplied
// with the values; as one, off by up to 2^-8, they make 1.1 to 1.4 times the error of the output's own rounding and cost less: us, one / two, cases below, 46.7 / 50.5, 85 / 91.5,
// 112 / 123, 223 / 248, 9.6 / 9.7 (the second product alone: its numbers computed and not multiplied take nothing).  That is what the sequences read by themselves get, and how many completions a prompt has should not show in their numbers.  The reference of a row
// moves when a score is beyond it by 8 (log2), and O is multiplied then.
//
// Items of at most 32 rows (64) stand in the 128 four times (twice), and each of the four softmax warps (pair of them) takes a quarter (half) of a tile's columns, with zeros
// for weights elsewhere and a reference of its own: a tile's exponentials, 8 clocks for each column of a warp, are shared between the warps.  The copies are
// parts of their own for the merge.
//
//   warp 0      TMA producer: a box for each cache block and 64 columns; keys and values of the tiles in one ring of stages
//   warp 1      MMA issuer: the next tile's scores while this one's become weights
//   warps 2-5   queries into shared memory, scores to weights, O to memory
//
// Bound by the pass over the cache: us with the merge, sequences x (shared + own tokens), 32 heads of 128: 16 x (50000 + 2000) 235 - 248 (its bytes at the copy rate 179; 203
// in this kernel by itself, the power limit holds the clocks of passes back to back), 32 x (4096 + 256) 50 (24; 2.5 of start, 1.5 between the kernels, 6.5 of merge), 67 in 8 groups x (8000 + 1001), 8 heads of the cache 88 - 92 (54); 40 heads, 48 in 3
// groups x (400 + 777) 118 - 123 (78: the ends of items, one after the other in each CTA), 128 in 4 groups x (512 + 10) 84 (8: 17 items to a CTA, 5300 clocks each); 12 heads of 64, 4 x
// (288 + 20) 9.7: launches and the chain of one item.  The products of rows that nobody has cost little: a tile's three are 768 clocks, its 32 KB take 1350 to come.  Two CTAs to an SM, so that one's loads are on their way while the other waits
// for its item's last ones.
//
// The tiles of all items stand in one row, places in front of each item for what it costs beside its tiles, and the CTAs take equal runs of it.  What a CTA finds for an item,
// O at its reference and the reference and the sum of each row, goes to memory at 128 c + (rows of the items before), c the CTA: a place of its own, since from each part to
// the next at least one of the two grows by the part's rows.  A second kernel puts the parts together.
//
// Every wait is bounded, as in latent_attention_t5.cu.
// Reference: none.
#include "../common/dependent.cuh"
#include "../common/fast_div.h"
#include "../common/ptx.cuh"
#include "../common/tma_host.h"
#include "../common/util.cuh"
#include "../common/wait_status.h"

#include <type_traits>

namespace llmctl {
using namespace ptx;

namespace decs {
constexpr int kTile = 64, kRows = 128, kThreads = 192, kCtas = 2 * kNumSMs;
constexpr float kLog2e = 1.4426950408889634f, kSlack = 8.f;

struct Work {
  const int* lens;
  const int* starts;               // [groups + 1]
  const int* shared;               // [groups]
  int batch, groups, per_head, kv_heads, limit, box;       // query heads of a cache head; tokens that the tables hold; rows of a copy
  int* found;                      // [groups + batch + 1][8]: of each entry what the merge has to know (Found)
  float* parts;                    // [capacity][D + 4]
  long long capacity;
  FastDiv by_head;                 // by per_head

  __device__ __forceinline__ int tokens(int b) const { return max(min(lens[b], limit), 0); }
  __device__ __forceinline__ int start(int g) const { return max(min(starts[g], batch), 0); }
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
// How often the rows of an item stand in the 128, and how many rows its parts are.
__device__ __forceinline__ int copies(int rows) { return rows <= 32 ? 4 : rows <= 64 ? 2 : 1; }
__device__ __forceinline__ int stored(int rows) { return rows * copies(rows); }
// Places in front of an item of an entry of so many rows: what it costs beside its tiles.  O of many rows takes 3400 clocks to leave, of one row 1000 (48 sequences of 3 groups, 400 tokens
// shared and 777 of their own, 40 heads: the CTAs with the groups' items ended 15 us after the others, at 105, and end with them now; us with 1 place for all 122, with 2 for
// those 117).  Stored
// side by side, [D / 4][rows], it leaves faster and is gathered slower (119; 32 sequences of 4096 + 256 tokens 47.5 -> 52).
__device__ __forceinline__ int front(int rows) { return rows >= 8 ? 2 : 1; }
// The items of one range of tokens: a group's shared ones (e < groups), or those that sequence e - groups has behind them.
struct Entry {
  int first, count;                // sequences; the first one's table is read
  int t0, t1, from, tiles;         // tokens; the first tile's first
  int rows, row_tiles;             // of queries, for a head of the cache
  __device__ __forceinline__ int items(const Work& w) const { return w.kv_heads * row_tiles; }
  __device__ __forceinline__ int places() const { return tiles + front(rows); }                       // of an item
  __device__ __forceinline__ int rows_of(int row_tile) const { return min(rows - row_tile * kRows, kRows); }
  __device__ __forceinline__ int stored_rows() const { return (row_tiles - 1) * kRows + stored(rows_of(row_tiles - 1)); }         // for a head of the cache
};
__device__ __forceinline__ Entry entry_of(const Work& w, int e) {
  Entry r;
  const bool own = e >= w.groups;
  const int mine = own ? w.lens[e - w.groups] : 0, g = own ? w.group_of(e - w.groups) : e;
  int first = 0, end = 0, shared = 0;
  if (g >= 0) {
    shared = w.shared[g];
    first = w.start(g), end = w.start(g + 1);
    shared = end - first < 2 ? 0 : max(min(shared, w.tokens(first)), 0);          // a group of one shares nothing
  }
  r.first = own ? e - w.groups : first;
  r.count = own ? 1 : max(end - first, 0);
  r.t0 = own ? shared : 0;
  r.t1 = own ? max(min(mine, w.limit), 0) : shared;
  r.from = r.t0 & ~(w.box - 1);             // (a power of two)
  r.tiles = r.t1 > r.t0 ? (r.t1 - r.from + kTile - 1) / kTile : 0;
  r.rows = r.count * w.per_head;
  r.row_tiles = (r.rows + kRows - 1) / kRows;
  return r;
}
struct alignas(16) Found {
  int places, rows;                // of the items before the entry
  int tiles, count, first;         // of it; tiles of the last one (behind all entries): nothing, places of all items
  int group;                       // of a sequence's own: the group that it has shared tokens with, or -1
  int none[2];
};
// Equal runs of `all` places.  (A quotient of at most some hundred: an approximate one is off by one at most.)
__device__ __forceinline__ int quotient(int n, int d) {
  const unsigned q = __float2uint_rz(__fdividef(static_cast<float>(n), static_cast<float>(d))), all = n, of = d;
  return static_cast<int>(q * of > all ? q - 1 : (q + 1) * of <= all ? q + 1 : q);
}
struct Runs {
  int run, longer;
  __device__ __forceinline__ explicit Runs(int all) : run(all / kCtas), longer(all % kCtas) {}
  __device__ __forceinline__ int begin(int c) const { return c * run + min(c, longer); }
  __device__ __forceinline__ int owner(int place) const {
    const int cut = longer * (run + 1);
    return place < cut ? quotient(place, run + 1) : longer + quotient(place - cut, max(run, 1));
  }
};
// A CTA's run, part by part: tiles t .. t + n of an item of entry e, n > 0.
struct Parts {
  Entry entry;
  int e, t, n, left;
  int head, row_tile;              // the item of the entry
  int rows_before;                 // of the items before this one
  __device__ __forceinline__ Parts(const Work& w, int e_, int in, int left_, int rows_before_) : e(e_), t(0), n(0), left(left_), head(0), row_tile(0), rows_before(rows_before_) {
    if (left == 0) return;
    entry = entry_of(w, e);
    if (entry.tiles == 0) {        // (lengths that change meanwhile)
      left = 0;
      return;
    }
    const int x = in / entry.places();
    head = x / entry.row_tiles;
    row_tile = x - head * entry.row_tiles;
    rows_before += head * entry.stored_rows() + row_tile * kRows;
    take(in - x * entry.places());     // (n = 0: the run ends in front of the item)
  }
  // The item's places from `from` on.
  __device__ __forceinline__ void take(int from) {
    const int places = min(entry.places() - from, left);
    left -= places;
    const int before = front(entry.rows);
    t = max(from - before, 0);
    n = max(places - max(before - from, 0), 0);
  }
  __device__ __forceinline__ bool more() const { return n > 0; }
  __device__ __forceinline__ int row0() const { return row_tile * kRows; }
  __device__ __forceinline__ int rows() const { return entry.rows_of(row_tile); }
  __device__ __forceinline__ void next(const Work& w) {
    n = 0;
    if (left == 0) return;
    rows_before += stored(rows());
    if (++row_tile == entry.row_tiles) row_tile = 0, ++head;
    if (head == w.kv_heads) {
      head = 0;
      do {
        if (++e >= w.groups + w.batch) {
          left = 0;
          return;
        }
        entry = entry_of(w, e);
      } while (entry.tiles == 0);
    }
    const int places = min(entry.places(), left);
    left -= places;
    t = 0;
    n = max(places - front(entry.rows), 0);            // 0: the run ends in front of the item
  }
};
constexpr int stage_bytes(int D) { return kTile * D * 2; }
constexpr int stages(int D) { return D == 64 ? 8 : 4; }        // of keys and values in turn
constexpr int smem_bytes(int D) { return kRows * D * 2 + stages(D) * stage_bytes(D) + 1024; }
}  // namespace decs

template <int D>
__global__ void __launch_bounds__(decs::kThreads, 2)
paged_attn_shared_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* q, long long q_stride,
                         const int* tables, int max_blocks, decs::Work w, int blocks, FastDiv by_block, float scale_log2, unsigned char* wait_byte) {
  using namespace decs;
  constexpr int kPanels = D / 64, kPanel = kTile * 128, kQPanel = kRows * 128, kStage = stage_bytes(D), kStages = stages(D), kQ = kRows * D * 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], empty[kStages], q_full, s_full, s_read, p_full, o_full;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag, scan[2][kThreads / 32], found[4];

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(&q_full, 4);
    mbar_init(&s_full, 1);
    mbar_init(&s_read, 4);
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
  const uint32_t tS = tmem_base_smem, tP = tS + kTile, tO = tS + 128;
  static_assert(2 * kTile <= 128 && 128 + D <= 256);
  wait_for_previous(q, tables, w.lens, w.starts, w.shared, w.found, w.parts);
  release_dependents();
  volatile int* abort = &abort_flag;

  // The run: places and rows before each entry, by all threads, an entry each; CTA 0 leaves them for the merge.
  const int entries = w.groups + w.batch, cta = blockIdx.x;
  if (threadIdx.x == 0) found[0] = 0, found[1] = 0, found[2] = 0;
  int all = 0, begin = 0, mine = 0;
  Entry x{};
  int own_t = 0, before_t = 0, before_r = 0, all_t = 0, all_r = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {     // sums of all, then where the run begins
    int tiles0 = 0, rows0 = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < entries; e0 += kThreads) {
      const int e = e0 + threadIdx.x;
      if (pass == 0 || entries > kThreads) {           // (else they are at hand)
        int t = 0, r = 0;
        if (e < entries) {
          x = entry_of(w, e);
          if (x.tiles > 0) t = x.items(w) * x.places(), r = w.kv_heads * x.stored_rows();
        }
        own_t = t;
        const int own_r = r;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(0xffffffffu, t, o), b = __shfl_up_sync(0xffffffffu, r, o);
          if (lane >= o) t += a, r += b;
        }
        if (lane == 31) scan[0][warp] = t, scan[1][warp] = r;
        __syncthreads();
        all_t = all_r = 0;
        for (int i = 0; i < kThreads / 32; ++i) {
          if (i == warp) before_t = all_t + t - own_t, before_r = all_r + r - own_r;
          all_t += scan[0][i], all_r += scan[1][i];
        }
        __syncthreads();
      }
      if (pass == 1 && e < entries) {
        const int at = tiles0 + before_t;
        if (begin >= at && begin < at + own_t) found[0] = e, found[1] = begin - at, found[2] = rows0 + before_r;
        if (cta == 0) reinterpret_cast<Found*>(w.found)[e] = Found{at, rows0 + before_r, x.tiles, x.rows, x.first, e < w.groups ? -1 : w.group_of(e - w.groups), {0, 0}};
      }
      tiles0 += all_t;
      rows0 += all_r;
    }
    if (pass == 0) {
      all = tiles0;
      const Runs runs(all);
      begin = runs.begin(cta);
      mine = runs.begin(cta + 1) - begin;
    }
  }
  if (cta == 0 && threadIdx.x == 0) w.found[8 * entries] = all;
  __syncthreads();
  Parts part(w, found[0], found[1], mine, found[2]);

  if (warp == 0) {
    // ------------------------------------ TMA producer: a lane per box ------------------------------------
    // A part's blocks are asked for 32 at a time, a lane each, one such piece ahead: a table's numbers take as long to come as the tiles that stand before them.
    const int boxes = kTile / w.box, box = lane & 15, panel = lane >> 4;
    auto divide = [&](int token, uint32_t& row) { return static_cast<int>(by_block.divide(static_cast<uint32_t>(token), row)); };
    auto first_block = [&](const Parts& p) {
      uint32_t row;
      return divide(p.entry.from + p.t * kTile, row);
    };
    auto last_block = [&](const Parts& p) {
      uint32_t row;
      return divide(min(p.entry.from + (p.t + p.n) * kTile, p.entry.t1) - 1, row);
    };
    Parts ahead = part;
    int piece = 0;                            // of `ahead`
    auto fetch = [&] {
      int id = -1;
      if (!ahead.more()) return id;
      const int at = first_block(ahead) + piece * 32 + lane, last = last_block(ahead);
      if (at <= last) id = tables[static_cast<long long>(ahead.entry.first) * max_blocks + at];
      ++piece;
      if (at - lane + 32 > last) {
        ahead.next(w);
        piece = 0;
      }
      return id;
    };
    int ids = fetch(), next_ids = fetch(), n = 0;
    for (; part.more(); part.next(w)) {
      const int head = part.head, b0 = first_block(part);
      int at = 0;                             // the piece that `ids` is
      for (int i = 0; i < part.n; ++i) {
        const int token = part.entry.from + (part.t + i) * kTile + box * w.box;
        const bool has = panel < kPanels && box < boxes && token < part.entry.t1;
        uint32_t row = 0;
        const int index = (has ? divide(token, row) : b0) - b0;
        if (__shfl_sync(0xffffffffu, index, 0) >= (at + 1) * 32) {
          ids = next_ids;
          next_ids = fetch();
          ++at;
        }
        const int here = __shfl_sync(0xffffffffu, ids, index & 31), there = __shfl_sync(0xffffffffu, next_ids, index & 31);
        int block = index < (at + 1) * 32 ? here : there;
        if (block < 0 || block >= blocks) block = blocks;       // outside of the cache: zeros
        const int bytes = __popc(__ballot_sync(0xffffffffu, has)) * w.box * 128;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const int st = n % kStages;
          if (n >= kStages) mbar_wait_or_abort(&empty[st], ((n / kStages) & 1u) ^ 1u, abort);
          __syncwarp();
          if (lane == 0) mbar_expect_tx(&full[st], bytes);
          __syncwarp();
          if (has) tma_load_4d(smem + kQ + st * kStage + panel * kPanel + box * w.box * 128, kv == 0 ? &tmK : &tmV, &full[st], panel * 64, head, static_cast<int>(row), block);
        }
      }
      for (const int last = (last_block(part) - b0) >> 5; at <= last; ++at) {
        ids = next_ids;
        next_ids = fetch();
      }
      if (__any_sync(0xffffffffu, *abort)) break;
    }
    if (__any_sync(0xffffffffu, *abort))      // copies still in flight land before the shared memory is given back
      for (int i = n > kStages ? n - kStages : 0; i < n; ++i) {
        int none = 0;
        mbar_wait_bounded(&full[i % kStages], (i / kStages) & 1u, &none);
      }
  } else if (warp == 1) {
    // ------------------------------------ MMA issuer ------------------------------------
    constexpr uint32_t id_s = make_idesc_bf16(kRows, kTile, 0u, 0u), id_o = make_idesc_bf16(kRows, D, 0u, 1u);
    const uint64_t q0 = make_smem_desc(smem_base, 16, 1024, 2), k0 = make_smem_desc(smem_base + kQ, 16, 1024, 2), v0 = make_smem_desc(smem_base + kQ, kPanel, 1024, 2);
    int n = 0, item = 0;                      // tiles, items so far
    auto scores = [&](int tile) {             // tile: of all
      const int st = 2 * tile % kStages;
      mbar_wait_or_abort(&full[st], (2 * tile / kStages) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      if (elect_one()) {
        const uint64_t k = k0 + (st * kStage >> 4);
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          umma_ss<1>(tS, q0 + (((c >> 2) * kQPanel + (c & 3) * 32) >> 4), k + (((c >> 2) * kPanel + (c & 3) * 32) >> 4), id_s, c != 0 ? 1u : 0u);
        umma_commit<1>(&empty[st]);
        umma_commit<1>(&s_full);
      }
    };
    for (; part.more(); part.next(w), ++item) {
      mbar_wait_or_abort(&q_full, item & 1u, abort);
      scores(n);
      for (int i = 0; i < part.n; ++i, ++n) {
        mbar_wait_or_abort(&s_read, n & 1u, abort);
        if (i + 1 < part.n) scores(n + 1);
        const int st = (2 * n + 1) % kStages;
        mbar_wait_or_abort(&full[st], ((2 * n + 1) / kStages) & 1u, abort);
        mbar_wait_or_abort(&p_full, n & 1u, abort);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = v0 + (st * kStage >> 4);
#pragma unroll
          for (int c = 0; c < kTile / 8; ++c)               // 16 tokens' weights, and their rests
            umma_ts<1>(tO, tP + c * 8, v + ((c >> 1) * 2048 >> 4), id_o, (i | c) != 0 ? 1u : 0u);
          umma_commit<1>(&empty[st]);
          umma_commit<1>(&o_full);
        }
      }
      if (__any_sync(0xffffffffu, *abort)) break;
    }
  } else {
    // ------------------------------------ a row of queries per thread ------------------------------------
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    int n = 0, item = 0;
    // Where the row stands: copy `copy` of the item's row `in`.
    struct Row {
      int copy, in;
    };
    auto row_of = [&](int rows) {
      const int f = copies(rows);
      return Row{f == 4 ? quad : f == 2 ? quad >> 1 : 0, f == 4 ? lane : f == 2 ? (quad & 1) * 32 + lane : row};
    };
    auto query = [&](const Parts& p, int in) {          // of the item's row
      uint32_t of_head;
      const int b = p.entry.first + static_cast<int>(w.by_head.divide(p.row0() + in, of_head));
      return reinterpret_cast<const uint4*>(q + static_cast<long long>(b) * q_stride + (p.head * w.per_head + of_head) * D);
    };
    // Items of at most 32 rows: a warp has a quarter of each row's queries and writes it to the four copies.  The next item's are asked for ahead.
    constexpr int kQuarter = D / 32;          // pieces of 16 bytes
    uint4 ahead[kQuarter] = {};
    auto ask = [&](const Parts& p) {
#pragma unroll
      for (int c = 0; c < kQuarter; ++c) ahead[c] = make_uint4(0, 0, 0, 0);
      if (p.more() && p.rows() <= 32 && lane < p.rows()) {
        const uint4* src = query(p, lane) + quad * kQuarter;
#pragma unroll
        for (int c = 0; c < kQuarter; ++c) ahead[c] = src[c];
      }
    };
    auto put = [&](int to_row, int c, uint4 x) { *reinterpret_cast<uint4*>(smem + to_row * 128 + (c >> 3) * kQPanel + (((c & 7) ^ (to_row & 7)) << 4)) = x; };
    // Puts an item's queries where the products read them.  The weights' columns that other warps have are zeros, and stay so from item to item of one form.
    int form = 0;
    auto begin_item = [&](const Parts& p) {
      const int rows = p.rows(), f = copies(rows);
      if (f == 4) {
#pragma unroll
        for (int c = 0; c < kQuarter; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k) put(k * 32 + lane, quad * kQuarter + c, ahead[c]);
      } else {
        const Row me = row_of(rows);
        const uint4* src = query(p, me.in < rows ? me.in : 0);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) put(row, c, me.in < rows ? src[c] : make_uint4(0, 0, 0, 0));
      }
      if (f != form) {
        if (n > 0) mbar_wait_or_abort(&o_full, (n - 1) & 1u, abort);
        __syncwarp();
        tc_fence_after();
        const uint32_t zero[8] = {};
#pragma unroll
        for (int c = 0; c < kTile; c += 8) tmem_st_x8(tP + lane_off + c, zero);
        tmem_st_wait();
        form = f;
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    };
    ask(part);
    if (part.more()) begin_item(part);
    while (part.more()) {
      const int rows = part.rows(), t1 = part.entry.t1, t0 = part.entry.t0, tiles = part.n, from0 = part.entry.from + part.t * kTile, f = copies(rows);
      const Row me = row_of(rows);
      const bool mine = me.in < rows, any = f == 4 || (f == 2 ? (quad & 1) : quad) * 32 < rows;
      int limit = t1;                         // of this row's tokens
      uint32_t of_head;
      if (mine) limit = min(w.tokens(part.entry.first + static_cast<int>(w.by_head.divide(part.row0() + me.in, of_head))), t1);
      const long long at = static_cast<long long>(kRows) * cta + part.rows_before + me.copy * rows + me.in;
      part.next(w);
      float m = -INFINITY, l = 0.f;

      // The tile before has been multiplied: O may be read and P written.  (All warps wait for each, since a phase more would look like one less.)
      auto before_done = [&](int i) {
        if (i != 0) mbar_wait_or_abort(&o_full, (n - 1) & 1u, abort);
        __syncwarp();
        tc_fence_after();
      };
      auto tile = [&](auto columns, int i, int from) {
        constexpr int C = decltype(columns)::value, kChunk = C == 16 ? 16 : 32;
        const uint32_t at_s = tS + lane_off + me.copy * C;
        const int lo = t0 - from - me.copy * C, hi = limit - from - me.copy * C;         // columns lo .. hi - 1 count
        const bool cut = __any_sync(0xffffffffu, lo > 0 || hi < C);
        // 64 columns are read twice, 32 at a time: they and the weights would not fit a thread's registers.
        uint32_t s[kChunk];
        auto read = [&](int c0) {
          if constexpr (C == 16) tmem_ld_x16(at_s, s);
          else tmem_ld_x32(at_s + c0, s);
          tmem_ld_wait();
          if (cut) {
#pragma unroll
            for (int c = 0; c < kChunk; ++c)
              if (c0 + c < lo || c0 + c >= hi) s[c] = 0xff800000u;
          }
        };
        auto have_read = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_read);
        };
        float top = -INFINITY;
#pragma unroll
        for (int c0 = 0; c0 < C; c0 += kChunk) {
          read(c0);
#pragma unroll
          for (int c = 0; c < kChunk; c += 2) top = max3(top, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
        }
        if constexpr (C == kChunk) have_read();
        top *= scale_log2;
        const bool moves = top > m + kSlack || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, moves)) {
          const float to = moves ? top : m, factor = moves ? ex2_approx(m - top) : 1.f;
          if (i != 0) {
            before_done(i);
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld_x16(tO + lane_off + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
              tmem_st_x16(tO + lane_off + c, o);
            }
          }
          l *= factor;
          m = to;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float l2 = 0.f;
        if constexpr (C != kChunk) before_done(i);
#pragma unroll 1
        for (int c0 = 0; c0 < C; c0 += kChunk) {
          if constexpr (C != kChunk) read(c0);
          if (C != kChunk && c0 + kChunk == C) have_read();
#pragma unroll
          for (int c1 = 0; c1 < kChunk; c1 += 16) {
            uint32_t p[16];                    // of 16 tokens eight columns of what bf16 holds, and eight of the rest
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float a = ex2_approx(fmaf(__uint_as_float(s[c1 + 2 * c]), scale_log2, -ref)), z = ex2_approx(fmaf(__uint_as_float(s[c1 + 2 * c + 1]), scale_log2, -ref));
              p[c] = pack_bf16x2(a, z);
              p[8 + c] = pack_bf16x2(a - __uint_as_float(p[c] << 16), z - __uint_as_float(p[c] & 0xffff0000u));
              add2(l, l2, a, z);
            }
            if (C == kChunk && c1 == 0) before_done(i);
            tmem_st_x16(tP + lane_off + me.copy * C + c0 + c1, p);
          }
        }
        l += l2;
        tmem_st_wait();
      };
      for (int i = 0; i < tiles; ++i, ++n) {
        const int from = from0 + i * kTile;
        mbar_wait_or_abort(&s_full, n & 1u, abort);
        __syncwarp();
        tc_fence_after();
        if (any) {
          if (f == 4) tile(std::integral_constant<int, 16>(), i, from);
          else if (f == 2) tile(std::integral_constant<int, 32>(), i, from);
          else tile(std::integral_constant<int, 64>(), i, from);
        } else {
          if (lane == 0) mbar_arrive(&s_read);
          before_done(i);
        }
        if (i == 0) ask(part);
        if (from + kTile > t1) {              // what stands behind the last token may be anything
          const int st = (2 * n + 1) % kStages;
          mbar_wait_or_abort(&full[st], ((2 * n + 1) / kStages) & 1u, abort);
          uint8_t* dst = smem + kQ + st * kStage + (t1 - from) * 128;
#pragma unroll 1
          for (int c = 0; c < kPanels; ++c)
            for (int i = row; i < (from + kTile - t1) * 8; i += kRows) *reinterpret_cast<uint4*>(dst + c * kPanel + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full);
      }
      // This item's scores have all been taken, so the next one's queries may stand in the place of its own, and their scores come while O is finished and read.
      if (part.more()) begin_item(part);
      mbar_wait_or_abort(&o_full, (n - 1) & 1u, abort);
      __syncwarp();
      tc_fence_after();
      if (any) {
        float* to = w.parts + at * (D + 4);
        const bool fits = mine && at >= 0 && at < w.capacity;          // (groups that overlap may count past 32 bits)
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
      ++item;
      if (__any_sync(0xffffffffu, *abort)) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<1>(tS, 256);
  if (threadIdx.x == 0 && abort_flag) report_wait(wait_byte);
}

// W warps (1 or 4) per sequence and query head: the parts of its group's shared tokens and of its own.  Each warp finds the parts' weights for itself, a lane to a part, and
// adds up every Wth part's row.  Grid: heads / (4 / W), rounded up, x sequences.
template <int D, int W>
__global__ void __launch_bounds__(128, W == 4 ? 8 : 5) paged_attn_shared_merge_kernel(decs::Work w, __nv_bfloat16* out) {
  using namespace decs;
  constexpr int kPer = D / 32, kUnderWay = W == 4 ? 4 : 8;
  __shared__ float rows_of_warps[W][D];
  wait_for_previous(w.found, w.parts, out);
  release_dependents();
  const int warp = W == 4 ? threadIdx.x >> 5 : 0, lane = threadIdx.x & 31, b = blockIdx.y, h = W == 4 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
  uint32_t of_head;
  const int head = static_cast<int>(w.by_head.divide(h, of_head));
  if (h >= w.kv_heads * w.per_head) return;
  const Found* found = reinterpret_cast<const Found*>(w.found);
  const int all = found[w.groups + w.batch].places;
  const Found own = found[w.groups + b];
  Found group = own;
  if (w.groups <= 32) {                      // a lane to each, beside the sequence's: one after the other they come 0.7 us later
    const Found x = found[min(lane, max(w.groups - 1, 0))];
    const int from = max(own.group, 0);
    group.places = __shfl_sync(0xffffffffu, x.places, from);
    group.rows = __shfl_sync(0xffffffffu, x.rows, from);
    group.tiles = __shfl_sync(0xffffffffu, x.tiles, from);
    group.count = __shfl_sync(0xffffffffu, x.count, from);
    group.first = __shfl_sync(0xffffffffu, x.first, from);
  } else if (own.group >= 0) {
    group = found[own.group];
  }
  if (own.group < 0) group.tiles = 0;
  const Runs runs(all);
  // An item's parts: the first one's row, how many CTAs have parts, how many copies of how many rows a part is.
  struct Item {
    long long first;
    int count, f, rows;
  };
  auto item = [&](const Found& x) {
    if (x.tiles == 0) return Item{0, 0, 1, 0};
    const int r = (b - x.first) * w.per_head + static_cast<int>(of_head), row_tile = r / kRows, row_tiles = (x.count + kRows - 1) / kRows, rows = min(x.count - row_tile * kRows, kRows);
    const int stored_rows = (row_tiles - 1) * kRows + stored(x.count - (row_tiles - 1) * kRows), f = copies(rows);
    const int place0 = x.places + (head * row_tiles + row_tile) * (x.tiles + front(x.count)) + front(x.count), c0 = runs.owner(place0);
    return Item{static_cast<long long>(kRows) * c0 + x.rows + head * stored_rows + row_tile * kRows + r % kRows, (runs.owner(place0 + x.tiles - 1) - c0 + 1) * f, f, rows};
  };
  const Item common = item(group), mine = item(own);
  const int parts = common.count + mine.count;
  float o[kPer] = {}, m = -INFINITY, l = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const int i = i0 + lane, n = min(parts - i0, 32);
    float2 ml = make_float2(-INFINITY, 0.f);
    long long at = 0;
    if (i < parts) {
      const bool first = i < common.count;
      const int j = first ? i : i - common.count, f = first ? common.f : mine.f, c = j / f;
      at = (first ? common.first : mine.first) + static_cast<long long>(kRows) * c + (j - c * f) * (first ? common.rows : mine.rows);
      if (at >= 0 && at < w.capacity) ml = *reinterpret_cast<const float2*>(w.parts + at * (D + 4) + D);
      else at = 0;
    }
    // Rows under way at once, the first ones beside their weights: of parts that do not count some other row is read and not used.
    float v[kUnderWay][kPer];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int k = 0; k < kUnderWay; ++k) {
        const float* row = w.parts + __shfl_sync(0xffffffffu, at, min(warp + W * (k0 + k), n - 1)) * (D + 4) + lane * kPer;
        if (W * (k0 + k) >= n) continue;
        if constexpr (kPer == 4) *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(row);
        else *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(row);
      }
    };
    fetch(0);
    const bool counts = !(ml.y == 0.f);      // else: no token that counts
    const float to = fmaxf(m, warp_max(counts ? ml.x : -INFINITY));
    const float z = !counts ? 0.f : ml.x == to ? 1.f : ex2_approx(ml.x - to), a = m == to ? 1.f : ex2_approx(m - to);
    l = l * a + warp_sum(counts ? ml.y * z : 0.f);
    m = to;
    const unsigned which = __ballot_sync(0xffffffffu, counts);
#pragma unroll
    for (int k = 0; k < kPer; ++k) o[k] *= a;
    for (int k0 = 0; k0 * W < n; k0 += kUnderWay) {
      if (k0 > 0) fetch(k0);
#pragma unroll
      for (int k = 0; k < kUnderWay; ++k) {
        const int part = warp + W * (k0 + k);
        const float factor = __shfl_sync(0xffffffffu, z, min(part, n - 1));
        const bool use = part < n && (which >> (part & 31) & 1u);
#pragma unroll
        for (int c = 0; c < kPer; ++c) o[c] = use ? fmaf(v[k][c], factor, o[c]) : o[c];
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* to = out + (static_cast<long long>(b) * w.kv_heads * w.per_head + h) * D;
  if constexpr (W == 1) {
#pragma unroll
    for (int c = 0; c < kPer; c += 2) *reinterpret_cast<__nv_bfloat162*>(to + lane * kPer + c) = __floats2bfloat162_rn(o[c] * inv, o[c + 1] * inv);
  } else {
#pragma unroll
    for (int c = 0; c < kPer; ++c) rows_of_warps[warp][lane * kPer + c] = o[c];
    __syncthreads();
    if (threadIdx.x < D) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) v += rows_of_warps[k][threadIdx.x];
      to[threadIdx.x] = __float2bfloat16(v * inv);
    }
  }
}

namespace {
// Floats of scratch: the sums before each entry, then the parts.
long long parts_at(int batch, int groups) { return 8LL * (groups + batch + 1); }
long long capacity_of(int batch, int heads) { return static_cast<long long>(decs::kRows) * decs::kCtas + 8LL * batch * heads; }
int box_rows(int block_size) {
  int box = 1;
  while (box < decs::kTile && block_size % (2 * box) == 0) box *= 2;
  return box;
}

template <int D>
cudaError_t launch(const CUtensorMap& k, const CUtensorMap& v, const __nv_bfloat16* q, long long q_stride, const int* tables, int max_blocks, const decs::Work& w, __nv_bfloat16* out,
                   int blocks, int block_size, float scale, unsigned char* byte, cudaStream_t s) {
  using namespace decs;
  const auto kernel = paged_attn_shared_kernel<D>;
  if (const cudaError_t e = allow_smem(kernel, smem_bytes(D)); e != cudaSuccess) return e;
  if (const cudaError_t e = launch_dependent(kernel, kCtas, kThreads, smem_bytes(D), s, k, v, q, q_stride, tables, max_blocks, w, blocks, FastDiv(block_size), scale * kLog2e, byte); e != cudaSuccess)
    return e;
  // Four warps to a sequence and head while all of them are on the chip at once, else one.
  const int heads = w.kv_heads * w.per_head;
  if (w.batch * heads <= 8 * kNumSMs) return launch_dependent(paged_attn_shared_merge_kernel<D, 4>, dim3(heads, w.batch), 128, 0, s, w, out);
  return launch_dependent(paged_attn_shared_merge_kernel<D, 1>, dim3((heads + 3) / 4, w.batch), 128, 0, s, w, out);
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
  LLMCTL_REQUIRE(2LL * batch * heads * ((limit >> 6) + 5) < (1LL << 31) && 8LL * batch * heads < (1LL << 30));
  const int box = box_rows(block_size);
  CUtensorMap k, v;
  const uint64_t D = head_dim, Hk = kv_heads, row = D * Hk;
  for (int i = 0; i < 2; ++i)
    if (const int e = get_tmap_4d_bf16(i ? &v : &k, i ? v_cache : k_cache, D, Hk, block_size, blocks, D, row, row * block_size, 64, 1, box, 1, 1); e != 0) LLMCTL_FAIL(e, "tensor map");
  unsigned char* const byte = wait_report(kWaitPagedShared);
  LLMCTL_REQUIRE(byte != nullptr);
  decs::Work w = {context_lens, group_starts, shared_lens, batch, groups, heads / kv_heads, kv_heads, static_cast<int>(limit), box, reinterpret_cast<int*>(scratch),
                  scratch + parts_at(batch, groups), capacity_of(batch, heads), FastDiv(heads / kv_heads)};
  const auto* qs = static_cast<const __nv_bfloat16*>(q);
  auto* o = static_cast<__nv_bfloat16*>(out);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  LLMCTL_CHECK(head_dim == 64 ? launch<64>(k, v, qs, q_stride, block_tables, max_blocks, w, o, blocks, block_size, scale, byte, s)
                              : launch<128>(k, v, qs, q_stride, block_tables, max_blocks, w, o, blocks, block_size, scale, byte, s));
  return 0;
}
