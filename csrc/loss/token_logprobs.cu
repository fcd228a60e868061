// Log probabilities of given tokens under rows of logits, each row's entropy and its most probable tokens; and the gradient of the logits.
//
//   m = max_j x_j,  s = sum_j exp(x_j - m),  l_j = (x_j - m) - log s,  p_j = exp(l_j)
//   logprob = l[token],   entropy H = -sum_j p_j l_j = log s - sum_j exp(x_j - m) (x_j - m) / s,   top: the largest l_j, of equal ones the lowest index first
//   dx_j = -p_j ((g + sum_i gt_i) + gH (l_j + H)) + g [j = token] + sum_i gt_i [j = id_i]        g, gH, gt: gradients of the three
//
// Forward: a row to a CTA, or to a cluster of up to 8 where rows are few, in one pass: every thread keeps a running maximum, the two sums over it and where its
// maximum stands.  The k-th largest of 64 groups' maxima bounds the k-th largest logit from below, so that only the units of threads whose own maximum
// reaches it are looked through again (of 32000 numbers some 25 are candidates for 20 places), and a candidate's rank is the number of
// larger ones.  All sums in fp32.
//
// 2000 x 50257 in 32 bits 68 us (5.9 TB/s: the pass over the logits bounds it), 4096 x 32000 bf16 48 us (5.4 TB/s; instructions and exponentials are as near: two
// thirds of either's rate), 64 x 32000 with 5 alternatives 6.3 us, one row with 20 6.9 us (the chain of a cluster's exchanges).
// Backward: 4096 x 32000 bf16 86 us (6.1 TB/s over logits and their gradient), in 32 bits 168 (6.2).
//
// Reference: none — the reference offers neither (its server returns text alone, reference llmctl/serve/server.py:57-75).
#include <type_traits>

#include "../common/dependent.cuh"
#include "../common/ptx.cuh"
#include "../common/util.cuh"

namespace llmctl {

namespace lp {
constexpr int kThreads = 256, kWarps = kThreads / 32, kGroups = 64, kMaxTop = kGroups, kMaxCandidates = 1024, kMaxCluster = 8, kAhead = 4;
constexpr int kResident = 4 * kNumSMs;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -200.f;             // 2^-200 is 0: what lies lower counts as this, so that -inf times its weight is 0 and no NaN
constexpr float kLow = -1e30f, kUsual = -1e29f;      // beside a maximum above kUsual numbers below kLow weigh nothing, and may be kLow
constexpr float kMost = 1e30f, kMostGrad = 1e7f;     // up to here differences to a maximum, and their products with the entropy's gradient, are finite with no floor

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T>
constexpr int kUnit = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void unpack(const uint4& raw, float (&f)[8]) { unpack8(*reinterpret_cast<const bf16x8*>(&raw), f); }
__device__ __forceinline__ void unpack(const uint4& raw, float (&f)[4]) {
  f[0] = __uint_as_float(raw.x), f[1] = __uint_as_float(raw.y), f[2] = __uint_as_float(raw.z), f[3] = __uint_as_float(raw.w);
}
// A unit of -inf
__device__ __forceinline__ uint4 nothing(const __nv_bfloat16*) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ uint4 nothing(const float*) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
// The same, but no number below kLow; NaN stays.
__device__ __forceinline__ void unpack_clamped(const uint4& raw, float (&f)[8]) {
  bf16x8 v = *reinterpret_cast<const bf16x8*>(&raw);
  const __nv_bfloat162 low = __float2bfloat162_rn(kLow);
#pragma unroll
  for (int i = 0; i < 4; ++i) v.v[i] = __hmax2_nan(v.v[i], low);
  unpack8(v, f);
}
__device__ __forceinline__ void unpack_clamped(const uint4& raw, float (&f)[4]) {
  unpack(raw, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = max_nan(f[i], kLow);
}
// NaN has no part.
__device__ __forceinline__ float largest(const uint4& raw, const __nv_bfloat16*) {
  const bf16x8 v = *reinterpret_cast<const bf16x8*>(&raw);
  const float2 m = __bfloat1622float2(__hmax2(__hmax2(v.v[0], v.v[1]), __hmax2(v.v[2], v.v[3])));
  return fmaxf(m.x, m.y);
}
__device__ __forceinline__ float largest(const uint4& raw, const float*) {
  return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
}
__device__ __forceinline__ void store_unit(__nv_bfloat16* p, const float (&f)[8]) { store8(p, pack8(f)); }
__device__ __forceinline__ void store_unit(float* p, const float (&f)[4]) { *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(f); }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float f) { *p = __float2bfloat16(f); }
__device__ __forceinline__ void store_one(float* p, float f) { *p = f; }

// A row as the numbers before its first 16-byte boundary, whole units, and the rest.
template <typename T>
struct Row {
  const T* p;
  int head, units, V;
  __device__ Row(const T* at, int n) : p(at), V(n) {
    head = min(n, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(at) & 15u)) & 15u) / static_cast<int>(sizeof(T)));
    units = (n - head) / kUnit<T>;
  }
  __device__ int tail() const { return head + units * kUnit<T>; }
};

// Larger numbers first, of equal ones (0 and -0 are) the one with the lower index; NaN counts as -inf.  0: none.
__device__ __forceinline__ unsigned long long make_key(float v, int index) {
  const uint32_t u = __float_as_uint(v != v ? -INFINITY : v + 0.f);
  const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(order) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int key_index(unsigned long long k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_number(unsigned long long k) {
  const uint32_t order = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
__device__ __forceinline__ unsigned long long key_max(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long reduce_key(unsigned long long k, int lanes) {
  for (int o = lanes / 2; o > 0; o >>= 1) k = key_max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

// (d0, d1) += (a0, a1) * (b0, b1)
__device__ __forceinline__ void fma2w(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rd, {%0, %1};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rd;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "+f"(d0), "+f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ float load_cluster_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long load_cluster_u64(uint32_t at) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void store_cluster_u64(uint32_t at, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ int add_cluster(uint32_t at, int v) {
  int old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.s32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
  return old;
}

// Running maximum m, sum of 2^u and of 2^u u over u = (x - m) log2 e.
struct Sums {
  float m = -INFINITY, s = 0.f, t = 0.f;
  __device__ __forceinline__ void move_to(float to) {          // to > m, or m if it is -inf
    const float u = max_nan((m - to) * kLog2e, kFloor), a = ptx::ex2_approx(u);
    t = (t + s * u) * a;
    s *= a;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {
    const float u = max_nan((x - (m == -INFINITY ? 0.f : m)) * kLog2e, kFloor), e = ptx::ex2_approx(u);
    s += e;
    t += e * u;
  }
  // Numbers above kLow beside a maximum between kUsual and kMost.
  template <int U>
  __device__ __forceinline__ void add_usual(const float (&x)[U]) {
    float s2[2] = {0.f, 0.f}, t2[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < U; j += 2) {
      float u0, u1;
      ptx::add2v(u0, u1, x[j], x[j + 1], -m, -m);
      ptx::mul2(u0, u1, u0, u1, kLog2e);
      const float e0 = ptx::ex2_approx(u0), e1 = ptx::ex2_approx(u1);
      ptx::add2(s2[0], s2[1], e0, e1);
      fma2w(t2[0], t2[1], e0, e1, u0, u1);
    }
    s += s2[0] + s2[1];
    t += t2[0] + t2[1];
  }
  __device__ __forceinline__ void join(float om, float os, float ot) {
    Sums o;
    o.m = om, o.s = os, o.t = ot;
    if (o.m > m) move_to(o.m);
    else if (m > o.m) o.move_to(m);
    s += o.s;
    t += o.t;
  }
};
}  // namespace lp

// Grid: clusters of `cluster` CTAs, one to a row.  As many CTAs to an SM as hide the loads of each other's turns, in few registers: 4096 x 32000 in 16 bits
// 4: 57.3 us, 6: 50.6, 8: 48.4; in 32 bits 4: 82.6, 5: 82.5, 6: 80.1, 8: 86.3, 2000 x 50257 4: 68.0, 5: 68.5, 6: 71.9.
template <typename T, bool kCluster>
__global__ void __launch_bounds__(lp::kThreads, sizeof(T) == 2 ? 8 : 5)
token_logprobs_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tokens, int V, int top, float* __restrict__ logprobs,
                      float* __restrict__ entropy, float* __restrict__ stats, long long* __restrict__ top_ids, float* __restrict__ top_logprobs, int cluster) {
  using namespace lp;
  constexpr int U = kUnit<T>;
  __shared__ float red[3][kWarps], sums[3];
  __shared__ unsigned long long group_key[kGroups], all_keys[kGroups], candidates[kMaxCandidates], bound;
  __shared__ int count, listed, list[kThreads];
  wait_for_previous(logits, tokens, logprobs, entropy, stats, top_ids, top_logprobs);
  release_dependents();
  const int part = kCluster ? static_cast<int>(ptx::cluster_ctarank()) : 0, parts = kCluster ? cluster : 1;
  const long long row = kCluster ? blockIdx.x / static_cast<unsigned>(parts) : blockIdx.x;
  const Row<T> r(logits + row * ld, V);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = kCluster ? (r.units + parts - 1) / parts : r.units, lo = part * per, hi = min(r.units, lo + per);       // this CTA's units
  const int head = part == 0 ? r.head : 0, tail = part == parts - 1 ? r.tail() : V;
  const long long token = tokens[row];
  float x_token = 0.f;
  const bool given = token >= 0 && token < V;
  if (tid == 0 && part == 0 && given) x_token = as_f32(r.p[token]);
  auto unit = [&](int i) { return r.p + r.head + static_cast<long long>(i) * U; };

  // Numbers are met in the order of their indices: before the first 16-byte boundary, units, the rest.  The reference moves once in kAhead units (some lane of a
  // warp has a new maximum in nearly each of a row's first, and the others wait: 4096 x 32000 76 us with a look at every unit, 64.9 so); the unit of the
  // maximum is kept, its place in it is looked up at the end.
  Sums a;
  int best = tid < head ? tid : -1, best_unit = tid >= head && lo + tid < hi ? lo + tid : -1;      // where the maximum stands, one of the two
  if (best < 0 && best_unit < 0 && tail + tid < V) best = tail + tid;
  auto one = [&](int at) {
    const float x = as_f32(r.p[at]);
    if (x > a.m) {
      a.move_to(x);
      best = at;
      best_unit = -1;
    }
    a.add(x);
  };
  if (tid < head) one(tid);
  auto turn = [&](int i0, auto whole) {       // kAhead units; not whole: those behind the last count as -inf
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) raw[k] = whole.value || i0 + k * kThreads < hi ? load_raw(unit(i0 + k * kThreads)) : nothing(r.p);
    float of[kAhead], most = -INFINITY;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      of[k] = largest(raw[k], r.p);
      most = fmaxf(most, of[k]);
    }
    if (most > a.m) {
      a.move_to(most);
      int k = 0;
#pragma unroll
      for (int e = kAhead - 1; e >= 0; --e)
        if (of[e] == most) k = e;
      best_unit = i0 + k * kThreads;
    }
    const bool usual = a.m > kUsual && a.m < kMost;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float x[U];
      if (usual) {
        unpack_clamped(raw[k], x);
        a.add_usual(x);
      } else {
        unpack(raw[k], x);
#pragma unroll
        for (int j = 0; j < U; ++j) a.add(x[j]);
      }
    }
  };
  int i0 = lo + tid;
  for (; i0 + (kAhead - 1) * kThreads < hi; i0 += kAhead * kThreads) turn(i0, std::true_type());
  if (i0 < hi) turn(i0, std::false_type());
  if (tail + tid < V) one(tail + tid);
  unsigned long long key = 0ull;              // of this thread's maximum
  if (top > 0 && best_unit >= 0) {
    float x[U];
    unpack(load_raw(unit(best_unit)), x);
    int j = 0;
#pragma unroll
    for (int e = U - 1; e >= 0; --e)
      if (x[e] == a.m) j = e;
    best = r.head + best_unit * U + j;
  }
  if (top > 0 && best >= 0) key = make_key(a.m, best);

  // One reference for the CTA, then plain sums (joining pairs of sums at each step of a tree was a third of the instructions at 32000 numbers).
  {
    const float m = ptx::warp_max_all(a.m);   // NaN has no part in it: it is in the sums
    if (lane == 0) red[0][warp] = m;
  }
  const int groups = kGroups / parts;         // of this CTA
  if (top > 0) {
    const unsigned long long k = reduce_key(key, kThreads / groups);
    if (tid % (kThreads / groups) == 0) group_key[tid / (kThreads / groups)] = k;
  }
  if (tid == 0) {
    count = listed = 0;
    bound = 0ull;
  }
  __syncthreads();
  Sums all;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all.m = fmaxf(all.m, red[0][w]);
  if (all.m > a.m) a.move_to(all.m);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  if (lane == 0) red[1][warp] = a.s, red[2][warp] = a.t;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    all.s += red[1][w];
    all.t += red[2][w];
  }
  if (kCluster) {
    if (tid == 0) sums[0] = all.m, sums[1] = all.s, sums[2] = all.t;
    ptx::cluster_sync();
    if (part == 0)
      for (int c = 1; c < parts; ++c) {
        const uint32_t at = ptx::mapa_u32(ptx::smem_u32(sums), c);
        all.join(load_cluster_f32(at), load_cluster_f32(at + 4), load_cluster_f32(at + 8));
      }
  }
  const float log2_s = log2f(all.s), log_s = log2_s * kLn2;
  if (tid == 0 && part == 0) {
    logprobs[row] = given ? (x_token - all.m) - log_s : 0.f;
    entropy[row] = kLn2 * (log2_s - all.t / all.s);
    if (stats != nullptr) {
      stats[2 * row] = all.m;
      stats[2 * row + 1] = log_s;
    }
  }
  if (top == 0) {
    if (kCluster) ptx::cluster_sync();        // nobody's shared memory goes before it was read
    return;
  }

  auto write = [&](int place, unsigned long long k) {
    top_ids[row * top + place] = key_index(k);
    top_logprobs[row * top + place] = (key_number(k) - all.m) - log_s;
  };
  // the top-th largest of the groups' maxima: keys are unlike but for groups without numbers
  if (tid < kGroups) all_keys[tid] = kCluster ? load_cluster_u64(ptx::mapa_u32(ptx::smem_u32(group_key + tid % groups), tid / groups)) : group_key[tid];
  __syncthreads();
  if (tid < kGroups) {
    const unsigned long long mine = all_keys[tid];
    int larger = 0;
#pragma unroll 16
    for (int i = 0; i < kGroups; ++i) larger += all_keys[i] > mine;
    if (larger == top - 1 && mine != 0ull) bound = mine;
    if (top == 1 && part == 0 && larger == 0 && mine != 0ull) write(0, mine);
  }
  if (top == 1) {
    if (kCluster) ptx::cluster_sync();
    return;
  }
  __syncthreads();
  const unsigned long long least = bound;
  if (key >= least && key != 0ull) list[atomicAdd(&listed, 1)] = tid;
  __syncthreads();
  // the candidates, in the first CTA's shared memory
  const uint32_t count_at = kCluster ? ptx::mapa_u32(ptx::smem_u32(&count), 0) : 0u, list_at = kCluster ? ptx::mapa_u32(ptx::smem_u32(candidates), 0) : 0u;
  auto collect = [&](float x, int at) {
    const unsigned long long k = make_key(x, at);
    if (k < least) return;
    const int i = kCluster ? add_cluster(count_at, 1) : atomicAdd(&count, 1);
    if (i >= kMaxCandidates) return;
    if (kCluster) store_cluster_u64(list_at + i * 8, k);
    else candidates[i] = k;
  };
  if (tid < head) collect(as_f32(r.p[tid]), tid);
  if (tail + tid < V) collect(as_f32(r.p[tail + tid]), tail + tid);
  const int each = (hi - lo + kThreads - 1) / kThreads;            // units of a thread
  for (int w = tid; w < listed * each; w += kThreads) {
    const int i = lo + list[w / each] + w % each * kThreads;
    if (i >= hi) continue;
    float x[U];
    unpack(load_raw(unit(i)), x);
#pragma unroll
    for (int j = 0; j < U; ++j) collect(x[j], r.head + i * U + j);
  }
  if (kCluster) ptx::cluster_sync();
  else __syncthreads();
  if (part != 0) return;
  const int n = count;
  if (n <= kMaxCandidates) {
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long mine = candidates[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += candidates[j] > mine;
      if (place < top) write(place, mine);
    }
    return;
  }
  // Rows whose largest numbers stand in few threads' units: one place after the other, each by a pass over the row.
  unsigned long long last = ~0ull;
  for (int place = 0; place < top; ++place) {
    unsigned long long k = 0ull;
    for (int i = tid; i < V; i += kThreads) {
      const unsigned long long c = make_key(as_f32(r.p[i]), i);
      if (c < last) k = key_max(k, c);
    }
    k = reduce_key(k, 32);
    __syncthreads();                          // the maxima of the place before have been read
    if (lane == 0) group_key[warp] = k;
    __syncthreads();
    last = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) last = key_max(last, group_key[w]);
    if (tid == 0) write(place, last);
  }
}

// Gradient of the logits, read and written once; the chosen places are written again at the end.  Grid: (rows, parts of a row).  d_top: rows of `top`, or null.
template <typename T>
__global__ void __launch_bounds__(lp::kThreads, 4)
token_logprobs_bwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tokens, int V, int top, const float* __restrict__ stats,
                          const float* __restrict__ entropy, const long long* __restrict__ top_ids, const float* __restrict__ d_logprobs,
                          const float* __restrict__ d_entropy, const float* __restrict__ d_top, T* __restrict__ dx, long long ldd) {
  using namespace lp;
  constexpr int U = kUnit<T>;
  wait_for_previous(logits, tokens, stats, entropy, top_ids, d_logprobs, d_entropy, d_top, dx);
  release_dependents();
  const long long row = blockIdx.x;
  const Row<T> r(logits + row * ld, V);
  T* out = dx + row * ldd;
  const int tid = threadIdx.x;
  const long long token = tokens[row];
  const bool given = token >= 0 && token < V;
  const float g = given && d_logprobs != nullptr ? d_logprobs[row] : 0.f, gh = d_entropy != nullptr ? d_entropy[row] : 0.f;
  float total = g;
  if (d_top != nullptr)
    for (int i = 0; i < top; ++i) total += d_top[row * top + i];
  const float m = stats[2 * row], log_s = stats[2 * row + 1], h = entropy[row], rest = -(total + gh * h);
  auto gradient = [&](float x) {
    const float l = max_nan((x - m) - log_s, kFloor);
    return ptx::ex2_approx(l * kLog2e) * fmaf(-gh, l, rest);
  };
  const int parts = gridDim.y, part = blockIdx.y, per = (r.units + parts - 1) / parts, lo = part * per, hi = min(r.units, lo + per);
  const int from = part == 0 ? 0 : r.head + lo * U, to = part == parts - 1 ? V : r.head + hi * U;        // this CTA's numbers
  const bool usual = m > kUsual && m < kMost && fabsf(gh) < kMostGrad;
  for (int i0 = lo + tid; i0 < hi; i0 += kAhead * kThreads) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k * kThreads < hi) raw[k] = load_raw(r.p + r.head + static_cast<long long>(i0 + k * kThreads) * U);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kThreads;
      if (i >= hi) break;
      float x[U];
      if (usual) {
        unpack_clamped(raw[k], x);
#pragma unroll
        for (int j = 0; j < U; j += 2) {
          float l0, l1, u0, u1;
          ptx::add2v(l0, l1, x[j], x[j + 1], -m, -m);
          ptx::add2v(l0, l1, l0, l1, -log_s, -log_s);
          ptx::mul2(u0, u1, l0, l1, kLog2e);
          ptx::fma2(l0, l1, l0, l1, -gh, rest);
          ptx::mul2v(x[j], x[j + 1], ptx::ex2_approx(u0), ptx::ex2_approx(u1), l0, l1);
        }
      } else {
        unpack(raw[k], x);
#pragma unroll
        for (int j = 0; j < U; ++j) x[j] = gradient(x[j]);
      }
      store_unit(out + r.head + static_cast<long long>(i) * U, x);
    }
  }
  if (part == 0 && tid < r.head) store_one(out + tid, gradient(as_f32(r.p[tid])));
  if (part == parts - 1 && r.tail() + tid < V) store_one(out + r.tail() + tid, gradient(as_f32(r.p[r.tail() + tid])));
  __syncthreads();
  if (d_top != nullptr && tid < top) {
    const long long id = top_ids[row * top + tid];
    if (id >= from && id < to) store_one(out + id, gradient(as_f32(r.p[id])) + d_top[row * top + tid] + (id == token ? g : 0.f));
  }
  if (tid == 0 && given && token >= from && token < to) {
    bool also = false;                        // among the most probable: written there
    if (d_top != nullptr)
      for (int i = 0; i < top; ++i) also |= top_ids[row * top + i] == token;
    if (!also) store_one(out + token, gradient(as_f32(r.p[token])) + g);
  }
}

namespace lp {
// CTAs to a row of the forward: its rounds between them (two or three, 0.5 us each) pay where a thread would have 24 units and more.  us by CTAs to a row, 20
// alternatives: one row of 32000 in 16 bits 1: 7.1, 4: 7.2; 50257 1: 9.5, 2: 8.2, 4: 7.3, 8: 8.0; 130000 1: 17.4, 4: 8.9, 8: 8.7; 256 rows of 32000 1: 8.9,
// 2: 11.5, of 50257 1: 12.9, 2: 14.0, of 130000 1: 28.5, 2: 24.0.
static int cluster_of(int rows, int V, int unit) {
  const int turns = V / unit / kThreads;
  int c = turns >= 48 ? kMaxCluster : turns >= 24 ? 4 : 1;
  while (c > 1 && static_cast<long long>(rows) * c > kResident) c /= 2;
  return c == 2 && turns < 48 ? 1 : c;
}
// CTAs to a row of the backward, which share nothing: as many as fit, of two turns of loads each.
static int parts_of(int rows, int V, int unit) {
  int c = 1;
  while (c < kMaxCluster && static_cast<long long>(rows) * 2 * c <= kResident && V / unit >= 2 * c * kThreads * 2) c *= 2;
  return c;
}
template <typename T>
static cudaError_t launch_logprobs(const void* logits, long long ld, const long long* tokens, int rows, int V, int top, float* logprobs, float* entropy,
                                   float* stats, long long* top_ids, float* top_logprobs, cudaStream_t s) {
  const int c = cluster_of(rows, V, kUnit<T>);
  if (c == 1)
    return launch_dependent(token_logprobs_kernel<T, false>, rows, kThreads, 0, s, (const T*)logits, ld, tokens, V, top, logprobs, entropy, stats, top_ids,
                            top_logprobs, 1);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(c);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * c);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, (const T*)logits, ld, tokens, V, top, logprobs, entropy, stats, top_ids, top_logprobs, c);
}
}  // namespace lp

}  // namespace llmctl

using namespace llmctl;

// logits: rows of V bf16 (or fp32) numbers, ld apart; tokens: int64, outside of 0 .. V - 1: none (its log probability is 0).  logprobs, entropy: fp32
// [rows]; stats: fp32 [rows, 2] (maximum, log of the sum over it) for the gradient, or null; top_ids (int64) and top_logprobs: [rows, top].
LLMCTL_API int llmctl_token_logprobs(const void* logits, int is_fp32, long long ld, const long long* tokens, int rows, int V, int top, float* logprobs,
                                     float* entropy, float* stats, long long* top_ids, float* top_logprobs, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE(rows >= 0 && V >= 1 && V <= 0x7fffffff - 4096 && top >= 0 && top <= lp::kMaxTop && top <= V && (top == 0 || (top_ids != nullptr && top_logprobs != nullptr)));
  LLMCTL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (is_fp32 ? 4 : 2) == 0);
  if (rows == 0) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  LLMCTL_CHECK(is_fp32 ? lp::launch_logprobs<float>(logits, ld, tokens, rows, V, top, logprobs, entropy, stats, top_ids, top_logprobs, s)
                       : lp::launch_logprobs<__nv_bfloat16>(logits, ld, tokens, rows, V, top, logprobs, entropy, stats, top_ids, top_logprobs, s));
  LLMCTL_RETURN_LAST();
}

// dx: rows of V numbers of the logits' type, ldd apart, that lie to 16-byte boundaries as the logits' do.  Gradients that are null are zero.
LLMCTL_API int llmctl_token_logprobs_bwd(const void* logits, int is_fp32, long long ld, const long long* tokens, int rows, int V, int top,
                                         const float* stats, const float* entropy, const long long* top_ids, const float* d_logprobs,
                                         const float* d_entropy, const float* d_top, void* dx, long long ldd, void* stream) {
  LLMCTL_BEGIN();
  const int size = is_fp32 ? 4 : 2;
  LLMCTL_REQUIRE(rows >= 0 && V >= 1 && top >= 0 && top <= lp::kMaxTop && (top == 0 || top_ids != nullptr));
  LLMCTL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0 && ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0 &&
                 (rows <= 1 || ((ld - ldd) * size & 15) == 0));
  if (rows == 0) return 0;
  if (top == 0) d_top = nullptr;
  const dim3 grid(rows, lp::parts_of(rows, V, is_fp32 ? lp::kUnit<float> : lp::kUnit<__nv_bfloat16>));
  if (is_fp32)
    LLMCTL_CHECK(launch_dependent(token_logprobs_bwd_kernel<float>, grid, lp::kThreads, 0, (cudaStream_t)stream, (const float*)logits, ld, tokens, V, top,
                                  stats, entropy, top_ids, d_logprobs, d_entropy, d_top, (float*)dx, ldd));
  else
    LLMCTL_CHECK(launch_dependent(token_logprobs_bwd_kernel<__nv_bfloat16>, grid, lp::kThreads, 0, (cudaStream_t)stream, (const __nv_bfloat16*)logits,
                                  ld, tokens, V, top, stats, entropy, top_ids, d_logprobs, d_entropy, d_top, (__nv_bfloat16*)dx, ldd));
  LLMCTL_RETURN_LAST();
}
