// Log probabilities of given tokens under rows of logits, each row's entropy and its most probable tokens; and the gradient of the logits.
//
//   m = max_j x_j,  s = sum_j exp(x_j - m),  l_j = (x_j - m) - log s,  p_j = exp(l_j)
//   logprob = l[token],   entropy H = -sum_j p_j l_j = log s - sum_j exp(x_j - m) (x_j - m) / s,   top: the largest l_j, of equal ones the lowest index first
//   dx_j = -p_j ((g + sum_i gt_i) + gH (l_j + H)) + g [j = token] + sum_i gt_i [j = id_i]        g, gH, gt: gradients of the three
//
// Forward: a CTA per row, one pass: every thread keeps a running maximum, the two sums over it and where its maximum stands.  The k-th largest of 64 groups'
// maxima bounds the k-th largest logit from below, so that only threads whose own maximum reaches it look through their numbers again (of the
// row's 32000 some 25 are candidates for 20 places), and a candidate's rank is the number of larger ones.  All sums in fp32.
//
// Reference: none — the reference offers neither (its server returns text alone, reference llmctl/serve/server.py:57-75).
#include "../common/dependent.cuh"
#include "../common/ptx.cuh"
#include "../common/util.cuh"

namespace llmctl {

namespace lp {
constexpr int kThreads = 512, kWarps = kThreads / 32, kGroups = 64, kMaxTop = kGroups, kMaxCandidates = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -200.f;             // 2^-200 is 0: what lies lower counts as this, so that -inf times its weight is 0 and no NaN

template <typename T>
constexpr int kUnit = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void load_unit(const __nv_bfloat16* p, float (&f)[8]) { unpack8(load8(p), f); }
__device__ __forceinline__ void load_unit(const float* p, float (&f)[4]) { *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p); }
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
__device__ __forceinline__ unsigned long long key_max(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
template <int kLanes>
__device__ __forceinline__ unsigned long long reduce_key(unsigned long long k) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) k = key_max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
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

template <typename T>
__global__ void __launch_bounds__(lp::kThreads, 2)
token_logprobs_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tokens, int V, int top, float* __restrict__ logprobs,
                      float* __restrict__ entropy, float* __restrict__ stats, long long* __restrict__ top_ids, float* __restrict__ top_logprobs) {
  using namespace lp;
  constexpr int U = kUnit<T>;
  __shared__ float red[3][kWarps];
  __shared__ unsigned long long group_key[kGroups], candidates[kMaxCandidates], bound;
  __shared__ int count;
  wait_for_previous(logits, tokens, logprobs, entropy, stats, top_ids, top_logprobs);
  release_dependents();
  const long long row = blockIdx.x;
  const Row<T> r(logits + row * ld, V);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long token = tokens[row];
  float x_token = 0.f;
  const bool given = token >= 0 && token < V;
  if (tid == 0 && given) x_token = as_f32(r.p[token]);

  // what this thread goes through, in the order of the indices: f(number, index) for single ones, g(unit, first index) for whole units
  auto walk = [&](auto&& f, auto&& g) {
    if (tid < r.head) f(as_f32(r.p[tid]), tid);
#pragma unroll 2
    for (int i = tid; i < r.units; i += kThreads) {
      float x[U];
      load_unit(r.p + r.head + i * U, x);
      g(x, r.head + i * U);
    }
    const int at = r.tail() + tid;
    if (at < V) f(as_f32(r.p[at]), at);
  };

  Sums a;
  int best = tid < r.head ? tid : tid < r.units ? r.head + tid * U : r.tail() + tid;      // where the maximum stands; >= V: no numbers
  walk(
      [&](float x, int at) {
        if (x > a.m) {
          a.move_to(x);
          best = at;
        }
        a.add(x);
      },
      [&](const float (&x)[U], int at) {
        float most = x[0];
#pragma unroll
        for (int j = 1; j < U; ++j) most = fmaxf(most, x[j]);
        if (most > a.m) {
          a.move_to(most);
          int j = 0;
#pragma unroll
          for (int i = U - 1; i >= 0; --i)
            if (x[i] == most) j = i;
          best = at + j;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) a.add(x[j]);
      });
  unsigned long long key = best < V ? make_key(a.m, best) : 0ull;

#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a.join(__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o));
  if (lane == 0) red[0][warp] = a.m, red[1][warp] = a.s, red[2][warp] = a.t;
  if (top > 0) {
    const unsigned long long k = reduce_key<kThreads / kGroups>(key);
    if (tid % (kThreads / kGroups) == 0) group_key[tid / (kThreads / kGroups)] = k;
  }
  if (tid == 0) {
    count = 0;
    bound = 0ull;
  }
  __syncthreads();
  Sums all;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all.join(red[0][w], red[1][w], red[2][w]);
  const float log2_s = log2f(all.s), log_s = log2_s * kLn2;
  if (tid == 0) {
    logprobs[row] = given ? (x_token - all.m) - log_s : 0.f;
    entropy[row] = kLn2 * (log2_s - all.t / all.s);
    if (stats != nullptr) {
      stats[2 * row] = all.m;
      stats[2 * row + 1] = log_s;
    }
  }
  if (top == 0) return;

  auto write = [&](int place, unsigned long long k) {
    const int index = key_index(k);
    top_ids[row * top + place] = index;
    top_logprobs[row * top + place] = (as_f32(r.p[index]) - all.m) - log_s;
  };
  if (tid < kGroups) {                        // the top-th largest of the groups' maxima: keys are unlike but for groups without numbers
    const unsigned long long mine = group_key[tid];
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < kGroups; ++i) larger += group_key[i] > mine;
    if (larger == top - 1 && mine != 0ull) bound = mine;
    if (top == 1 && larger == 0 && mine != 0ull) write(0, mine);
  }
  if (top == 1) return;
  __syncthreads();
  const unsigned long long least = bound;
  auto collect = [&](float x, int at) {
    const unsigned long long k = make_key(x, at);
    if (k >= least) {
      const int i = atomicAdd(&count, 1);
      if (i < kMaxCandidates) candidates[i] = k;
    }
  };
  if (key >= least && key != 0ull)
    walk(collect, [&](const float (&x)[U], int at) {
#pragma unroll
      for (int j = 0; j < U; ++j) collect(x[j], at + j);
    });
  __syncthreads();
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
  // Rows whose largest numbers stand in few threads' places: one after the other, each from the thread that has it.
  for (int place = 0; place < top; ++place) {
    const unsigned long long k = reduce_key<32>(key);
    __syncthreads();                          // the candidates, or the maxima of the place before, have been read
    if (lane == 0) candidates[warp] = k;
    __syncthreads();
    unsigned long long chosen = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) chosen = key_max(chosen, candidates[w]);
    if (chosen == key) {
      write(place, key);
      unsigned long long next = 0ull;
      auto look = [&](float x, int at) {
        const unsigned long long c = make_key(x, at);
        if (c < chosen) next = key_max(next, c);
      };
      walk(look, [&](const float (&x)[U], int at) {
#pragma unroll
        for (int j = 0; j < U; ++j) look(x[j], at + j);
      });
      key = next;
    }
  }
}

// Gradient of the logits: a CTA per row, read and written once; the chosen places are written again at the end.  d_top: rows of `top`, or null.
template <typename T>
__global__ void __launch_bounds__(lp::kThreads, 2)
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
  const float m = stats[2 * row], log_s = stats[2 * row + 1], h = entropy[row];
  auto gradient = [&](float x) {
    const float l = max_nan((x - m) - log_s, kFloor), p = ptx::ex2_approx(l * kLog2e);
    return -p * (total + gh * (l + h));
  };
  if (tid < r.head) store_one(out + tid, gradient(as_f32(r.p[tid])));
#pragma unroll 2
  for (int i = tid; i < r.units; i += kThreads) {
    float x[U];
    load_unit(r.p + r.head + i * U, x);
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = gradient(x[j]);
    store_unit(out + r.head + i * U, x);
  }
  const int at = r.tail() + tid;
  if (at < V) store_one(out + at, gradient(as_f32(r.p[at])));
  __syncthreads();
  if (d_top != nullptr && tid < top) {
    const long long id = top_ids[row * top + tid];
    if (id >= 0 && id < V) store_one(out + id, gradient(as_f32(r.p[id])) + d_top[row * top + tid] + (id == token ? g : 0.f));
  }
  if (tid == 0 && given) {
    bool also = false;                        // among the most probable: written there
    if (d_top != nullptr)
      for (int i = 0; i < top; ++i) also |= top_ids[row * top + i] == token;
    if (!also) store_one(out + token, gradient(as_f32(r.p[token])) + g);
  }
}

}  // namespace llmctl

using namespace llmctl;

// logits: rows of V bf16 (or fp32) numbers, ld apart; tokens: int64, outside of 0 .. V - 1: none (its log probability is 0).  logprobs, entropy: fp32
// [rows]; stats: fp32 [rows, 2] (maximum, log of the sum over it) for the gradient, or null; top_ids (int64) and top_logprobs: [rows, top].
LLMCTL_API int llmctl_token_logprobs(const void* logits, int is_fp32, long long ld, const long long* tokens, int rows, int V, int top, float* logprobs,
                                     float* entropy, float* stats, long long* top_ids, float* top_logprobs, void* stream) {
  LLMCTL_BEGIN();
  LLMCTL_REQUIRE(rows >= 0 && V >= 1 && top >= 0 && top <= lp::kMaxTop && top <= V && (top == 0 || (top_ids != nullptr && top_logprobs != nullptr)));
  LLMCTL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (is_fp32 ? 4 : 2) == 0);
  if (rows == 0) return 0;
  if (is_fp32)
    LLMCTL_CHECK(launch_dependent(token_logprobs_kernel<float>, rows, lp::kThreads, 0, (cudaStream_t)stream, (const float*)logits, ld, tokens, V, top,
                                  logprobs, entropy, stats, top_ids, top_logprobs));
  else
    LLMCTL_CHECK(launch_dependent(token_logprobs_kernel<__nv_bfloat16>, rows, lp::kThreads, 0, (cudaStream_t)stream, (const __nv_bfloat16*)logits, ld,
                                  tokens, V, top, logprobs, entropy, stats, top_ids, top_logprobs));
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
  if (is_fp32)
    LLMCTL_CHECK(launch_dependent(token_logprobs_bwd_kernel<float>, rows, lp::kThreads, 0, (cudaStream_t)stream, (const float*)logits, ld, tokens, V, top,
                                  stats, entropy, top_ids, d_logprobs, d_entropy, d_top, (float*)dx, ldd));
  else
    LLMCTL_CHECK(launch_dependent(token_logprobs_bwd_kernel<__nv_bfloat16>, rows, lp::kThreads, 0, (cudaStream_t)stream, (const __nv_bfloat16*)logits,
                                  ld, tokens, V, top, stats, entropy, top_ids, d_logprobs, d_entropy, d_top, (__nv_bfloat16*)dx, ldd));
  LLMCTL_RETURN_LAST();
}
