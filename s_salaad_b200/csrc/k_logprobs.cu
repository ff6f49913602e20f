// Log probabilities of given tokens, entropy and the k best tokens of every
// row of logits [rows, vocab], in one pass over the logits.
//
//   lse = log Σ_j e^x_j,   logprob = x_target - lse,   H = lse - Σ_j p_j x_j
//
// Bound by reading the logits once; in 16-bit types the exp2 rate (16 per clock
// and SM) and the instructions are close behind.  Each thread streams 16-byte
// vectors and keeps a reference m within 8 of the maximum and the sums s = Σ 2^t
// and u = Σ t 2^t with t = (x - m)·log2 e; the triples join associatively: over
// a thread's batches, a block and a cluster of CTAs that share a row (few rows:
// up to 8 CTAs per row through distributed shared memory, one launch, no
// workspace; many rows: one CTA per row).  t is one multiply-add for two
// elements (against the rounded product m·log2 e, whose error is taken back at
// the end), and -inf is raised to a finite value so that it adds 0 to u; where
// that is not exact (a part whose greatest logit is -inf or of the order of the
// type's lowest or greatest value) the part is summed again element by element.
//
// The k best need no second pass over the row: each thread also keeps its
// greatest value and the vector that held it, and (in shared memory) the
// greatest value of each of up to 64 groups of its vectors.  The k-th greatest
// of 64 sets of threads' values is a lower bound of the k-th greatest element,
// which leaves about k groups (44 for k = 32) that can hold a better one; only
// they are read again, all at once, and their elements from the bound on are
// ranked by counting.  (Reading all vectors of the k threads again cost 14 us of
// the 41 us that a row of 151936 took: they have left L2 by then.)
// Elements are ordered by value, then by lower index, as unique 64-bit keys.
//
// 2048 rows of 151936, bf16, 622 MB: 103 us without best tokens (6.0 TB/s), 119
// us with 20; in long runs, at the power cap, 110 and 124.
#include <cooperative_groups.h>
#include <type_traits>

#include "internal.hpp"

namespace slr {

__device__ unsigned g_status_logprobs;

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;       // vectors in flight per thread
static_assert(kWarps == 4 && kBatch == 4, "the sets of threads, the groups of batches");
constexpr int kPerSm = 8;       // CTAs per SM
constexpr int kCandidates = 512;
constexpr int kEligible = 512;
// Groups per thread; 8 CTAs per SM share what L1 leaves: 40 groups of fp32 were 15 % slower.
template <typename T> constexpr int kGroups = sizeof(T) == 4 ? 20 : 64;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Sums {
  float m, s, u;  // m: the reference of s and u; -inf: nothing but -inf (s = 0) or NaN so far
};
// (a - b) log2 e, finite: a product with a sum of 0 stays 0.  The difference
// is taken first: logits of the type's lowest value times log2 e overflow.
__device__ __forceinline__ float log2_gap(float a, float b) { return fmaxf((a - b) * kLog2e, -1e30f); }
// Unique key of element i: greater for a greater value, then for a lower
// index.  NaN ranks with -inf; -0 with +0.
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t i) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  const uint32_t o = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t o = uint32_t(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

using Key = unsigned long long;
__device__ __forceinline__ Key max_key(Key a, Key b) { return a > b ? a : b; }

// Bitonic networks over a warp's 32 keys (one per lane), greatest first.
template <typename K> __device__ __forceinline__ K merge_step(K k, int j, bool descending) {
  const K other = __shfl_xor_sync(0xffffffffu, k, j);
  const bool low_lane = ((threadIdx.x & 31) & j) == 0;
  return low_lane == descending ? max(k, other) : min(k, other);
}
__device__ __forceinline__ uint32_t warp_sort(uint32_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int j = size >> 1; j; j >>= 1) k = merge_step(k, j, (lane & size) == 0);
  return k;
}
// The 32 greatest of two sorted lists, sorted: a's lane i against b's lane 31 - i.
template <typename K> __device__ __forceinline__ K warp_merge(K a, K b_reversed) {
  K k = max(a, b_reversed);
#pragma unroll
  for (int j = 16; j; j >>= 1) k = merge_step(k, j, true);
  return k;
}

// Room for `count` entries of every lane behind *counter (shared memory, one
// atomic per warp): this lane's first.
__device__ __forceinline__ int warp_reserve(int count, int* counter) {
  const int lane = threadIdx.x & 31;
  int incl = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  int base = 0;
  if (lane == 31 && incl) base = atomicAdd(counter, incl);
  return __shfl_sync(0xffffffffu, base, 31) + incl - count;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int E = 4;
  static constexpr float kClip = -1e38f;  // stands for anything below
  static constexpr float kLow = -1e37f, kHigh = 1e37f;
  __device__ static void to_floats(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  __device__ static void clipped(const uint4& v, float* f) {
    to_floats(v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(f[i]) : "f"(kClip));  // NaN stays
  }
  // the greatest element; NaN is passed over
  using Top = float;
  __device__ static Top top(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  __device__ static Top greater(Top a, Top b) { return fmaxf(a, b); }
  __device__ static float of_top(Top a) { return a; }
  __device__ static Top none() { return -INFINITY; }
};
template <typename T, typename P> struct Vec16 {
  static constexpr int E = 8;
  __device__ static P as(uint32_t w) { return *reinterpret_cast<P*>(&w); }
  __device__ static void unpack(const P* p, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of an fp32
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p + i);
        f[2 * i] = __uint_as_float(w << 16), f[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        f[2 * i] = to_f(p[i].x), f[2 * i + 1] = to_f(p[i].y);
      }
    }
  }
  __device__ static void to_floats(const uint4& v, float* f) {
    const P p[4] = {as(v.x), as(v.y), as(v.z), as(v.w)};
    unpack(p, f);
  }
  __device__ static void clipped(const uint4& v, float* f) {
    const P low = {from_f<T>(Vec<T>::kClip), from_f<T>(Vec<T>::kClip)};
    const P p[4] = {__hmax2_nan(as(v.x), low), __hmax2_nan(as(v.y), low), __hmax2_nan(as(v.z), low),
                    __hmax2_nan(as(v.w), low)};
    unpack(p, f);
  }
  using Top = P;
  __device__ static Top top(const uint4& v) {
    return __hmax2(__hmax2(as(v.x), as(v.y)), __hmax2(as(v.z), as(v.w)));
  }
  __device__ static Top greater(Top a, Top b) { return __hmax2(a, b); }
  __device__ static float of_top(Top a) { return fmaxf(to_f(a.x), to_f(a.y)); }
  __device__ static Top none() { return {from_f<T>(-INFINITY), from_f<T>(-INFINITY)}; }
};
template <> struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16, __nv_bfloat162> {
  static constexpr float kClip = -1e38f, kLow = -1e37f, kHigh = 1e37f;
};
template <> struct Vec<__half> : Vec16<__half, __half2> {
  static constexpr float kClip = -65504.f, kLow = -6e4f, kHigh = 1e37f;
};

// A row as the 16-byte vectors on 16-byte boundaries inside it (vector j:
// elements [head + j E, head + j E + E)) and up to 2 (E - 1) elements at its
// ends.
template <typename T> struct Row {
  static constexpr int E = Vec<T>::E;
  const T* x;
  int head, vectors, edges;
  __device__ Row(const T* p, int vocab) : x(p) {
    const int shift = int((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
    head = min(vocab, (E - shift) % E);
    vectors = (vocab - head) / E;
    edges = vocab - vectors * E;
  }
  __device__ const uint4* at(int j) const { return reinterpret_cast<const uint4*>(x + head) + j; }
  __device__ uint4 load(int j) const { return __ldg(at(j)); }
  __device__ int first_of(int j) const { return head + j * E; }
  // element index of edge e < edges
  __device__ int edge(int e) const { return e < head ? e : e + vectors * E; }
};

template <typename T> struct Shared {
  Sums sums[kWarps];
  Key lists[kWarps][32];  // sets of threads (and the warps' best in the slow search)
  Key cand[kCandidates];
  Key best[32];       // this CTA's list, greatest first
  Sums mine;
  uint32_t values[32], tau_value, tau_index[2];
  int n_cand, n_elig;
  T group[kGroups<T>][kThreads];      // greatest value of each thread's groups of batches
  unsigned short elig[kEligible];  // groups to read again
};

template <typename T>
__global__ void __launch_bounds__(kThreads, kPerSm) logprobs_kernel(const LogprobArgs a) {
  using V = Vec<T>;
  constexpr int E = V::E;
  __shared__ Shared<T> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / parts;
  pdl_wait_primary();
  pdl_launch_dependents();
  const Row<T> row(static_cast<const T*>(a.logits) + r * a.row_stride, int(a.vocab));
  const int per = (row.vectors + parts - 1) / parts;
  const int v0 = min(row.vectors, part * per), v1 = min(row.vectors, v0 + per);
  const bool edge = part == 0 && tid < row.edges;  // this thread also has an element at the row's ends
  const float edge_x = edge ? to_f(row.x[row.edge(tid)]) : -INFINITY;
  if (tid == 0) sh.n_cand = 0, sh.n_elig = 0;

  // ---- one pass: sums, and each thread's greatest value with the elements it was found among
  Sums st = {-INFINITY, 0.f, 0.f};
  float best = -INFINITY;
  // where it was: the batch, and of 16-bit types its vectors' greatest (fp32: the vector at once)
  constexpr bool kLate = sizeof(T) == 2;
  int best_at = 0;
  typename V::Top best_top[kLate ? kBatch : 1];
#pragma unroll
  for (int b = 0; b < (kLate ? kBatch : 1); ++b) best_top[b] = V::none();
  const int batches = max(1, (v1 - v0 + kThreads * kBatch - 1) / (kThreads * kBatch));
  const int group_log = 32 - __clz((batches + kGroups<T> - 1) / kGroups<T> * 2 - 1) - 1;  // batches: a power of two
  float in_group = -INFINITY;
  // log2 e times the maximum, rounded; 0 (every 2^t is 0 then) until there is one that the product holds
  auto base = [&] { return st.m > V::kLow ? __fmul_rn(st.m, kLog2e) : 0.f; };
  // The sums are exact against the rounded base, so it is bases that are
  // subtracted here, and rest() is taken back at the end of the pass: left in
  // the sums, the rounding of a base of 10^4 would be 5e-4 of every result.
  auto rebase = [&](float d) {
    const float f = ex2(d);
    st.u = f * (st.u + st.s * d);
    st.s *= f;
  };
  auto raise = [&](float to) {
    const float from = base();
    const bool any = st.m > V::kLow;  // else the sums are 0
    st.m = to;
    if (any) rebase(fmaxf(from - base(), -1e30f));
  };
  auto rest = [&] { return st.m > V::kLow ? fmaf(st.m, kLog2e, -base()) : 0.f; };
  auto batch = [&](const uint4* v, const int it) {
    typename V::Top top[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) top[b] = V::top(v[b]);
    typename V::Top all = top[0];
#pragma unroll
    for (int b = 1; b < kBatch; ++b) all = V::greater(all, top[b]);
    const float most = V::of_top(all);
    // m follows the maximum within 8 (2^t up to 3000): a new greatest value of
    // one lane, which most batches have, then rarely costs the warp a rescaling
    if (most > st.m + 8.f) raise(most);
    if (a.top) {
      in_group = fmaxf((it & ((1 << group_log) - 1)) ? in_group : -INFINITY, most);  // NaN alone counts as -inf
      sh.group[it >> group_log][tid] = from_f<T>(in_group);  // exact
      const bool up = most > best;
      best = up ? most : best;
      int at = it * kBatch;
      if constexpr (kLate) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) best_top[b] = up ? top[b] : best_top[b];
      } else {
        at += V::of_top(top[0]) == most ? 0 : V::of_top(top[1]) == most ? 1 : V::of_top(top[2]) == most ? 2 : 3;
      }
      best_at = up ? at : best_at;
    }
    const float m2 = base();
    const Pair scale2 = pair(kLog2e, kLog2e), base2 = pair(-m2, -m2);
    Pair s2 = 0, u2 = 0;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float x[E];
      V::clipped(v[b], x);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const Pair t2 = fma2(pair(x[e], x[e + 1]), scale2, base2);
        float t0, t1;
        unpair(t2, t0, t1);
        const Pair p2 = pair(ex2(t0), ex2(t1));
        s2 = add2(s2, p2);
        u2 = fma2(p2, t2, u2);
      }
    }
    float s0, s1, u0, u1;
    unpair(s2, s0, s1);
    unpair(u2, u0, u1);
    st.s += s0 + s1;
    st.u += u0 + u1;
  };
  constexpr int kSpan = kBatch * kThreads;
  const int mine = v1 - v0 > tid ? (v1 - v0 - tid + kThreads - 1) / kThreads : 0;  // vectors of this thread
  const int n_whole = mine / kBatch, n_batch = (mine + kBatch - 1) / kBatch;
  const uint4* src = row.at(v0 + tid);
  auto fetch = [&](uint4* v) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) v[b] = __ldg(src + b * kThreads);
    src += kSpan;
  };
  // the next batch is under way while one is summed
  if (n_whole) {
    uint4 v[kBatch], next[kBatch];
    fetch(v);
    int it = 0;
    for (; it + 2 < n_whole; it += 2) {
      fetch(next);
      batch(v, it);
      fetch(v);
      batch(next, it + 1);
    }
    if (it + 1 < n_whole) fetch(next);
    batch(v, it);
    if (it + 1 < n_whole) batch(next, it + 1);
  }
  if (n_batch > n_whole) {
    uint4 v[kBatch];
    const typename V::Top none = V::none();
    const uint32_t word = *reinterpret_cast<const uint32_t*>(&none);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      v[b] = n_whole * kBatch + b < mine ? __ldg(src + b * kThreads) : make_uint4(word, word, word, word);
    batch(v, n_whole);
  }
  // index of the last element of the vector that held the greatest value; -1: no element
  int best_last = -1;
  if (mine) {
    if constexpr (kLate) {
      int b = 0;
#pragma unroll
      for (int i = kBatch - 1; i >= 0; --i)
        if (V::of_top(best_top[i]) == best) b = best == -INFINITY ? 0 : i;
      best_at += b;
    }
    best_last = row.first_of(v0 + tid + best_at * kThreads) + E - 1;
  }
  if (edge) {
    if (edge_x > st.m + 8.f) raise(edge_x);
    const float x = edge_x < V::kClip ? V::kClip : edge_x;
    const float t = fmaf(x, kLog2e, -base()), p = ex2(t);
    st.s += p;
    st.u = fmaf(p, t, st.u);
    if (edge_x > best || best_last < 0) {
      best = edge_x == edge_x ? edge_x : -INFINITY;
      best_last = row.edge(tid);
    }
  }
  rebase(-rest());
  // the triples of a warp (or of its first lanes) as one, in every lane
  auto warp_join = [&](Sums x) {
    float top = x.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float d = x.m == -INFINITY ? 0.f : log2_gap(x.m, top), f = x.m == -INFINITY ? 0.f : ex2(d);
    x.u = f * (x.u + x.s * d);
    x.s *= f;
    x.m = top;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      x.s += __shfl_xor_sync(0xffffffffu, x.s, o);
      x.u += __shfl_xor_sync(0xffffffffu, x.u, o);
    }
    return x;
  };
  auto block_join = [&] {
    st = warp_join(st);
    if (lane == 0) sh.sums[w] = st;
    __syncthreads();
  };
  block_join();
  float most = sh.sums[0].m;
#pragma unroll
  for (int i = 1; i < kWarps; ++i) most = fmaxf(most, sh.sums[i].m);
  if (!(most > V::kLow && most < V::kHigh)) {
    // element by element, without raising -inf and with the difference first
    __syncthreads();
    st = {most, 0.f, 0.f};
    auto one = [&](float x) {
      const float t = (x - (most == -INFINITY ? 0.f : most)) * kLog2e, p = ex2(t);
      st.s += p;
      st.u = fmaf(p, fmaxf(t, -1e30f), st.u);
    };
    for (int i = v0 + tid; i < v1; i += kThreads) {
      float x[E];
      V::to_floats(row.load(i), x);
#pragma unroll
      for (int e = 0; e < E; ++e) one(x[e]);
    }
    if (edge) one(edge_x);
    block_join();
  }

  // ---- the k best of this CTA's part
  const int k = a.top;
  if (k) {
    const bool has = best_last >= 0;
    // 64 sets of two threads: their values sorted by two warps, merged by one
    const Key own = has ? key_of(best, best_last) : 0ull;
    if (w >= 2) sh.lists[w - 2][lane] = own;
    __syncthreads();
    if (w < 2) {
      const Key set = max_key(own, sh.lists[w][lane]);
      const uint32_t value = uint32_t(set >> 32), sorted = warp_sort(value);
      if (w == 1) sh.values[lane] = sorted;
      named_bar_sync(1, 64);
      if (w == 0) {
        const uint32_t both = warp_merge(sorted, sh.values[31 - lane]);
        if (lane == k - 1) sh.tau_value = both;  // 0 when fewer than k sets have elements: all are candidates
      }
      named_bar_sync(1, 64);
      // of equal values the highest index: all of these sets count
      const bool equal = value == sh.tau_value;
      const uint32_t low = __reduce_min_sync(0xffffffffu, equal ? uint32_t(set) : 0xffffffffu);
      if (lane == 0) sh.tau_index[w] = low;
    }
    __syncthreads();
    const Key tau =
        sh.tau_value ? static_cast<Key>(sh.tau_value) << 32 | min(sh.tau_index[0], sh.tau_index[1]) : 0ull;
    const float tau_x = tau ? value_of(tau) : -INFINITY;
    const int groups = (n_batch + (1 << group_log) - 1) >> group_log;
#pragma unroll 4
    for (int g = 0; g < groups; ++g)
      if (to_f(sh.group[g][tid]) >= tau_x) {  // about k of all threads' groups
        const int at = atomicAdd(&sh.n_elig, 1);
        if (at < kEligible) sh.elig[at] = static_cast<unsigned short>(g * kThreads + tid);
      }
    __syncthreads();
    // whether an element is a candidate (NaN counts as -inf)
    auto passes = [&](float x, int i) {
      const float y = x == x ? x : -INFINITY;
      return y > tau_x || (y == tau_x && key_of(y, i) >= tau);
    };
    // four reads in flight per thread: the latency of DRAM counts here
    const int sub_log = group_log + 2;
    const bool all = sh.n_elig > kEligible;  // many equal values: every vector
    const int items = all ? v1 - v0 : sh.n_elig << sub_log;
    for (int q0 = tid; q0 - lane < items; q0 += 4 * kThreads) {
      uint4 v[4];
      int at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = q0 + i * kThreads;
        at[i] = v1;
        if (q < items && all) {
          at[i] = v0 + q;
        } else if (q < items) {
          const int e = sh.elig[q >> sub_log];
          at[i] = v0 + (((e / kThreads) << sub_log) + (q & ((1 << sub_log) - 1))) * kThreads + e % kThreads;
        }
        if (at[i] < v1) v[i] = row.load(at[i]);
      }
      unsigned mask = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (at[i] >= v1 || V::of_top(V::top(v[i])) < tau_x) continue;  // all NaN goes on
        float x[E];
        V::to_floats(v[i], x);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (passes(x[e], row.first_of(at[i]) + e)) mask |= 1u << (i * E + e);
      }
      __syncwarp();
      int to = warp_reserve(__popc(mask), &sh.n_cand);
      for (; mask; mask &= mask - 1, ++to) {
        const int b = __ffs(mask) - 1, i = b / E;
        const int idx = row.first_of(i == 0 ? at[0] : i == 1 ? at[1] : i == 2 ? at[2] : at[3]) + b % E;
        if (to < kCandidates) sh.cand[to] = key_of(to_f(row.x[idx]), idx);
      }
      __syncwarp();
    }
    if (edge && passes(edge_x, row.edge(tid))) {
      const int to = atomicAdd(&sh.n_cand, 1);
      if (to < kCandidates) sh.cand[to] = key_of(edge_x, row.edge(tid));
    }
    __syncthreads();
    const int n = sh.n_cand;
    if (n <= kCandidates) {
      for (int c = tid; c < n; c += kThreads) {
        const Key mine = sh.cand[c];
        int rank = 0;
        for (int q = 0; q < n; ++q) rank += sh.cand[q] > mine;
        if (rank < 32) sh.best[rank] = mine;
      }
      if (tid >= n && tid < 32) sh.best[tid] = 0ull;
    } else {
      // more candidates than the buffer holds (long runs of nearly equal
      // values in a few threads): one element per round, the greatest below the last
      Key prev = ~0ull;
      for (int i = 0; i < 32; ++i) {
        Key top = 0ull;
        if (i < k)
          for (int v = v0 + tid; v < v1; v += kThreads) {
            float x[E];
            V::to_floats(row.load(v), x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const Key key = key_of(x[e], row.first_of(v) + e);
              if (key < prev) top = max_key(top, key);
            }
          }
        if (i < k && edge) {
          const Key key = key_of(edge_x, row.edge(tid));
          if (key < prev) top = max_key(top, key);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = max_key(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) sh.lists[w][0] = top;
        __syncthreads();
        for (int q = 0; q < kWarps; ++q) top = max_key(top, sh.lists[q][0]);
        if (tid == 0) sh.best[i] = top;
        prev = top;
        __syncthreads();
      }
    }
  }
    if (w == 0) {
      const Sums all = warp_join(lane < kWarps ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f});
      if (lane == 0) sh.mine = all;
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    if (part == 0) {
      // the parts' lists, merged pairwise by one warp each
      Key list = 0ull;
      if (k) {
        int n = parts;
        if (w < (n + 1) / 2) list = cluster.map_shared_rank(sh.best, w)[lane];
        if (n > 1 && w < n / 2) list = warp_merge(list, cluster.map_shared_rank(sh.best, w + n / 2)[31 - lane]);
        for (n /= 2; n > 1; n /= 2) {
          if (w >= n / 2 && w < n) sh.lists[w][lane] = list;
          __syncthreads();
          if (w < n / 2) list = warp_merge(list, sh.lists[w + n / 2][31 - lane]);
        }
      }
    if (w == 0) {
      const Sums all =
          parts == 1 ? sh.mine
                     : warp_join(lane < parts ? *cluster.map_shared_rank(&sh.mine, lane) : Sums{-INFINITY, 0.f, 0.f});
      const float log_s = log2f(all.s);
      const bool none = !(all.s > 0.f);  // no finite logit, or a NaN
      const float nan = __int_as_float(0x7fffffff);
      auto logprob = [&](float x) { return none ? nan : (x - all.m) - kLn2 * log_s; };
      if (lane == 0) {
        if (a.entropy) a.entropy[r] = none ? nan : kLn2 * (log_s - all.u / all.s);
        if (a.targets) {
          const int64_t t = a.targets[r];
          if (t >= a.vocab) atomicOr(&g_status_logprobs, SLR_BAD_INDEX_BIT);
          a.logprob[r] = t < 0 ? 0.f : t >= a.vocab ? nan : logprob(to_f(row.x[t]));
        }
      }
      if (lane < k) {
        // a token whatever the row holds: callers take the ids as indexes
        a.top_ids[r * k + lane] = min(int64_t(0xffffffffu - uint32_t(list)), a.vocab - 1);
        a.top_logprobs[r * k + lane] = logprob(value_of(list));
      }
    }
  }
  if (parts > 1) cluster.sync();  // the parts stay until they have been read
}

template <typename T> int launch(const LogprobArgs& a, cudaStream_t s) {
  // CTAs per row: until there are four per SM, each with at least one batch
  // (151936 tokens, bf16, 20 best: 296 rows with 2 CTAs each 31 us, 1: 38, 4:
  // 42; 740 rows with 1 CTA 52 us, 2: 65)
  int dev = 0, sms = 0;
  SLR_CHECK_CUDA(cudaGetDevice(&dev));
  SLR_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  int parts = 1;
  while (parts < 8 && a.rows * parts < 4 * sms && a.vocab / Vec<T>::E >= int64_t(2) * parts * kThreads) parts *= 2;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // waits for the kernel before it first
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, a));
  return SLR_OK;
}

}  // namespace

int launch_logprobs(const LogprobArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case SLR_F32: return launch<float>(a, s);
    case SLR_F16: return launch<__half>(a, s);
    default: return launch<__nv_bfloat16>(a, s);
  }
}

int read_and_clear_status_logprobs(unsigned* out) {
  unsigned v = 0, zero = 0;
  SLR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_status_logprobs, sizeof(v)));
  if (v) SLR_CHECK_CUDA(cudaMemcpyToSymbol(g_status_logprobs, &zero, sizeof(zero)));
  *out = v;
  return SLR_OK;
}

}  // namespace slr
