// Log probabilities of given tokens, entropy and the k best tokens of every
// row of logits [rows, vocab], in one pass over the logits.
//
//   lse = log Σ_j e^x_j,   logprob = x_target - lse,   H = lse - Σ_j p_j x_j
//
// Bound by reading the logits once (16-bit types: close to the exp2 rate too).
// Each thread streams 16-byte vectors and keeps a running maximum m and the
// sums s = Σ 2^t and u = Σ t 2^t with t = (x - m)·log2 e; the triples join
// associatively: over a thread's batches, a block and a cluster of CTAs that
// share a row (few rows: up to 8 CTAs per row through distributed shared
// memory, one launch, no workspace; many rows: one CTA per row).
//
// The k best need no second pass over the row: each thread also keeps its
// greatest value and the vector that held it.  The k-th greatest of these
// (a lower bound of the k-th greatest element) leaves about k threads that
// can hold a better element; only their vectors are read again (from L2).
// Elements are ordered by value, then by lower index, as unique 64-bit keys.
#include <cooperative_groups.h>

#include <type_traits>

#include "internal.hpp"

namespace slr {

__device__ unsigned g_status_logprobs;

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;       // vectors in flight per thread
constexpr int kCandidates = 512;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Sums {
  float m, s, u;  // m = -inf: nothing but -inf (s = 0) or NaN so far
};
// (a - b) log2 e, finite: a product with a sum of 0 stays 0.  The difference
// is taken first: logits of the type's lowest value times log2 e overflow.
__device__ __forceinline__ float log2_gap(float a, float b) { return fmaxf((a - b) * kLog2e, -1e30f); }
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = a.m == -INFINITY ? 0.f : log2_gap(a.m, r.m), db = b.m == -INFINITY ? 0.f : log2_gap(b.m, r.m);
  const float fa = a.m == -INFINITY ? 0.f : ex2(da), fb = b.m == -INFINITY ? 0.f : ex2(db);
  r.s = a.s * fa + b.s * fb;
  r.u = fa * (a.u + a.s * da) + fb * (b.u + b.s * db);
  return r;
}

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
__device__ __forceinline__ Key merge_step(Key k, int j, bool descending) {
  const Key other = __shfl_xor_sync(0xffffffffu, k, j);
  const bool low_lane = ((threadIdx.x & 31) & j) == 0;
  return (low_lane == descending) == (k > other) ? k : other;
}
__device__ __forceinline__ Key warp_sort(Key k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int j = size >> 1; j; j >>= 1) k = merge_step(k, j, (lane & size) == 0);
  return k;
}
// The 32 greatest of two sorted lists, sorted: a's lane i against b's lane 31 - i.
__device__ __forceinline__ Key warp_merge(Key a, Key b_reversed) {
  Key k = max_key(a, b_reversed);
#pragma unroll
  for (int j = 16; j; j >>= 1) k = merge_step(k, j, true);
  return k;
}

template <typename T> struct Vec {
  static constexpr int E = 16 / int(sizeof(T));
  __device__ static void to_floats(const uint4& v, float* f) {
    if constexpr (std::is_same<T, float>::value) {
      f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 p;
        if constexpr (std::is_same<T, __half>::value) p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
      }
    }
  }
  // the greatest element; NaN is passed over
  __device__ static float greatest(const uint4& v) {
    if constexpr (std::is_same<T, float>::value) {
      return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
      using P = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
      const P a = *reinterpret_cast<const P*>(&v.x), b = *reinterpret_cast<const P*>(&v.y);
      const P c = *reinterpret_cast<const P*>(&v.z), d = *reinterpret_cast<const P*>(&v.w);
      const P m = __hmax2(__hmax2(a, b), __hmax2(c, d));
      return fmaxf(to_f(m.x), to_f(m.y));
    }
  }
};

// A row as 16-byte vectors on 16-byte boundaries: vector j holds elements
// [j * E - shift, j * E - shift + E), of which those outside [0, vocab) do
// not exist (only the first and the last vector can have such).
template <typename T> struct Row {
  static constexpr int E = Vec<T>::E;
  const T* x;
  int64_t vocab;
  int shift;
  __device__ uint4 load(int64_t j) const {
    const int64_t i = j * E - shift;
    if (i >= 0 && i + E <= vocab) return __ldg(reinterpret_cast<const uint4*>(x + i));
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = i + e >= 0 && i + e < vocab ? x[i + e] : from_f<T>(-INFINITY);
    uint4 v;
    memcpy(&v, t, 16);
    return v;
  }
};

struct Shared {
  Sums sums[kWarps];
  Key lists[kWarps][32];
  Key cand[kCandidates];
  Key best[32];       // this CTA's list, greatest first
  Sums mine;
  Key tau, next;
  int n_cand, n_elig, valid;
  int elig[kThreads];
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobArgs a) {
  constexpr int E = Vec<T>::E;
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int64_t r = blockIdx.x / parts;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  Row<T> row;
  row.x = static_cast<const T*>(a.logits) + r * a.row_stride;
  row.vocab = a.vocab;
  row.shift = int((reinterpret_cast<uintptr_t>(row.x) & 15u) / sizeof(T));
  const int64_t vectors = (a.vocab + row.shift + E - 1) / E;
  const int64_t per = (vectors + parts - 1) / parts;
  const int64_t v0 = part * per, v1 = v0 + per < vectors ? v0 + per : vectors;
  if (tid == 0) sh.n_cand = 0, sh.n_elig = 0;

  // ---- one pass: sums and each thread's greatest value
  Sums st = {-INFINITY, 0.f, 0.f};
  float best = -INFINITY;
  int64_t best_vec = v0 + tid;
  for (int64_t j = v0 + tid; j < v1; j += kThreads * kBatch) {
    uint4 v[kBatch];
    float top[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t jb = j + b * kThreads;
      if (jb < v1) v[b] = row.load(jb);
      else {
        const T none = from_f<T>(-INFINITY);
        T t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = none;
        memcpy(&v[b], t, 16);
      }
    }
    float most = -INFINITY;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      top[b] = Vec<T>::greatest(v[b]);
      most = fmaxf(most, top[b]);
      if (top[b] > best) {
        best = top[b];
        best_vec = j + b * kThreads;
      }
    }
    if (most > st.m) {
      const float d = st.m == -INFINITY ? 0.f : log2_gap(st.m, most), f = st.m == -INFINITY ? 0.f : ex2(d);
      st.u = f * (st.u + st.s * d);
      st.s *= f;
      st.m = most;
    }
    const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float x[E];
      Vec<T>::to_floats(v[b], x);
      float s = 0.f, u = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float t = (x[e] - base) * kLog2e;
        const float p = ex2(t);
        s += p;
        u = fmaf(p, fmaxf(t, -1e30f), u);  // 0 · -inf counts as 0
      }
      st.s += s;
      st.u += u;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Sums other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.u = __shfl_xor_sync(0xffffffffu, st.u, o);
    st = join(st, other);
  }
  if (lane == 0) sh.sums[w] = st;

  // ---- the k best of this CTA's part
  const int k = a.top;
  if (k) {
    const bool has = v0 + tid < v1;
    const int64_t i0 = best_vec * E - row.shift;
    const uint32_t first = uint32_t(i0 < 0 ? 0 : i0), last = uint32_t(i0 + E - 1 < a.vocab ? i0 + E - 1 : a.vocab - 1);
    Key mine = warp_sort(has ? key_of(best, last) : 0ull);
    for (int n = kWarps; n > 1; n >>= 1) {
      if (w < n) sh.lists[w][lane] = mine;
      __syncthreads();
      if (w < n / 2) mine = warp_merge(mine, sh.lists[w + n / 2][31 - lane]);
      __syncthreads();
    }
    if (tid == k - 1) sh.tau = mine;  // 0 when fewer than k threads have elements: all are candidates
    __syncthreads();
    const Key tau = sh.tau;
    if (has && key_of(best, first) >= tau) sh.elig[atomicAdd(&sh.n_elig, 1)] = tid;
    __syncthreads();
    const int n_elig = sh.n_elig;
    for (int q = w; q < n_elig; q += kWarps)
      for (int64_t j = v0 + sh.elig[q] + int64_t(lane) * kThreads; j < v1; j += 32 * kThreads) {
        float x[E];
        Vec<T>::to_floats(row.load(j), x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t i = j * E - row.shift + e;
          const Key key = key_of(x[e], uint32_t(i));
          if (i >= 0 && i < a.vocab && key >= tau) {
            const int at = atomicAdd(&sh.n_cand, 1);
            if (at < kCandidates) sh.cand[at] = key;
          }
        }
      }
    __syncthreads();
    const int n = sh.n_cand;
    if (n <= kCandidates) {
      if (w == 0) {
        Key list = 0ull;
        for (int c = 0; c < n; c += 32) {
          const Key chunk = warp_sort(c + lane < n ? sh.cand[c + lane] : 0ull);
          const Key rev = __shfl_sync(0xffffffffu, chunk, 31 - lane);
          list = warp_merge(list, rev);
        }
        sh.best[lane] = list;
      }
    } else {
      // more candidates than the buffer holds (long runs of nearly equal
      // values in a few threads): one element per round, the greatest below the last
      Key prev = ~0ull;
      for (int i = 0; i < 32; ++i) {
        Key top = 0ull;
        if (i < k)
          for (int64_t j = v0 + tid; j < v1; j += kThreads) {
            float x[E];
            Vec<T>::to_floats(row.load(j), x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int64_t at = j * E - row.shift + e;
              const Key key = key_of(x[e], uint32_t(at));
              if (at >= 0 && at < a.vocab && key < prev) top = max_key(top, key);
            }
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
  __syncthreads();
  if (tid == 0) {
    Sums all = sh.sums[0];
    for (int i = 1; i < kWarps; ++i) all = join(all, sh.sums[i]);
    sh.mine = all;
  }
  if (parts > 1) cluster.sync();
  else __syncthreads();
  if (part == 0 && w == 0) {
    Sums all = sh.mine;
    for (int p = 1; p < parts; ++p) all = join(all, *cluster.map_shared_rank(&sh.mine, p));
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
    if (k) {
      Key list = sh.best[lane];
      for (int p = 1; p < parts; ++p) list = warp_merge(list, cluster.map_shared_rank(sh.best, p)[31 - lane]);
      if (lane < k) {
        a.top_ids[r * k + lane] = int64_t(0xffffffffu - uint32_t(list));
        a.top_logprobs[r * k + lane] = logprob(value_of(list));
      }
    }
  }
  if (parts > 1) cluster.sync();  // the parts stay until they have been read
}

template <typename T> int launch(const LogprobArgs& a, cudaStream_t s) {
  // CTAs per row: enough to give every SM work, each with at least one batch
  int dev = 0, sms = 0;
  SLR_CHECK_CUDA(cudaGetDevice(&dev));
  SLR_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  int parts = 1;
  while (parts < 8 && a.rows * parts < 4 * sms && a.vocab / Vec<T>::E >= int64_t(2) * parts * kThreads) parts *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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
