// Attention of one new token per row over a paged key-value cache.
//
//   s_t = scale · q·K_t,  o = Σ_t e^(s_t - m) V_t / Σ_t e^(s_t - m),  m = max_t s_t
//
// over the T = lens[b] tokens of row b; token t lies in page table[b, t / page_size]
// at slot t % page_size.  Every K and V element is used for the few query
// heads of its group only, so the kernel is bound by reading the cache once.
//
// Split: the tokens of every (row, block of query heads of one key head)
// are cut into tiles, all tiles of the call form one list, and each CTA takes
// an equal contiguous part of it (computed on the device from lens, so the
// launch does not depend on the lengths and can be replayed from a graph).
// A (row, head block) that lies inside one CTA's part is written directly; the
// others leave (o, m, l) per part in the workspace and attend_join_kernel joins
// them in part order, so results do not depend on timing.
//
// Inside a CTA each warp owns a slice of every tile and streams it through
// its own ring of cp.async stages (no CTA barrier until the end of a row); the
// page number of a stage is fetched one stage ahead.  Running maximum and sum
// are per warp and joined through shared memory at the end of a row.
// 16-bit types: Q·Kᵀ and P·V on mma.sync with the query heads of the group as
// the 16 rows of the MMA (the work is far below tcgen05's tile of 128 rows and
// the tensor pipe is not the bound).  fp32: FFMA.
#include <atomic>
#include <type_traits>

#include "internal.hpp"

namespace slr {

__device__ unsigned g_status_attend;

namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

struct AttendK {
  const void* k;
  const void* v;
  int64_t page_stride, head_stride, token_stride;
  const int32_t* table;
  const int32_t* lens;
  const void* q;
  int64_t q_row, q_head;
  void* out;
  int64_t o_row, o_head;
  float* lse;        // [rows, heads] or null
  float* part_o;     // [2 * ctas][GT][DP]
  float2* part_ml;   // [2 * ctas][GT]
  int32_t* prefix;   // [rows + 1] tiles before each row
  int rows, kv_heads, group, hblocks, dim, page_size, max_pages, num_pages, ctas;
  float scale_log2;
};

// Tiles that one CTA takes of a list of n: an equal part, but not less than
// min_tiles (a join costs more than a few tiles in a row).
__device__ __forceinline__ int64_t tiles_per_cta(int64_t n, int ctas, int min_tiles) {
  const int64_t per = (n + ctas - 1) / ctas;
  return per < min_tiles ? min_tiles : per;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
  // src-size 0 writes 16 zero bytes and reads nothing
  const int n = fill ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T> struct pair_of;
template <> struct pair_of<__nv_bfloat16> {
  __device__ static uint32_t pack(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ static float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u)); }
};
template <> struct pair_of<__half> {
  __device__ static uint32_t pack(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ static float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
};

// Shape of one instance: DP head dimension padded to a power of two, W warps,
// TT tokens per warp and tile, NS stages per warp, GT query heads per CTA, RB
// rows of them joined per round.
template <typename T, int DP_> struct Cfg {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int DP = DP_;
  static constexpr int W = 4;
  static constexpr int TT = kF32 ? 8 : 16;
  static constexpr int NS = DP == 64 ? 4 : 3;
  static constexpr int GT = kF32 ? 8 : 16;
  static constexpr int RB = kF32 ? 4 : 8;
  static constexpr int kTile = W * TT;
  static constexpr int kRow = DP * int(sizeof(T));     // bytes of a token's row
  static constexpr int kHalf = TT * kRow;              // K (or V) bytes of a stage
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = W * NS * kStage;
  static constexpr int kBuf = (W - 1) * RB * DP * 4;   // other warps' o at the end of a row
  static constexpr int kMl = W * GT * 8;
  static constexpr int kQ = kF32 ? GT * DP * 4 : 0;
  static constexpr int kP = kF32 ? W * TT * GT * 4 : 0;
  static constexpr int kCnt = W * NS * 4;
  static constexpr int kFixed = kRing + kBuf + kMl + kQ + kP + kCnt + 64;
  static constexpr int kMinTiles = kF32 ? 4 : 2;
};

// Place in the list of tiles: row b, head block h, tile of the row.
struct Cursor {
  int b, h, tile, ntiles, len;
};

template <int kTile>
__device__ __forceinline__ void cursor_next(Cursor& c, const int* lens, int rows, int hb) {
  if (++c.tile < c.ntiles) return;
  c.tile = 0;
  if (++c.h < hb) return;
  c.h = 0;
  do {
    ++c.b;
  } while (c.b < rows && lens[c.b] == 0);
  c.len = c.b < rows ? lens[c.b] : 0;
  c.ntiles = (c.len + kTile - 1) / kTile;
}

template <typename T, int DP_>
__global__ void __launch_bounds__(Cfg<T, DP_>::W * 32) attend_kernel(const AttendK a) {
  using C = Cfg<T, DP_>;
  constexpr int DP = C::DP, W = C::W, TT = C::TT, NS = C::NS, GT = C::GT, RB = C::RB;
  constexpr int kThreads = W * 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float* buf = reinterpret_cast<float*>(smem + C::kRing);
  float2* ml = reinterpret_cast<float2*>(smem + C::kRing + C::kBuf);
  float* qs = reinterpret_cast<float*>(smem + C::kRing + C::kBuf + C::kMl);
  float* ps = reinterpret_cast<float*>(smem + C::kRing + C::kBuf + C::kMl + C::kQ);
  int* cnt = reinterpret_cast<int*>(smem + C::kRing + C::kBuf + C::kMl + C::kQ + C::kP);
  int* scratch = cnt + W * NS;                       // 16 words
  int* lens = reinterpret_cast<int*>(smem + C::kFixed);  // [rows]

  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int hb = a.kv_heads * a.hblocks;
  pdl_wait_primary();
  pdl_launch_dependents();

  // ---- this CTA's part of the list of tiles
  const int64_t cap = int64_t(a.max_pages) * a.page_size;
  const int chunk = (a.rows + kThreads - 1) / kThreads;
  const int r0 = tid * chunk, r1 = min(a.rows, r0 + chunk);
  int mine = 0;
  bool bad = false;
  for (int r = r0; r < r1; ++r) {
    int64_t n = a.lens[r];
    if (n < 0 || n > cap) {
      bad = true;
      n = n < 0 ? 0 : cap;
    }
    lens[r] = int(n);
    mine += int((n + C::kTile - 1) / C::kTile);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) scratch[w] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i < w) before += scratch[i];
    total += scratch[i];
  }
  const int64_t n_all = int64_t(total) * hb;
  const int64_t per = tiles_per_cta(n_all, a.ctas, C::kMinTiles);
  const int64_t t_begin = int64_t(blockIdx.x) * per;
  const int64_t t_end = t_begin + per < n_all ? t_begin + per : n_all;
  for (int r = r0; r < r1; ++r) {
    if (blockIdx.x == 0) a.prefix[r] = before;
    const int nt = (lens[r] + C::kTile - 1) / C::kTile;
    if (nt && int64_t(before) * hb <= t_begin && t_begin < int64_t(before + nt) * hb) {
      scratch[8] = r;
      scratch[9] = before;
    }
    before += nt;
  }
  if (blockIdx.x == 0) {
    if (tid == 0) a.prefix[a.rows] = total;
    if (bad) atomicOr(&g_status_attend, SLR_BAD_INDEX_BIT);
  }
  __syncthreads();
  if (t_begin >= t_end) return;
  Cursor c;
  c.b = scratch[8];
  c.len = lens[c.b];
  c.ntiles = (c.len + C::kTile - 1) / C::kTile;
  {
    const int64_t in_row = t_begin - int64_t(scratch[9]) * hb;
    c.h = int(in_row / c.ntiles);
    c.tile = int(in_row - int64_t(c.h) * c.ntiles);
  }
  const int n = int(t_end - t_begin);
  // where the first row's tiles start relative to this CTA's part
  int64_t seg_start = t_begin - c.tile;

  // ---- the ring
  const uint32_t ring_w = smem_u32(ring) + w * NS * C::kStage;
  int* cnt_w = cnt + w * NS;
  Cursor f = c;
  auto fetch_page = [&](const Cursor& u) -> int {
    const int t0 = u.tile * C::kTile + w * TT;
    return t0 < u.len ? a.table[int64_t(u.b) * a.max_pages + t0 / a.page_size] : 0;
  };
  int page = fetch_page(f);
  int loaded = 0, load_slot = 0;
  auto load_stage = [&]() {
    if (loaded < n) {
      const int t0 = f.tile * C::kTile + w * TT;
      int valid = min(TT, f.len - t0);
      if (valid > 0 && (page < 0 || page >= a.num_pages)) {
        if (lane == 0) atomicOr(&g_status_attend, SLR_BAD_INDEX_BIT);
        valid = 0;
      }
      if (lane == 0) cnt_w[load_slot] = valid;
      if (valid > 0) {
        const int64_t off = int64_t(page) * a.page_stride + int64_t(f.h / a.hblocks) * a.head_stride +
                            int64_t(t0 % a.page_size) * a.token_stride;
        const T* ks = static_cast<const T*>(a.k) + off;
        const T* vs = static_cast<const T*>(a.v) + off;
        constexpr int E = 16 / int(sizeof(T));   // elements of a 16-byte chunk
        constexpr int CH = DP / E;               // chunks of a row
        const uint32_t base = ring_w + load_slot * C::kStage;
#pragma unroll
        for (int i = 0; i < TT * CH / 32; ++i) {
          const int idx = i * 32 + lane;
          const int row = idx / CH, ch = idx % CH;
          const bool in = row < valid && ch * E < a.dim;
          const uint32_t dst = base + row * C::kRow + ((ch ^ (row & 7)) << 4);
          const int64_t src = in ? row * a.token_stride + ch * E : 0;
          cp_async16(dst, ks + src, in);
          cp_async16(dst + C::kHalf, vs + src, in);
        }
      }
      ++loaded;
      if (loaded < n) {
        cursor_next<C::kTile>(f, lens, a.rows, hb);
        page = fetch_page(f);
      }
      load_slot = load_slot + 1 == NS ? 0 : load_slot + 1;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load_stage();

  // ---- running softmax of this warp: log2-domain maximum, sum, output
  // 16-bit: rows lane/4 and lane/4 + 8 (index 0, 1), columns of the MMA tiles.
  // fp32: every lane all GT heads, DP / 32 columns each.
  constexpr int kRows = C::kF32 ? GT : 2;
  constexpr int kOut = C::kF32 ? GT * (DP / 32) : DP / 2;
  float m[kRows], l[kRows], o[kOut];
  uint32_t qf[C::kF32 ? 1 : DP / 4];
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < kRows; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int i = 0; i < kOut; ++i) o[i] = 0.f;
  };
  auto load_q = [&]() {
    const int kvh = c.h / a.hblocks, g0 = (c.h % a.hblocks) * GT;
    const T* q = static_cast<const T*>(a.q) + int64_t(c.b) * a.q_row + int64_t(kvh * a.group + g0) * a.q_head;
    const int heads = min(GT, a.group - g0);
    if constexpr (C::kF32) {
      for (int i = tid; i < GT * DP; i += kThreads) {
        const int g = i / DP, d = i % DP;
        qs[i] = g < heads && d < a.dim ? q[g * a.q_head + d] : 0.f;
      }
      __syncthreads();
    } else {
      const unsigned short* qu = reinterpret_cast<const unsigned short*>(q);
#pragma unroll
      for (int i = 0; i < DP / 4; ++i) {
        const int g = (lane >> 2) + (i & 1) * 8, d = (i >> 2) * 16 + (i & 2) * 4 + (lane & 3) * 2;
        uint32_t v = 0;
        if (g < heads && d < a.dim) {
          const unsigned short* p = qu + g * a.q_head + d;
          v = uint32_t(p[0]) | (uint32_t(p[1]) << 16);
        }
        qf[i] = v;
      }
    }
  };

  auto step = [&](uint32_t base, int valid, bool two) {
    if constexpr (!C::kF32) {
      float s[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const int row = ((lane >> 4) << 3) + (lane & 7), ch = ks * 2 + ((lane >> 3) & 1);
        uint32_t b0, b1, b2, b3;
        ldsm_x4(base + row * C::kRow + ((ch ^ (row & 7)) << 4), b0, b1, b2, b3);
        mma16816<T>::run(s[0], qf + ks * 4, b0, b1);
        mma16816<T>::run(s[1], qf + ks * 4, b2, b3);
      }
      // With scale < 0 the largest product is the smallest score: the maximum is taken after scaling.
      float mn[2], f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = j * 8 + (lane & 3) * 2 + e;
            x = fmaxf(x, t < valid ? s[j][r * 2 + e] * a.scale_log2 : -INFINITY);
          }
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mn[r] = fmaxf(m[r], x);
      }
      const bool grew = mn[0] > m[0] || mn[1] > m[1];
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          f[r] = mn[r] == -INFINITY ? 1.f : exp2f(m[r] - mn[r]);
          l[r] *= f[r];
          m[r] = mn[r];
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i * 4 + 0] *= f[0];
          o[i * 4 + 1] *= f[0];
          o[i * 4 + 2] *= f[1];
          o[i * 4 + 3] *= f[1];
        }
      }
      // P as the sum of two 16-bit numbers (hi + lo): one alone would add an
      // error of the size of the output's own rounding.
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float base_m = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float p0 = 0.f, p1 = 0.f;
          if (r == 0 || two) {
            const int t = j * 8 + (lane & 3) * 2;
            if (t < valid) p0 = exp2f(fmaf(s[j][r * 2], a.scale_log2, -base_m));
            if (t + 1 < valid) p1 = exp2f(fmaf(s[j][r * 2 + 1], a.scale_log2, -base_m));
          }
          l[r] += p0 + p1;
          const uint32_t h = pair_of<T>::pack(p0, p1);
          const float2 back = pair_of<T>::unpack(h);
          hi[j * 2 + r] = h;
          lo[j * 2 + r] = pair_of<T>::pack(p0 - back.x, p1 - back.y);
        }
      }
#pragma unroll
      for (int nt = 0; nt < DP / 16; ++nt) {
        const int row = (((lane >> 3) & 1) << 3) + (lane & 7), ch = nt * 2 + (lane >> 4);
        uint32_t b0, b1, b2, b3;
        ldsm_x4_trans(base + C::kHalf + row * C::kRow + ((ch ^ (row & 7)) << 4), b0, b1, b2, b3);
        mma16816<T>::run(o + nt * 8, hi, b0, b1);
        mma16816<T>::run(o + nt * 8 + 4, hi, b2, b3);
        mma16816<T>::run(o + nt * 8, lo, b0, b1);
        mma16816<T>::run(o + nt * 8 + 4, lo, b2, b3);
      }
    } else {
      // lane = token (lane & 7) x quarter of the head dimension (lane >> 3)
      const int t = lane & 7, qt = lane >> 3;
      const int heads = min(GT, a.group - (c.h % a.hblocks) * GT);
      float s[GT] = {};
      const uint8_t* kr = ring + (base - smem_u32(ring)) + t * C::kRow;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const int ch = qt * (DP / 16) + i;
        const float4 kv = *reinterpret_cast<const float4*>(kr + ((ch ^ t) << 4));
#pragma unroll
        for (int g = 0; g < GT; ++g)
          if (g < heads) {
            const float4 qv = *reinterpret_cast<const float4*>(qs + g * DP + ch * 4);
            s[g] = fmaf(qv.x, kv.x, s[g]);
            s[g] = fmaf(qv.y, kv.y, s[g]);
            s[g] = fmaf(qv.z, kv.z, s[g]);
            s[g] = fmaf(qv.w, kv.w, s[g]);
          }
      }
      float* pw = ps + w * TT * GT;
#pragma unroll
      for (int g = 0; g < GT; ++g)
        if (g < heads) {
          s[g] += __shfl_xor_sync(0xffffffffu, s[g], 8);
          s[g] += __shfl_xor_sync(0xffffffffu, s[g], 16);
          float x = t < valid ? s[g] * a.scale_log2 : -INFINITY;
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          const float mn = fmaxf(m[g], x);
          if (mn > m[g]) {
            const float fac = exp2f(m[g] - mn);
            l[g] *= fac;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[g * (DP / 32) + i] *= fac;
            m[g] = mn;
          }
          const float base_m = m[g] == -INFINITY ? 0.f : m[g];
          const float p = t < valid ? exp2f(fmaf(s[g], a.scale_log2, -base_m)) : 0.f;
          if (qt == 0) {
            l[g] += p;
            pw[t * GT + g] = p;
          }
        }
      __syncwarp();
      const uint8_t* vr = ring + (base - smem_u32(ring)) + C::kHalf;
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        if (tt >= valid) break;
        float vv[DP / 32];
        if constexpr (DP == 64) {
          const float2 x = *reinterpret_cast<const float2*>(vr + tt * C::kRow + (((lane >> 1) ^ tt) << 4) + (lane & 1) * 8);
          vv[0] = x.x, vv[1] = x.y;
        } else {
#pragma unroll
          for (int j = 0; j < DP / 128; ++j) {
            const float4 x = *reinterpret_cast<const float4*>(vr + tt * C::kRow + (((j * 32 + lane) ^ tt) << 4));
            vv[j * 4] = x.x, vv[j * 4 + 1] = x.y, vv[j * 4 + 2] = x.z, vv[j * 4 + 3] = x.w;
          }
        }
        const float4 pa = *reinterpret_cast<const float4*>(pw + tt * GT);
        const float4 pb = *reinterpret_cast<const float4*>(pw + tt * GT + 4);
        const float pg[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
        for (int g = 0; g < GT; ++g)
          if (g < heads)
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[g * (DP / 32) + i] = fmaf(pg[g], vv[i], o[g * (DP / 32) + i]);
      }
      __syncwarp();
    }
  };

  // One value pair of (row g, columns d, d + 1) or one column group of the
  // joined output to its place.
  auto finish = [&](int64_t seg0, int64_t seg1) {
    const bool whole = seg0 >= t_begin && seg1 <= t_end;
    const int slot = 2 * int(blockIdx.x) + (seg0 >= t_begin ? 1 : 0);
    const int kvh = c.h / a.hblocks, g0 = (c.h % a.hblocks) * GT;
    const int heads = min(GT, a.group - g0);
    // the sum of a row over the lanes that share it
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if constexpr (C::kF32) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 4);
        l[r] = __shfl_sync(0xffffffffu, l[r], 0);
      }
    }
    __syncthreads();  // warp 0 has read the previous row's buffers
    if constexpr (C::kF32) {
      if (lane == 0)
#pragma unroll
        for (int g = 0; g < GT; ++g) ml[w * GT + g] = make_float2(m[g], l[g]);
    } else if ((lane & 3) == 0) {
      ml[w * GT + (lane >> 2)] = make_float2(m[0], l[0]);
      ml[w * GT + (lane >> 2) + 8] = make_float2(m[1], l[1]);
    }
#pragma unroll
    for (int rb = 0; rb < GT / RB; ++rb) {
      if (rb * RB >= heads) break;
      if (rb) __syncthreads();
      if (w) {
        float* dst = buf + (w - 1) * RB * DP;
        if constexpr (C::kF32) {
#pragma unroll
          for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
              const int d = DP == 64 ? lane * 2 + i : (i / 4) * 128 + lane * 4 + (i & 3);
              dst[r * DP + d] = o[(rb * RB + r) * (DP / 32) + i];
            }
        } else {
#pragma unroll
          for (int i = 0; i < DP / 8; ++i)
            *reinterpret_cast<float2*>(dst + (lane >> 2) * DP + i * 8 + (lane & 3) * 2) =
                make_float2(o[i * 4 + rb * 2], o[i * 4 + rb * 2 + 1]);
        }
      }
      __syncthreads();
      if (w == 0) {
        constexpr int kMine = C::kF32 ? RB : 1;
#pragma unroll
        for (int r = 0; r < kMine; ++r) {
          const int lr = C::kF32 ? r : (lane >> 2), g = rb * RB + lr;
          float M = -INFINITY, L = 0.f, fac[W];
#pragma unroll
          for (int i = 0; i < W; ++i) M = fmaxf(M, ml[i * GT + g].x);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const float2 x = ml[i * GT + g];
            fac[i] = x.x == -INFINITY ? (x.y != x.y ? x.y : 0.f) : exp2f(x.x - M);
            L += x.y * fac[i];
          }
          if (g < heads) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            T* out = static_cast<T*>(a.out) + int64_t(c.b) * a.o_row + int64_t(kvh * a.group + g0 + g) * a.o_head;
            float* po = a.part_o + (int64_t(slot) * GT + g) * DP;
            const bool one = C::kF32 ? lane == 0 : (lane & 3) == 0;
            if (one && !whole) a.part_ml[int64_t(slot) * GT + g] = make_float2(M, L);
            if (one && whole && a.lse)
              a.lse[int64_t(c.b) * a.kv_heads * a.group + kvh * a.group + g0 + g] =
                  L == 0.f ? -INFINITY : kLn2 * (M + log2f(L));
            if constexpr (C::kF32) {
#pragma unroll
              for (int i = 0; i < DP / 32; ++i) {
                const int d = DP == 64 ? lane * 2 + i : (i / 4) * 128 + lane * 4 + (i & 3);
                float y = o[g * (DP / 32) + i] * fac[0];
#pragma unroll
                for (int j = 1; j < W; ++j) y = fmaf(buf[((j - 1) * RB + lr) * DP + d], fac[j], y);
                if (!whole) po[d] = y;
                else if (d < a.dim) out[d] = y * inv;
              }
            } else {
#pragma unroll
              for (int i = 0; i < DP / 8; ++i) {
                const int d = i * 8 + (lane & 3) * 2;
                float y0 = o[i * 4 + rb * 2] * fac[0], y1 = o[i * 4 + rb * 2 + 1] * fac[0];
#pragma unroll
                for (int j = 1; j < W; ++j) {
                  const float2 x = *reinterpret_cast<const float2*>(buf + ((j - 1) * RB + lr) * DP + d);
                  y0 = fmaf(x.x, fac[j], y0);
                  y1 = fmaf(x.y, fac[j], y1);
                }
                if (!whole) *reinterpret_cast<float2*>(po + d) = make_float2(y0, y1);
                else if (d < a.dim) {
                  out[d] = from_f<T>(y0 * inv);
                  out[d + 1] = from_f<T>(y1 * inv);
                }
              }
            }
          }
        }
      }
    }
  };

  reset();
  load_q();
  int slot = 0;
  for (int it = 0; it < n; ++it) {
    load_stage();
    cp_async_wait<NS - 1>();
    __syncwarp();
    const int valid = cnt_w[slot];
    if (valid > 0) step(ring_w + slot * C::kStage, valid, a.group > 8);
    __syncwarp();  // the slot may be refilled
    slot = slot + 1 == NS ? 0 : slot + 1;
    if (c.tile + 1 == c.ntiles || it + 1 == n) {
      finish(seg_start, seg_start + c.ntiles);
      if (it + 1 < n) {
        seg_start += c.ntiles;
        cursor_next<C::kTile>(c, lens, a.rows, hb);
        reset();
        load_q();
      }
    } else {
      ++c.tile;
    }
  }
  cp_async_wait<0>();
}

// Joins the parts of every (row, head block) that was split, in part order,
// and writes rows of length 0.  One CTA per row and `per_cta` query heads of a
// block; its warps take the parts in turn.
template <typename T, int DP_>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendK a, int per_cta) {
  using C = Cfg<T, DP_>;
  constexpr int DP = C::DP, GT = C::GT, V = DP / 32;
  __shared__ float s_o[8][DP];
  __shared__ float2 s_ml[8];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hb = a.kv_heads * a.hblocks;
  const int groups = (min(GT, a.group) + per_cta - 1) / per_cta;
  const int h = blockIdx.x / groups, g_first = (blockIdx.x % groups) * per_cta, b = blockIdx.y;
  const int kvh = h / a.hblocks, g0 = (h % a.hblocks) * GT;
  const int heads = min(GT, a.group - g0);
  pdl_wait_primary();
  const int p0 = a.prefix[b], p1 = a.prefix[b + 1];
  const int64_t per = tiles_per_cta(int64_t(a.prefix[a.rows]) * hb, a.ctas, C::kMinTiles);
  const int tiles = p1 - p0;
  const int64_t t0 = int64_t(p0) * hb + int64_t(h) * tiles, t1 = t0 + tiles;
  const int c0 = tiles ? int(t0 / per) : 0, c1 = tiles ? int((t1 - 1) / per) : 0;
  if (tiles && c0 == c1) return;
  for (int g = g_first; g < min(heads, g_first + per_cta); ++g) {
    const int head = kvh * a.group + g0 + g;
    T* out = static_cast<T*>(a.out) + int64_t(b) * a.o_row + int64_t(head) * a.o_head;
    float* lse = a.lse ? a.lse + int64_t(b) * a.kv_heads * a.group + head : nullptr;
    if (!tiles) {
      for (int d = threadIdx.x; d < a.dim; d += blockDim.x) out[d] = from_f<T>(0.f);
      if (lse && threadIdx.x == 0) *lse = -INFINITY;
      continue;
    }
    float M = -INFINITY, L = 0.f, acc[V] = {};
#pragma unroll 4
    for (int c = c0 + w; c <= c1; c += 8) {
      const int64_t slot = 2 * int64_t(c) + (c == c0 ? 1 : 0);
      const float2 x = a.part_ml[slot * GT + g];
      const float* src = a.part_o + (slot * GT + g) * DP + lane * V;
      float y[V];
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float2 z = *reinterpret_cast<const float2*>(src + i);
        y[i] = z.x, y[i + 1] = z.y;
      }
      const float mn = fmaxf(M, x.x);
      const float fa = M == -INFINITY ? 0.f : exp2f(M - mn);
      const float fb = x.x == -INFINITY ? (x.y != x.y ? x.y : 0.f) : exp2f(x.x - mn);
      L = L * fa + x.y * fb;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = acc[i] * fa + y[i] * fb;
      M = mn;
    }
    if (lane == 0) s_ml[w] = make_float2(M, L);
#pragma unroll
    for (int i = 0; i < V; ++i) s_o[w][lane * V + i] = acc[i];
    __syncthreads();
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) mm = fmaxf(mm, s_ml[i].x);
    float fac[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      fac[i] = s_ml[i].x == -INFINITY ? (s_ml[i].y != s_ml[i].y ? s_ml[i].y : 0.f) : exp2f(s_ml[i].x - mm);
      ll += s_ml[i].y * fac[i];
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
      float y = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) y = fmaf(s_o[i][d], fac[i], y);
      out[d] = from_f<T>(y * inv);
    }
    if (lse && threadIdx.x == 0) *lse = ll == 0.f ? -INFINITY : kLn2 * (mm + log2f(ll));
    __syncthreads();
  }
}

template <typename T, int DP>
struct Inst {
  using C = Cfg<T, DP>;

  // CTAs of a launch over `rows` rows: all that fit the device at once.  The
  // occupancy is asked for once per device and size class of the row table.
  static int prepare(int rows, size_t* smem, int* ctas) {
    constexpr int kDevices = 32;
    static std::atomic<int> known[2][kDevices];
    const int cls = rows <= 256 ? 0 : 1;
    *smem = C::kFixed + (cls ? kAttendMaxRows : 256) * 4;
    int dev = 0;
    SLR_CHECK_CUDA(cudaGetDevice(&dev));
    int n = dev < kDevices ? known[cls][dev].load(std::memory_order_acquire) : 0;
    if (n == 0) {
      int occ = 0, sms = 0;
      SLR_CHECK_CUDA(cudaFuncSetAttribute(attend_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::kFixed + kAttendMaxRows * 4));
      SLR_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, attend_kernel<T, DP>, C::W * 32, *smem));
      SLR_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
      if (occ < 1) return fail(SLR_ERR_UNSUPPORTED, "attend: the kernel does not fit this device");
      n = sms * occ;
      if (dev < kDevices) known[cls][dev].store(n, std::memory_order_release);
    }
    *ctas = n;
    return SLR_OK;
  }

  static int launch(const AttendArgs& x, cudaStream_t s) {
    AttendK a = {};
    size_t smem = 0;
    int rc = prepare(x.rows, &smem, &a.ctas);
    if (rc) return rc;
    a.k = x.k;
    a.v = x.v;
    a.page_stride = x.page_stride;
    a.head_stride = x.head_stride;
    a.token_stride = x.token_stride;
    a.table = x.table;
    a.lens = x.lens;
    a.q = x.q;
    a.q_row = x.q_row;
    a.q_head = x.q_head;
    a.out = x.out;
    a.o_row = x.o_row;
    a.o_head = x.o_head;
    a.lse = x.lse;
    a.rows = x.rows;
    a.kv_heads = x.kv_heads;
    a.group = x.heads / x.kv_heads;
    a.hblocks = int(ceil_div(a.group, C::GT));
    a.dim = x.dim;
    a.page_size = x.page_size;
    a.max_pages = x.max_pages;
    a.num_pages = x.num_pages;
    a.scale_log2 = x.scale * kLog2e;
    // no more CTAs than tiles that rows of the greatest length could have
    const int64_t most = int64_t(a.rows) * a.kv_heads * a.hblocks *
                         ceil_div(int64_t(a.max_pages) * a.page_size, C::kTile * C::kMinTiles);
    if (most < a.ctas) a.ctas = int(most < 1 ? 1 : most);
    uint8_t* ws = static_cast<uint8_t*>(x.workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + size_t(2 * a.ctas) * C::GT * DP * 4);
    a.prefix = reinterpret_cast<int32_t*>(ws + size_t(2 * a.ctas) * C::GT * (DP * 4 + 8));
    if (need(a.ctas, a.rows) > x.workspace_bytes)
      return fail(SLR_ERR_WORKSPACE, "attend: workspace too small, need " + std::to_string(need(a.ctas, a.rows)) + " bytes");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.ctas);
    cfg.blockDim = dim3(C::W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_kernel<T, DP>, a));
    // heads of a block share a joining CTA when there are enough rows to fill the GPU
    const int gt = std::min(C::GT, a.group);
    const int per_cta = int64_t(a.rows) * x.heads <= 8 * 148 ? 1 : gt;
    cfg.gridDim = dim3(a.kv_heads * a.hblocks * int(ceil_div(gt, per_cta)), a.rows);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_join_kernel<T, DP>, a, per_cta));
    return SLR_OK;
  }

  static size_t need(int ctas, int rows) {
    return size_t(2 * ctas) * C::GT * (DP * 4 + 8) + size_t(rows + 1) * 4;
  }
  static int size(int rows, size_t* out) {
    size_t smem = 0;
    int ctas = 0;
    int rc = prepare(rows, &smem, &ctas);
    *out = rc ? 0 : need(ctas, rows);
    return rc;
  }
};

template <typename F> int by_shape(int dtype, int dim, F&& f) {
  const int dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  switch (dtype) {
    case SLR_F32: return dp == 64 ? f(Inst<float, 64>{}) : dp == 128 ? f(Inst<float, 128>{}) : f(Inst<float, 256>{});
    case SLR_F16: return dp == 64 ? f(Inst<__half, 64>{}) : dp == 128 ? f(Inst<__half, 128>{}) : f(Inst<__half, 256>{});
    default:
      return dp == 64 ? f(Inst<__nv_bfloat16, 64>{})
                      : dp == 128 ? f(Inst<__nv_bfloat16, 128>{}) : f(Inst<__nv_bfloat16, 256>{});
  }
}

}  // namespace

int attend_workspace_size(int dtype, int dim, int rows, size_t* bytes) {
  return by_shape(dtype, dim, [&](auto inst) { return decltype(inst)::size(rows, bytes); });
}

int launch_attend(const AttendArgs& a, cudaStream_t s) {
  return by_shape(a.dtype, a.dim, [&](auto inst) { return decltype(inst)::launch(a, s); });
}

int read_and_clear_status_attend(unsigned* out) {
  unsigned v = 0, zero = 0;
  SLR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_status_attend, sizeof(v)));
  if (v) SLR_CHECK_CUDA(cudaMemcpyToSymbol(g_status_attend, &zero, sizeof(zero)));
  *out = v;
  return SLR_OK;
}

}  // namespace slr
