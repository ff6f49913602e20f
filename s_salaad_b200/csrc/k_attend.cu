// Attention of one new token per row over a paged key-value cache.
//
//   s_t = scale · q·K_t,  o = Σ_t e^(s_t - m) V_t / Σ_t e^(s_t - m),  m = max_t s_t
//
// over the T = lens[b] tokens of row b; token t lies in page table[b, t / page_size]
// at slot t % page_size.  Every K and V element is used for the few query
// heads of its group only, so the kernel is bound by reading the cache once.
//
// Split: the tokens of every (row, block of query heads of one key head)
// are cut into tiles, all tiles of the call form one list (with kEndCost empty
// places behind each row's: the end of a row costs about as much time as that
// many tiles), and each warp takes an equal contiguous part of it (computed on
// the device from lens, so the launch does not depend on the lengths and can be
// replayed from a graph).  48 rows of up to 6007 tokens, 32/8 heads of 128,
// bf16, 591 MB: 103 us, 5.7 TB/s.
// A (row, head block) that lies inside one warp's part is written directly; the
// others leave (o, m, l) per part in the workspace and attend_join_kernel joins
// them in part order, so results do not depend on timing.
//
// Few and short rows (the whole call is latency) take a cluster of 1 to 8 CTAs
// per (row, head block) instead: its warps share the tiles and join through
// shared memory, in one launch without workspace (one row of 100 tokens, 8
// heads of 64: 3.2 us instead of 9.4).
//
// A warp streams its tiles through its own ring of cp.async stages, across the
// ends of rows, and waits for no other warp; the page number of a stage is
// fetched one stage ahead, the q of the next row (or head block) one row ahead.
// 16-bit types: Sᵀ = K·Qᵀ and Oᵀ = Vᵀ·Pᵀ on mma.sync, 8 query heads as the MMA's
// columns (a group is far below tcgen05's tile of 128, and the tensor pipe is
// 16 % busy in fp16, 20 % in bf16).  fp32: FFMA.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "internal.hpp"

namespace slr {

__device__ unsigned g_status_attend;

namespace {

namespace cg = cooperative_groups;

// A warp takes at least this many places.  One row of 512 tokens, 8 key heads of
// 128, bf16: 2 places 10.4 us, 4: 11.9, 1: 9.5, but then 16000 tokens of one key
// head are 1000 parts to join: 18.2 us, 2: 14.5.
constexpr int kMinTiles = 2;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

// The reference of the exponentials follows the running maximum within this
// many powers of two: most tiles then need one vote instead of a maximum over
// the lanes and a rescaling.
constexpr float kSlack = 8.f;
// ... and lies this many below the maximum where the weights become fp16, whose
// steps are 2^-24 at the small end: the greatest weight is 2^7 to 2^15 (fp16 ends
// at 2^16), so small ones are held to 2^-32 of it. It cancels in the output.
template <typename T> constexpr float kBelow = std::is_same<T, __half>::value ? 7.f : 0.f;

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
  float* part_o;     // [2 * workers][GT][DP]
  float2* part_ml;   // [2 * workers][GT]
  int32_t* prefix;   // [rows + 1] places before each row
  int rows, kv_heads, group, hblocks, dim, page_size, page_shift, max_pages, num_pages, workers;
  int q_wide, o_pairs;  // q can be read in 16 bytes (fp32) or two elements, out written in two elements
  float scale_log2;
};

// A row's end (its output, the next row's q from DRAM) takes the time of some
// tiles.  8 rows of 1 to 4100 tokens, 32 heads, bf16: 1 place 77 us, 2: 58, 3:
// 52.5, 4: 52.7, 6: 53; 400 rows of 1 to 700 tokens: 129, 118, 109.5, 113, 111.
constexpr int kEndCost = 3;
__device__ __forceinline__ int places(int tiles) { return tiles ? tiles + kEndCost : 0; }

// Places that one warp takes of a list of n: an equal part, but not less than
// kMinTiles (a join costs more than a few tiles in a row).
__device__ __forceinline__ int64_t tiles_per_worker(int64_t n, int workers) {
  const int64_t per = (n + workers - 1) / workers;
  return per < kMinTiles ? kMinTiles : per;
}

// 16 bytes, or (n = 0) 16 zero bytes without reading.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Transposes an 8 x 8 matrix of 16-bit elements held one row per four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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

// Shape of one instance: DP head dimension padded to a power of two, GT query
// heads per warp, W warps, TT tokens per tile, NS stages per warp.  DP = 128: 3
// CTAs of 64 KB, two stages per warp (2 x 131071 tokens, fp16: 152.6 us; 2 CTAs
// with three stages 158.5); DP = 64: four stages of 4 KB (12000 tokens, bf16: 98
// us, three 104.5, six 115).
template <typename T, int DP_, int GT_> struct Cfg {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int DP = DP_, GT = GT_;
  static constexpr int W = 4;
  static constexpr int TT = kF32 ? 8 : 16;
  static constexpr int NS = DP == 64 && !(kF32 && GT == 8) ? 4 : 2;
  static constexpr int kRow = DP * int(sizeof(T));     // bytes of a token's row
  static constexpr int kHalf = TT * kRow;              // K (or V) bytes of a stage
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = W * NS * kStage;
  static constexpr bool kQRegs = GT * DP <= 256;       // fp32: a lane's quarter of q in registers
  static constexpr int kQ = kF32 && !kQRegs ? W * GT * DP * 4 : 0;
  static constexpr int kP = kF32 ? W * TT * GT * 4 : 0;
  static constexpr int kCnt = W * NS * 4;
  static constexpr int kFixed = kRing + kQ + kP + kCnt + 64 + GT * 8;
};

// Place in the list of tiles: row b, head block h, tile of the row.
struct Cursor {
  int b, h, tile, ntiles, len;
  int64_t seg;  // place of its first tile
  __device__ int64_t place() const { return seg + tile; }
};

template <int TT>
__device__ __forceinline__ void cursor_next(Cursor& c, const int* lens, int rows, int hb) {
  if (++c.tile < c.ntiles) return;
  c.tile = 0;
  c.seg += places(c.ntiles);
  if (++c.h < hb) return;
  c.h = 0;
  do {
    ++c.b;
  } while (c.b < rows && lens[c.b] == 0);
  c.len = c.b < rows ? lens[c.b] : 0;
  c.ntiles = (c.len + TT - 1) / TT;
}

// To the first tile of the next (row, head block).
template <int TT>
__device__ __forceinline__ void cursor_skip(Cursor& c, const int* lens, int rows, int hb) {
  c.tile = c.ntiles - 1;
  cursor_next<TT>(c, lens, rows, hb);
}

// kSmall: a cluster = (row, head block), the tiles of the row dealt to its warps
// in equal parts.
template <typename T, int DP_, int GT_, bool kSmall>
__global__ void __launch_bounds__(Cfg<T, DP_, GT_>::W * 32) attend_kernel(const AttendK a) {
  using C = Cfg<T, DP_, GT_>;
  constexpr int DP = C::DP, W = C::W, TT = C::TT, NS = C::NS, GT = C::GT;
  constexpr int kThreads = W * 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float* qs = reinterpret_cast<float*>(smem + C::kRing) + (threadIdx.x >> 5) * GT * DP;  // this warp's
  float* ps = reinterpret_cast<float*>(smem + C::kRing + C::kQ);
  int* cnt = reinterpret_cast<int*>(smem + C::kRing + C::kQ + C::kP);
  int* scratch = cnt + W * NS;                       // 16 words
  float2* ml = reinterpret_cast<float2*>(scratch + 16);  // kSmall: [GT] maximum and sum of the CTA
  int* lens = reinterpret_cast<int*>(smem + C::kFixed);  // [rows]

  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int hb = a.kv_heads * a.hblocks;
  pdl_wait_primary();
  pdl_launch_dependents();

  // ---- this warp's part of the list of tiles
  const int64_t cap = int64_t(a.max_pages) * a.page_size;
  Cursor c;
  int64_t t_begin, t_end;
  int worker = 0;
  bool active = true;
  if constexpr (kSmall) {
    const int cs = int(cg::this_cluster().num_blocks()), rank = int(cg::this_cluster().block_rank());
    c.b = int(blockIdx.x) / cs / hb;
    c.h = int(blockIdx.x) / cs % hb;
    int64_t n = a.lens[c.b];
    if (n < 0 || n > cap) {
      if (tid == 0 && rank == 0) atomicOr(&g_status_attend, SLR_BAD_INDEX_BIT);
      n = n < 0 ? 0 : cap;
    }
    c.len = int(n);
    c.ntiles = (c.len + TT - 1) / TT;
    const int per = (c.ntiles + W * cs - 1) / (W * cs);
    c.seg = 0;
    c.tile = (rank * W + w) * per;
    t_begin = c.tile;
    t_end = min(c.ntiles, c.tile + per);
    active = t_begin < t_end;
  } else {
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
      mine += places(int((n + TT - 1) / TT));
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
    const int64_t per = tiles_per_worker(n_all, a.workers);
    for (int r = r0; r < r1; ++r) {
      if (blockIdx.x == 0) a.prefix[r] = before;
      const int nt = places((lens[r] + TT - 1) / TT);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int64_t t = (int64_t(blockIdx.x) * W + i) * per;
        if (int64_t(before) * hb <= t && t < int64_t(before + nt) * hb) {
          scratch[4 + 2 * i] = r;
          scratch[5 + 2 * i] = before;
        }
      }
      before += nt;
    }
    if (blockIdx.x == 0) {
      if (tid == 0) a.prefix[a.rows] = total;
      if (bad) atomicOr(&g_status_attend, SLR_BAD_INDEX_BIT);
    }
    __syncthreads();
    worker = int(blockIdx.x) * W + w;
    t_begin = worker * per;
    t_end = t_begin + per < n_all ? t_begin + per : n_all;
    if (t_begin >= t_end) return;  // no barrier of the CTA from here on
    c.b = scratch[4 + 2 * w];
    c.len = lens[c.b];
    c.ntiles = (c.len + TT - 1) / TT;
    {
      const int64_t row0 = int64_t(scratch[5 + 2 * w]) * hb, per_head = places(c.ntiles);
      c.h = int((t_begin - row0) / per_head);
      c.seg = row0 + c.h * per_head;
      c.tile = int(t_begin - c.seg);
      // between two rows: on to the next
      if (c.tile >= c.ntiles) cursor_skip<TT>(c, lens, a.rows, hb);
    }
    if (c.place() >= t_end || c.b >= a.rows) return;
  }

  // ---- the ring
  // Chunk `ch` of a token's row lies at ch ^ (row & 7): the eight rows of an
  // ldmatrix (or the lanes of a 16-byte read) meet all banks once.
  const uint32_t ring_w = smem_u32(ring) + w * NS * C::kStage;
  int* cnt_w = cnt + w * NS;
  auto kv_head = [&](int h) { return a.hblocks == 1 ? h : h / a.hblocks; };
  auto page_of = [&](int t) { return a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size; };
  Cursor f = c;
  auto fetch_page = [&](const Cursor& u) -> int {
    const int t0 = u.tile * TT;
    return t0 < u.len ? a.table[int64_t(u.b) * a.max_pages + page_of(t0)] : 0;
  };
  constexpr int E = 16 / int(sizeof(T));             // elements of a 16-byte chunk
  constexpr int CH = DP / E;                         // chunks of a row
  constexpr int kRowStep = CH <= 32 ? 32 / CH : 1;   // rows that a warp-wide load covers
  constexpr int kColStep = CH <= 32 ? 1 : CH / 32;   // warp-wide loads of one row
  const int lrow = lane / CH, lch = lane % CH;
  const uint32_t ldst = lrow * C::kRow + ((lch ^ lrow) << 4);
  const int64_t lsrc = lrow * a.token_stride + lch * E;
  // one lane per 128 bytes of a block's q
  auto prefetch_q = [&]() {
    constexpr int kLine = 128 / int(sizeof(T)), kLines = DP / kLine;
    const int kvh = kv_head(f.h), g0 = (f.h - kvh * a.hblocks) * GT;
    const T* q = static_cast<const T*>(a.q) + int64_t(f.b) * a.q_row + int64_t(kvh * a.group + g0) * a.q_head;
#pragma unroll
    for (int i = 0; i < GT * kLines; i += 32) {
      const int g = (i + lane) / kLines, d = (i + lane) % kLines * kLine;
      if (g < GT && g0 + g < a.group && d < a.dim) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + g * a.q_head + d));
    }
  };
  int page = active ? fetch_page(f) : 0;
  int load_slot = 0;
  bool more = active;  // tiles left to load
  auto load_stage = [&]() {
    if (more) {
      const int t0 = f.tile * TT;
      int valid = min(TT, f.len - t0);
      if (valid > 0 && (page < 0 || page >= a.num_pages)) {
        if (lane == 0) atomicOr(&g_status_attend, SLR_BAD_INDEX_BIT);
        valid = 0;
      }
      if (lane == 0) cnt_w[load_slot] = valid;
      if (valid > 0) {
        const int64_t off = int64_t(page) * a.page_stride + int64_t(kv_head(f.h)) * a.head_stride +
                            int64_t(t0 - page_of(t0) * a.page_size) * a.token_stride + lsrc;
        const T* ks = static_cast<const T*>(a.k) + off;
        const T* vs = static_cast<const T*>(a.v) + off;
        const uint32_t dst = ring_w + load_slot * C::kStage + ldst;
        if (valid == TT && a.dim == DP) {
#pragma unroll
          for (int i = 0; i < TT / kRowStep; ++i) {
#pragma unroll
            for (int j = 0; j < kColStep; ++j) {
              const uint32_t d = (dst + i * kRowStep * C::kRow + j * 512) ^ (((i * kRowStep) & 7) << 4);
              cp_async16(d, ks + j * 32 * E, 16);
              cp_async16(d + C::kHalf, vs + j * 32 * E, 16);
            }
            ks += kRowStep * a.token_stride;
            vs += kRowStep * a.token_stride;
          }
        } else {
          const T* k0 = static_cast<const T*>(a.k);
          const T* v0 = static_cast<const T*>(a.v);
#pragma unroll
          for (int i = 0; i < TT / kRowStep; ++i) {
#pragma unroll
            for (int j = 0; j < kColStep; ++j) {
              const bool in = lrow + i * kRowStep < valid && (lch + j * 32) * E < a.dim;
              const uint32_t d = (dst + i * kRowStep * C::kRow + j * 512) ^ (((i * kRowStep) & 7) << 4);
              cp_async16(d, in ? ks + j * 32 * E : k0, in ? 16 : 0);
              cp_async16(d + C::kHalf, in ? vs + j * 32 * E : v0, in ? 16 : 0);
            }
            ks += kRowStep * a.token_stride;
            vs += kRowStep * a.token_stride;
          }
        }
      }
      if constexpr (kSmall) {
        more = ++f.tile < t_end;
        if (more) page = fetch_page(f);
      } else {
        cursor_next<TT>(f, lens, a.rows, hb);
        more = f.b < a.rows && f.place() < t_end;
        if (more) {
          page = fetch_page(f);
          if (f.tile == 0) prefetch_q();
        }
      }
      load_slot = load_slot + 1 == NS ? 0 : load_slot + 1;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load_stage();

  // ---- running softmax of this warp: log2-domain reference, sum, output
  // 16-bit: the MMAs compute Sᵀ = K · Qᵀ (16 tokens x 8 heads) and Oᵀ = Vᵀ · Pᵀ
  // (16 columns x 8 heads), so a lane has heads 2 (lane % 4) and + 1 of every
  // 8 in both; groups of up to 8 heads waste no MMA on empty rows.
  // fp32: every lane all GT heads, DP / 32 columns each.
  constexpr int NT = C::kF32 ? 1 : GT / 8;
  constexpr int kStat = C::kF32 ? GT : 2 * NT;
  constexpr int kOut = C::kF32 ? GT * (DP / 32) : NT * DP / 4;
  float m[kStat], l[kStat], o[kOut];
  constexpr int kQf = C::kF32 ? 1 : NT * DP / 8, kQr = C::kF32 && C::kQRegs ? GT * DP / 4 : 1;
  constexpr bool kAhead = kSmall ? false : C::kF32 ? kQr > 1 && kQr <= 32 : kQf <= 32;  // the next q fits the registers too
  uint32_t qf[kQf], qf_next[kAhead && !C::kF32 ? kQf : 1];
  float qr[kQr], qr_next[kAhead && C::kF32 ? kQr : 1];
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < kStat; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int i = 0; i < kOut; ++i) o[i] = 0.f;
  };
  // q of the (row, head block) at u into registers (this warp's shared memory for wide fp32 groups)
  auto load_q = [&](const Cursor& u, uint32_t* to16, float* to32) {
    const int kvh = kv_head(u.h), g0 = (u.h - kvh * a.hblocks) * GT;
    const T* q = static_cast<const T*>(a.q) + int64_t(u.b) * a.q_row + int64_t(kvh * a.group + g0) * a.q_head;
    const int heads = min(GT, a.group - g0);
    if constexpr (C::kF32) {
      if constexpr (C::kQRegs) {
#pragma unroll
        for (int i = 0; i < kQr; i += 4) {
          const int g = i / (DP / 4), d = (lane >> 3) * (DP / 4) + i % (DP / 4);
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (g < heads && d < a.dim) {  // head_dim is a multiple of 8
            const float* p = q + g * a.q_head + d;
            v = a.q_wide ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
          }
          to32[i] = v.x, to32[i + 1] = v.y, to32[i + 2] = v.z, to32[i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < GT * DP / 128; ++i) {
          const int at = i * 128 + lane * 4, g = at / DP, d = at % DP;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (g < heads && d < a.dim) {  // head_dim is a multiple of 8
            const float* p = q + g * a.q_head + d;
            v = a.q_wide ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
          }
          *reinterpret_cast<float4*>(qs + at) = v;
        }
        __syncwarp();
      }
    } else {
      const unsigned short* qu = reinterpret_cast<const unsigned short*>(q);
#pragma unroll
      for (int i = 0; i < kQf; ++i) {
        // i = (k-step, head tile, half of the k-step)
        const int g = (i >> 1) % NT * 8 + (lane >> 2), d = (i / (2 * NT)) * 16 + (i & 1) * 8 + (lane & 3) * 2;
        uint32_t v = 0;
        if (g < heads && d < a.dim) {
          const unsigned short* p = qu + g * a.q_head + d;
          v = a.q_wide ? *reinterpret_cast<const uint32_t*>(p) : uint32_t(p[0]) | (uint32_t(p[1]) << 16);
        }
        to16[i] = v;
      }
    }
  };
  // the q that comes after the one in use, if it is still this warp's
  auto load_next_q = [&]() {
    if constexpr (kAhead)
      if (c.seg + places(c.ntiles) < t_end) {
        Cursor u = c;
        cursor_skip<TT>(u, lens, a.rows, hb);
        if (u.b < a.rows) load_q(u, qf_next, qr_next);
      }
  };
  auto take_next_q = [&]() {
    if constexpr (!kAhead) load_q(c, qf, qr);
    else if constexpr (C::kF32) {
#pragma unroll
      for (int i = 0; i < kQr; ++i) qr[i] = qr_next[i];
    } else {
#pragma unroll
      for (int i = 0; i < kQf; ++i) qf[i] = qf_next[i];
    }
  };

  auto step = [&](uint32_t base, int valid) {
    if constexpr (!C::kF32) {
      const int r8 = lane & 7;
      float s[NT][2][4] = {};
      {
        const uint32_t at = base + (((lane >> 3) & 1) * 8 + r8) * C::kRow + (((lane >> 4) ^ r8) << 4);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          uint32_t k[4];
          ldsm_x4(at ^ (ks << 5), k[0], k[1], k[2], k[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)  // two chains: half the latency
            mma16816<T>::run(s[nt][ks & 1], k, qf[(ks * NT + nt) * 2], qf[(ks * NT + nt) * 2 + 1]);
        }
      }
      // With scale < 0 the largest product is the smallest score: the maximum is taken after scaling.
      float mn[kStat];
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][0][e] = __fmul_rn(s[nt][0][e] + s[nt][1][e], a.scale_log2);  // not fused, see below
          if (valid < TT && (lane >> 2) + (e >> 1) * 8 >= valid) s[nt][0][e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mn[nt * 2 + e] = fmaxf(s[nt][0][e], s[nt][0][e + 2]) - kBelow<T>;
          grew |= mn[nt * 2 + e] > m[nt * 2 + e] + kSlack;
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float fac[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = nt * 2 + e;
            float x = fmaxf(m[i], mn[i]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            fac[e] = x == m[i] ? 1.f : ex2(m[i] - x);
            l[i] *= fac[e];
            m[i] = x;
          }
#pragma unroll
          for (int i = 0; i < DP / 4; ++i) o[nt * (DP / 4) + i] *= fac[i & 1];
        }
      }
      // The scaled score is rounded before the reference, which is one of them,
      // is taken from it: at scores of 10^8 the rounding of a fused product
      // against it would be a power of two that overflows.
      // P as a sum of 16-bit numbers, each the rounding of what the ones before
      // leave: one alone would add an error of the size of the output's own
      // rounding.  Two fp16 keep 22 bits, three bf16 all 24; two bf16 would keep
      // 16, which rounds one output in 500 the other way (48 rows of up to 6007
      // tokens: 102.4 us with two, 103.5 with three; 24 rows, groups of 16 heads
      // of 256: 108.5, 112.6; two columns of tiles side by side gain nothing).
      constexpr int kParts = std::is_same<T, __half>::value ? 2 : 3;
      uint32_t part[NT][2][kParts];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float top = m[nt * 2 + (e & 1)];
          p[e] = ex2(s[nt][0][e] - (top == -INFINITY ? 0.f : top));
          // at scores of 10^7 the reference's own steps can put it farther below
          if constexpr (kBelow<T> != 0.f) asm("min.NaN.f32 %0, %0, %1;" : "+f"(p[e]) : "f"(65504.f));
          l[nt * 2 + (e & 1)] += p[e];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x0 = p[j * 2], x1 = p[j * 2 + 1];
#pragma unroll
          for (int i = 0; i < kParts; ++i) {
            const uint32_t h = pair_of<T>::pack(x0, x1);
            const float2 back = pair_of<T>::unpack(h);
            part[nt][j][i] = transpose8(h);
            x0 -= back.x, x1 -= back.y;
          }
        }
      }
      const uint32_t at = base + C::kHalf + ((lane >> 4) * 8 + r8) * C::kRow + ((((lane >> 3) & 1) ^ r8) << 4);
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) {
        uint32_t v[4];
        ldsm_x4_trans(at ^ (dt << 5), v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < kParts; ++i)
            mma16816<T>::run(o + nt * (DP / 4) + dt * 4, v, part[nt][0][i], part[nt][1][i]);
        }
      }
    } else {
      // lane = token (lane & 7) x quarter of the head dimension (lane >> 3)
      const int t = lane & 7, qt = lane >> 3;
      Pair s2[GT] = {};  // even and odd columns
      const uint8_t* stage = ring + (base - smem_u32(ring));
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const int ch = qt * (DP / 16) + i;
        const ulonglong2 kv = *reinterpret_cast<const ulonglong2*>(stage + t * C::kRow + ((ch ^ t) << 4));
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          ulonglong2 qv;
          if constexpr (C::kQRegs) {
            const float* x = qr + g * (DP / 4) + i * 4;
            qv = make_ulonglong2(pair(x[0], x[1]), pair(x[2], x[3]));
          } else {
            qv = *reinterpret_cast<const ulonglong2*>(qs + g * DP + ch * 4);
          }
          s2[g] = fma2(qv.x, kv.x, s2[g]);
          s2[g] = fma2(qv.y, kv.y, s2[g]);
        }
      }
      float s[GT];
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        float even, odd;
        unpair(s2[g], even, odd);
        s[g] = even + odd;
      }
      float* pw = ps + w * TT * GT;
      bool grew = false;
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        s[g] += __shfl_xor_sync(0xffffffffu, s[g], 8);
        s[g] += __shfl_xor_sync(0xffffffffu, s[g], 16);
        s[g] = __fmul_rn(s[g], a.scale_log2);  // rounded before the reference is taken from it, as above
        grew |= t < valid && s[g] > m[g] + kSlack;
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          float x = t < valid ? fmaxf(m[g], s[g]) : m[g];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          const float fac = x == m[g] ? 1.f : ex2(m[g] - x);
          l[g] *= fac;
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) o[g * (DP / 32) + i] *= fac;
          m[g] = x;
        }
      }
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        const float p = t < valid ? ex2(s[g] - (m[g] == -INFINITY ? 0.f : m[g])) : 0.f;
        if (qt == 0) {
          l[g] += p;
          pw[t * GT + g] = p;
        }
      }
      __syncwarp();
      const uint8_t* vr = stage + C::kHalf;
      auto add = [&](int tt) {
        Pair vv[DP / 64];
        float pg[GT];
        if constexpr (DP == 64) {
          vv[0] = *reinterpret_cast<const Pair*>(vr + tt * C::kRow + (((lane >> 1) ^ tt) << 4) + (lane & 1) * 8);
        } else {
#pragma unroll
          for (int j = 0; j < DP / 128; ++j) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(vr + tt * C::kRow + (((j * 32 + lane) ^ tt) << 4));
            vv[j * 2] = x.x, vv[j * 2 + 1] = x.y;
          }
        }
        if constexpr (GT % 4 == 0) {
#pragma unroll
          for (int g = 0; g < GT; g += 4) {
            const float4 x = *reinterpret_cast<const float4*>(pw + tt * GT + g);
            pg[g] = x.x, pg[g + 1] = x.y, pg[g + 2] = x.z, pg[g + 3] = x.w;
          }
        } else {
#pragma unroll
          for (int g = 0; g < GT; ++g) pg[g] = pw[tt * GT + g];
        }
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          const Pair p2 = pair(pg[g], pg[g]);
#pragma unroll
          for (int i = 0; i < DP / 64; ++i) {
            float* at = o + g * (DP / 32) + i * 2;
            unpair(fma2(p2, vv[i], pair(at[0], at[1])), at[0], at[1]);
          }
        }
      };
      // rows behind the length are zeros in the stage, their p is 0
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) add(tt);
      __syncwarp();
    }
  };

  // End of a row's tiles (or of this warp's part): the result is written as
  // output, or as one part of a split row to the workspace.
  auto finish = [&](int64_t seg0, int64_t seg1) {
    const bool whole = seg0 >= t_begin && seg1 <= t_end;
    const int64_t part = 2 * int64_t(worker) + (seg0 >= t_begin ? 1 : 0);
    const int kvh = kv_head(c.h), g0 = (c.h - kvh * a.hblocks) * GT;
    const int heads = min(GT, a.group - g0);
    const int64_t head0 = int64_t(kvh) * a.group + g0;
    T* out = static_cast<T*>(a.out) + int64_t(c.b) * a.o_row + head0 * a.o_head;
    float* po = a.part_o + part * GT * DP;
    // the sum of a head over the lanes that share it
#pragma unroll
    for (int i = 0; i < kStat; ++i)
#pragma unroll
      for (int x = C::kF32 ? 1 : 4; x < (C::kF32 ? 8 : 32); x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    if constexpr (C::kF32) {
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        l[g] = __shfl_sync(0xffffffffu, l[g], 0);
        if (g >= heads) break;
        const float inv = l[g] == 0.f ? 0.f : 1.f / l[g];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const int d = DP == 64 ? lane * 2 + i : (i / 4) * 128 + lane * 4 + (i & 3);
          const float y = o[g * (DP / 32) + i];
          if (!whole) po[g * DP + d] = y;
          else if (d < a.dim) out[g * a.o_head + d] = y * inv;
        }
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt * 8 >= heads) break;
        const float inv0 = l[nt * 2] == 0.f ? 0.f : 1.f / l[nt * 2];
        const float inv1 = l[nt * 2 + 1] == 0.f ? 0.f : 1.f / l[nt * 2 + 1];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          const float y0 = o[nt * (DP / 4) + i * 2], y1 = o[nt * (DP / 4) + i * 2 + 1];
          if (whole) {
            // heads across lanes, two columns in each
            const uint32_t v = transpose8(pair_of<T>::pack(y0 * inv0, y1 * inv1));
            const int g = nt * 8 + (lane >> 2), d = i * 8 + (lane & 3) * 2;
            if (g < heads && d < a.dim) {
              unsigned short* dst = reinterpret_cast<unsigned short*>(out) + g * a.o_head + d;
              if (a.o_pairs) *reinterpret_cast<uint32_t*>(dst) = v;
              else dst[0] = static_cast<unsigned short>(v), dst[1] = static_cast<unsigned short>(v >> 16);
            }
          } else {
            float* dst = po + (nt * 8 + (lane & 3) * 2) * DP + i * 8 + (lane >> 2);
            if (nt * 8 + (lane & 3) * 2 < heads) dst[0] = y0;
            if (nt * 8 + (lane & 3) * 2 + 1 < heads) dst[DP] = y1;
          }
        }
      }
    }
    // one lane per head: its maximum and sum
    if (C::kF32 ? lane == 0 : lane < 4) {
#pragma unroll
      for (int i = 0; i < kStat; ++i) {
        const int g = C::kF32 ? i : (i >> 1) * 8 + lane * 2 + (i & 1);
        if (g >= heads) continue;
        if (!whole) a.part_ml[part * GT + g] = make_float2(m[i], l[i]);
        else if (a.lse)
          a.lse[int64_t(c.b) * a.kv_heads * a.group + head0 + g] =
              l[i] == 0.f ? -INFINITY : kLn2 * ((m[i] == -INFINITY ? 0.f : m[i]) + log2f(l[i]));
      }
    }
  };

  // kSmall: the warps' results joined through the place of their rings
  auto finish_small = [&]() {
    cp_async_wait<0>();
#pragma unroll
    for (int i = 0; i < kStat; ++i)
#pragma unroll
      for (int x = C::kF32 ? 1 : 4; x < (C::kF32 ? 8 : 32); x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    __syncwarp();
    constexpr int kO = DP + 4;  // floats of a head's row (bank offset 4)
    static_assert(GT * kO * 4 + GT * 8 <= NS * C::kStage, "a warp's rows take its ring's place");
    float* mine = reinterpret_cast<float*>(ring + w * NS * C::kStage);
    if constexpr (C::kF32) {
#pragma unroll
      for (int g = 0; g < GT; ++g) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
          mine[g * kO + (DP == 64 ? lane * 2 + i : (i / 4) * 128 + lane * 4 + (i & 3))] = o[g * (DP / 32) + i];
        if (lane == 0) mine[GT * kO + 2 * g] = m[g], mine[GT * kO + 2 * g + 1] = l[g];
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < DP / 4; ++i)
          mine[(nt * 8 + (lane & 3) * 2 + (i & 1)) * kO + (i >> 2) * 16 + ((i >> 1) & 1) * 8 + (lane >> 2)] =
              o[nt * (DP / 4) + i];
      if (lane < 4)
#pragma unroll
        for (int i = 0; i < kStat; ++i) {
          const int g = (i >> 1) * 8 + lane * 2 + (i & 1);
          mine[GT * kO + 2 * g] = m[i], mine[GT * kO + 2 * g + 1] = l[i];
        }
    }
    __syncthreads();
    const int kvh = kv_head(c.h), g0 = (c.h - kvh * a.hblocks) * GT;
    const int heads = min(GT, a.group - g0);
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = int(cluster.num_blocks());
    float* part = reinterpret_cast<float*>(ring);
    constexpr int kPart = NS * C::kStage / 4;
    auto write = [&](int g, int d, float top, float sum, float y) {
      const int head = kvh * a.group + g0 + g;
      if (d < a.dim)
        static_cast<T*>(a.out)[int64_t(c.b) * a.o_row + int64_t(head) * a.o_head + d] =
            from_f<T>(sum == 0.f ? 0.f : y / sum);
      if (d == 0 && a.lse)
        a.lse[int64_t(c.b) * a.kv_heads * a.group + head] =
            sum == 0.f ? -INFINITY : kLn2 * ((top == -INFINITY ? 0.f : top) + log2f(sum));
    };
    // a part without a finite score has sum 0, or NaN if a score was NaN
    auto weight = [](float m, float l, float top) { return m == -INFINITY ? (l != l ? l : 0.f) : ex2(m - top); };
    for (int i = tid; i < heads * DP; i += kThreads) {
      const int g = i / DP, d = i % DP;
      float top = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) top = fmaxf(top, part[j * kPart + GT * kO + 2 * g]);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float pl = part[j * kPart + GT * kO + 2 * g + 1];
        const float fac = weight(part[j * kPart + GT * kO + 2 * g], pl, top);
        sum = fmaf(pl, fac, sum);
        y = fmaf(part[j * kPart + g * kO + d], fac, y);
      }
      if (cs == 1) {
        write(g, d, top, sum, y);
      } else {
        part[g * kO + d] = y;  // read by this thread alone
        if (d == 0) ml[g] = make_float2(top, sum);
      }
    }
    if (cs == 1) return;
    cluster.sync();
    for (int i = int(cluster.block_rank()) * kThreads + tid; i < heads * DP; i += cs * kThreads) {
      const int g = i / DP, d = i % DP;
      float top = -INFINITY, sum = 0.f, y = 0.f;
      for (int j = 0; j < cs; ++j) top = fmaxf(top, cluster.map_shared_rank(ml, j)[g].x);
      for (int j = 0; j < cs; ++j) {
        const float2 x = cluster.map_shared_rank(ml, j)[g];
        const float fac = weight(x.x, x.y, top);
        sum = fmaf(x.y, fac, sum);
        y = fmaf(cluster.map_shared_rank(part, j)[g * kO + d], fac, y);
      }
      write(g, d, top, sum, y);
    }
    cluster.sync();  // the parts stay until they have been read
  };

  reset();
  if (active) load_q(c, qf, qr);
  if constexpr (kSmall) {
    int slot = 0;
    for (int64_t t = t_begin; t < t_end; ++t) {
      load_stage();
      cp_async_wait<NS - 1>();
      __syncwarp();
      const int valid = cnt_w[slot];
      if (valid > 0) step(ring_w + slot * C::kStage, valid);
      __syncwarp();  // the slot may be refilled
      slot = slot + 1 == NS ? 0 : slot + 1;
    }
    finish_small();
    return;
  }
  load_next_q();
  int slot = 0;
  while (true) {
    load_stage();
    cp_async_wait<NS - 1>();
    __syncwarp();
    const int valid = cnt_w[slot];
    if (valid > 0) step(ring_w + slot * C::kStage, valid);
    __syncwarp();  // the slot may be refilled
    slot = slot + 1 == NS ? 0 : slot + 1;
    if (c.tile + 1 < c.ntiles && c.place() + 1 < t_end) {
      ++c.tile;
      continue;
    }
    finish(c.seg, c.seg + c.ntiles);
    cursor_skip<TT>(c, lens, a.rows, hb);
    if (c.b >= a.rows || c.place() >= t_end) break;
    reset();
    take_next_q();
    load_next_q();
  }
  cp_async_wait<0>();
}

// Joins the parts of every (row, head) that was split, in part order, and
// writes rows of length 0.  `wph` warps (a power of two) share a head: each
// joins every wph-th part, then the first joins theirs.
template <typename T, int DP_, int GT_>
__global__ void __launch_bounds__(1024) attend_join_kernel(const AttendK a, int wph) {
  using C = Cfg<T, DP_, GT_>;
  constexpr int DP = C::DP, GT = C::GT, V = DP / 32;
  __shared__ float s_o[32][DP];
  __shared__ float2 s_ml[32];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int hb = a.kv_heads * a.hblocks, n_heads = a.kv_heads * a.group;
  const int64_t item = int64_t(blockIdx.x) * (warps / wph) + w / wph;  // (row, head)
  const int sub = w % wph;
  const bool in = item < int64_t(a.rows) * n_heads;
  const int b = in ? int(item / n_heads) : 0, head = in ? int(item % n_heads) : 0;
  const int kvh = head / a.group, hg = head % a.group, h = kvh * a.hblocks + hg / GT, g = hg % GT;
  pdl_wait_primary();
  const int p0 = a.prefix[b], p1 = a.prefix[b + 1];
  const int64_t per = tiles_per_worker(int64_t(a.prefix[a.rows]) * hb, a.workers);
  const int tiles = in && p1 > p0 ? p1 - p0 - kEndCost : 0;
  const int64_t t0 = int64_t(p0) * hb + int64_t(h) * places(tiles), t1 = t0 + tiles;
  const int c0 = tiles ? int(t0 / per) : 0, c1 = tiles ? int((t1 - 1) / per) : 0;
  const bool split = c0 != c1;
  float M = -INFINITY, L = 0.f, acc[V] = {};
  auto add = [&](const float2 x, const float* y) {
    const float mn = fmaxf(M, x.x);
    const float fa = M == -INFINITY ? 0.f : ex2(M - mn);
    // a part without a finite score has sum 0, or NaN if a score was NaN
    const float fb = x.x == -INFINITY ? (x.y != x.y ? x.y : 0.f) : ex2(x.x - mn);
    L = L * fa + x.y * fb;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = acc[i] * fa + y[i] * fb;
    M = mn;
  };
  if (split) {
    constexpr int U = 4;
    for (int c = c0 + sub; c <= c1; c += U * wph) {
      float2 x[U];
      float y[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * wph <= c1) {
          const int64_t slot = 2 * int64_t(c + u * wph) + (c + u * wph == c0 ? 1 : 0);
          x[u] = a.part_ml[slot * GT + g];
          const float* src = a.part_o + (slot * GT + g) * DP + lane * V;
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float2 z = *reinterpret_cast<const float2*>(src + i);
            y[u][i] = z.x, y[u][i + 1] = z.y;
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * wph <= c1) add(x[u], y[u]);
    }
  }
  if (wph > 1) {
    if (lane == 0) s_ml[w] = make_float2(M, L);
#pragma unroll
    for (int i = 0; i < V; ++i) s_o[w][lane * V + i] = acc[i];
    __syncthreads();
    if (sub) return;
    for (int i = 1; i < wph; ++i) {
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = s_o[w + i][lane * V + j];
      add(s_ml[w + i], y);
    }
  }
  if (!in || (tiles && !split)) return;
  T* out = static_cast<T*>(a.out) + int64_t(b) * a.o_row + int64_t(head) * a.o_head + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane * V + i < a.dim) out[i] = from_f<T>(L == 0.f ? 0.f : acc[i] / L);
  if (lane == 0 && a.lse)
    a.lse[int64_t(b) * n_heads + head] = L == 0.f ? -INFINITY : kLn2 * ((M == -INFINITY ? 0.f : M) + log2f(L));
}

template <typename T, int DP, int GT>
struct Inst {
  using C = Cfg<T, DP, GT>;

  // CTAs of a launch over `rows` rows: all that fit the device at once.  The
  // occupancy is asked for once per device and size class of the row table.
  static int prepare(int rows, size_t* smem, int* workers) {
    constexpr int kDevices = 32;
    static std::atomic<int> known[2][kDevices];
    const int cls = rows <= 256 ? 0 : 1;
    *smem = C::kFixed + (cls ? kAttendMaxRows : 256) * 4;
    int dev = 0;
    SLR_CHECK_CUDA(cudaGetDevice(&dev));
    int n = dev < kDevices ? known[cls][dev].load(std::memory_order_acquire) : 0;
    if (n == 0) {
      int occ = 0, sms = 0;
      SLR_CHECK_CUDA(cudaFuncSetAttribute(attend_kernel<T, DP, GT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::kFixed + kAttendMaxRows * 4));
      SLR_CHECK_CUDA(cudaFuncSetAttribute(attend_kernel<T, DP, GT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::kFixed + kAttendMaxRows * 4));
      SLR_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, attend_kernel<T, DP, GT, false>, C::W * 32, *smem));
      SLR_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
      if (occ < 1) return fail(SLR_ERR_UNSUPPORTED, "attend: the kernel does not fit this device");
      n = sms * occ;
      if (dev < kDevices) known[cls][dev].store(n, std::memory_order_release);
    }
    *workers = n * C::W;
    return SLR_OK;
  }

  static int launch(const AttendArgs& x, cudaStream_t s) {
    AttendK a = {};
    size_t smem = 0;
    int rc = prepare(x.rows, &smem, &a.workers);
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
    a.page_shift = (x.page_size & (x.page_size - 1)) == 0 ? __builtin_ctz(x.page_size) : -1;
    a.max_pages = x.max_pages;
    a.num_pages = x.num_pages;
    a.scale_log2 = x.scale * kLog2e;
    const int64_t kw = C::kF32 ? 4 : 2;
    a.q_wide = a.q_row % kw == 0 && a.q_head % kw == 0 && reinterpret_cast<uintptr_t>(a.q) % (kw * sizeof(T)) == 0;
    a.o_pairs = a.o_row % 2 == 0 && a.o_head % 2 == 0 && reinterpret_cast<uintptr_t>(a.out) % 4 == 0;
    const int64_t longest = int64_t(a.max_pages) * a.page_size;
    const int small = small_cluster(x.rows, a.kv_heads * a.hblocks, longest, a.workers / C::W);
    a.workers = useful(a.workers, x.rows, a.kv_heads * a.hblocks, longest);
    uint8_t* ws = static_cast<uint8_t*>(x.workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + size_t(2 * a.workers) * C::GT * DP * 4);
    a.prefix = reinterpret_cast<int32_t*>(ws + size_t(2 * a.workers) * C::GT * (DP * 4 + 8));
    if (!small && (!ws || need(a.workers, a.rows) > x.workspace_bytes))
      return fail(SLR_ERR_WORKSPACE,
                  "attend: workspace is NULL or too small, need " + std::to_string(need(a.workers, a.rows)) + " bytes");
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(std::max(small, 1));
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(small ? a.rows * a.kv_heads * a.hblocks * small : a.workers / C::W);
    cfg.blockDim = dim3(C::W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (small) {
      cfg.numAttrs = 2;
      SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_kernel<T, DP, GT, true>, a));
      return SLR_OK;
    }
    SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_kernel<T, DP, GT, false>, a));
    // warps per head of the join: a fourth of the parts that an even split of
    // the longest possible rows gives each (they are read four at a time)
    int wph = 1;
    while (wph < 32 && int64_t(wph) * 4 * a.rows * a.kv_heads * a.hblocks < a.workers) wph *= 2;
    const int warps = std::max(wph, 8);
    cfg.gridDim = dim3(unsigned(ceil_div(int64_t(a.rows) * x.heads, warps / wph)));
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = 0;
    SLR_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attend_join_kernel<T, DP, GT>, a, wph));
    return SLR_OK;
  }

  // CTAs per (row, head block) when the call is small, else 0.  All CTAs run at
  // once; the cluster grows until a row of the greatest length gives a warp 2
  // tiles (a tile takes 0.3 to 0.4 us, a cluster 1.2 us more than one CTA).
  // Where it cannot grow for want of SMs, up to 8 tiles are taken (256 CTAs, 512
  // tokens, 32 heads of 128: 11 us, split 16; 1024 ragged tokens would wait for
  // the longest).  Clusters of 8 take up to 16, 8192 tokens, since rows are
  // mostly shorter than their table (one row, 8 key heads of 128: 100 tokens 5.6
  // us, split 11.4; 4000 tokens 11.4, split 13.2; at 16000 it would be 29, split 18).
  static int small_cluster(int rows, int hb, int64_t longest, int ctas) {
    constexpr int64_t kTokens = 2 * C::W * C::TT;
    int cs = 1;
    while (cs < 8 && longest > kTokens * cs && int64_t(rows) * hb * cs * 2 <= ctas) cs *= 2;
    return int64_t(rows) * hb * cs <= ctas && longest <= kTokens * cs * (cs == 8 ? 8 : 4) ? cs : 0;
  }
  // No more warps than shares of tiles that rows of the greatest length could have.
  static int useful(int workers, int rows, int hb, int64_t longest) {
    const int64_t most = int64_t(rows) * hb * ceil_div(longest, int64_t(C::TT) * kMinTiles);
    return most < workers ? int(round_up(std::max<int64_t>(most, 1), C::W)) : workers;
  }
  static size_t need(int workers, int rows) {
    return size_t(2 * workers) * C::GT * (DP * 4 + 8) + size_t(rows + 1) * 4;
  }
  static int size(int rows, int kv_heads, int group, int64_t longest, size_t* out) {
    size_t smem = 0;
    int workers = 0;
    int rc = prepare(rows, &smem, &workers);
    const int hb = kv_heads * int(ceil_div(group, GT));
    const bool small = !rc && small_cluster(rows, hb, longest, workers / C::W);
    *out = rc || small ? 0 : need(useful(workers, rows, hb, longest), rows);
    return rc;
  }
};

// Query heads per CTA: the group, rounded up to what the arithmetic offers (8
// or 16 columns of an MMA; 1, 2, 4 or 8 accumulators per lane in fp32).
template <typename T, int DP, typename F> int by_group(int group, F&& f) {
  if constexpr (std::is_same<T, float>::value) {
    if (group == 1) return f(Inst<T, DP, 1>{});
    if (group == 2) return f(Inst<T, DP, 2>{});
    if (group <= 4) return f(Inst<T, DP, 4>{});
    return f(Inst<T, DP, 8>{});
  } else {
    return group <= 8 ? f(Inst<T, DP, 8>{}) : f(Inst<T, DP, 16>{});
  }
}
template <typename T, typename F> int by_dim(int dim, int group, F&& f) {
  return dim <= 64 ? by_group<T, 64>(group, f) : dim <= 128 ? by_group<T, 128>(group, f) : by_group<T, 256>(group, f);
}
template <typename F> int by_shape(int dtype, int dim, int group, F&& f) {
  switch (dtype) {
    case SLR_F32: return by_dim<float>(dim, group, f);
    case SLR_F16: return by_dim<__half>(dim, group, f);
    default: return by_dim<__nv_bfloat16>(dim, group, f);
  }
}

}  // namespace

int attend_workspace_size(int dtype, int dim, int rows, int kv_heads, int group, int64_t longest, size_t* bytes) {
  return by_shape(dtype, dim, group,
                  [&](auto inst) { return decltype(inst)::size(rows, kv_heads, group, longest, bytes); });
}

int launch_attend(const AttendArgs& a, cudaStream_t s) {
  return by_shape(a.dtype, a.dim, a.heads / a.kv_heads, [&](auto inst) { return decltype(inst)::launch(a, s); });
}

int read_and_clear_status_attend(unsigned* out) {
  unsigned v = 0, zero = 0;
  SLR_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_status_attend, sizeof(v)));
  if (v) SLR_CHECK_CUDA(cudaMemcpyToSymbol(g_status_attend, &zero, sizeof(zero)));
  *out = v;
  return SLR_OK;
}

}  // namespace slr
