// The products of the gated feed-forward layer (ffn.cu) on the tensor cores:
//   kUp        g = x Wg^T and u = x Wu^T of the same tile, h = f(g) u (and f(g), u f'(g) kept for the backward);
//   kDh        dh = dy Wd, of which only du = dh f(g) and dg = dh u f'(g) leave the SM;
//   kProducts  plain products: y = h Wd^T; or dWg = dg^T x, dWu = du^T x, dWd = dy^T h and dx = dg Wg + du Wu in one launch.
//
// One persistent kernel per kind, a pair of CTAs (cta_group::2) per tile of 256 rows and 256 columns, as in the loss (loss_tc.cu, which has what
// was measured about stages and boxes): each CTA holds 128 rows of A, 128 columns of B and 128 x 256 sums.  kUp: the even CTA's 128 columns are
// Wg's, the odd one's Wu's for the same 128 hidden columns, so a thread of either CTA has g and u of its row side by side in TMEM.
// A stage is 128 summands (float32: 64 in three parts); sums are double buffered in TMEM: a tile's epilogue runs under the next one's products.
//
// The tensor core adds by truncation (loss_tc.cu), so where a sum is long its chain is cut (LONG): formed chunk by chunk, the chunks' sums
// added in registers.
//
// What the backward needs of g and u are a = f(g) and b = u f'(g): du = dh a, dg = dh b.  They are formed where g and u are, under products that
// take twice as long per hidden value as those under which dh is used (65,536 x 768 x 2,048: with g and u kept the dh kernel took 324 us).  Kept in
// bf16 they would bring one more rounding of 2^-9 to results that have one in dg and one in their own type (2.4e-3 of dx, 2.9e-3 with it); so
// they are kept with 2^-12: as fp16 times a power of two per 32 values of a row, which puts the largest of them just below fp16's limit;
// beside float16's own 2^-12, and float32's, as float32.  They lie as the lanes write and read them, [32 rows][32 columns][a, b][16 bytes of each lane].
//
// Warps: 0 producer, 1 MMA issuer (even CTA) and TMEM owner, 2-9 epilogue: two warps per quarter of the rows.  Every wait is bounded (ptx.cuh);
// no multicast loads.
#include <cfloat>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ffn.cuh"
#include "ptx.cuh"

namespace nlfa {
namespace ffn {
namespace {

constexpr int kThreads = 320;
constexpr int kEpilogueWarps = 8;
constexpr int kBlockBytes = 128 * 128;                        // 128 rows of 64 columns
template <int PARTS>
struct Ring {
  static constexpr int kStages = PARTS == 3 ? 2 : 3;
  static constexpr int kSummands = summands(PARTS);
  static constexpr int kBlocks = PARTS == 3 ? 3 : kSummands / 64;
  static constexpr int kOperandBytes = kBlocks * kBlockBytes;   // one CTA's half of an operand
  static constexpr int kStageBytes = 2 * kOperandBytes;
  static_assert(kStages * kStageBytes <= 12 * kBlockBytes, "stages");
};
constexpr int kMostStages = 3;
constexpr int kStagingBytes = 4096;                           // per epilogue warp: 32 rows of 128 bytes
constexpr int kStaging = 12 * kBlockBytes;
constexpr int kBars = kStaging + kEpilogueWarps * kStagingBytes;
constexpr int kNumBars = 2 * kMostStages + 4;
constexpr int kTmemSlot = kBars + 8 * kNumBars;
constexpr int kAbort = kTmemSlot + 4;
constexpr int kSmem = kAbort + 4 + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");

enum { FULL = 0, EMPTY = kMostStages, ACC_FULL = 2 * kMostStages, ACC_EMPTY = ACC_FULL + 2 };

// float32 operands are sums of three bf16 parts; the products of parts, smallest first (what is left out is below 2^-24)
__device__ __forceinline__ int part_a(int pair) { return (0x001012 >> (4 * pair)) & 15; }   // 2 1 0 1 0 0
__device__ __forceinline__ int part_b(int pair) { return (0x010210 >> (4 * pair)) & 15; }   // 0 1 2 0 1 0

__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

struct Tile {
  int m0, n0;
  int k0, k1;                       // its stages: all, or of a shared tile this pair's
  int seg;                          // kProducts
  int slot;                         // where a share of a tile goes (-1: the tile is whole)
};

// kProducts: tile v of a group
__device__ __forceinline__ void place(const Params& p, const Group& g, int v, Tile& t) {
  t.seg = g.seg0;
  while (t.seg + 1 < g.seg1 && v >= p.seg[t.seg].tiles) v -= p.seg[t.seg++].tiles;
  const int m = v / p.seg[t.seg].tiles_n;
  t.m0 = m * kRowTile;
  t.n0 = (v - m * p.seg[t.seg].tiles_n) * kColTile;
}

// The tiles of one pair of CTAs, in order; every role walks the same list.
template <int MODE, int PARTS>
struct Walk {
  const Params& p;
  int u, stride, units, row_tiles, col_tiles, k;

  __device__ Walk(const Params& p_, int pair, int n_pairs) : p(p_), u(pair - n_pairs), stride(n_pairs) {
    if (MODE == kProducts) {
      units = p.units;
    } else {
      row_tiles = ceil_div(p.rows, kRowTile);
      col_tiles = ceil_div(p.cols, MODE == kUp ? kColTile / 2 : kColTile);
      units = row_tiles * col_tiles;
      k = ceil_div(p.k, summands(PARTS));
    }
  }
  __device__ bool next(Tile& t) {
    u += stride;
    if (u >= units) return false;
    t.slot = -1;
    t.k0 = 0;
    if (MODE != kProducts) {
      // eight row tiles at a time past all columns: their x (or dy) and the weight stay in L2
      const int group = 8 * col_tiles, g = u / group, v = u - g * group;
      const int size = row_tiles - 8 * g < 8 ? row_tiles - 8 * g : 8;
      const int c = v / size;
      t.m0 = (8 * g + v - c * size) * kRowTile;
      t.n0 = c * (MODE == kUp ? kColTile / 2 : kColTile);
      t.k1 = k;
      return true;
    }
    const Group& g = p.group[p.groups > 1 && u >= p.group[0].end ? 1 : 0];
    int v = u - g.first;
    t.k1 = g.k;
    if (v >= g.whole) {
      const int i = v - g.whole, part = i / g.rest;
      v = g.whole + i - part * g.rest;
      if (g.parts > 1) {
        t.k0 = static_cast<int>(static_cast<long long>(g.k) * part / g.parts);
        t.k1 = static_cast<int>(static_cast<long long>(g.k) * (part + 1) / g.parts);
        t.slot = g.slot + i;
      }
    }
    place(p, g, v, t);
    return true;
  }
};

// What row m of a segment's sums is multiplied with: 1 / f of a power of two.
__device__ __forceinline__ float factor_of(const Segment& s, int m) {
  return s.scale != nullptr && m < s.m_end ? __int_as_float(0x7f000000 - __float_as_int(s.scale[s.by_row ? m : 0])) : 1.f;
}

// Four values of row m, columns n .. of a segment's result
__device__ __forceinline__ void put(const Segment& s, int m, int n, float (&v)[4]) {
  if (m >= s.m_end || n >= s.n_end) return;
  const bool vec = s.n_end % 4 == 0;
  const int count = s.n_end - n < 4 ? s.n_end - n : 4;
  const size_t at = static_cast<size_t>(m) * s.n_end + n;
  if (s.dtype == NLFA_DTYPE_F32) {
    float* o = static_cast<float*>(s.to) + at;
    if (vec) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    else for (int e = 0; e < count; ++e) o[e] = v[e];
  } else if (s.dtype == NLFA_DTYPE_BF16) {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(s.to) + at;
    if (vec) *reinterpret_cast<uint2*>(o) = make_uint2(Pack2<__nv_bfloat16>::pack(v[0], v[1]), Pack2<__nv_bfloat16>::pack(v[2], v[3]));
    else for (int e = 0; e < count; ++e) o[e] = __float2bfloat16_rn(v[e]);
  } else {
    __half* o = static_cast<__half*>(s.to) + at;
    if (vec) *reinterpret_cast<uint2*>(o) = make_uint2(Pack2<__half>::pack(v[0], v[1]), Pack2<__half>::pack(v[2], v[3]));
    else for (int e = 0; e < count; ++e) o[e] = __float2half_rn(v[e]);
  }
}

// The shares of a tile formed in parts (blockIdx.x), added in order; 4 rows a CTA.
constexpr int kFoldThreads = 256, kFoldRows = 4;
__global__ void __launch_bounds__(kFoldThreads)
fold_kernel(const __grid_constant__ Params p) {
  grid_dep_wait();
  grid_dep_release();
  int i = blockIdx.x, which = 0;
  const int split = p.group[0].parts > 1 ? p.group[0].rest : 0;
  if (i >= split) { i -= split; which = 1; }
  const Group& g = p.group[which];
  Tile t;
  place(p, g, g.whole + i, t);
  const Segment& s = p.seg[t.seg];
  const int c = 4 * (threadIdx.x & 63), r = blockIdx.y * kFoldRows + (threadIdx.x >> 6);
  if (t.n0 + c >= s.n_end || t.m0 + r >= s.m_end) return;
  const float* shares = p.shares + (static_cast<size_t>(g.slot) + i) * (kRowTile * kColTile) + c;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int part = 0; part < g.parts; ++part) {
    const float4 x = *reinterpret_cast<const float4*>(shares + (static_cast<size_t>(part) * g.rest * kRowTile + r) * kColTile);
    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
  }
  const float factor = factor_of(s, t.m0 + r);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] *= factor;
  put(s, t.m0 + r, t.n0 + c, v);
}

// ---- the activation: f(g), and f'(g).  EXACT (float32): no approximate exponential or quotient

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <bool EXACT> __device__ __forceinline__ float logistic(float g) {
  return EXACT ? 1.f / (1.f + expf(-g)) : reciprocal(1.f + fast_exp2(-kLog2e * g));
}
template <int ACT, bool EXACT> __device__ __forceinline__ void activate(float g, float& a, float& da) {
  if (ACT == NLFA_FFN_SILU) {
    const float p = logistic<EXACT>(g);
    a = g * p;
    da = fmaf(a, 1.f - p, p);
  } else if (ACT == NLFA_FFN_GELU) {
    const float p = fmaf(0.5f, erff(g * 0.70710678118654752f), 0.5f);
    const float e = EXACT ? expf(-0.5f * g * g) : fast_exp2(-0.5f * kLog2e * g * g);
    a = g * p;
    da = fmaf(g * 0.39894228040143268f, e, p);
  } else {
    a = g < 0.f ? 0.f : g;                                    // (NaN stays)
    da = g > 0.f ? 1.f : 0.f;
  }
}

// ---- kept a and b: this thread's 32 values of one of them (WIDE: float32)

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

template <bool WIDE> __device__ __forceinline__ void keep(uint8_t* at, int8_t* exponent, const float (&v)[32]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(at + 512 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 32; j += 2) top = fmax3(top, fabsf(v[j]), fabsf(v[j + 1]));
    if (!(top < INFINITY)) {                                  // the largest finite one
      top = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (fabsf(v[j]) < INFINITY) top = fmaxf(top, fabsf(v[j]));
    }
    // top < 2^(e + 15), and 2^e a normal float
    const int e = max(((__float_as_int(top) >> 23) & 255) - 127 - 14, -126);
    *exponent = static_cast<int8_t>(e);
    const float f = power_of_two(-e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 w;
      w.x = Pack2<__half>::pack(v[8 * i] * f, v[8 * i + 1] * f);
      w.y = Pack2<__half>::pack(v[8 * i + 2] * f, v[8 * i + 3] * f);
      w.z = Pack2<__half>::pack(v[8 * i + 4] * f, v[8 * i + 5] * f);
      w.w = Pack2<__half>::pack(v[8 * i + 6] * f, v[8 * i + 7] * f);
      *reinterpret_cast<uint4*>(at + 512 * i) = w;
    }
  }
}
// Eight of them, those at 8 i, each times v's.
template <bool WIDE> __device__ __forceinline__ void times_kept(const uint8_t* at, int i, const float (&v)[8], float f, float (&out)[8]) {
  if constexpr (WIDE) {
    const float4 x = *reinterpret_cast<const float4*>(at + 1024 * i), y = *reinterpret_cast<const float4*>(at + 1024 * i + 512);
    out[0] = v[0] * x.x; out[1] = v[1] * x.y; out[2] = v[2] * x.z; out[3] = v[3] * x.w;
    out[4] = v[4] * y.x; out[5] = v[5] * y.y; out[6] = v[6] * y.z; out[7] = v[7] * y.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(at + 512 * i);
    const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = __half22float2(h[j]);
      unpack_f2(fmul2(fmul2(pack_f2(v[2 * j], v[2 * j + 1]), pack_f2(f, f)), pack_f2(x.x, x.y)), out[2 * j], out[2 * j + 1]);
    }
  }
}

// 32 columns of a row in parts, each the nearest value to what is left: [part][64 columns][rows][64]
template <typename T> __device__ __forceinline__ float round_to(float x);
template <> __device__ __forceinline__ float round_to<__nv_bfloat16>(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
template <> __device__ __forceinline__ float round_to<__half>(float x) { return __half2float(__float2half_rn(x)); }
template <typename T>
__device__ __forceinline__ void store_parts(void* to, size_t plane, int n_rows, int row, int col, float (&v)[32], int parts = 3) {
  T* o = static_cast<T*>(to) + (static_cast<size_t>(col / 64) * n_rows + row) * 64 + col % 64;
  for (int part = 0; part < parts; ++part, o += plane) {
#pragma unroll
    for (int j = 0; j < 32; j += 8)
      *reinterpret_cast<uint4*>(o + j) = make_uint4(Pack2<T>::pack(v[j], v[j + 1]), Pack2<T>::pack(v[j + 2], v[j + 3]),
                                                    Pack2<T>::pack(v[j + 4], v[j + 5]), Pack2<T>::pack(v[j + 6], v[j + 7]));
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] -= round_to<T>(v[j]);
  }
}

// ---- epilogues: a thread has row `lane` of its warp's 32 and 128 of the tile's columns

// The columns of a thread's row: in TMEM, or (LONG) summed from the chunks' sums in registers.  kUp: 64 of g's, then 64 of u's.
template <int MODE, bool LONG>
struct Sums {
  uint32_t acc;                     // of the thread's first column
  float v[LONG ? 128 : 1];
  // where its 16 columns c are, from the first
  __device__ static constexpr int column(int c) { return MODE == kUp && c >= 4 ? 128 + 16 * (c - 4) : 16 * c; }
  __device__ __forceinline__ void get(int c32, float (&r)[32]) const {
    if constexpr (LONG) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c32 == c) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = v[32 * c + j];
        }
    } else {
      uint32_t w[32];
      tmem_ld32(acc + column(2 * c32), w);
      tc_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = __uint_as_float(w[j]);
    }
  }
};

template <typename T, int MODE, bool LONG, int PARTS, int ACT>
__global__ void __launch_bounds__(kThreads, 1)
ffn_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  constexpr bool kBf16 = Pack2<T>::kIsBf16;
  using R = Ring<PARTS>;
  constexpr int kStages = R::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  auto bar = [&](int i) -> uint32_t { return base + kBars + 8u * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kAbort);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + kTmemSlot);
  const WaitCtx wctx{abort_flag, p.status};

  if (threadIdx.x >= 32 && threadIdx.x < 32 + kMostMaps) tma_prefetch_desc(&maps.m[threadIdx.x - 32]);
  if (threadIdx.x == 0) {
    *abort_flag = (*reinterpret_cast<volatile unsigned*>(p.status) != STATUS_OK) ? 1 : 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(FULL + s), 1);
      mbar_init(bar(EMPTY + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ACC_FULL + i), 1);
      mbar_init(bar(ACC_EMPTY + i), 2 * kEpilogueWarps);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(base + kTmemSlot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const bool dead = *abort_flag != 0;
  grid_dep_wait();
  grid_dep_release();

  if (dead) {
    // a give-up recorded earlier makes this launch a no-op
  } else if (warp == 0) {
    // ============================== producer ================================
    if (lane == 0) {
      Walk<MODE, PARTS> walk(p, pair, n_pairs);
      Tile t;
      int it = 0;
      bool ok = true;
      const uint32_t full0 = cluster_addr(bar(FULL), 0);       // loads of both CTAs are counted on the even one's
      while (ok && walk.next(t)) {
        const Segment* seg = MODE == kProducts ? &p.seg[t.seg] : nullptr;
        const int a0 = t.m0 + 128 * rank, b0 = MODE == kUp ? t.n0 : t.n0 + 128 * rank;
        for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
          const int s = it % kStages;
          if (!(ok = mbar_wait(bar(EMPTY + s), ((it / kStages) & 1) ^ 1, wctx, 100))) break;
          const uint32_t st = base + s * R::kStageBytes, full = full0 + 8u * s;
          if (rank == 0) mbar_arrive_expect_tx(bar(FULL + s), 2 * R::kStageBytes);
          // boxes at (row, block of 64 columns, plane): the sum runs along the columns, or (MN-major) along the rows
          auto load = [&](uint32_t dst, const CUtensorMap* map, bool mn, int at, int k, int plane) {
            tma_load_4d_pair(dst, map, full, 0, mn ? k : at, (mn ? at : k) / 64, plane);
          };
          if (MODE == kUp) {
            const int k = kb * R::kSummands;
            load(st, &maps.m[0], false, a0, k, 0);
            load(st + R::kOperandBytes, &maps.m[1 + rank], false, b0, k, 0);
          } else if (MODE == kDh) {
            const int k = kb * R::kSummands;
            load(st, &maps.m[0], false, a0, k, 0);
            load(st + R::kOperandBytes, &maps.m[1], true, b0, k, 0);
          } else {
            const int sub = kb / seg->k_sub, k = (kb - sub * seg->k_sub) * R::kSummands;
            load(st, &maps.m[seg->a_map], seg->a_mn, a0, k, seg->a_plane[sub]);
            load(st + R::kOperandBytes, &maps.m[seg->b_map[sub]], seg->b_mn, b0, k, seg->b_plane[sub]);
          }
        }
      }
      // the last loads of this CTA have been consumed before it may leave (after a give-up: have had time to land)
      for (int i = 0; ok && i < kStages; ++i, ++it) ok = mbar_wait(bar(EMPTY + it % kStages), ((it / kStages) & 1) ^ 1, wctx, 101);
      if (!ok) for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    // ============================= MMA issuer ===============================
    if (rank == 0) {
      const uint32_t leader = elect_one() ? 1u : 0u;
      Walk<MODE, PARTS> walk(p, pair, n_pairs);
      Tile t;
      int it = 0, sums = 0;                                    // sums: filled TMEM buffers so far
      bool ok = true;
      while (ok && walk.next(t)) {
        const bool a_mn = MODE == kProducts && p.seg[t.seg].a_mn, b_mn = MODE == kDh || (MODE == kProducts && p.seg[t.seg].b_mn);
        const uint32_t idesc = make_idesc(kBf16, 256, kColTile, a_mn, b_mn);
        // 16 summands on: 32 bytes along a row, then the next block of 64 columns; or (MN-major) 16 rows
        constexpr uint32_t kMnBlock = PARTS == 3 ? kBlockBytes / 2 : kBlockBytes;     // (of 64 summands: 64 rows)
        const uint32_t a_lbo = a_mn ? kMnBlock : 16u, b_lbo = b_mn ? kMnBlock : 16u;
        const int chunk = LONG ? p.chunk : t.k1 - t.k0;
        for (int k0 = t.k0; ok && k0 < t.k1; k0 += chunk, ++sums) {
          const int buf = sums & 1;
          if (!(ok = mbar_wait(bar(ACC_EMPTY + buf), ((sums >> 1) & 1) ^ 1, wctx, 102))) break;
          tc_fence_after();
          const int stages = t.k1 - k0 < chunk ? t.k1 - k0 : chunk;
          for (int kb = 0; kb < stages; ++kb, ++it) {
            const int s = it % kStages;
            if (!(ok = mbar_wait(bar(FULL + s), (it / kStages) & 1, wctx, 103))) break;
            tc_fence_after();
            const uint32_t a = base + s * R::kStageBytes, b = a + R::kOperandBytes;
#pragma unroll
            for (int pr = 0; pr < (PARTS == 3 ? 6 : 1); ++pr) {
              const uint32_t a_part = PARTS == 3 ? part_a(pr) * kBlockBytes : 0u, b_part = PARTS == 3 ? part_b(pr) * kBlockBytes : 0u;
#pragma unroll
              for (int kk = 0; kk < R::kSummands / 16; ++kk) {
                const uint32_t along = (kk / 4) * kBlockBytes + (kk % 4) * 32u;
                umma_ss_pair(leader, tmem + buf * kColTile, make_smem_desc(a + a_part + (a_mn ? kk * 2048u : along), a_lbo, 1024),
                             make_smem_desc(b + b_part + (b_mn ? kk * 2048u : along), b_lbo, 1024), idesc,
                             (kb > 0 || pr > 0 || kk > 0) ? 1u : 0u);
              }
            }
            umma_commit_pair(leader, bar(EMPTY + s));
          }
          if (ok) umma_commit_pair(leader, bar(ACC_FULL + buf));
        }
      }
    }
  } else {
    // ============================== epilogue ================================
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t staging = base + kStaging + (warp - 2) * kStagingBytes;
    const uint32_t acc_empty0 = cluster_addr(bar(ACC_EMPTY), 0);
    constexpr int kOwn = MODE == kUp ? 64 : 128;               // hidden columns (or columns) of a warp
    Walk<MODE, PARTS> walk(p, pair, n_pairs);
    Tile t;
    int sums = 0;
    bool ok = true;
    const size_t plane = static_cast<size_t>(p.n_rows) * p.f_pad;
    Sums<MODE, LONG> l;
    auto release = [&](int buf) {                              // this warp has read its part of the buffer
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + 8u * buf);
    };
    // eight columns of the staging tile: 16 bytes of this lane's row, swizzled as the tensor maps have it
    auto stage = [&](int chunk, const float (&v)[8]) {
      st_shared_v4(staging + lane * 128 + static_cast<uint32_t>(chunk ^ (lane & 7)) * 16, Pack2<T>::pack(v[0], v[1]), Pack2<T>::pack(v[2], v[3]),
                   Pack2<T>::pack(v[4], v[5]), Pack2<T>::pack(v[6], v[7]));
    };
    auto staging_free = [&]() {
      if (lane == 0) tma_store_wait_read();
      __syncwarp();
    };
    auto store_staged = [&](const CUtensorMap* map, int row, int col, int to_plane) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_4d(map, staging, 0, row, col / 64, to_plane);
        tma_store_commit();
      }
    };
    // kept a and b: of 32 rows and 32 columns a, then b
    constexpr bool kWide = PARTS == 3 || !kBf16;
    constexpr int kKeptBytes = kWide ? 4096 : 2048;
    auto kept_at = [&](int row, int col) -> size_t { return (static_cast<size_t>(row / 32) * (p.f_pad / 32) + col / 32) * 2; };
    while (walk.next(t)) {
      const int row0 = t.m0 + 128 * rank + 32 * q, row = row0 + lane;
      const float scale = !kBf16 && MODE != kProducts && row < p.rows ? p.scale[row] : 1.f;
      int buf = 0;
      if constexpr (LONG) {
#pragma unroll
        for (int j = 0; j < 128; ++j) l.v[j] = 0.f;
        for (int k0 = t.k0; k0 < t.k1; k0 += p.chunk, ++sums) {
          buf = sums & 1;
          if (!(ok = mbar_wait(bar(ACC_FULL + buf), (sums >> 1) & 1, wctx, 104))) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t r[16];
            tmem_ld16(tmem_addr(tmem, 32 * q, buf * kColTile + kOwn * half + Sums<MODE, LONG>::column(c)), r);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j += 2)
              unpack_f2(fadd2(pack_f2(l.v[16 * c + j], l.v[16 * c + j + 1]), pack_f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]))),
                        l.v[16 * c + j], l.v[16 * c + j + 1]);
          }
          release(buf);
        }
      } else {
        buf = sums & 1;
        ok = mbar_wait(bar(ACC_FULL + buf), (sums >> 1) & 1, wctx, 104);
        tc_fence_after();
        l.acc = tmem_addr(tmem, 32 * q, buf * kColTile + kOwn * half);
        ++sums;
      }
      if (!ok) break;
      const int c0 = t.n0 + kOwn * half;
      // kUp gives the buffer back as soon as its last columns are in registers: the release waits for all that this thread has stored before (351 -> 328 us;
      // the dh kernel and the products are slower so, 248 -> 258 and 161 -> 166).
      if constexpr (MODE == kUp) {
        if (c0 < p.f_pad) {
          if (PARTS == 1) staging_free();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float g[32], u[32];
            l.get(c, g);
            l.get(2 + c, u);
            if (!LONG && c == 1) release(buf);
            if (p.kept != nullptr) {
              const size_t at = kept_at(row0, c0 + 32 * c);
              float f[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float slope;
                activate<ACT, PARTS == 3>(g[j], f[j], slope);
                g[j] = f[j] * u[j];
                u[j] *= slope;
              }
              keep<kWide>(p.kept + at * kKeptBytes + 16 * lane, p.exponents + 32 * at + lane, f);
              keep<kWide>(p.kept + (at + 1) * kKeptBytes + 16 * lane, p.exponents + 32 * (at + 1) + lane, u);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float f, slope;
                activate<ACT, PARTS == 3>(g[j], f, slope);
                g[j] = f * u[j];
              }
            }
            if (!kBf16) {
#pragma unroll
              for (int j = 0; j < 32; ++j) g[j] *= scale;
            }
            if (PARTS == 3) {
              store_parts<T>(p.h, plane, p.n_rows, row, c0 + 32 * c, g);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v[8] = {g[8 * i], g[8 * i + 1], g[8 * i + 2], g[8 * i + 3], g[8 * i + 4], g[8 * i + 5], g[8 * i + 6], g[8 * i + 7]};
                stage(4 * c + i, v);
              }
            }
          }
          if (PARTS == 1) store_staged(&maps.m[3], row0, c0, 0);
        } else if (!LONG) {
          release(buf);
        }
      } else if constexpr (MODE == kDh) {
#pragma unroll (LONG ? 2 : 1)
        for (int c2 = 0; c2 < 2; ++c2) {
          const int col0 = c0 + 64 * c2;
          if (col0 >= p.f_pad) break;
          uint32_t held[PARTS == 1 ? 32 : 1];                  // du of these columns, packed
          if (PARTS == 1) staging_free();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const size_t at = kept_at(row0, col0 + 32 * c);
            const uint8_t* as = p.kept + at * kKeptBytes + 16 * lane;
            const uint8_t* bs = as + kKeptBytes;
            float fa = 1.f, fb = 1.f;
            if (!kWide) {
              fa = power_of_two(p.exponents[32 * at + lane]);
              fb = power_of_two(p.exponents[32 * (at + 1) + lane]);
            }
            float d[32], e[PARTS == 3 ? 32 : 1];
            l.get(2 * c2 + c, d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v[8], dg[8], du[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = kBf16 ? d[8 * i + j] : d[8 * i + j] * scale;
              times_kept<kWide>(as, i, v, fa, du);
              times_kept<kWide>(bs, i, v, fb, dg);
              if constexpr (PARTS == 1) {
                stage(4 * c + i, dg);
#pragma unroll
                for (int j = 0; j < 4; ++j) held[16 * c + 4 * i + j] = Pack2<T>::pack(du[2 * j], du[2 * j + 1]);
              } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  d[8 * i + j] = dg[j];
                  e[8 * i + j] = du[j];
                }
              }
            }
            if constexpr (PARTS == 3) {
              store_parts<T>(p.dg, plane, p.n_rows, row, col0 + 32 * c, d);
              store_parts<T>(p.du, plane, p.n_rows, row, col0 + 32 * c, e);
            }
          }
          if constexpr (PARTS == 1) {
            store_staged(&maps.m[2], row0, col0, 0);
            staging_free();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              st_shared_v4(staging + lane * 128 + static_cast<uint32_t>(i ^ (lane & 7)) * 16, held[4 * i], held[4 * i + 1], held[4 * i + 2], held[4 * i + 3]);
            store_staged(&maps.m[2], row0, col0, 1);
          }
        }
      } else {
        // 32 x 32 values through shared memory, so that a row's columns leave side by side
        const Segment& seg = p.seg[t.seg];
        const int local = 128 * rank + 32 * q;
        const float factor = kBf16 || t.slot >= 0 ? 1.f : factor_of(seg, row);
        float* share = t.slot < 0 ? nullptr : p.shares + (static_cast<size_t>(t.slot) * kRowTile + local) * kColTile;
#pragma unroll (LONG ? 4 : 1)
        for (int c = 0; c < 4; ++c) {
          const int col = c0 + 32 * c;
          if (col >= seg.n_end) break;
          float r[32];
          l.get(c, r);
          if (!kBf16) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] *= factor;
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            st_shared_v4(staging + lane * 128 + (((j / 4) ^ (lane & 7)) * 16), __float_as_uint(r[j]), __float_as_uint(r[j + 1]),
                         __float_as_uint(r[j + 2]), __float_as_uint(r[j + 3]));
          __syncwarp();
          const int cc = col + 4 * (lane & 7);
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const int lr = 4 * i + (lane >> 3);
            uint32_t w0, w1, w2, w3;
            ld_shared_v4(staging + lr * 128 + (((lane & 7) ^ (lr & 7)) * 16), w0, w1, w2, w3);
            float v[4] = {__uint_as_float(w0), __uint_as_float(w1), __uint_as_float(w2), __uint_as_float(w3)};
            if (share != nullptr) *reinterpret_cast<float4*>(share + static_cast<size_t>(lr) * kColTile + (cc - t.n0)) = make_float4(v[0], v[1], v[2], v[3]);
            else put(seg, t.m0 + local + lr, cc, v);
          }
          __syncwarp();
        }
      }
      if (!LONG && MODE != kUp) release(buf);
    }
    if (MODE != kProducts && lane == 0) tma_store_wait_all();
  }

  tc_fence_before();
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---- few tiles: the products in float32 first, formed in parts by all pairs of CTAs (ffn.cu: apart), then this; a warp has 32 rows of 32 columns
constexpr int kApartThreads = 256;
struct Block {
  int row, col;                     // this thread's row, the block's first column
  size_t kept;                      // the block's place among what is kept
  __device__ bool next(const Params& p, int& i) {
    const int cols = p.f_pad / 32;
    if (i >= p.n_rows / 32 * cols) return false;
    row = i / cols * 32 + (threadIdx.x & 31);
    col = i % cols * 32;
    kept = static_cast<size_t>(i) * 2;
    i += gridDim.x * (kApartThreads / 32);
    return true;
  }
  __device__ float scale(const Params& p) const { return p.scale != nullptr && row < p.rows ? p.scale[row] : 1.f; }
  __device__ void load(const Params& p, const float* from, float (&v)[32]) const {
    const float* s = from + static_cast<size_t>(row) * p.cols + col;
    if (row < p.rows && p.cols % 4 == 0 && col + 32 <= p.cols) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 x = *reinterpret_cast<const float4*>(s + j);
        v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = row < p.rows && col + j < p.cols ? s[j] : 0.f;
    }
  }
};

template <typename T, int PLANES>
__global__ void __launch_bounds__(kApartThreads)
hidden_kernel(const __grid_constant__ Params p, int parts, const float* __restrict__ gs, const float* __restrict__ us) {
  constexpr bool kWide = PLANES == 3 || !Pack2<T>::kIsBf16;
  constexpr int kKeptBytes = kWide ? 4096 : 2048;
  grid_dep_wait();
  grid_dep_release();
  const int lane = threadIdx.x & 31;
  int i = blockIdx.x * (kApartThreads / 32) + (threadIdx.x >> 5);
  Block b;
  while (b.next(p, i)) {
    float g[32], u[32], f[32];
    b.load(p, gs, g);
    b.load(p, us, u);
    const float scale = b.scale(p);
    auto walk = [&](auto act) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        float slope;
        activate<decltype(act)::value, PLANES == 3>(g[j], f[j], slope);
        g[j] = f[j] * u[j];
        u[j] *= slope;
      }
    };
    if (p.activation == NLFA_FFN_SILU) walk(std::integral_constant<int, NLFA_FFN_SILU>{});
    else if (p.activation == NLFA_FFN_GELU) walk(std::integral_constant<int, NLFA_FFN_GELU>{});
    else walk(std::integral_constant<int, NLFA_FFN_RELU>{});
    if (p.kept != nullptr) {
      keep<kWide>(p.kept + b.kept * kKeptBytes + 16 * lane, p.exponents + 32 * b.kept + lane, f);
      keep<kWide>(p.kept + (b.kept + 1) * kKeptBytes + 16 * lane, p.exponents + 32 * (b.kept + 1) + lane, u);
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) g[j] *= scale;
    store_parts<T>(p.h, static_cast<size_t>(p.n_rows) * p.f_pad, p.n_rows, b.row, b.col, g, parts);
  }
}

template <typename T, int PLANES>
__global__ void __launch_bounds__(kApartThreads)
grads_kernel(const __grid_constant__ Params p, int parts, const float* __restrict__ dh) {
  constexpr bool kWide = PLANES == 3 || !Pack2<T>::kIsBf16;
  constexpr int kKeptBytes = kWide ? 4096 : 2048;
  grid_dep_wait();
  grid_dep_release();
  const int lane = threadIdx.x & 31;
  int i = blockIdx.x * (kApartThreads / 32) + (threadIdx.x >> 5);
  Block b;
  while (b.next(p, i)) {
    float d[32], e[32];
    b.load(p, dh, d);
    const float scale = b.scale(p);
    const uint8_t* as = p.kept + b.kept * kKeptBytes + 16 * lane;
    float fa = 1.f, fb = 1.f;
    if (!kWide) {
      fa = power_of_two(p.exponents[32 * b.kept + lane]);
      fb = power_of_two(p.exponents[32 * (b.kept + 1) + lane]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v[8], dg[8], du[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = d[8 * k + j] * scale;
      times_kept<kWide>(as, k, v, fa, du);
      times_kept<kWide>(as + kKeptBytes, k, v, fb, dg);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        d[8 * k + j] = dg[j];
        e[8 * k + j] = du[j];
      }
    }
    const size_t plane = static_cast<size_t>(p.n_rows) * p.f_pad;
    store_parts<T>(p.dg, plane, p.n_rows, b.row, b.col, d, parts);
    store_parts<T>(p.du, plane, p.n_rows, b.row, b.col, e, parts);
  }
}

int checked(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

template <typename T, int MODE, bool LONG, int PARTS, int ACT>
int launch_one(const Params& p, const Maps& maps, cudaStream_t stream) {
  auto* kernel = ffn_kernel<T, MODE, LONG, PARTS, ACT>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem);
  if (rc != NLFA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2u * static_cast<unsigned>(pairs()));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;           // (a pair lies along x)
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap_launches(kOverlapRowwise) ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, p);
  if (MODE == kProducts && e == cudaSuccess) {
    int odd = 0;
    for (int i = 0; i < p.groups; ++i)
      if (p.group[i].parts > 1) odd += p.group[i].rest;
    if (odd > 0)
      e = launch_kernel(fold_kernel, dim3(static_cast<unsigned>(odd), kRowTile / kFoldRows), dim3(kFoldThreads), 0, stream,
                        overlap_launches(kOverlapRowwise), p);
  }
  return checked(e);
}

template <typename T, int MODE, int PARTS, int ACT>
int launch_chains(bool chains, const Params& p, const Maps& maps, cudaStream_t stream) {
  if constexpr (PARTS == 1)
    if (!chains) return launch_one<T, MODE, false, PARTS, ACT>(p, maps, stream);
  return launch_one<T, MODE, true, PARTS, ACT>(p, maps, stream);
}
template <typename T, int PARTS>
int launch_mode(int mode, bool chains, const Params& p, const Maps& maps, cudaStream_t stream) {
  if (mode == kProducts) return launch_chains<T, kProducts, PARTS, NLFA_FFN_SILU>(chains, p, maps, stream);
  auto act = [&](auto a) {
    constexpr int kAct = decltype(a)::value;
    return mode == kUp ? launch_chains<T, kUp, PARTS, kAct>(chains, p, maps, stream) : launch_chains<T, kDh, PARTS, kAct>(chains, p, maps, stream);
  };
  if (p.activation == NLFA_FFN_SILU) return act(std::integral_constant<int, NLFA_FFN_SILU>{});
  if (p.activation == NLFA_FFN_GELU) return act(std::integral_constant<int, NLFA_FFN_GELU>{});
  return act(std::integral_constant<int, NLFA_FFN_RELU>{});
}

unsigned apart_ctas(const Params& p) {
  const int need = ceil_div(p.n_rows / 32 * (p.f_pad / 32), kApartThreads / 32), most = 4 * sm_count();
  return static_cast<unsigned>(need < most ? need : most);
}

}  // namespace

int launch_hidden(int dtype, int planes, int parts, const Params& p, const float* g, const float* u, cudaStream_t stream) {
  auto go = [&](auto* kernel) {
    return checked(launch_kernel(kernel, dim3(apart_ctas(p)), dim3(kApartThreads), 0, stream, overlap_launches(kOverlapRowwise), p, parts, g, u));
  };
  if (planes == 3) return go(hidden_kernel<__nv_bfloat16, 3>);
  return dtype == NLFA_DTYPE_F16 ? go(hidden_kernel<__half, 1>) : go(hidden_kernel<__nv_bfloat16, 1>);
}
int launch_grads(int dtype, int planes, int parts, const Params& p, const float* dh, cudaStream_t stream) {
  auto go = [&](auto* kernel) {
    return checked(launch_kernel(kernel, dim3(apart_ctas(p)), dim3(kApartThreads), 0, stream, overlap_launches(kOverlapRowwise), p, parts, dh));
  };
  if (planes == 3) return go(grads_kernel<__nv_bfloat16, 3>);
  return dtype == NLFA_DTYPE_F16 ? go(grads_kernel<__half, 1>) : go(grads_kernel<__nv_bfloat16, 1>);
}

int pairs() { return sm_count() > 1 ? sm_count() / 2 : 1; }     // (without a device: sizes are still asked for)

int launch_product(int mode, int dtype, int planes, bool chains, const Params& p, const Maps& maps, cudaStream_t stream) {
  if (planes == 3) return launch_mode<__nv_bfloat16, 3>(mode, true, p, maps, stream);
  if (dtype == NLFA_DTYPE_F16) return launch_mode<__half, 1>(mode, chains, p, maps, stream);
  return launch_mode<__nv_bfloat16, 1>(mode, chains, p, maps, stream);
}

}  // namespace ffn
}  // namespace nlfa
