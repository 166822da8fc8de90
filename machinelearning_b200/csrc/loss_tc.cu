// The products of the linear cross entropy (loss.cu) on the tensor cores:
//   kLse       l = x W^T, of which only each row's running maximum and sum of exponentials, both without the target's, leave the SM, and
//              the target's l;
//   kGrad      l again for a piece of the vocabulary, dl = r (exp(l - lse) - [v == target]), written in 16 bits;
//   kProducts  dx (+)= dl W and dW = dl^T x of that piece, both in one launch;
//   kFew       kLse of up to 64 rows with the operands exchanged: l^T = W x^T, 256 words x 64 rows a tile.
//
// One persistent kernel per kind, a pair of CTAs (cta_group::2) per 256 x 256 tile: each CTA holds 128 rows of A, 128
// columns of B and 128 x 256 of the sums, so an operand byte brought into shared memory serves twice the columns
// of a single CTA's tile.  A stage is 128 summands, each operand of it one box of 32 KB: 128 rows x 2 blocks of 64 columns, K-major or
// MN-major by what its coordinates mean.  (Loads bound these kernels, and how many there are counts as much as their bytes:
// forward of 16,384 x 50,304 x 768 at 1,490 TFLOP/s with boxes of 8 KB, 1,583 with 16 KB, 1,605 with
// 32 KB; with half of the bytes 1,780.)  Sums are double buffered in TMEM (2 x 256 columns): the epilogue of a tile runs under the next one's products.
//
// The tensor core adds to its sums by truncation: a chain of K / 16 steps over positive summands comes out low by 6.6e-7 of
// its value at K = 768, 1.1e-5 at 4,096 and 7.7e-5 at 16,384 (measured; a float32 product on the CUDA cores is off by 5e-8).  Where that shows,
// the chain is cut (LONG; where: loss.cu): a tile's sum is formed chunk by chunk, and the chunks' sums are added in registers.
//
// Warps: 0 producer, 1 MMA issuer (even CTA) and TMEM owner, 2-9 epilogue: two warps per quarter of the rows, 128 columns
// each.  Every wait is bounded (ptx.cuh); no multicast loads.
#include <cfloat>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "loss.cuh"
#include "ptx.cuh"

namespace nlfa {
namespace loss {
namespace {

constexpr int kThreads = 320;
constexpr int kEpilogueWarps = 8;
constexpr int kBlockBytes = 128 * 128;                        // 128 rows of 64 columns
// PARTS = 1: three stages of 128 summands.  PARTS = 3 (float32 operands, sums of three bf16 parts): two stages of 64 summands in all
// parts, each of which is multiplied with two or three of the other operand's: a pair of parts a stage loads everything twice.
// kFew: four stages, A as above, B 32 rows of a CTA.
template <int MODE, int PARTS>
struct Ring {
  static constexpr int kStages = PARTS == 3 ? 2 : MODE == kFew ? 4 : 3;
  static constexpr int kSummands = summands(PARTS);
  static constexpr int kBlocks = PARTS == 3 ? 3 : kSummands / 64;
  static constexpr int kOperandBytes = kBlocks * kBlockBytes;   // one CTA's half of A
  static constexpr int kBBlockBytes = MODE == kFew ? kBlockBytes / 4 : kBlockBytes;
  static constexpr int kStageBytes = kOperandBytes + kBlocks * kBBlockBytes;
  static_assert(kStages * kStageBytes <= 12 * kBlockBytes, "stages");
};
constexpr int kMostStages = 4;
constexpr int kStagingBytes = 4096;                           // per epilogue warp
constexpr int kStaging = 12 * kBlockBytes;
constexpr int kBars = kStaging + kEpilogueWarps * kStagingBytes;
constexpr int kNumBars = 2 * kMostStages + 4;
constexpr int kTmemSlot = kBars + 8 * kNumBars;
constexpr int kAbort = kTmemSlot + 4;
constexpr int kPlan = kAbort + 4;
constexpr int kSmem = kPlan + 128 + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");

enum { FULL = 0, EMPTY = kMostStages, ACC_FULL = 2 * kMostStages, ACC_EMPTY = ACC_FULL + 2 };

// float32 operands are sums of three bf16 parts; the products of parts, smallest first (what is left out is below 2^-24)
__device__ __forceinline__ int part_a(int pair) { return (0x001012 >> (4 * pair)) & 15; }   // 2 1 0 1 0 0
__device__ __forceinline__ int part_b(int pair) { return (0x010210 >> (4 * pair)) & 15; }   // 0 1 2 0 1 0

__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// A tile: where it lies in A's rows and B's columns, how many stages its sum takes, which operands it has.
struct Tile {
  int m0, n0;
  int k0, k1;                       // its blocks of summands (a stage each): all, or of a shared tile this pair's
  int length;                       // kProducts: blocks per part of dl (the parts follow one another)
  int dw;                           // kProducts: a tile of dW (else of dx)
  int first, last;                  // kLse: first / last tile of a unit
  int slot;                         // kLse: which part of the vocabulary; kProducts: where a share of a tile goes (-1: the tile is whole)
};

// kProducts: the units are dW's tiles and then dx's, handed out in turn: whole tiles, as many of each kind as all pairs of CTAs get,
// and the rest, whose sums are cut into parts so that every pair is busy (loss.cu: choose_parts; fold_kernel adds the shares).  Parts of one
// index stand together: they read the same summands, from L2.  Backward with whole tiles only, and as it is: 65,536 rows x 50,304 words
// x 768 13.5 and 12.4 ms, 4,096 rows 0.86 and 0.82, 300 rows 0.38 and 0.15.  (The rest as one line of stages cut into equal lengths balances
// better, but every pair then reads summands of its own from HBM: slower than whole tiles at 16,384 rows.)
struct Plan {
  int d_tiles, kw, kx, again;
  int chunk;                        // stages per chain
  int dw_whole, dw_rest, dw_parts, dx_whole, dx_rest, dx_parts;
  int u1, u2, u3, u4;               // ends of the four kinds of units
  int dx_slot;                      // dx's first share
  __device__ Plan(const Params& p, int rows, int pairs) {
    const int row_tiles = rows > 0 ? ceil_div(rows, kRowTile) : 1;
    d_tiles = ceil_div(p.d, kColTile);
    const int dw_tiles = p.want_dw ? ceil_div(p.v1 - p.v0, kColTile) * d_tiles : 0, dx_tiles = p.want_dx ? row_tiles * d_tiles : 0;
    again = p.planes == 1 ? dl_parts(p.planes, p.per_row, rows) : 1;
    chunk = again == 2 ? 8 : p.chunk;                          // (loss.cu: product_chain)
    kw = again * row_tiles * (kRowTile / summands(p.planes));
    kx = again * ceil_div(p.v1 - p.v0, summands(p.planes));
    dw_whole = dw_tiles / pairs * pairs;
    dx_whole = dx_tiles / pairs * pairs;
    dw_rest = dw_tiles - dw_whole;
    dx_rest = dx_tiles - dx_whole;
    dw_parts = p.parts->dw[p.last];
    dx_parts = p.parts->dx[p.last];
    u1 = dw_whole;
    u2 = u1 + dw_rest * dw_parts;
    u3 = u2 + dx_whole;
    u4 = u3 + dx_rest * dx_parts;
    dx_slot = kPartsPerPair * pairs;
  }
  __device__ bool unit(int u, Tile& t) const {
    if (u >= u4) return false;
    t.dw = u < u2;
    const int first = t.dw ? 0 : u2, whole = t.dw ? dw_whole : dx_whole, rest = t.dw ? dw_rest : dx_rest;
    const int parts = t.dw ? dw_parts : dx_parts, k = t.dw ? kw : kx, i = u - first - whole;
    int v = u - first;
    t.k0 = 0;
    t.k1 = k;
    t.length = k / again;
    t.slot = -1;
    if (i >= 0) {
      const int part = i / rest;
      v = whole + i - part * rest;
      if (parts > 1) {
        t.k0 = static_cast<int>(static_cast<long long>(k) * part / parts);
        t.k1 = static_cast<int>(static_cast<long long>(k) * (part + 1) / parts);
        t.slot = (t.dw ? 0 : dx_slot) + i;
      }
    }
    place(v, t);
    return true;
  }
  __device__ void place(int v, Tile& t) const {
    const int m = v / d_tiles;
    t.m0 = m * kRowTile;                                       // dW: columns of dl, from the piece's first
    t.n0 = (v - m * d_tiles) * kColTile;
  }
};

static_assert(sizeof(Plan) <= 128, "its place in shared memory");

// The tiles of one pair of CTAs, in order; every role walks the same list.
template <int MODE>
struct Walk {
  const Params& p;
  int rows, row_tiles, stride, u, units;
  int n, n_end;                     // kLse: column tiles left in the unit
  int col_tiles, splits;
  const Plan* plan;                 // kProducts: in shared memory

  __device__ Walk(const Params& p_, int pair, int n_pairs, const Plan* plan_) : p(p_), rows(p_.head->count), stride(n_pairs), plan(plan_) {
    row_tiles = rows > 0 ? ceil_div(rows, kRowTile) : 1;        // (no row: one tile of zeros, which leaves zero gradients)
    u = pair - n_pairs;
    n = n_end = 0;
    splits = 1;
    if (MODE == kLse) {
      splits = p.head->splits;
      col_tiles = ceil_div(p.V, kColTile);
      units = row_tiles * splits;
    } else if (MODE == kFew) {
      // a run of W's tiles for every pair
      col_tiles = ceil_div(p.V, kRowTile);
      n = static_cast<int>(static_cast<long long>(col_tiles) * pair / n_pairs);
      n_end = static_cast<int>(static_cast<long long>(col_tiles) * (pair + 1) / n_pairs);
    } else if (MODE == kGrad) {
      col_tiles = ceil_div(p.v1 - p.v0, kColTile);
      units = row_tiles * col_tiles;
    }
  }

  __device__ int chunk() const { return MODE == kProducts ? plan->chunk : p.chunk; }
  __device__ bool next(Tile& t) {
    t.k0 = 0;
    if (MODE != kProducts) t.k1 = ceil_div(p.d, summands(p.planes));
    if (MODE == kLse) {
      t.first = 0;
      if (n == n_end) {
        u += stride;
        if (u >= units) return false;
        // neighbouring pairs: the same part of the vocabulary, other rows, so that W is read from L2
        const int part = u / row_tiles;
        t.m0 = (u - part * row_tiles) * kRowTile;
        t.slot = part;
        n = static_cast<int>(static_cast<long long>(col_tiles) * part / splits);
        n_end = static_cast<int>(static_cast<long long>(col_tiles) * (part + 1) / splits);
        t.first = 1;
      }
      t.n0 = n * kColTile;
      t.last = ++n == n_end;
      return true;
    }
    if (MODE == kFew) {
      if (n == n_end) return false;
      t.m0 = n++ * kRowTile;
      t.n0 = 0;
      return true;
    }
    u += stride;
    if (MODE == kGrad) {
      if (u >= units) return false;
      // eight row tiles at a time past all columns of the piece
      const int group = 8 * col_tiles, g = u / group, v = u - g * group;
      const int size = row_tiles - 8 * g < 8 ? row_tiles - 8 * g : 8;
      const int c = v / size;
      t.m0 = (8 * g + v - c * size) * kRowTile;
      t.n0 = p.v0 + c * kColTile;
      return true;
    }
    return plan->unit(u, t);
  }
};

template <typename T>
__device__ __forceinline__ float round_to(float x);
template <>
__device__ __forceinline__ float round_to<__nv_bfloat16>(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
template <>
__device__ __forceinline__ float round_to<__half>(float x) { return __half2float(__float2half_rn(x)); }

// Where a product's values go: four of row `m` of its tiles' rows, columns cc ..
struct Out {
  const Params& p;
  int dw, dtype, m_end;
  float alpha;
  void* to;
  bool vec;
  __device__ Out(const Params& p_, int dw_, int rows) : p(p_), dw(dw_) {
    dtype = dw ? p.dw_dtype : p.dx_dtype;
    m_end = dw ? p.v1 - p.v0 : rows;
    alpha = *p.alpha;
    to = dw ? p.dw : p.dx;
    vec = p.d % 4 == 0;
  }
  __device__ __forceinline__ void put(int m, int cc, float (&v)[4]) const {
    if (m >= m_end || cc >= p.d) return;
    const int n = p.d - cc < 4 ? p.d - cc : 4;
    size_t at = static_cast<size_t>(dw ? p.v0 + m : m) * p.d + cc;
    if (!dw && !(p.first && p.last)) {                         // dx is summed over the pieces
      float* sum = p.dx_sum + at;
      if (vec) {
        float4* s4 = reinterpret_cast<float4*>(sum);
        if (!p.first) {
          const float4 b = *s4;
          v[0] += b.x; v[1] += b.y; v[2] += b.z; v[3] += b.w;
        }
        if (!p.last) *s4 = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        for (int e = 0; e < n; ++e) {
          if (!p.first) v[e] += sum[e];
          if (!p.last) sum[e] = v[e];
        }
      }
      if (!p.last) return;
    }
    if (!dw) at = static_cast<size_t>(p.row_of[m]) * p.d + cc;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= alpha;
    if (dtype == NLFA_DTYPE_F32) {
      float* o = static_cast<float*>(to) + at;
      if (vec) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
      else for (int e = 0; e < n; ++e) o[e] = v[e];
    } else if (dtype == NLFA_DTYPE_BF16) {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(to) + at;
      if (vec) *reinterpret_cast<uint2*>(o) = make_uint2(Pack2<__nv_bfloat16>::pack(v[0], v[1]), Pack2<__nv_bfloat16>::pack(v[2], v[3]));
      else for (int e = 0; e < n; ++e) o[e] = __float2bfloat16_rn(v[e]);
    } else {
      __half* o = static_cast<__half*>(to) + at;
      if (vec) *reinterpret_cast<uint2*>(o) = make_uint2(Pack2<__half>::pack(v[0], v[1]), Pack2<__half>::pack(v[2], v[3]));
      else for (int e = 0; e < n; ++e) o[e] = __float2half_rn(v[e]);
    }
  }
};

// The shares of a tile formed in parts (blockIdx.x), added in order; 4 rows a CTA.
constexpr int kFoldThreads = 256, kFoldRows = 4;
__global__ void __launch_bounds__(kFoldThreads)
fold_kernel(const Params p, int pairs) {
  grid_dep_wait();
  grid_dep_release();
  const Plan plan(p, p.head->count, pairs);
  int i = blockIdx.x;
  Tile t;
  t.dw = i < plan.dw_rest;
  if (!t.dw) i -= plan.dw_rest;
  const int rest = t.dw ? plan.dw_rest : plan.dx_rest, parts = t.dw ? plan.dw_parts : plan.dx_parts;
  if (i >= rest || parts < 2) return;
  plan.place((t.dw ? plan.dw_whole : plan.dx_whole) + i, t);
  const Out out(p, t.dw, p.head->count);
  const int cc = 4 * (threadIdx.x & 63);
  if (t.n0 + cc >= p.d) return;
  const float* shares = p.shares + (static_cast<size_t>(t.dw ? 0 : plan.dx_slot) + i) * (kRowTile * kColTile) + cc;
  const int r = blockIdx.y * kFoldRows + (threadIdx.x >> 6);
  if (t.m0 + r >= out.m_end) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int part = 0; part < parts; ++part) {
    const float4 x = *reinterpret_cast<const float4*>(shares + (static_cast<size_t>(part) * rest * kRowTile + r) * kColTile);
    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
  }
  out.put(t.m0 + r, t.n0 + cc, v);
}

// ---- epilogues: a thread has row `lane` of its warp's 32 and, 32 at a time, 128 columns

// The columns of a thread's row: in TMEM, or (LONG) summed from the chunks' sums in registers.
template <bool LONG, int COLS>
struct Sums {
  uint32_t acc;
  float v[LONG ? COLS : 1];
  __device__ __forceinline__ void get(int col, uint32_t (&r)[32]) const {
    if constexpr (LONG) {
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c)
        if (col == 32 * c) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(v[32 * c + j]);
        }
    } else {
      tmem_ld32(acc + col, r);
      tc_wait_ld();
    }
  }
};

template <typename T, int MODE, bool LONG, int PARTS>
__global__ void __launch_bounds__(kThreads, 1)
loss_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
            const __grid_constant__ CUtensorMap tm_ds, const __grid_constant__ CUtensorMap tm_out, const Params p) {
  constexpr bool kBf16 = Pack2<T>::kIsBf16;
  using R = Ring<MODE, PARTS>;
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

  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
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
  if (MODE == kFew && p.w_stands && threadIdx.x == 0) {
    // while the rows are packed, W comes into L2: what this CTA loads first, 0.5 MB (all CTAs: 78 of the 126 MB)
    const int tiles = ceil_div(p.V, kRowTile), n_end = static_cast<int>(static_cast<long long>(tiles) * (pair + 1) / n_pairs);
    int left = 16;
    for (int n = static_cast<int>(static_cast<long long>(tiles) * pair / n_pairs); n < n_end && left > 0; ++n)
      for (int k = 0; k < p.d && left > 0; k += R::kSummands, --left) tma_prefetch_4d(&tm_w, 0, n * kRowTile + 128 * rank, k / 64, 0);
  }
  grid_dep_wait();
  grid_dep_release();
  Plan* plan = reinterpret_cast<Plan*>(gen + kPlan);
  if constexpr (MODE == kProducts) {
    if (threadIdx.x == 0) *plan = Plan(p, p.head->count, n_pairs);
    __syncthreads();
  }

  if (dead) {
    // a give-up recorded earlier makes this launch a no-op
  } else if (warp == 0) {
    // ============================== producer ================================
    if (lane == 0) {
      Walk<MODE> walk(p, pair, n_pairs, plan);
      Tile t;
      int it = 0;
      bool ok = true;
      const uint32_t full0 = cluster_addr(bar(FULL), 0);       // loads of both CTAs are counted on the even one's
      auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t full, int row, int col) {
        tma_load_4d_pair(dst, map, full, 0, row, col / 64, 0);
      };
      while (ok && walk.next(t)) {
        const CUtensorMap* ma = MODE == kFew ? &tm_w : MODE != kProducts ? &tm_x : t.dw ? &tm_out : &tm_ds;
        const CUtensorMap* mb = MODE == kFew || (MODE == kProducts && t.dw) ? &tm_x : &tm_w;
        const int a0 = t.m0 + 128 * rank, b0 = t.n0 + (MODE == kFew ? kFewRows / 2 : 128) * rank;
        for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
          const int s = it % kStages;
          if (!(ok = mbar_wait(bar(EMPTY + s), ((it / kStages) & 1) ^ 1, wctx, 90))) break;
          const uint32_t st = base + s * R::kStageBytes, full = full0 + 8u * s;
          if (rank == 0) mbar_arrive_expect_tx(bar(FULL + s), 2 * R::kStageBytes);
          // boxes at (row, block of 64 columns): the sum runs along the columns, or (MN-major) along the rows
          const bool second = MODE == kProducts && PARTS == 1 && kb >= t.length;            // part of dl
          const int k = (kb - (second ? t.length : 0)) * R::kSummands, part = second ? p.dl_second : 0;
          if (MODE == kProducts && t.dw) load(st, ma, full, part + k, a0);
          else load(st, ma, full, part + a0, k);
          if (MODE != kProducts) load(st + R::kOperandBytes, mb, full, b0, k);
          else load(st + R::kOperandBytes, mb, full, (t.dw ? 0 : p.v0) + k, b0);
        }
      }
      // the last loads of this CTA have been consumed before it may leave (after a give-up: have had time to land)
      for (int i = 0; ok && i < kStages; ++i, ++it) ok = mbar_wait(bar(EMPTY + it % kStages), ((it / kStages) & 1) ^ 1, wctx, 91);
      if (!ok) for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    // ============================= MMA issuer ===============================
    if (rank == 0) {
      const uint32_t leader = elect_one() ? 1u : 0u;
      Walk<MODE> walk(p, pair, n_pairs, plan);
      Tile t;
      int it = 0, sums = 0;                                    // sums: filled TMEM buffers so far
      bool ok = true;
      while (ok && walk.next(t)) {
        const bool a_mn = MODE == kProducts && t.dw, b_mn = MODE == kProducts;
        constexpr int kN = MODE == kFew ? kFewRows : kColTile;
        const uint32_t idesc = a_mn ? make_idesc(kBf16, 256, kN, true, b_mn) : make_idesc(kBf16, 256, kN, false, b_mn);
        // 16 summands on: 32 bytes along a row, then the next block of 64 columns; or (MN-major) 16 rows
        constexpr uint32_t kMnBlock = PARTS == 3 ? kBlockBytes / 2 : kBlockBytes;     // (of 64 summands: 64 rows)
        const uint32_t a_lbo = a_mn ? kMnBlock : 16u, b_lbo = b_mn ? kMnBlock : 16u;
        const int chunk = LONG ? walk.chunk() : t.k1 - t.k0;
        for (int k0 = t.k0; ok && k0 < t.k1; k0 += chunk, ++sums) {
          const int buf = sums & 1;
          if (!(ok = mbar_wait(bar(ACC_EMPTY + buf), ((sums >> 1) & 1) ^ 1, wctx, 92))) break;
          tc_fence_after();
          const int stages = t.k1 - k0 < chunk ? t.k1 - k0 : chunk;
          for (int kb = 0; kb < stages; ++kb, ++it) {
            const int s = it % kStages;
            if (!(ok = mbar_wait(bar(FULL + s), (it / kStages) & 1, wctx, 93))) break;
            tc_fence_after();
            const uint32_t a = base + s * R::kStageBytes, b = a + R::kOperandBytes;
#pragma unroll
            for (int pr = 0; pr < (PARTS == 3 ? 6 : 1); ++pr) {
              const uint32_t a_part = PARTS == 3 ? part_a(pr) * kBlockBytes : 0u, b_part = PARTS == 3 ? part_b(pr) * R::kBBlockBytes : 0u;
#pragma unroll
              for (int kk = 0; kk < R::kSummands / 16; ++kk) {
                const uint32_t along_a = a_mn ? kk * 2048u : (kk / 4) * kBlockBytes + (kk % 4) * 32u;
                const uint32_t along_b = b_mn ? kk * 2048u : (kk / 4) * R::kBBlockBytes + (kk % 4) * 32u;
                umma_ss_pair(leader, tmem + buf * kColTile, make_smem_desc(a + a_part + along_a, a_lbo, 1024),
                             make_smem_desc(b + b_part + along_b, b_lbo, 1024), idesc,
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
    Walk<MODE> walk(p, pair, n_pairs, plan);
    Tile t;
    float run_max = 0.f, run_sum = 0.f;
    int sums = 0;
    bool ok = true;
    constexpr int kMine = kFewRows / 2;                        // kFew: a thread has one word and, of each tile, this many rows
    float few_max[MODE == kFew ? kMine : 1], few_sum[MODE == kFew ? kMine : 1];
    int few_target = -1;
    if constexpr (MODE == kFew) {
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        few_max[j] = -FLT_MAX;
        few_sum[j] = 0.f;
      }
      few_target = p.target[kMine * half + lane];
    }
    constexpr int kCols = MODE == kFew ? kMine : 128;
    Sums<LONG, kCols> l;
    auto release = [&](int buf) {                              // this warp has read its part of the buffer
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + 8u * buf);
    };
    while (walk.next(t)) {
      const int row0 = t.m0 + 128 * rank + 32 * q, row = row0 + lane;
      int target = -1;
      float lse = 0.f, rest2 = 0.f, scale = 0.f, own = 0.f;
      if (MODE == kLse || MODE == kGrad) target = p.target[row];
      if (MODE == kGrad) {
        lse = p.lse[row];
        rest2 = p.lse_rest[row] * kLog2e;
        scale = p.row_scale[row];
        own = p.own[row] * scale;                              // dl of the row's target
      }
      if (MODE == kLse && t.first) { run_max = -INFINITY; run_sum = 0.f; }
      int buf = 0;
      if constexpr (LONG) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) l.v[j] = 0.f;
        for (int k0 = t.k0; k0 < t.k1; k0 += walk.chunk(), ++sums) {
          buf = sums & 1;
          if (!(ok = mbar_wait(bar(ACC_FULL + buf), (sums >> 1) & 1, wctx, 94))) break;
          tc_fence_after();
          // 16 columns at a time beside the 128 in registers: what spills goes to L2, since L1 has next to nothing left.  The products spill 304
          // bytes with 32 and nothing with 16 (backward of 300 rows 160 and 147 us, of 1,000 x 5,003 x 384 in float32 99.8 and 94.6).
#pragma unroll
          for (int c = 0; c < kCols / 16; ++c) {
            uint32_t r[16];
            tmem_ld16(tmem_addr(tmem, 32 * q, buf * kColTile + kCols * half + 16 * c), r);
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
        ok = mbar_wait(bar(ACC_FULL + buf), (sums >> 1) & 1, wctx, 94);
        tc_fence_after();
        l.acc = tmem_addr(tmem, 32 * q, buf * kColTile + kCols * half);
        ++sums;
      }
      if (!ok) break;
      const int c0 = t.n0 + 128 * half;

      if constexpr (MODE == kFew) {
        uint32_t r[32];
        l.get(0, r);
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          if (kMine * half + j >= walk.rows) break;
          float x = row < p.V ? __uint_as_float(r[j]) : -INFINITY;
          if (__shfl_sync(0xffffffffu, few_target, j) == row) {
            p.at_target[kMine * half + j] = x;
            x = -INFINITY;
          }
          const float top = fmaxf(few_max[j], x);
          few_sum[j] = fmaf(few_sum[j], fast_exp2((few_max[j] - top) * kLog2e), fast_exp2((x - top) * kLog2e));
          few_max[j] = top;
        }
      } else if constexpr (MODE == kLse) {
#pragma unroll (LONG ? 4 : 1)
        for (int c = 0; c < 4; ++c) {
          const int col = c0 + 32 * c;
          if (col >= p.V) break;
          uint32_t r[32];
          l.get(32 * c, r);
          if (col + 32 > p.V) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col + j >= p.V) r[j] = __float_as_uint(-INFINITY);
          }
          const unsigned at = static_cast<unsigned>(target - col);
          if (__any_sync(0xffffffffu, at < 32u)) {
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (at == static_cast<unsigned>(j)) {
                v = __uint_as_float(r[j]);
                r[j] = __float_as_uint(-INFINITY);
              }
            if (at < 32u) p.at_target[row] = v;
          }
          float top = __uint_as_float(r[0]);
#pragma unroll
          for (int j = 1; j < 31; j += 2) top = fmax3(top, __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
          top = fmaxf(fmaxf(top, __uint_as_float(r[31])), run_max);
          // The difference is formed before it is scaled: fma(l, log2 e, -top log2 e) is off by the rounding of top log2 e,
          // in every summand alike.  (every logit so far -inf: nothing to subtract)
          const float shift = top == -INFINITY ? 0.f : top;
          const uint64_t minus = pack_f2(-shift, -shift), by = pack_f2(kLog2e, kLog2e);
          uint64_t part[2] = {0ull, 0ull};
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float a, b;
            unpack_f2(fmul2(fadd2(pack_f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), minus), by), a, b);
            part[j / 2 & 1] = fadd2(part[j / 2 & 1], pack_f2(fast_exp2(a), fast_exp2(b)));
          }
          float a, b;
          unpack_f2(fadd2(part[0], part[1]), a, b);
          run_sum = fmaf(run_sum, fast_exp2((run_max - shift) * kLog2e), a + b);
          run_max = top;
        }
        if (t.last) p.partial[static_cast<size_t>(2 * t.slot + half) * p.n_rows + row] = make_float2(run_max, run_sum);
      } else if constexpr (MODE == kGrad) {
#pragma unroll (LONG ? 2 : 1)
        for (int c2 = 0; c2 < 2; ++c2) {
          // 64 columns: a row of the staging tile (128 bytes, swizzled as the tensor map has it)
          float lo[2][32];                                     // what is left of the values after the parts written so far
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = c0 + 64 * c2 + 32 * h;
            uint32_t r[32];
            l.get(64 * c2 + 32 * h, r);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float a, b;
              unpack_f2(ffma2(fadd2(pack_f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), pack_f2(-lse, -lse)),
                              pack_f2(kLog2e, kLog2e), pack_f2(-rest2, -rest2)), a, b);
              unpack_f2(fmul2(pack_f2(fast_exp2(a), fast_exp2(b)), pack_f2(scale, scale)), lo[h][j], lo[h][j + 1]);
            }
            if (col + 32 > p.V) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j >= p.V) lo[h][j] = 0.f;
            }
            const unsigned at = static_cast<unsigned>(target - col);
            // (three parts leave no registers: the backward of 1,000 x 5,003 x 384 takes 95 us with a product and sum here, 101 with a choice; in
            // one part, 16,384 x 50,304 x 768: 3.27 and 3.15 ms.  p is finite unless own is NaN too)
            if (__any_sync(0xffffffffu, at < 32u)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (at == static_cast<unsigned>(j)) lo[h][j] = PARTS == 3 ? fmaf(lo[h][j], 0.f, own) : own;
            }
            if (__any_sync(0xffffffffu, target == -1)) {     // behind the last row: zeros, whatever W holds (0 inf would not be)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (target == -1) lo[h][j] = 0.f;
            }
          }
          const int held = dl_parts(PARTS, p.per_row, walk.rows);
#pragma unroll 1
          for (int part = 0; part < held; ++part) {
            if (lane == 0) tma_store_wait_read();
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < 32; j += 8) {
                const float* v = lo[h] + j;
                const uint32_t chunk = static_cast<uint32_t>((4 * h + j / 8) ^ (lane & 7));
                st_shared_v4(staging + lane * 128 + chunk * 16, Pack2<T>::pack(v[0], v[1]), Pack2<T>::pack(v[2], v[3]),
                             Pack2<T>::pack(v[4], v[5]), Pack2<T>::pack(v[6], v[7]));
              }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_4d(&tm_out, staging, 0, row0 + (PARTS == 1 && part > 0 ? p.dl_second : 0), (c0 + 64 * c2 - p.v0) / 64, PARTS == 1 ? 0 : part);
              tma_store_commit();
            }
            if (part + 1 < held) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 32; ++j) lo[h][j] -= round_to<T>(lo[h][j]);
            }
          }
        }
      } else {
        // 32 x 32 values through shared memory, so that a row's columns leave side by side
        const Out out(p, t.dw, walk.rows);
        const int local = 128 * rank + 32 * q;
        float* share = t.slot < 0 ? nullptr : p.shares + (static_cast<size_t>(t.slot) * kRowTile + local) * kColTile;
#pragma unroll (LONG ? 4 : 1)
        for (int c = 0; c < 4; ++c) {
          const int col = c0 + 32 * c;
          if (col >= p.d) break;
          uint32_t r[32];
          l.get(32 * c, r);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            st_shared_v4(staging + lane * 128 + (((j / 4) ^ (lane & 7)) * 16), r[j], r[j + 1], r[j + 2], r[j + 3]);
          __syncwarp();
          const int cc = col + 4 * (lane & 7);
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const int lr = 4 * i + (lane >> 3);
            uint32_t w0, w1, w2, w3;
            ld_shared_v4(staging + lr * 128 + (((lane & 7) ^ (lr & 7)) * 16), w0, w1, w2, w3);
            float v[4] = {__uint_as_float(w0), __uint_as_float(w1), __uint_as_float(w2), __uint_as_float(w3)};
            if (share != nullptr) *reinterpret_cast<float4*>(share + static_cast<size_t>(lr) * kColTile + (cc - t.n0)) = make_float4(v[0], v[1], v[2], v[3]);
            else out.put(t.m0 + local + lr, cc, v);
          }
          __syncwarp();
        }
      }
      if (!LONG) release(buf);
    }
    if constexpr (MODE == kFew) {
      // the 128 words of a CTA's four warps as one part (a pair without tiles has an empty one)
      float2* parts = reinterpret_cast<float2*>(gen + kStaging);          // [quarter][row]
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        if (kMine * half + j >= walk.rows) break;
        float top = few_max[j];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        float sum = few_sum[j] * fast_exp2((few_max[j] - top) * kLog2e);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane == 0) parts[kFewRows * q + kMine * half + j] = make_float2(top, sum);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory");
      const int row = kMine * half + lane;
      if (q == 0 && row < walk.rows) {
        float2 all = parts[row];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          const float2 x = parts[kFewRows * i + row];
          const float top = fmaxf(all.x, x.x);
          all = make_float2(top, fmaf(all.y, fast_exp2((all.x - top) * kLog2e), x.y * fast_exp2((x.x - top) * kLog2e)));
        }
        p.partial[static_cast<size_t>(2 * pair + rank) * p.n_rows + row] = all;
      }
    }
    if (MODE == kGrad && lane == 0) tma_store_wait_all();
  }

  tc_fence_before();
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

template <typename T, int MODE, bool LONG, int PARTS = 1>
int launch_one(const Params& p, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& ds, const CUtensorMap& out,
               cudaStream_t stream) {
  auto* kernel = loss_kernel<T, MODE, LONG, PARTS>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem);
  if (rc != NLFA_OK) return rc;
  const int pairs = most_pairs();
  // (a pair has to lie along x: along y the launch is refused)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2u * static_cast<unsigned>(pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap_launches(kOverlapRowwise) ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, x, w, ds, out, p);
  if (MODE == kProducts && e == cudaSuccess) {
    const int d_tiles = ceil_div(p.d, kColTile), dw_rest = p.want_dw ? ceil_div(p.v1 - p.v0, kColTile) * d_tiles % pairs : 0;
    const int dx_tiles = p.want_dx ? p.n_rows / kRowTile * d_tiles : 0, most = dw_rest + (dx_tiles < pairs ? dx_tiles : pairs);
    e = launch_kernel(fold_kernel, dim3(static_cast<unsigned>(most > 0 ? most : 1), kRowTile / kFoldRows), dim3(kFoldThreads), 0,
                      stream, overlap_launches(kOverlapRowwise), p, pairs);
  }
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

}  // namespace

int most_pairs() { return sm_count() / 2; }
size_t share_bytes() { return static_cast<size_t>(2 * kPartsPerPair * most_pairs()) * kRowTile * kColTile * sizeof(float); }

int launch_product(int mode, int dtype, const Params& p, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& ds,
                   const CUtensorMap& ds_out, cudaStream_t stream) {
  const bool bf16 = dtype == NLFA_DTYPE_BF16;
#define NLFA_GO(...) launch_one<__VA_ARGS__>(p, x, w, ds, ds_out, stream)
  if (p.planes == 3)                                          // float32 operands: parts in bf16
    return mode == kFew ? NLFA_GO(__nv_bfloat16, kFew, true, 3)
           : mode == kLse ? NLFA_GO(__nv_bfloat16, kLse, true, 3)
           : mode == kGrad ? NLFA_GO(__nv_bfloat16, kGrad, true, 3)
                           : NLFA_GO(__nv_bfloat16, kProducts, true, 3);
  if (mode == kFew && p.chunk > 0) return bf16 ? NLFA_GO(__nv_bfloat16, kFew, true) : NLFA_GO(__half, kFew, true);
  if (mode == kFew) return bf16 ? NLFA_GO(__nv_bfloat16, kFew, false) : NLFA_GO(__half, kFew, false);
  if (mode == kLse && p.chunk > 0) return bf16 ? NLFA_GO(__nv_bfloat16, kLse, true) : NLFA_GO(__half, kLse, true);
  if (mode == kLse) return bf16 ? NLFA_GO(__nv_bfloat16, kLse, false) : NLFA_GO(__half, kLse, false);
  if (mode == kGrad && p.chunk > 0) return bf16 ? NLFA_GO(__nv_bfloat16, kGrad, true) : NLFA_GO(__half, kGrad, true);
  if (mode == kGrad) return bf16 ? NLFA_GO(__nv_bfloat16, kGrad, false) : NLFA_GO(__half, kGrad, false);
  return bf16 ? NLFA_GO(__nv_bfloat16, kProducts, true) : NLFA_GO(__half, kProducts, true);
#undef NLFA_GO
}

}  // namespace loss
}  // namespace nlfa
