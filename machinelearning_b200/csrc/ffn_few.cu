// The gated feed-forward layer for a few tokens (decoding): bound by one pass over the weights, and by latency.
//
// Two launches: h = f(x Wg^T) (x Wu^T) in float32, then y = h Wd^T.  A warp has 16 rows of a weight and a run of the sum: each lane loads 16 bytes (8 summands) of
// two rows at a time straight into the operand registers of mma.sync m16n8k16 -- the order of the summands is free, so a lane's 8 consecutive ones
// serve as its places of two products, for weight and tokens alike.  A tensor-memory kernel's set-up and tiles of 256 rows cost more than
// the whole sum here (8 x 768 x 2,048: 30 us in the kernels of ffn_tc.cu, 6.7 here).  The runs of a tile's sum are added through shared memory, in order.
// All loads of a run are in flight at once; the second launch has its weights on the way before the first one's h is there.
//
// Types: every operand is a sum of bf16 parts, split in registers: bf16 one, float16 two (exact), float32 three (to 2^-24), h two (2^-17), beside float32 three; the products
// of parts down to the type's own rounding, the leading parts' last.  The tensor core truncates what it adds to, so a long chain of one sign comes out low: chains end
// after 32 summands in float32, 128 in 16 bits, and their sums are added in registers.  So h is not rounded to 16 bits, nor kept to float16's range.
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ffn.cuh"
#include "ptx.cuh"

namespace nlfa {
namespace ffn {
namespace {

constexpr int kRows = 16;                     // of a weight, per CTA (kUp: of both)
constexpr int kUpWarps = 8, kDownWarps = 16;
constexpr int kDeep = 4;                      // steps of 32 summands in flight

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight values as they lie.
template <typename S> struct Eight { uint4 r[sizeof(S) / 2]; };
template <typename S> __device__ __forceinline__ void load(Eight<S>& e, const S* p, bool on) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(S)) / 2; ++i) e.r[i] = on ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ float2 pair_of(const Eight<__nv_bfloat16>& e, int i) {
  return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&e)[i]);
}
__device__ __forceinline__ float2 pair_of(const Eight<__half>& e, int i) { return __half22float2(reinterpret_cast<const __half2*>(&e)[i]); }
__device__ __forceinline__ float2 pair_of(const Eight<float>& e, int i) { return reinterpret_cast<const float2*>(&e)[i]; }

// What a value is in the type C of the products, and its bf16 parts.
template <typename C> struct Parts;
template <> struct Parts<__nv_bfloat16> { static constexpr int kCount = 1, kHidden = 2; };
template <> struct Parts<__half> { static constexpr int kCount = 2, kHidden = 2; };
template <> struct Parts<float> { static constexpr int kCount = 3, kHidden = 3; };
template <typename C> __device__ __forceinline__ float as(float x) { return x; }
template <> __device__ __forceinline__ float as<__nv_bfloat16>(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
template <> __device__ __forceinline__ float as<__half>(float x) { return __half2float(__float2half_rn(x)); }

// part[i][j]: part i of the pair j of eight values
template <typename S, typename C, int PARTS> __device__ __forceinline__ void split(const Eight<S>& e, uint32_t (&part)[PARTS][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (std::is_same_v<S, __nv_bfloat16> && PARTS == 1) {
      part[0][j] = reinterpret_cast<const uint32_t*>(&e)[j];
    } else {
      float2 v = pair_of(e, j);
      if constexpr (!std::is_same_v<S, C>) v = make_float2(as<C>(v.x), as<C>(v.y));
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        part[i][j] = *reinterpret_cast<const uint32_t*>(&h);
        const float2 f = __bfloat1622float2(h);
        v.x -= f.x;
        v.y -= f.y;
      }
    }
  }
}

// acc += the parts' products that count, smallest first
template <int WP, int XP>
__device__ __forceinline__ void product(float (&acc)[4], const uint32_t (&lo)[WP][4], const uint32_t (&hi)[WP][4], const uint32_t (&x)[XP][4]) {
#pragma unroll
  for (int i = WP - 1; i >= 0; --i)
#pragma unroll
    for (int j = XP - 1; j >= 0; --j) {
      if (i + j >= (WP > XP ? WP : XP)) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a[4] = {lo[i][2 * h], hi[i][2 * h], lo[i][2 * h + 1], hi[i][2 * h + 1]};
        mma(acc, a, x[j][2 * h], x[j][2 * h + 1]);
      }
    }
}

// Rows [row, row + 16) of w [rows, k] times the tokens, steps [s0, s1) of 32 summands: each lane's sums.  X: as the tokens lie.
template <typename S> struct Ahead {
  Eight<S> lo[kDeep], hi[kDeep];
};
template <typename S>
__device__ __forceinline__ void ask(Ahead<S>& a, int i, const S* lo, const S* hi, int step, int s1, int k) {
  const int at = 32 * step + 8 * (threadIdx.x & 3);
  const bool on = step < s1 && at < k;
  load(a.lo[i], lo + at, on);
  load(a.hi[i], hi + at, on);
}
// CW, CX: the types that weights and tokens are rounded to.
template <typename S, typename X, typename CW, typename CX, int WP, int XP, int NT>
__device__ __forceinline__ void run(float (&sum)[NT][4], Ahead<S>& ahead, const S* lo, const S* hi, const X* x, int n, int s0, int s1, int k) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  // the tokens of a step, one step ahead (of 32 tokens there are no registers for that: 64 of them 13.7 us so, 11.8 without)
  constexpr bool kAhead = NT < 4;
  Eight<X> xs[NT];
  auto tokens = [&](int step) {
    const int at = 32 * step + 8 * t;
#pragma unroll
    for (int j = 0; j < NT; ++j) load(xs[j], x + static_cast<size_t>(8 * j + g) * k + at, step < s1 && 8 * j + g < n && at < k);
  };
  float acc[NT][4] = {};
  auto cut = [&]() {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum[j][i] += acc[j][i];
        acc[j][i] = 0.f;
      }
  };
  if (kAhead) tokens(s0);
  for (int s = s0; s < s1; s += kDeep) {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      if (s + i >= s1) break;
      if (!kAhead) tokens(s + i);
      uint32_t wl[WP][4], wh[WP][4];
      split<S, CW, WP>(ahead.lo[i], wl);
      split<S, CW, WP>(ahead.hi[i], wh);
      ask(ahead, i, lo, hi, s + i + kDeep, s1, k);
      if constexpr (kAhead) {
        uint32_t xp[NT][XP][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) split<X, CX, XP>(xs[j], xp[j]);
        tokens(s + i + 1);
#pragma unroll
        for (int j = 0; j < NT; ++j) product<WP, XP>(acc[j], wl, wh, xp[j]);
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t xp[XP][4];
          split<X, CX, XP>(xs[j], xp);
          product<WP, XP>(acc[j], wl, wh, xp);
        }
      }
      if (WP == 3) cut();
    }
    if (WP != 3) cut();
  }
}

// The sums of a tile's runs, [warp][token][16 rows], with a row's padding against bank conflicts
constexpr int kPitch = kRows + 1;
template <int NT> __device__ __forceinline__ void leave(float* sums, const float (&sum)[NT][4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sums[(warp * 8 * NT + 8 * j + 2 * (lane & 3) + (i & 1)) * kPitch + (lane >> 2) + 8 * (i >> 1)] = sum[j][i];
}

struct FewParams {
  const void *x, *gate, *up, *down;
  float* h;
  void* y;
  int n, d, F, o, x_dtype, activation, out_dtype;
  int turns;
  // This CTA's rows of the weights (the CTAs that read the same ones stand side by side), and its tokens, up to `most`.
  __device__ __forceinline__ int turn(int most) {
    const int tile = blockIdx.x / turns, first = most * (blockIdx.x - tile * turns);
    x = static_cast<const uint8_t*>(x) + static_cast<size_t>(first) * d * (x_dtype == NLFA_DTYPE_F32 ? 4 : 2);
    h += static_cast<size_t>(first) * F;
    y = static_cast<uint8_t*>(y) + static_cast<size_t>(first) * o * (out_dtype == NLFA_DTYPE_F32 ? 4 : 2);
    n = min(n - first, most);
    return tile * kRows;
  }
};

__device__ __forceinline__ float activated(float g, int activation) {
  if (activation == NLFA_FFN_SILU) return g / (1.f + expf(-g));
  if (activation == NLFA_FFN_GELU) return g * fmaf(0.5f, erff(g * 0.70710678118654752f), 0.5f);
  return g < 0.f ? 0.f : g;
}

template <typename S, typename C, int NT>
__global__ void __launch_bounds__(32 * kUpWarps)
few_up_kernel(FewParams p) {
  const int row0 = p.turn(8 * NT);
  __shared__ float sums[kUpWarps * 8 * NT * kPitch];
  constexpr int kHalf = kUpWarps / 2, WP = Parts<C>::kCount;
  const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2;
  const int steps = (p.d + 31) / 32, q = warp % kHalf, s0 = steps * q / kHalf, s1 = steps * (q + 1) / kHalf;
  const S* w = static_cast<const S*>(warp < kHalf ? p.gate : p.up);
  // (rows behind the last one: the last one again, and nothing is written)
  const S* lo = w + static_cast<size_t>(min(row0 + g, p.F - 1)) * p.d;
  const S* hi = w + static_cast<size_t>(min(row0 + g + 8, p.F - 1)) * p.d;
  grid_dep_wait();
  grid_dep_release();
  Ahead<S> ahead;
#pragma unroll
  for (int i = 0; i < kDeep; ++i) ask(ahead, i, lo, hi, s0 + i, s1, p.d);
  float sum[NT][4] = {};
  if (p.x_dtype == NLFA_DTYPE_F32) run<S, float, C, C, WP, WP, NT>(sum, ahead, lo, hi, static_cast<const float*>(p.x), p.n, s0, s1, p.d);
  else if (p.x_dtype == NLFA_DTYPE_F16) run<S, __half, C, C, WP, WP, NT>(sum, ahead, lo, hi, static_cast<const __half*>(p.x), p.n, s0, s1, p.d);
  else run<S, __nv_bfloat16, C, C, WP, WP, NT>(sum, ahead, lo, hi, static_cast<const __nv_bfloat16*>(p.x), p.n, s0, s1, p.d);
  leave<NT>(sums, sum);
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * p.n; i += 32 * kUpWarps) {
    const int token = i / kRows, r = i % kRows;
    if (row0 + r >= p.F) continue;
    float gate = 0.f, up = 0.f;
#pragma unroll
    for (int v = 0; v < kHalf; ++v) {
      gate += sums[(v * 8 * NT + token) * kPitch + r];
      up += sums[((v + kHalf) * 8 * NT + token) * kPitch + r];
    }
    p.h[static_cast<size_t>(token) * p.F + row0 + r] = activated(gate, p.activation) * up;
  }
}

template <typename S, typename C, int NT>
__global__ void __launch_bounds__(32 * kDownWarps)
few_down_kernel(FewParams p) {
  const int row0 = p.turn(8 * NT);
  __shared__ float sums[kDownWarps * 8 * NT * kPitch];
  const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2;
  const int steps = (p.F + 31) / 32, s0 = steps * warp / kDownWarps, s1 = steps * (warp + 1) / kDownWarps;
  const S* lo = static_cast<const S*>(p.down) + static_cast<size_t>(min(row0 + g, p.o - 1)) * p.F;
  const S* hi = static_cast<const S*>(p.down) + static_cast<size_t>(min(row0 + g + 8, p.o - 1)) * p.F;
  // the first weights, before h is there: the launch in front of this one has let it start after everything in front of itself was done
  Ahead<S> ahead;
#pragma unroll
  for (int i = 0; i < kDeep; ++i) ask(ahead, i, lo, hi, s0 + i, s1, p.F);
  grid_dep_wait();
  grid_dep_release();
  float sum[NT][4] = {};
  run<S, float, C, float, Parts<C>::kCount, Parts<C>::kHidden, NT>(sum, ahead, lo, hi, p.h, p.n, s0, s1, p.F);
  leave<NT>(sums, sum);
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * p.n; i += 32 * kDownWarps) {
    const int token = i / kRows, r = i % kRows;
    if (row0 + r >= p.o) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += sums[(w * 8 * NT + token) * kPitch + r];
    const size_t at = static_cast<size_t>(token) * p.o + row0 + r;
    if (p.out_dtype == NLFA_DTYPE_F32) static_cast<float*>(p.y)[at] = v;
    else if (p.out_dtype == NLFA_DTYPE_F16) static_cast<__half*>(p.y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  }
}

template <typename S, typename C, int NT>
int launch_few(FewParams p, cudaStream_t st) {
  const bool overlap = overlap_launches(kOverlapRowwise);
  p.turns = (p.n + 8 * NT - 1) / (8 * NT);
  auto tiles = [&](int rows) { return dim3(static_cast<unsigned>((rows + kRows - 1) / kRows * p.turns)); };
  cudaError_t e = launch_kernel(few_up_kernel<S, C, NT>, tiles(p.F), dim3(32 * kUpWarps), 0, st, overlap, p);
  if (e == cudaSuccess)
    e = launch_kernel(few_down_kernel<S, C, NT>, tiles(p.o), dim3(32 * kDownWarps), 0, st, overlap, p);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}
template <typename S, typename C>
int launch_tokens(const FewParams& p, cudaStream_t st) {
  if (p.n <= 8) return launch_few<S, C, 1>(p, st);
  // (bf16, 768 x 2,048: two turns of 16 for 32 tokens 8.3 us, one of 32 10.9; two of 32 for 64 11.1, four of 16 15.2)
  return p.n <= 32 ? launch_few<S, C, 2>(p, st) : launch_few<S, C, 4>(p, st);
}

}  // namespace

// (weights and products of one type, or float32 weights that are rounded to it)
bool few_types(int w_dtype, int dtype) { return w_dtype == dtype || w_dtype == NLFA_DTYPE_F32; }

int launch_few_tokens(const void* x, int x_dtype, const void* gate, const void* up, const void* down, int w_dtype, int dtype, int activation, int n,
                      int d, int F, int o, float* h, void* y, cudaStream_t st) {
  const FewParams p{x, gate, up, down, h, y, n, d, F, o, x_dtype, activation, dtype, 1};
  if (dtype == NLFA_DTYPE_F32) return launch_tokens<float, float>(p, st);
  if (dtype == NLFA_DTYPE_F16) return w_dtype == dtype ? launch_tokens<__half, __half>(p, st) : launch_tokens<float, __half>(p, st);
  return w_dtype == dtype ? launch_tokens<__nv_bfloat16, __nv_bfloat16>(p, st) : launch_tokens<float, __nv_bfloat16>(p, st);
}

}  // namespace ffn
}  // namespace nlfa
