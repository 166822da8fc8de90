// Token embedding: out_i = s w[id_i], and the table's gradient dw_v = s sum_{i: id_i = v} g_i.
//
// Both directions move rows and are bound by HBM.  The gradient adds the rows of a token in the order of their positions, so
// that the same call gives the same bits: the ids are sorted first (sort_ids_kernel: one cluster, a stable radix sort whose
// digit counts cross between its CTAs through distributed shared memory: no launch per pass and no waiting on flags),
// then warps add runs of sorted positions (add_rows_kernel).  A token's rows that cross from one run into the next are added from the
// runs' partial sums afterwards (join_rows_kernel), in order.  The rows of tokens that do not occur have been zeroed beside the sort.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"
#include "rowwise.cuh"

namespace nlfa {
namespace embedding {
namespace {

constexpr int kBlock = 256, kWarps = kBlock / 32;
constexpr int kSortThreads = 1024;
constexpr int kMostDigitBits = 9;

// W bytes of a row: 16, 8, 4 or 2, what its alignment allows
template <int W> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T as_type(float x);
template <> __device__ __forceinline__ float as_type<float>(float x) { return x; }
template <> __device__ __forceinline__ __half as_type<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int W>
struct Vec {
  static constexpr int N = W / static_cast<int>(sizeof(T));
  union {
    typename Word<W>::type w;
    T e[N];
  };
  __device__ Vec() {}
};

// A thread moves words of a row; `per_row` words of W bytes, four of them in flight.
template <typename T, int W, typename I>
__global__ void __launch_bounds__(kBlock)
lookup_kernel(const I* __restrict__ ids, const T* __restrict__ w, T* __restrict__ out, int n, int V, int per_row, FastDiv div, float scale) {
  using Word_ = typename Word<W>::type;
  using V_ = Vec<T, W>;
  constexpr int U = 4;
  grid_dep_wait();
  grid_dep_release();
  // (per CTA a run of words that fits 31 bits, wherever it starts)
  const long long total = static_cast<long long>(n) * per_row;
  const long long first = static_cast<long long>(blockIdx.x) * (kBlock * U);
  const int row0 = static_cast<int>(first / per_row), col0 = static_cast<int>(first - static_cast<long long>(row0) * per_row);
  V_ v[U];
  long long at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * kBlock + threadIdx.x;
    at[u] = first + i;
    if (at[u] >= total) continue;
    const int step = div.div(col0 + i), row = row0 + step, col = col0 + i - step * per_row;
    const long long id = static_cast<long long>(ids[row]);
    if (id >= 0 && id < V) v[u].w = reinterpret_cast<const Word_*>(w)[id * per_row + col];
    else {
#pragma unroll
      for (int e = 0; e < V_::N; ++e) v[u].e[e] = as_type<T>(__int_as_float(0x7fffffff));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] >= total) continue;
    if (scale != 1.f) {
#pragma unroll
      for (int e = 0; e < V_::N; ++e) v[u].e[e] = as_type<T>(as_float(v[u].e[e]) * scale);
    }
    reinterpret_cast<Word_*>(out)[at[u]] = v[u].w;
  }
}

// ------------------------------------------------------------------------------------------------ sort

// (id, position) by id, positions in order; ids without a gradient (outside the table, padding) become V and end up last.
// begin[v], end[v]: where v's positions lie; begin = -1 where there are none.  The first cluster of
// the grid: each of its CTAs has a run of the positions, each warp of it a run of that.  The other clusters write zeros over dw
// meanwhile (it is the larger part of the memory traffic where the table is; the sort is all latency).
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
sort_ids_kernel(const I* __restrict__ ids, int n, int V, long long padding, uint2* pairs, int* __restrict__ begin,
                int* __restrict__ end, int passes, int digit_bits, int ctas, uint8_t* __restrict__ dw, long long dw_bytes) {
  extern __shared__ int smem[];
  constexpr int U = 8;
  const int digits = 1 << digit_bits;
  int* count = smem;                                   // [warp][digit]
  int* total = smem + (blockDim.x / 32) * digits;             // [digit], read by the other CTAs
  int* base = total + digits;
  __shared__ int warp_sum[32];
  grid_dep_wait();
  grid_dep_release();
  const int rank = static_cast<int>(cluster_rank()), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int threads = blockDim.x, warps = threads / 32;
  if (blockIdx.x > 0) {
    const long long i0 = ((static_cast<long long>(blockIdx.x) - 1) * ctas + rank) * threads + threadIdx.x;
    const long long step = static_cast<long long>(gridDim.x - 1) * ctas * threads;
    const int head = static_cast<int>(-reinterpret_cast<uintptr_t>(dw) & 15u);             // to a 16-byte border, in whole elements
    const long long body = dw_bytes > head ? (dw_bytes - head) / 16 : 0, tail = dw_bytes > head ? head + 16 * body : 0;
    uint4* words = reinterpret_cast<uint4*>(dw + head);
#pragma unroll 8
    for (long long i = i0; i < body; i += step) words[i] = make_uint4(0u, 0u, 0u, 0u);
    for (long long b = 2 * i0; b < 16 && b < dw_bytes; b += 2 * step) {
      if (b < head || tail == 0) *reinterpret_cast<uint16_t*>(dw + b) = 0;
      if (tail + b < dw_bytes) *reinterpret_cast<uint16_t*>(dw + tail + b) = 0;
    }
    return;
  }
  const unsigned below = (1u << lane) - 1u;
  const int per_round = ctas * threads;
  const int run = static_cast<int>((static_cast<long long>(n) + per_round - 1) / per_round) * 32;
  const long long lo = static_cast<long long>(run) * (rank * warps + warp);
  const int from = lo < n ? static_cast<int>(lo) : n, to = n - from < run ? n : from + run;

  for (int v = rank * threads + threadIdx.x; v < V; v += per_round) begin[v] = -1;

  uint2 *src = pairs, *dst = pairs + n;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    // the keys of U x 32 positions; behind the run: no digit
    auto load_keys = [&](int i0, uint32_t (&k)[U]) {
      if (pass > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = i0 + 32 * u + lane < to ? __ldcg(&src[i0 + 32 * u + lane].x) : 0xffffffffu;
      } else {
        long long id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = i0 + 32 * u + lane < to ? static_cast<long long>(ids[i0 + 32 * u + lane]) : 0ll;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t key = id[u] >= 0 && id[u] < V && id[u] != padding ? static_cast<uint32_t>(id[u]) : static_cast<uint32_t>(V);
          k[u] = i0 + 32 * u + lane < to ? key : 0xffffffffu;
        }
      }
    };
    auto digit_of = [&](uint32_t key) { return key == 0xffffffffu ? key : (key >> shift) & (digits - 1); };
    // the lanes with this lane's digit, bit by bit (with match.any in its place the sort of 131,072 ids took 46.7 us, so 40)
    auto same_digit = [&](uint32_t d) {
      const unsigned valid = __ballot_sync(0xffffffffu, d != 0xffffffffu);
      unsigned same = d != 0xffffffffu ? valid : ~valid;
      for (int b = 0; b < digit_bits; ++b) {
        const bool bit = d >> b & 1u;
        const unsigned set = __ballot_sync(0xffffffffu, bit);
        same &= bit ? set : ~set;
      }
      return same;
    };
    for (int i = threadIdx.x; i < warps * digits; i += threads) count[i] = 0;
    __syncthreads();
    int* mine = count + warp * digits;
    for (int i0 = from; i0 < to; i0 += 32 * U) {
      uint32_t k[U];
      load_keys(i0, k);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + 32 * u >= to) break;
        const uint32_t d = digit_of(k[u]);
        const unsigned same = same_digit(d);
        if (d != 0xffffffffu && (same & below) == 0) mine[d] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += threads) {
      int sum = 0;
#pragma unroll 8
      for (int w = 0; w < warps; ++w) {
        const int c = count[w * digits + d];
        count[w * digits + d] = sum;
        sum += c;
      }
      total[d] = sum;
    }
    cluster_arrive();
    cluster_wait();
    int carry = 0;                                       // positions of the digits below d0
    for (int d0 = 0; d0 < digits; d0 += threads) {
      const int d = d0 + threadIdx.x;
      int before = 0, all = 0;
      if (d < digits) {
#pragma unroll 8
        for (int r = 0; r < ctas; ++r) {
          int v;
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(smem_u32(total + d), r)) : "memory");
          if (r < rank) before += v;
          all += v;
        }
      }
      int inclusive = all;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inclusive, off);
        if (lane >= off) inclusive += o;
      }
      if (lane == 31) warp_sum[warp] = inclusive;
      __syncthreads();
      int ahead = 0, sum = 0;
      for (int w = 0; w < warps; ++w) {
        const int v = warp_sum[w];
        if (w < warp) ahead += v;
        sum += v;
      }
      if (d < digits) base[d] = carry + ahead + inclusive - all + before;
      carry += sum;
      __syncthreads();
    }
    for (int i0 = from; i0 < to; i0 += 32 * U) {
      uint32_t k[U], at[U];
      load_keys(i0, k);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + 32 * u + lane;
        at[u] = pass > 0 ? (i < to ? __ldcg(&src[i].y) : 0u) : static_cast<uint32_t>(i);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + 32 * u >= to) break;
        const uint32_t d = digit_of(k[u]);
        const unsigned same = same_digit(d);
        const bool in = d != 0xffffffffu;
        int to_place = 0;
        if (in) to_place = base[d] + mine[d] + __popc(same & below);
        __syncwarp();
        if (in && (same & below) == 0) mine[d] += __popc(same);
        __syncwarp();
        if (in) dst[to_place] = make_uint2(k[u], at[u]);      // (one store: the scattered sectors are what this loop waits for)
      }
    }
    // the next pass reads what the other CTAs wrote, and overwrites what they read
    cluster_arrive();
    cluster_wait();
    uint2* t = src;
    src = dst;
    dst = t;
  }
#pragma unroll 4
  for (int i = from + lane; i < to; i += 32) {
    const uint32_t key = __ldcg(&src[i].x), prev = i > 0 ? __ldcg(&src[i - 1].x) : 0xffffffffu, next = i + 1 < n ? __ldcg(&src[i + 1].x) : 0xffffffffu;
    if (key >= static_cast<uint32_t>(V)) continue;
    if (prev != key) begin[key] = i;
    if (next != key) end[key] = i + 1;
  }
}

// ------------------------------------------------------------------------------------------------ sums

template <typename T, int W>
struct Row {
  using V = Vec<T, W>;
  static constexpr int N = V::N;
  // scaled and rounded once
  static __device__ __forceinline__ void store(T* p, const float (&s)[N], float scale) {
    V v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.e[e] = as_type<T>(s[e] * scale);
    *reinterpret_cast<typename Word<W>::type*>(p) = v.w;
  }
};

// A warp adds a run of `run` sorted positions, a slab of 32 words of each row.  partial [runs][2][d]: what a run has of a token that
// began in an earlier run, and of one that goes on in the next.  Where tokens end is found for 32 positions at once, so that a row costs its
// load and its additions (131,072 rows of 1,024 in bf16: 78 us, 4.5 TB/s; 86 with both tokens compared at each row, 91 with the next rows requested before
// these are added, which takes the registers of a CTA).
template <typename T, int W>
__global__ void __launch_bounds__(kBlock)
add_rows_kernel(const T* __restrict__ g, const uint2* __restrict__ pairs, T* __restrict__ dw,
                float* __restrict__ partial, int n, int V, int d, int run, int runs, int slabs, float scale) {
  using R = Row<T, W>;
  constexpr int N = R::N, U = 8;
  grid_dep_wait();
  grid_dep_release();
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (unit >= static_cast<long long>(runs) * slabs) return;
  const int c = static_cast<int>(unit / slabs), slab = static_cast<int>(unit - static_cast<long long>(c) * slabs);
  const int col = (slab * 32 + lane) * N;
  const bool in = col < d;
  const int from = c * run, to = n - from < run ? n : from + run;
  const uint32_t before = from > 0 ? pairs[from - 1].x : 0xffffffffu, after = to < n ? pairs[to].x : 0xffffffffu;
  const T* rows = g + (in ? col : 0);
  float sum[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = 0.f;
  bool first = true;                                       // the token at hand is the run's first
  for (int i0 = from; i0 < to; i0 += 32) {
    const int i = i0 + lane;
    const uint2 at = i < to ? pairs[i] : make_uint2(0xffffffffu, 0u);
    const uint32_t key = at.x, place = at.y;
    const uint32_t next = i + 1 < to ? pairs[i + 1].x : 0xffffffffu;         // (behind the run: another)
    const int live = __popc(__ballot_sync(0xffffffffu, key < static_cast<uint32_t>(V)));   // (those without a gradient stand last)
    const unsigned ends = __ballot_sync(0xffffffffu, next != key);
    for (int j0 = 0; j0 < live; j0 += U) {
      typename R::V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t p = __shfl_sync(0xffffffffu, place, (j0 + u) & 31);
        if (j0 + u < live) v[u].w = *reinterpret_cast<const typename Word<W>::type*>(rows + static_cast<size_t>(p) * d);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u;
        if (j >= live) break;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += as_float(v[u].e[e]);
        if (!(ends >> j & 1u)) continue;
        const uint32_t k = __shfl_sync(0xffffffffu, key, j);
        const bool came = first && k == before, goes = i0 + j + 1 == to && k == after;
        if (in) {
          if (came || goes) {
            float* o = partial + (static_cast<size_t>(2 * c) + (came ? 0 : 1)) * d + col;
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = sum[e];
          } else {
            R::store(dw + static_cast<size_t>(k) * d + col, sum, scale);
          }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.f;
        first = false;
      }
    }
    if (live < 32) break;
  }
}

// Tokens that begin in run c and go on: their shares of run c and of those behind, in order.  A warp per run; where there are many
// shares the CTA's warps take an eighth each.
template <typename T, int W>
__global__ void __launch_bounds__(kBlock)
join_rows_kernel(const uint2* __restrict__ pairs, const int* __restrict__ begin, const int* __restrict__ end, const float* __restrict__ partial,
                 T* __restrict__ dw, int n, int V, int d, int run, int runs, float scale) {
  using R = Row<T, W>;
  constexpr int N = R::N, kAlone = 8;
  __shared__ float shares[kWarps][32 * N];
  __shared__ int long_last[kWarps];
  grid_dep_wait();
  grid_dep_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (runs + kWarps - 1) / kWarps, slab = static_cast<int>(blockIdx.x) / groups, group = static_cast<int>(blockIdx.x) - slab * groups;
  const int col = (slab * 32 + lane) * N;
  const bool in = col < d;
  const int c = group * kWarps + warp;
  uint32_t key = 0xffffffffu;
  int last = 0;                                            // the last run with a share
  if (c + 1 < runs) {
    key = pairs[(c + 1) * run - 1].x;
    if (key >= static_cast<uint32_t>(V) || pairs[(c + 1) * run].x != key || begin[key] < c * run) key = 0xffffffffu;
    else last = (end[key] - 1) / run;
  }
  auto share = [&](int r, int which, float (&s)[N]) {
    const float* o = partial + (static_cast<size_t>(2 * r) + which) * d + col;
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += o[e];
  };
  const bool alone = key != 0xffffffffu && last - c <= kAlone;
  if (alone && in) {
    float s[N];
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] = 0.f;
    share(c, 1, s);
#pragma unroll 8
    for (int r = c + 1; r <= last; ++r) share(r, 0, s);
    R::store(dw + static_cast<size_t>(key) * d + col, s, scale);
  }
  if (lane == 0) long_last[warp] = key != 0xffffffffu && !alone ? last : -1;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    const int l = long_last[w];
    if (l < 0) continue;
    const int c0 = group * kWarps + w, many = l - c0;                     // shares of runs c0 + 1 .. l
    const int lo = c0 + 1 + static_cast<int>(static_cast<long long>(many) * warp / kWarps);
    const int hi = c0 + 1 + static_cast<int>(static_cast<long long>(many) * (warp + 1) / kWarps);
    float s[N];
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] = 0.f;
    if (in) {
      if (warp == 0) share(c0, 1, s);
#pragma unroll 8
      for (int r = lo; r < hi; ++r) share(r, 0, s);
#pragma unroll
      for (int e = 0; e < N; ++e) shares[warp][lane * N + e] = s[e];
    }
    __syncthreads();
    if (warp == w && in) {
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = 0.f;
      for (int x = 0; x < kWarps; ++x)
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += shares[x][lane * N + e];
      R::store(dw + static_cast<size_t>(key) * d + col, s, scale);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ host

size_t up(size_t v) { return (v + 255) / 256 * 256; }

int checked(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

int check(int n, int V, int d, int dtype) {
  if (n < 0 || V < 1 || d < 1 || n > (1 << 30) || V > (1 << 30) || d > (1 << 24)) return NLFA_ERR_BAD_SHAPE;
  return rowwise::dtype_ok(dtype) ? NLFA_OK : NLFA_ERR_BAD_DTYPE;
}

int element_bytes(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }

// Widest word that divides a row and both bases.
int word_bytes(long long row_bytes, const void* a, const void* b) {
  const unsigned long long all = static_cast<unsigned long long>(row_bytes) | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// Sorted positions per warp: enough warps for the GPU (148 SMs as a constant: the runs decide the order of additions and the size of the
// scratch, so neither depends on the device that is asked), and few partial sums when there are many positions.
int run_length(int n, int d) {
  const long long warps = 64ll * 148, slabs = (d + 127) / 128;
  int run = 16;
  while (run < 128 && n * slabs / (2 * run) >= warps) run *= 2;
  return run;
}

struct Scratch {
  size_t pairs, begin, end, partial, bytes;
};
Scratch scratch_layout(int n, int V, int d) {
  Scratch s{};
  size_t at = 0;
  s.pairs = at; at = up(at + static_cast<size_t>(n) * 16);         // two of (id, position), from one pass to the next
  s.begin = at; at = up(at + static_cast<size_t>(V) * 4);
  s.end = at; at = up(at + static_cast<size_t>(V) * 4);
  s.partial = at; at = up(at + (static_cast<size_t>(n) / run_length(n, d) + 1) * 2 * d * 4);
  s.bytes = at;
  return s;
}

template <typename T, int W, typename I>
int lookup(const void* ids, const void* w, void* out, int n, int V, int d, float scale, cudaStream_t st) {
  const int per_row = d / Vec<T, W>::N;
  const long long ctas = (static_cast<long long>(n) * per_row + 4 * kBlock - 1) / (4 * kBlock);
  if (ctas > 0x7fffffffll) return NLFA_ERR_BAD_SHAPE;
  return checked(launch_kernel(lookup_kernel<T, W, I>, dim3(static_cast<unsigned>(ctas)), dim3(kBlock), 0, st, overlap_launches(kOverlapRowwise),
                               static_cast<const I*>(ids), static_cast<const T*>(w), static_cast<T*>(out), n, V, per_row,
                               FastDiv(per_row), scale));
}

template <typename T, int W>
int gradient(const void* g, const Scratch& s, uint8_t* scratch, int sorted, void* dw, int n, int V, int d, float scale, cudaStream_t st) {
  const int slabs = (d / Vec<T, W>::N + 31) / 32, run = run_length(n, d), runs = (n + run - 1) / run;
  const uint2* pairs = reinterpret_cast<const uint2*>(scratch + s.pairs) + static_cast<size_t>(sorted) * n;
  const int *begin = reinterpret_cast<const int*>(scratch + s.begin), *end = reinterpret_cast<const int*>(scratch + s.end);
  float* partial = reinterpret_cast<float*>(scratch + s.partial);
  const bool overlap = overlap_launches(kOverlapRowwise);
  const long long units = static_cast<long long>(runs) * slabs, ctas = (units + kWarps - 1) / kWarps;
  const long long join = static_cast<long long>((runs + kWarps - 1) / kWarps) * slabs;
  if (join > 0x7fffffffll) return NLFA_ERR_BAD_SHAPE;      // (no fewer than `ctas`)
  if (n == 0) return NLFA_OK;                              // (the zeros are written)
  int rc = checked(launch_kernel(add_rows_kernel<T, W>, dim3(static_cast<unsigned>(ctas)), dim3(kBlock), 0, st, overlap, static_cast<const T*>(g),
                                 pairs, static_cast<T*>(dw), partial, n, V, d, run, runs, slabs, scale));
  if (rc != NLFA_OK || runs < 2) return rc;
  return checked(launch_kernel(join_rows_kernel<T, W>, dim3(static_cast<unsigned>(join)), dim3(kBlock), 0, st, overlap, pairs, begin, end, partial,
                               static_cast<T*>(dw), n, V, d, run, runs, scale));
}

}  // namespace
}  // namespace embedding
}  // namespace nlfa

using namespace nlfa;
using namespace nlfa::embedding;

extern "C" {

int nlfa_embedding_fwd(const void* ids, int id_bytes, const void* w, int dtype, void* out, int n, int V, int d, float scale, void* stream) {
  const int rc = check(n, V, d, dtype);
  if (rc != NLFA_OK) return rc;
  if (id_bytes != 4 && id_bytes != 8) return NLFA_ERR_BAD_ARGUMENT;
  if (n == 0) return NLFA_OK;
  if (!ids || !w || !out) return NLFA_ERR_NULL_POINTER;
  const int bytes = element_bytes(dtype);
  if ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) % bytes != 0 || reinterpret_cast<uintptr_t>(ids) % id_bytes != 0)
    return NLFA_ERR_MISALIGNED;
  const int word = word_bytes(static_cast<long long>(d) * bytes, w, out);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define NLFA_GO(T, W) (id_bytes == 8 ? lookup<T, W, long long>(ids, w, out, n, V, d, scale, st) : lookup<T, W, int>(ids, w, out, n, V, d, scale, st))
#define NLFA_16(T) (word == 16 ? NLFA_GO(T, 16) : word == 8 ? NLFA_GO(T, 8) : word == 4 ? NLFA_GO(T, 4) : NLFA_GO(T, 2))
  if (dtype == NLFA_DTYPE_F32) return word == 16 ? NLFA_GO(float, 16) : word == 8 ? NLFA_GO(float, 8) : NLFA_GO(float, 4);
  return dtype == NLFA_DTYPE_F16 ? NLFA_16(__half) : NLFA_16(__nv_bfloat16);
#undef NLFA_16
#undef NLFA_GO
}

size_t nlfa_embedding_scratch_bytes(int n, int V, int d) {
  return check(n, V, d, NLFA_DTYPE_F32) == NLFA_OK ? scratch_layout(n, V, d).bytes : 0;
}

int nlfa_embedding_bwd(const void* g, int dtype, const void* ids, int id_bytes, void* dw, int n, int V, int d, float scale,
                       long long padding_idx, void* scratch, size_t scratch_bytes, void* stream) {
  int rc = check(n, V, d, dtype);
  if (rc != NLFA_OK) return rc;
  if (id_bytes != 4 && id_bytes != 8) return NLFA_ERR_BAD_ARGUMENT;
  if (!dw || !scratch || (n > 0 && (!g || !ids))) return NLFA_ERR_NULL_POINTER;
  if (!rowwise::aligned16(scratch)) return NLFA_ERR_MISALIGNED;
  const int bytes = element_bytes(dtype);
  if ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(dw)) % bytes != 0 || reinterpret_cast<uintptr_t>(ids) % id_bytes != 0)
    return NLFA_ERR_MISALIGNED;
  const Scratch s = scratch_layout(n, V, d);
  if (scratch_bytes < s.bytes) return NLFA_ERR_SCRATCH_TOO_SMALL;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  // digits of equal width that cover 0 .. V
  int bits = 1;
  while (bits < 31 && (static_cast<unsigned>(V) >> bits) != 0) ++bits;
  const int passes = (bits + kMostDigitBits - 1) / kMostDigitBits, digit_bits = (bits + passes - 1) / passes;
  // few positions: fewer warps, whose counts are added one after the other
  const int threads = n <= 32768 ? 256 : kSortThreads;
  const size_t smem = static_cast<size_t>(threads / 32 + 2) * (1u << digit_bits) * sizeof(int);
  auto sort = [&](auto* typed, auto* kernel) {
    const int r = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), (kSortThreads / 32 + 2) * (1 << kMostDigitBits) * static_cast<int>(sizeof(int)));
    if (r != NLFA_OK) return r;
    const int ctas = resident_clusters(reinterpret_cast<const void*>(kernel), kSortThreads, (kSortThreads / 32 + 2) * (1 << kMostDigitBits) * 4, 16) > 0 ? 16 : 8;
    const long long dw_bytes = static_cast<long long>(V) * d * bytes, each = 16ll * threads * ctas * 8;   // (eight words a thread)
    const long long most = 8 * (kSortThreads / threads), want = dw_bytes / each;
    const int clusters = static_cast<int>(want < 1 ? 1 : want > most ? most : want);
    return checked(launch_cluster(kernel, dim3(static_cast<unsigned>(1 + clusters), static_cast<unsigned>(ctas)), dim3(static_cast<unsigned>(threads)), smem, st, overlap_launches(kOverlapRowwise), ctas,
                                  typed, n, V, padding_idx, reinterpret_cast<uint2*>(at + s.pairs),
                                  reinterpret_cast<int*>(at + s.begin), reinterpret_cast<int*>(at + s.end), passes, digit_bits, ctas, static_cast<uint8_t*>(dw), dw_bytes));
  };
  rc = id_bytes == 8 ? sort(static_cast<const long long*>(ids), sort_ids_kernel<long long>) : sort(static_cast<const int*>(ids), sort_ids_kernel<int>);
  if (rc != NLFA_OK) return rc;
  const int word = word_bytes(static_cast<long long>(d) * bytes, g, dw), sorted = passes & 1;
#define NLFA_GO(T, W) gradient<T, W>(g, s, at, sorted, dw, n, V, d, scale, st)
#define NLFA_16(T) (word == 16 ? NLFA_GO(T, 16) : word == 8 ? NLFA_GO(T, 8) : word == 4 ? NLFA_GO(T, 4) : NLFA_GO(T, 2))
  if (dtype == NLFA_DTYPE_F32) return word == 16 ? NLFA_GO(float, 16) : word == 8 ? NLFA_GO(float, 8) : NLFA_GO(float, 4);
  return dtype == NLFA_DTYPE_F16 ? NLFA_16(__half) : NLFA_16(__nv_bfloat16);
#undef NLFA_16
#undef NLFA_GO
}

}  // extern "C"
