// Linear cross entropy: the loss of a language model's head without its logits.
//
//   l_iv = x_i . w_v,  lse_i = log sum_v exp(l_iv),  loss_i = lse_i - l_i,t(i)
//   dl_iv = g_i (exp(l_iv - lse_i) - [v == t(i)]),  dx = dl W,  dW = dl^T x
//
// The logits of N = 65,536 tokens over 50,304 words are 13 GB in float32.  The forward (loss_tc.cu) keeps each row's maximum
// and sum; the backward goes through the vocabulary in pieces, forms dl of a piece in a workspace and multiplies it
// both ways: four products of 2 N V d operations in all.  This file has what goes before and after: the rows that have a
// target, packed (rows without one cost nothing and reach nothing, whatever they hold); 16-bit copies of operands that the products
// cannot read as they are (float32: sums of three bf16 parts, exact to 2^-24); the sum of the losses.
#include <climits>
#include <cmath>
#include <type_traits>

#include "loss.cuh"
#include "rowwise.cuh"

namespace nlfa {

unsigned* status_block();      // api.cu

namespace loss {
namespace {

using rowwise::aligned16;
using rowwise::dtype_ok;
using rowwise::last_cta;

constexpr int kScanCtas = 8, kScanThreads = 1024;
constexpr int kBlock = 256;

// ------------------------------------------------------------------------------------------------ 16-bit operands

template <typename T> __device__ __forceinline__ float load1(const T* p) { return static_cast<float>(*p); }

// Eight columns (from c) of row `from` of src [*, d] (-1: zeros) to row r of dst [planes][d_pad / 64][n_rows][64]; planes = 3: dst = a + b + c,
// each the nearest bf16 value to what is left (of infinity: NaN; and its products with the other operand's small parts would be NaN whatever was left).
template <typename S, typename T>
__device__ __forceinline__ void copy_chunk(const S* __restrict__ src, T* __restrict__ dst, int from, int r, int c, int n_rows, int d, int d_pad,
                                           int planes, int vec) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if (from >= 0 && c < d) {
    const S* s = src + static_cast<size_t>(from) * d + c;
    if (vec) rowwise::Elem<S>::load(s, v);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < d) v[j] = load1(s + j);
    }
  }
  T* o = dst + (static_cast<size_t>(c / 64) * n_rows + r) * 64 + c % 64;
  for (int part = 0; part < planes; ++part) {
    rowwise::Elem<T>::store(o, v);
    o += static_cast<size_t>(n_rows) * d_pad;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] -= rowwise::Elem<T>::round(v[j]);
  }
}

// Rows from row_of (or r itself), zeros behind the last one up to a whole tile and behind column d.
template <typename S, typename T>
__global__ void __launch_bounds__(kBlock)
copy_rows_kernel(const S* __restrict__ src, T* __restrict__ dst, const Head* head, const int* __restrict__ row_of, int n_src,
                 int n_rows, int d, int d_pad, int planes, int vec) {
  grid_dep_wait();
  grid_dep_release();
  int end = n_src;
  if (row_of != nullptr) {
    const int all = head->count;
    end = all < kRowTile ? kRowTile : (all + kRowTile - 1) / kRowTile * kRowTile;
  }
  const int chunks = d_pad / 8;
  const long long total = static_cast<long long>(end) * chunks;
  for (long long i = static_cast<long long>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kBlock) {
    const int r = static_cast<int>(i / chunks), c = 8 * static_cast<int>(i - static_cast<long long>(r) * chunks);
    copy_chunk(src, dst, row_of != nullptr ? row_of[r] : r, r, c, n_rows, d, d_pad, planes, vec);
  }
}

// ------------------------------------------------------------------------------------------------ rows with a target

template <typename I>
__device__ __forceinline__ bool counts(I t, long long ignore) { return static_cast<long long>(t) != ignore; }

// One cluster: each CTA takes a run of the rows, counts those that have a target, learns the counts in front of its own from
// the others, and writes its rows' numbers in order.  Rows behind the last one, up to a whole tile, are set empty.
template <typename I>
__global__ void __launch_bounds__(kScanThreads)
pack_rows_kernel(const I* __restrict__ targets, int n, int n_rows, int V, long long ignore, Head* head, int* __restrict__ row_of,
                 int* __restrict__ target, float* __restrict__ at_target, float* __restrict__ each, int col_tiles, int pairs,
                 int max_splits) {
  __shared__ int warp_count[32];
  __shared__ int total;
  grid_dep_wait();
  grid_dep_release();
  const int rank = static_cast<int>(cluster_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int run = ((n + kScanCtas - 1) / kScanCtas + kScanThreads - 1) / kScanThreads * kScanThreads;
  const long long lo = static_cast<long long>(run) * rank;
  const int from = lo < n ? static_cast<int>(lo) : n, to = n - from < run ? n : from + run;

  int mine = 0;
  for (int i = from + threadIdx.x; i < to; i += kScanThreads) mine += counts(targets[i], ignore) ? 1 : 0;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
  if (lane == 0) warp_count[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    int v = warp_count[lane];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if (lane == 0) total = v;
  }
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  int at = 0, all = 0;
  for (int r = 0; r < kScanCtas; ++r) {
    int v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(smem_u32(&total), r)) : "memory");
    if (r < rank) at += v;
    all += v;
  }
  cluster_arrive();                        // (the others' shared memory is no longer read)

  for (int i0 = from; i0 < to; i0 += kScanThreads) {
    const int i = i0 + threadIdx.x;
    const bool in = i < to;
    const long long t = in ? static_cast<long long>(targets[i]) : 0;
    const bool has = in && counts(t, ignore);
    const unsigned b = __ballot_sync(0xffffffffu, has);
    __syncthreads();
    if (lane == 0) warp_count[warp] = __popc(b);
    __syncthreads();
    int before = 0, sum = 0;
    for (int w = 0; w < 32; ++w) {
      const int c = warp_count[w];
      if (w < warp) before += c;
      sum += c;
    }
    if (has) {
      const int r = at + before + __popc(b & ((1u << lane) - 1u));
      row_of[r] = i;
      // a target outside the vocabulary: its logit stays NaN, and so do its loss and its gradients (-2: see scale_rows)
      target[r] = t >= 0 && t < V ? static_cast<int>(t) : -2;
      at_target[r] = __int_as_float(0x7fffffff);
    } else if (in && each != nullptr) {
      each[i] = 0.f;
    }
    at += sum;
  }
  // rows up to the end of the last tile
  const int end = all < kRowTile ? kRowTile : (all + kRowTile - 1) / kRowTile * kRowTile;
  for (int r = all + rank * kScanThreads + threadIdx.x; r < end; r += kScanCtas * kScanThreads) {
    row_of[r] = -1;
    target[r] = -1;
    at_target[r] = 0.f;
  }
  if (rank == 0 && warp == 0) {
    // Parts of the vocabulary per row tile, so that the pairs of CTAs end together: the fewest column tiles for the busiest
    // pair, counted with one more per unit for its start; of equals the fewest parts.
    const int row_tiles = end / kRowTile;
    long long best = LLONG_MAX;
    for (int s = 1 + lane; s <= max_splits; s += 32) {
      const long long units = (static_cast<long long>(row_tiles) * s + pairs - 1) / pairs;
      const long long cost = units * ((col_tiles + s - 1) / s) * 4 + units;
      if (cost < (best >> 12)) best = (cost << 12) | s;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const long long o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o < best ? o : best;
    }
    if (lane == 0) {
      head->count = all;
      head->splits = static_cast<int>(best & 4095);
    }
  }
  cluster_wait();
}

// Up to kFewRows rows, packed and copied in one launch: every CTA finds the rows for itself and copies its part of the tile.
template <typename I, typename S, typename T>
__global__ void __launch_bounds__(kBlock)
pack_few_kernel(const I* __restrict__ targets, int n, int V, long long ignore, Head* head, int* __restrict__ row_of, int* __restrict__ target,
                float* __restrict__ at_target, float* __restrict__ each, const S* __restrict__ x, T* __restrict__ copy, int n_rows, int d, int d_pad,
                int planes, int vec) {
  __shared__ int source[kFewRows];
  __shared__ unsigned has[kFewRows / 32];
  grid_dep_wait();
  grid_dep_release();
  const int i = threadIdx.x, lane = i & 31;
  const bool in = i < n;
  const long long t = in ? static_cast<long long>(targets[i]) : 0;
  const bool mine = in && counts(t, ignore);
  if (i < kFewRows) {
    const unsigned b = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) has[i / 32] = b;
  }
  __syncthreads();
  int all = 0, r = 0;                      // rows with a target, and those in front of this one
  for (int w = 0; w < kFewRows / 32; ++w) {
    if (w < i / 32) r += __popc(has[w]);
    if (w == i / 32) r += __popc(has[w] & ((1u << lane) - 1u));
    all += __popc(has[w]);
  }
  if (mine) source[r] = i;
  if (blockIdx.x == 0) {
    if (mine) {
      row_of[r] = i;
      target[r] = t >= 0 && t < V ? static_cast<int>(t) : -2;
      at_target[r] = __int_as_float(0x7fffffff);
    } else if (in && each != nullptr) {
      each[i] = 0.f;
    }
    if (i >= all && i < kRowTile) {
      row_of[i] = -1;
      target[i] = -1;
      at_target[i] = 0.f;
    }
    if (i == 0) {
      head->count = all;
      head->splits = 1;
    }
  }
  __syncthreads();
  const int chunks = d_pad / 8;
  for (int c = blockIdx.x * kBlock + i; c < kRowTile * chunks; c += gridDim.x * kBlock) {
    const int row = c / chunks;
    copy_chunk(x, copy, row < all ? source[row] : -1, row, 8 * (c - row * chunks), n_rows, d, d_pad, planes, vec);
  }
}

// ------------------------------------------------------------------------------------------------ losses

// (max, sum) of a row's parts, the target left out of them, and the target's logit t -> lse, loss, and own = p - 1 of the target.  With
// e = sum_{v != t} exp(l_v - t):  lse = t + log(1 + e),  loss = log(1 + e),  own = -e / (1 + e).  (A sum that held the target's own 1 would keep
// of e what 2^-24 leaves: at e = 1e-7 own would be off by a fifth, and at 5e-8 nothing would be left of it.)  Rows behind the last one get
// lse = +inf: their probabilities are zero.  `lanes` threads per row (a power of two up to 32): few rows have many parts.
__global__ void __launch_bounds__(kBlock)
finish_kernel(const Head* head, const float2* __restrict__ partial, const float* __restrict__ at_target, const int* __restrict__ row_of,
              int n_rows, float* __restrict__ lse, float* __restrict__ lse_rest, float* __restrict__ own, float* __restrict__ each, float* __restrict__ out, double* sums,
              unsigned* ticket, int mean, int lanes, int few_parts) {
  __shared__ double warp_sum[kBlock / 32];
  __shared__ int last;
  grid_dep_wait();
  grid_dep_release();
  const int all = head->count, parts = few_parts > 0 ? few_parts : 2 * head->splits;
  const int end = all < kRowTile ? kRowTile : (all + kRowTile - 1) / kRowTile * kRowTile;
  const int mine = threadIdx.x & (lanes - 1), rows = kBlock / lanes;
  double sum = 0.0;
  for (int r0 = blockIdx.x * rows; r0 < end; r0 += gridDim.x * rows) {
    const int r = r0 + threadIdx.x / lanes;               // (end is a multiple of rows: whole warps stay together)
    const bool live = r < all;
    float top = -INFINITY;
    if (live) {
#pragma unroll 4
      for (int s = mine; s < parts; s += lanes) top = fmaxf(top, partial[static_cast<size_t>(s) * n_rows + r].x);
    }
    for (int off = lanes / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float shift = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    if (live) {
#pragma unroll 4
      for (int s = mine; s < parts; s += lanes) {
        const float2 q = partial[static_cast<size_t>(s) * n_rows + r];
        total += q.y * expf(q.x - shift);
      }
    }
    for (int off = lanes / 2; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (mine != 0) continue;
    if (!live) {
      lse[r] = INFINITY;
      lse_rest[r] = own[r] = 0.f;
      continue;
    }
    const float t = at_target[r];
    float base = t, rest, loss, p_less_1;
    if (t > top) {
      const float e = total * expf(top - t), bad = t - t;   // (a logit of +inf: NaN, as its softmax is)
      rest = log1pf(e);
      loss = rest + bad;
      p_less_1 = -e / (1.f + e) + bad;
    } else {
      const float with_t = total + expf(t - top);
      base = top;
      rest = logf(with_t);
      loss = (top - t) + rest;
      p_less_1 = -total / with_t;
    }
    const float whole = base + rest;
    lse[r] = whole;
    lse_rest[r] = rest - (whole - base);                   // (NaN where lse is not finite)
    own[r] = p_less_1;
    if (each != nullptr) each[row_of[r]] = loss;
    sum += loss;
  }
  if (out == nullptr) return;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kBlock / 32; ++w) t += warp_sum[w];
    sums[blockIdx.x] = t;
  }
  if (!last_cta(ticket, gridDim.x, &last)) return;
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (unsigned i = 0; i < gridDim.x; ++i) t += __ldcg(sums + i);
    *out = static_cast<float>(mean ? t / all : t);       // (no target at all: 0 / 0)
  }
}

// ------------------------------------------------------------------------------------------------ backward

// The largest finite |grad| (1 if there is none): one CTA.
__global__ void __launch_bounds__(1024)
largest_kernel(const Head* head, const float* __restrict__ grad, const int* __restrict__ row_of, float* __restrict__ largest) {
  __shared__ float warp_top[32];
  grid_dep_wait();
  grid_dep_release();
  float top = 0.f;
#pragma unroll 4
  for (int r = threadIdx.x; r < head->count; r += 1024) {
    const float g = fabsf(grad[row_of[r]]);
    if (g > top && g < INFINITY) top = g;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 32; ++w) top = fmaxf(top, warp_top[w]);
  *largest = top > 0.f ? top : 1.f;
}

// In how many parts the sums of `rest` tiles of k stages are formed, by one warp: the fewest stages for the busiest pair of CTAs, with
// `share` more for every share written and added.  The units are handed out in turn behind `ahead` units of `length` stages.
__device__ int choose_parts(int rest, int k, int pairs, int share, int ahead, int length) {
  const int lane = threadIdx.x & 31, most = rest > 0 ? kPartsPerPair * pairs / rest : 1;
  long long best = LLONG_MAX;
  for (int s = 1 + lane; s <= most && s <= k; s += 32) {
    const int end = ahead + rest * s, mine = (k + s - 1) / s + (s > 1 ? share : 0);
    long long cost = 0;
    for (int i = 0; i < 3; ++i) {                          // the first pair, and the first that gets one unit less of either kind
      const int b = i == 0 ? 0 : (i == 1 ? ahead : end) % pairs;
      const int first = (ahead + pairs - 1 - b) / pairs, both = (end + pairs - 1 - b) / pairs;
      const long long c = static_cast<long long>(first) * length + static_cast<long long>(both - first) * mine;
      cost = c > cost ? c : cost;
    }
    cost += s > 1 ? s : 0;
    if (cost < best >> 8) best = cost << 8 | s;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const long long o = __shfl_xor_sync(0xffffffffu, best, off);
    best = o < best ? o : best;
  }
  return best == LLONG_MAX ? 1 : static_cast<int>(best & 255);
}

// Factors of dl: g_i = alpha row_scale_i.  `grad` is one value, which alpha takes, or one per row of the call (per_row), which row_scale
// takes.  fp16: small probabilities would not be normal numbers, so dl is held times 2^14 (`unit`) over the largest |g| (`largest`).
// Rows of dx that have no target become zeros on the way.
template <typename I>
__global__ void __launch_bounds__(kBlock)
scale_rows_kernel(const Head* head, const float* __restrict__ grad, int per_row, int mean, const int* __restrict__ row_of,
                  const int* __restrict__ target, float* __restrict__ row_scale, float* __restrict__ alpha, Parts* parts, const float* __restrict__ largest,
                  float unit, const I* __restrict__ targets, int n, long long ignore, uint8_t* __restrict__ dx, long long row_bytes, int V,
                  int d, int piece, int want_dw, int pairs, int planes) {
  grid_dep_wait();
  grid_dep_release();
  const int all = head->count, stride = gridDim.x * kBlock;
  const int end = all < kRowTile ? kRowTile : (all + kRowTile - 1) / kRowTile * kRowTile;
  const float top = largest != nullptr ? *largest : 1.f;
  for (int r = blockIdx.x * kBlock + threadIdx.x; r < end; r += stride) {
    float s = 0.f;
    if (r < all) {
      s = per_row ? grad[row_of[r]] / top * unit : unit;
      if (target[r] == -2) s = __int_as_float(0x7fffffff);
    }
    row_scale[r] = s;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const float g = per_row ? top : mean ? *grad / static_cast<float>(all) : *grad;
    *alpha = all > 0 ? g / unit : 0.f;                    // (no target: gradients of zero, not 0 / 0)
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x < 32) {
    const int again = planes == 1 ? dl_parts(planes, per_row, all) : 1;
    const int k = summands(planes), share = planes == 3 ? 1 : 4;          // (a stage of three parts is three times as long)
    const int d_tiles = (d + kColTile - 1) / kColTile, rest_x = dx != nullptr ? end / kRowTile * d_tiles % pairs : 0;
    for (int last = 0; last < 2; ++last) {
      const int cols = last ? V - (V - 1) / piece * piece : piece;
      const int rest_w = want_dw ? (cols + kColTile - 1) / kColTile * d_tiles % pairs : 0;
      const int kw = again * end / k, parts_w = choose_parts(rest_w, kw, pairs, share, 0, 0);
      const int length = (kw + parts_w - 1) / parts_w + (parts_w > 1 ? share : 0);
      const int parts_x = choose_parts(rest_x, again * ((cols + k - 1) / k), pairs, share, rest_w * parts_w, length);
      if (threadIdx.x == 0) {
        parts->dw[last] = parts_w;
        parts->dx[last] = parts_x;
      }
    }
  }
  if (dx == nullptr || all == n) return;
  const int lane = threadIdx.x & 31;
  for (int r = blockIdx.x * (kBlock / 32) + (threadIdx.x >> 5); r < n; r += gridDim.x * (kBlock / 32)) {
    if (counts(targets[r], ignore)) continue;
    uint8_t* o = dx + static_cast<size_t>(r) * row_bytes;
    if ((row_bytes & 15) == 0)
      for (long long i = 16 * lane; i < row_bytes; i += 512) *reinterpret_cast<uint4*>(o + i) = make_uint4(0u, 0u, 0u, 0u);
    else
      for (long long i = 2 * lane; i < row_bytes; i += 64) *reinterpret_cast<uint16_t*>(o + i) = 0;
  }
}

// ------------------------------------------------------------------------------------------------ host

struct Call {
  int x_dtype, w_dtype, dtype;      // dtype: what the products read (NLFA_DTYPE_BF16 for float32: three parts)
  int n, V, d;
};

size_t up(size_t v) { return (v + 255) / 256 * 256; }
int element_bytes(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }
bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_call(const Call& c) {
  if (c.n < 0 || c.V < 1 || c.d < 1 || c.n > (1 << 30) || c.V > (1 << 30) || c.d > (1 << 24)) return NLFA_ERR_BAD_SHAPE;
  if (!dtype_ok(c.x_dtype) || !dtype_ok(c.w_dtype) || !dtype_ok(c.dtype)) return NLFA_ERR_BAD_DTYPE;
  return NLFA_OK;
}

Layout layout(const Call& c, bool w_aligned) {
  Layout l{};
  l.n_rows = c.n < kRowTile ? kRowTile : (c.n + kRowTile - 1) / kRowTile * kRowTile;
  l.d_pad = (c.d + 63) / 64 * 64;
  l.x_planes = c.dtype == NLFA_DTYPE_F32 ? 3 : 1;
  l.copy_w = l.x_planes == 3 || c.w_dtype != c.dtype || c.d % 64 != 0 || !w_aligned;
  size_t at = 256;                                        // the head
  const size_t rows = static_cast<size_t>(l.n_rows) * 4;
  l.row_of = at; at = up(at + rows);
  l.target = at; at = up(at + rows);
  l.lse = at; at = up(at + rows);
  l.lse_rest = at; at = up(at + rows);
  l.own = at; at = up(at + rows);
  l.x = at; at = up(at + static_cast<size_t>(l.x_planes) * l.n_rows * l.d_pad * 2);
  l.w = at; if (l.copy_w) at = up(at + static_cast<size_t>(l.x_planes) * c.V * l.d_pad * 2);
  l.tape_bytes = at;
  // parts of the vocabulary: enough for every pair of CTAs when there is one row tile, few when there are many
  const int col_tiles = (c.V + kColTile - 1) / kColTile, row_tiles = l.n_rows / kRowTile;
  int most = 256 / row_tiles > 8 ? 256 / row_tiles : 8;
  l.max_splits = most < col_tiles ? most : col_tiles;
  l.max_parts = c.n <= kFewRows ? 2 * most_pairs() : 2 * l.max_splits;
  at = 0;
  l.partial = at; at = up(at + static_cast<size_t>(l.max_parts) * l.n_rows * sizeof(float2));
  l.at_target = at; at = up(at + rows);
  l.sums = at; at = up(at + 1024 * sizeof(double));
  l.ticket = at; at = up(at + 4);
  l.fwd_bytes = at;
  return l;
}

// The backward's pieces of the vocabulary: dl of one takes at most this (65,536 x 50,304 x 768: backward 13.7 ms with 512 MiB, 12.4 with
// 1 GiB and with 4: between pieces the GPU runs empty, and dx is summed in memory).
constexpr size_t kMostDl = 1024ull << 20;

struct BwdLayout {
  int piece;                        // columns, a multiple of kColTile
  int dl_rows, dl_second;           // rows of dl's buffer, and where the second part begins if there is one: only the device knows (dl_parts)
  size_t row_scale, alpha, parts, dl, shares, dx_sum, bytes;
};
BwdLayout bwd_layout(const Call& c, const Layout& l) {
  BwdLayout b{};
  b.dl_second = l.n_rows < kTwoParts ? l.n_rows : kTwoParts;
  b.dl_rows = l.x_planes == 3 || l.n_rows > 2 * b.dl_second ? l.n_rows : 2 * b.dl_second;
  const size_t column = static_cast<size_t>(l.x_planes) * b.dl_rows * 2;
  const int col_tiles = (c.V + kColTile - 1) / kColTile;
  size_t most = kMostDl / (column * kColTile);
  if (most < 1) most = 1;
  const int pieces = static_cast<int>((col_tiles + most - 1) / most);
  b.piece = (col_tiles + pieces - 1) / pieces * kColTile;
  size_t at = 0;
  b.row_scale = at; at = up(at + static_cast<size_t>(l.n_rows) * 4);
  b.alpha = at; at = up(at + 8);                          // (and the largest |grad|)
  b.parts = at; at = up(at + sizeof(Parts));
  b.dl = at; at = up(at + column * b.piece);
  b.shares = at; at = up(at + share_bytes());
  b.dx_sum = at; if (pieces > 1) at = up(at + static_cast<size_t>(l.n_rows) * c.d * 4);
  b.bytes = at;
  return b;
}

// What lies in tape and scratch lies in blocks, [planes][blocks of 64 columns][rows][64], so that a box is contiguous; the caller's w is
// [rows][cols].  Either as (64 columns, rows, blocks of 64 columns, planes), cols a multiple of 64.
int box_map(CUtensorMap* map, const void* base, int dtype, long long cols, long long rows, int planes, int box_rows, int box_blocks,
            int box_planes, bool blocked) {
  const unsigned long long pitch = static_cast<unsigned long long>(cols) * 2, r = static_cast<unsigned long long>(rows);
  const unsigned long long dims[4] = {64ull, r, pitch / 128, static_cast<unsigned long long>(planes)};
  const unsigned long long strides[3] = {blocked ? 128ull : pitch, blocked ? 128ull * r : 128ull, pitch * r};
  const unsigned box[4] = {64u, static_cast<unsigned>(box_rows), static_cast<unsigned>(box_blocks), static_cast<unsigned>(box_planes)};
  return make_map(map, base, dtype, dims, strides, box);
}
// One CTA's half of an operand, a stage of it, in all its parts: 128 rows, the summands along the columns ...
int column_map(CUtensorMap* map, const void* base, int dtype, long long cols, long long rows, int planes, bool blocked = true) {
  return box_map(map, base, dtype, cols, rows, planes, 128, summands(planes) / 64, planes == 3 ? 3 : 1, blocked);
}
// ... or 128 columns, the summands along the rows.
int row_map(CUtensorMap* map, const void* base, int dtype, long long cols, long long rows, int planes, bool blocked = true) {
  return box_map(map, base, dtype, cols, rows, planes, summands(planes), 2, planes == 3 ? 3 : 1, blocked);
}

int checked(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

template <typename S, typename T>
int copy_rows_typed(const void* src, void* dst, const Head* head, const int* row_of, int n_src, int n_rows, int d, int d_pad,
                    int planes, cudaStream_t st) {
  const int vec = d % 8 == 0 && aligned16(src) ? 1 : 0;
  const long long work = static_cast<long long>(row_of != nullptr ? n_rows : n_src) * (d_pad / 8);
  const long long most = 16ll * sm_count();
  const long long need = (work + kBlock - 1) / kBlock;
  return checked(launch_kernel(copy_rows_kernel<S, T>, dim3(static_cast<unsigned>(need < most ? need : most)), dim3(kBlock), 0, st,
                               overlap_launches(kOverlapRowwise), static_cast<const S*>(src), static_cast<T*>(dst), head, row_of,
                               n_src, n_rows, d, d_pad, planes, vec));
}
int copy_rows(const void* src, int src_dtype, void* dst, int dtype, const Head* head, const int* row_of, int n_src, int n_rows,
              int d, int d_pad, int planes, cudaStream_t st) {
#define NLFA_TO(S) (dtype == NLFA_DTYPE_F16 ? copy_rows_typed<S, __half>(src, dst, head, row_of, n_src, n_rows, d, d_pad, planes, st) \
                                            : copy_rows_typed<S, __nv_bfloat16>(src, dst, head, row_of, n_src, n_rows, d, d_pad, planes, st))
  if (src_dtype == NLFA_DTYPE_F32) return NLFA_TO(float);
  if (src_dtype == NLFA_DTYPE_F16) return NLFA_TO(__half);
  return NLFA_TO(__nv_bfloat16);
#undef NLFA_TO
}

struct Pointers {
  uint8_t* tape;
  const Layout& l;
  Head* head() const { return reinterpret_cast<Head*>(tape); }
  int* row_of() const { return reinterpret_cast<int*>(tape + l.row_of); }
  int* target() const { return reinterpret_cast<int*>(tape + l.target); }
  float* lse() const { return reinterpret_cast<float*>(tape + l.lse); }
  float* lse_rest() const { return reinterpret_cast<float*>(tape + l.lse_rest); }
  float* own() const { return reinterpret_cast<float*>(tape + l.own); }
};

Params params(const Call& c, const Layout& l, const Pointers& t, unsigned* status) {
  Params p{};
  p.head = t.head();
  p.V = c.V;
  p.d = c.d;
  p.d_pad = l.d_pad;
  p.planes = l.x_planes;
  p.n_rows = l.n_rows;
  p.target = t.target();
  p.lse = t.lse();
  p.lse_rest = t.lse_rest();
  p.own = t.own();
  p.row_of = t.row_of();
  p.status = status;
  return p;
}

// Stages per chain of the tensor core (loss_tc.cu) where logits are formed, in the forward and again in the backward: exp(l - lse) would
// show any difference between the two.  Chains of 64 summands for float32, of 384 for few rows (whose losses are not averaged; 22.5 us
// with one chain, 24.3 so, 25.9 with 256, for 8 rows of 50,304 x 768), else of up to 1,024.
int logit_chain(const Call& c, const Layout& l) {
  return l.x_planes == 3 ? 1 : c.n <= kFewRows ? (c.d > 384 ? 3 : 0) : c.d > 1024 ? 8 : 0;
}
// ... and in the products with dl, whose sums run over rows or words without end.  Where dl is held in one part its roundings leave 2^-8 / sqrt(3)
// (bf16; 2^-11 in fp16) over sqrt(4,096) of a sum of as many values of one sign, 3.5e-5 (4.4e-6): a chain of 4,096 summands, low by 1.1e-5,
// hides under that, in fp16 one of 2,048.  In two parts nothing hides it: 1,024 (loss_tc.cu: Plan).  (65,536 x 50,304 x 768, forward and backward: 16.05 ms with one chain
// however long, 16.25 with 4,096; 16.7 with 2,048; 17.1 with 1,024: adding costs power.
// One chain over a piece of 131,072 words of one sign left dx low by 8.5e-5.)
int product_chain(const Layout& l, int dtype) { return l.x_planes == 3 ? 1 : dtype == NLFA_DTYPE_F16 ? 16 : 32; }

int run_fwd(const Call& c, const void* x, const void* w, const void* targets, int target_bytes, long long ignore, int reduction,
            float* out, uint8_t* tape, uint8_t* scratch, cudaStream_t st) {
  const Layout l = layout(c, aligned16(w));
  const Pointers t{tape, l};
  unsigned* status = status_block();
  if (!status) return NLFA_ERR_CUDA;
  const int dtype = c.dtype == NLFA_DTYPE_F32 ? NLFA_DTYPE_BF16 : c.dtype;
  float* at_target = reinterpret_cast<float*>(scratch + l.at_target);
  float* each = reduction == NLFA_REDUCE_NONE ? out : nullptr;
  const bool overlap = overlap_launches(kOverlapRowwise);
  const int col_tiles = (c.V + kColTile - 1) / kColTile;
  const bool few = c.n <= kFewRows;
  const int vec = c.d % 8 == 0 && aligned16(x) ? 1 : 0;
  auto pack_few = [&](auto* kernel, auto* typed, auto* from, auto* to) {
    const int need = (kRowTile * (l.d_pad / 8) + kBlock - 1) / kBlock, ctas = need < sm_count() ? need : sm_count();
    return checked(launch_kernel(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kBlock), 0, st, overlap, typed, c.n, c.V, ignore, t.head(),
                                 t.row_of(), t.target(), at_target, each, from, to, l.n_rows, c.d, l.d_pad, l.x_planes, vec));
  };
  auto pack = [&](auto* typed) {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(typed)>>;
    auto from = [&](auto* rows) {
      using S = std::remove_const_t<std::remove_pointer_t<decltype(rows)>>;
      return dtype == NLFA_DTYPE_F16 ? pack_few(pack_few_kernel<I, S, __half>, typed, rows, reinterpret_cast<__half*>(tape + l.x))
                                     : pack_few(pack_few_kernel<I, S, __nv_bfloat16>, typed, rows, reinterpret_cast<__nv_bfloat16*>(tape + l.x));
    };
    if (few)
      return c.x_dtype == NLFA_DTYPE_F32 ? from(static_cast<const float*>(x))
             : c.x_dtype == NLFA_DTYPE_F16 ? from(static_cast<const __half*>(x)) : from(static_cast<const __nv_bfloat16*>(x));
    return checked(launch_cluster(pack_rows_kernel<I>, dim3(1, kScanCtas), dim3(kScanThreads), 0, st, overlap, kScanCtas, typed, c.n, l.n_rows,
                                  c.V, ignore, t.head(), t.row_of(), t.target(), at_target, each, col_tiles, most_pairs(), l.max_splits));
  };
  int rc = target_bytes == 8 ? pack(static_cast<const long long*>(targets)) : pack(static_cast<const int*>(targets));
  if (rc != NLFA_OK) return rc;
  if (l.copy_w) {
    rc = copy_rows(w, c.w_dtype, tape + l.w, dtype, nullptr, nullptr, c.V, c.V, c.d, l.d_pad, l.x_planes, st);
    if (rc != NLFA_OK) return rc;
  }
  if (!few) rc = copy_rows(x, c.x_dtype, tape + l.x, dtype, t.head(), t.row_of(), c.n, l.n_rows, c.d, l.d_pad, l.x_planes, st);
  if (rc != NLFA_OK) return rc;
  CUtensorMap mx, mw;
  rc = few ? box_map(&mx, tape + l.x, dtype, l.d_pad, l.n_rows, l.x_planes, kFewRows / 2, summands(l.x_planes) / 64, l.x_planes, true)
           : column_map(&mx, tape + l.x, dtype, l.d_pad, l.n_rows, l.x_planes);
  if (rc == NLFA_OK) rc = column_map(&mw, l.copy_w ? tape + l.w : w, dtype, l.d_pad, c.V, l.x_planes, l.copy_w);
  if (rc != NLFA_OK) return rc;
  Params p = params(c, l, t, status);
  p.chunk = logit_chain(c, l);
  p.partial = reinterpret_cast<float2*>(scratch + l.partial);
  p.w_stands = l.copy_w ? 0 : 1;
  p.at_target = at_target;
  // few rows: W is read once, as the operand with 256 rows a tile; a tile of 256 rows of x would be read again for each of W's
  rc = launch_product(few ? kFew : kLse, dtype, p, mx, mw, mx, mx, st);
  if (rc != NLFA_OK) return rc;
  unsigned* ticket = nullptr;
  bool captured = false;
  if (each == nullptr) {
    rc = launch_ticket(st, reinterpret_cast<unsigned*>(scratch + l.ticket), &ticket, &captured);
    if (rc != NLFA_OK) return rc;
  }
  int lanes = 1;
  while (lanes < 32 && l.max_parts > 4 * lanes) lanes *= 2;
  const int need = l.n_rows / (kBlock / lanes), ctas = need < 1024 ? need : 1024;
  return checked(launch_kernel(finish_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kBlock), 0, st, !captured && overlap, t.head(),
                               p.partial, at_target, t.row_of(), l.n_rows, t.lse(), t.lse_rest(), t.own(), each, each != nullptr ? nullptr : out,
                               reinterpret_cast<double*>(scratch + l.sums), ticket, reduction == NLFA_REDUCE_MEAN ? 1 : 0, lanes, few ? l.max_parts : 0));
}

int run_bwd(const Call& c, const float* grad, const void* w, const void* targets, int target_bytes, long long ignore, int reduction,
            uint8_t* tape, void* dx, void* dw, uint8_t* scratch, cudaStream_t st) {
  const Layout l = layout(c, aligned16(w));
  const BwdLayout b = bwd_layout(c, l);
  const Pointers t{tape, l};
  unsigned* status = status_block();
  if (!status) return NLFA_ERR_CUDA;
  const int dtype = c.dtype == NLFA_DTYPE_F32 ? NLFA_DTYPE_BF16 : c.dtype;
  const bool overlap = overlap_launches(kOverlapRowwise);
  float* row_scale = reinterpret_cast<float*>(scratch + b.row_scale);
  float* alpha = reinterpret_cast<float*>(scratch + b.alpha);
  Parts* parts = reinterpret_cast<Parts*>(scratch + b.parts);
  const int per_row = reduction == NLFA_REDUCE_NONE ? 1 : 0;
  float* largest = per_row && dtype == NLFA_DTYPE_F16 ? alpha + 1 : nullptr;
  int rc = NLFA_OK;
  if (largest != nullptr)
    rc = checked(launch_kernel(largest_kernel, dim3(1), dim3(1024), 0, st, overlap, t.head(), grad, t.row_of(), largest));
  if (rc != NLFA_OK) return rc;
  const long long row_bytes = static_cast<long long>(c.d) * element_bytes(c.x_dtype);
  const int need = l.n_rows / (kBlock / 32), most = 4 * sm_count();
  auto scale = [&](auto* typed, auto* kernel) {
    return checked(launch_kernel(kernel, dim3(static_cast<unsigned>(need < most ? need : most)), dim3(kBlock), 0, st, overlap, t.head(), grad,
                                 per_row, reduction == NLFA_REDUCE_MEAN ? 1 : 0, t.row_of(), t.target(), row_scale, alpha, parts, largest,
                                 dtype == NLFA_DTYPE_F16 ? 16384.f : 1.f, typed, c.n, ignore, static_cast<uint8_t*>(dx), row_bytes, c.V, c.d, b.piece, dw != nullptr ? 1 : 0,
                                 most_pairs(), l.x_planes));
  };
  rc = target_bytes == 8 ? scale(static_cast<const long long*>(targets), scale_rows_kernel<long long>)
                         : scale(static_cast<const int*>(targets), scale_rows_kernel<int>);
  if (rc != NLFA_OK) return rc;
  CUtensorMap x_columns, w_columns, out, x_rows, w_rows, dl_columns, dl_rows;
  const void* wp = l.copy_w ? tape + l.w : w;
  rc = column_map(&x_columns, tape + l.x, dtype, l.d_pad, l.n_rows, l.x_planes);
  if (rc == NLFA_OK) rc = column_map(&w_columns, wp, dtype, l.d_pad, c.V, l.x_planes, l.copy_w);
  if (rc == NLFA_OK) rc = row_map(&x_rows, tape + l.x, dtype, l.d_pad, l.n_rows, l.x_planes);
  if (rc == NLFA_OK) rc = row_map(&w_rows, wp, dtype, l.d_pad, c.V, l.x_planes, l.copy_w);
  if (rc == NLFA_OK) rc = column_map(&dl_columns, scratch + b.dl, dtype, b.piece, b.dl_rows, l.x_planes);
  if (rc == NLFA_OK) rc = row_map(&dl_rows, scratch + b.dl, dtype, b.piece, b.dl_rows, l.x_planes);
  if (rc == NLFA_OK) rc = box_map(&out, scratch + b.dl, dtype, b.piece, b.dl_rows, l.x_planes, 32, 1, 1, true);
  if (rc != NLFA_OK) return rc;
  Params p = params(c, l, t, status);
  p.per_row = per_row;
  p.dl_second = b.dl_second;
  p.row_scale = row_scale;
  p.alpha = alpha;
  p.parts = parts;
  p.dx = dx;
  p.dw = dw;
  p.dx_dtype = c.x_dtype;
  p.dw_dtype = c.w_dtype;
  p.shares = reinterpret_cast<float*>(scratch + b.shares);
  p.dx_sum = reinterpret_cast<float*>(scratch + b.dx_sum);
  p.want_dx = dx != nullptr;
  p.want_dw = dw != nullptr;
  for (int v = 0; v < c.V; v += b.piece) {
    p.v0 = v;
    p.v1 = c.V - v < b.piece ? c.V : v + b.piece;
    p.first = v == 0;
    p.last = p.v1 == c.V;
    p.chunk = logit_chain(c, l);
    rc = launch_product(kGrad, dtype, p, x_columns, w_columns, out, out, st);
    p.chunk = product_chain(l, dtype);
    if (rc == NLFA_OK) rc = launch_product(kProducts, dtype, p, x_rows, w_rows, dl_columns, dl_rows, st);
    if (rc != NLFA_OK) return rc;
  }
  return NLFA_OK;
}

}  // namespace
}  // namespace loss
}  // namespace nlfa

using namespace nlfa;
using namespace nlfa::loss;
using rowwise::aligned16;

extern "C" {

size_t nlfa_linear_ce_tape_bytes(const void* w, int n, int V, int d, int x_dtype, int w_dtype, int dtype) {
  const Call c{x_dtype, w_dtype, dtype, n, V, d};
  return check_call(c) == NLFA_OK ? layout(c, aligned16(w)).tape_bytes : 0;
}
size_t nlfa_linear_ce_scratch_bytes(int n, int V, int d, int x_dtype, int w_dtype, int dtype, int backward) {
  const Call c{x_dtype, w_dtype, dtype, n, V, d};
  if (check_call(c) != NLFA_OK) return 0;
  const Layout l = layout(c, false);
  return backward ? bwd_layout(c, l).bytes : l.fwd_bytes;
}

int nlfa_linear_ce_fwd(const void* x, int x_dtype, const void* w, int w_dtype, int dtype, const void* targets, int target_bytes,
                       int n, int V, int d, long long ignore_index, int reduction, float* loss, void* tape, size_t tape_bytes,
                       void* scratch, size_t scratch_bytes, void* stream) {
  const Call c{x_dtype, w_dtype, dtype, n, V, d};
  const int rc = check_call(c);
  if (rc != NLFA_OK) return rc;
  if ((target_bytes != 4 && target_bytes != 8) || reduction < NLFA_REDUCE_NONE || reduction > NLFA_REDUCE_SUM) return NLFA_ERR_BAD_ARGUMENT;
  if (!w || !tape || !scratch || (n > 0 && (!x || !targets)) || (!loss && !(n == 0 && reduction == NLFA_REDUCE_NONE)))
    return NLFA_ERR_NULL_POINTER;
  if (!aligned16(tape) || !aligned16(scratch) || !aligned_to(x, element_bytes(x_dtype)) || !aligned_to(w, element_bytes(w_dtype)) ||
      !aligned_to(targets, target_bytes) || !aligned_to(loss, 4))
    return NLFA_ERR_MISALIGNED;
  const Layout l = layout(c, aligned16(w));
  if (tape_bytes < l.tape_bytes || scratch_bytes < l.fwd_bytes) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (!nlfa_device_supported()) return NLFA_ERR_NOT_SM100;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  return run_fwd(c, x, w, targets, target_bytes, ignore_index, reduction, loss, static_cast<uint8_t*>(tape),
                 static_cast<uint8_t*>(scratch), static_cast<cudaStream_t>(stream));
}

int nlfa_linear_ce_bwd(const float* grad, const void* w, int w_dtype, int x_dtype, int dtype, const void* targets, int target_bytes,
                       int n, int V, int d, long long ignore_index, int reduction, void* tape, size_t tape_bytes, void* dx, void* dw,
                       void* scratch, size_t scratch_bytes, void* stream) {
  const Call c{x_dtype, w_dtype, dtype, n, V, d};
  const int rc = check_call(c);
  if (rc != NLFA_OK) return rc;
  if ((target_bytes != 4 && target_bytes != 8) || reduction < NLFA_REDUCE_NONE || reduction > NLFA_REDUCE_SUM) return NLFA_ERR_BAD_ARGUMENT;
  if (!dx && !dw) return NLFA_OK;
  if (!w || !tape || !scratch || (n > 0 && !targets) || (!grad && (n > 0 || reduction != NLFA_REDUCE_NONE))) return NLFA_ERR_NULL_POINTER;
  if (!aligned16(tape) || !aligned16(scratch) || !aligned16(dx) || !aligned16(dw) || !aligned_to(w, element_bytes(w_dtype)) ||
      !aligned_to(targets, target_bytes) || !aligned_to(grad, 4))
    return NLFA_ERR_MISALIGNED;
  const Layout l = layout(c, aligned16(w));
  if (tape_bytes < l.tape_bytes || scratch_bytes < bwd_layout(c, l).bytes) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (!nlfa_device_supported()) return NLFA_ERR_NOT_SM100;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  return run_bwd(c, grad, w, targets, target_bytes, ignore_index, reduction, static_cast<uint8_t*>(tape), dx, dw,
                 static_cast<uint8_t*>(scratch), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
