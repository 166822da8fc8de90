// The norm of many tensors as of one vector, and their clip:  n = (sum g^2)^(1/2) or max |g|,  c = min(1, max_norm / (n + 1e-6)),
// g <- c g where c < 1 (or out <- c g).
//
// Bound by HBM: one read for the norm, one read and one write where the gradients change.  The tensors come as a table in the
// launch's parameters (nothing is copied to the device, and a captured launch keeps its table); a CTA takes pieces of 32 KB
// of whichever tensor.  Squares are added eight at a time in float32 and the eights in float64; an eight whose sum leaves float32's
// safe range is squared in float64 (gradients of 1e20, or of 1e-20, have a norm).  The sums of the CTAs are added in order by the one that ends
// last, so the same call gives the same bits.  The clip goes through the pieces backwards: what the norm read last is still in L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"
#include "ptx.cuh"
#include "rowwise.cuh"

namespace nlfa {
namespace clip {
namespace {

constexpr int kBlock = 256;
constexpr int kPieceBytes = 32768;              // of a gradient
constexpr int kCtasPerSm = 6;
constexpr int kMostTables = 64;                 // launches of one call

template <int K>
struct Table {
  int count, pieces;
  int first[K];                                 // first piece of a tensor
  unsigned char dtype[K], out_dtype[K];
  long long n[K];
  const void* src[K];
  void* dst[K];
};

struct Piece {
  const void* src;
  void* dst;
  long long n, from, to;                        // whole vectors of [from, to); [0, head) and [to, n) too for its first / last piece
  int head, dtype, out_dtype;
  bool first, last;
};

__device__ __forceinline__ int element_bytes(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }

template <int K>
__device__ __forceinline__ Piece piece_of(const Table<K>& t, int piece) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  Piece p;
  p.src = t.src[lo];
  p.dst = t.dst[lo];
  p.n = t.n[lo];
  p.dtype = t.dtype[lo];
  p.out_dtype = t.out_dtype[lo];
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(p.src) & 15u);
  p.head = skew == 0 ? 0 : (16 - skew) / element_bytes(p.dtype);
  if (p.head > p.n) p.head = static_cast<int>(p.n);
  const int at = piece - t.first[lo], size = kPieceBytes / element_bytes(p.dtype);
  p.from = p.head + static_cast<long long>(at) * size;
  p.to = p.from + size;
  p.first = at == 0;
  p.last = p.to >= p.n;
  if (p.last) p.to = p.n;
  return p;
}

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__half x) { return __half2float(x); }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }

struct Square {
  double sum = 0.0;
  __device__ __forceinline__ void add(const float (&v)[8]) {
    float s = 0.f, any = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s = fmaf(v[i], v[i], s);
      any = fmaxf(any, fabsf(v[i]));
    }
    if (s < 1e37f && s > 1e-28f) sum += static_cast<double>(s);
    else if (any > 0.f || !(s == 0.f)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), sum);
    }
  }
  __device__ __forceinline__ void add(float v) { sum = fma(static_cast<double>(v), static_cast<double>(v), sum); }
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
  static __device__ __forceinline__ double finish(double s) { return sqrt(s); }
};
struct Largest {
  double sum = 0.0;                             // a float's value
  unsigned bits = 0u;                           // of |x|: NaN above infinity above all others
  __device__ __forceinline__ void add(const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) add(v[i]);
  }
  __device__ __forceinline__ void add(float v) {
    const unsigned b = __float_as_uint(v) & 0x7fffffffu;
    bits = b > bits ? b : bits;
  }
  static __device__ __forceinline__ double join(double a, double b) { return a > b || a != a ? a : b; }
  static __device__ __forceinline__ double finish(double s) { return s; }
};

// 16 bytes of a gradient a thread and step, as many steps of a piece in flight.
constexpr int kSteps = kPieceBytes / 16 / kBlock;

template <typename S, typename Norm>
__device__ __forceinline__ void add_words(const uint4 (&raw)[kSteps], Norm& acc) {
  constexpr int N = 16 / sizeof(S);
#pragma unroll
  for (int u = 0; u < kSteps; u += 8 / N) {
    float v[8];
#pragma unroll
    for (int w = 0; w < 8 / N; ++w) {
      S e[N];
      *reinterpret_cast<uint4*>(e) = raw[u + w];
#pragma unroll
      for (int j = 0; j < N; ++j) v[N * w + j] = value(e[j]);
    }
    acc.add(v);
  }
}
template <typename S, typename Norm>
__device__ __forceinline__ void add_ends(const Piece& p, Norm& acc) {
  constexpr int N = 16 / sizeof(S);
  const S* src = static_cast<const S*>(p.src);
  if (p.first && static_cast<int>(threadIdx.x) < p.head) acc.add(value(src[threadIdx.x]));
  if (p.last) {
    const long long i = p.from + (p.to - p.from) / N * N + threadIdx.x;
    if (i < p.to) acc.add(value(src[i]));
  }
}
__device__ __forceinline__ void load_words(const Piece& p, uint4 (&raw)[kSteps]) {
  const int bytes = element_bytes(p.dtype), words = static_cast<int>((p.to - p.from) * bytes / 16);
  const uint4* body = reinterpret_cast<const uint4*>(static_cast<const char*>(p.src) + p.from * bytes);
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    const int i = u * kBlock + threadIdx.x;
    raw[u] = i < words ? body[i] : make_uint4(0u, 0u, 0u, 0u);
  }
}

struct Result {
  float norm, factor;
};

template <int K, typename Norm>
__global__ void __launch_bounds__(kBlock)
norm_kernel(const __grid_constant__ Table<K> t, double* __restrict__ partial, int done, int last_table, float max_norm, Result* result,
            float* __restrict__ norm_out, unsigned* ticket) {
  __shared__ double warp_sum[kBlock / 32];
  __shared__ int last;
  grid_dep_wait();
  grid_dep_release();
  Norm acc;
  const int step = gridDim.x;
  for (int i = blockIdx.x; i < t.pieces; i += step) {
    const Piece p = piece_of(t, i);
    uint4 raw[kSteps];
    load_words(p, raw);
    if (p.dtype == NLFA_DTYPE_F32) { add_ends<float>(p, acc); add_words<float>(raw, acc); }
    else if (p.dtype == NLFA_DTYPE_F16) { add_ends<__half>(p, acc); add_words<__half>(raw, acc); }
    else { add_ends<__nv_bfloat16>(p, acc); add_words<__nv_bfloat16>(raw, acc); }
  }
  auto block = [&](double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = Norm::join(v, __shfl_xor_sync(0xffffffffu, v, off));
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_sum[0];
#pragma unroll
    for (int w = 1; w < kBlock / 32; ++w) v = Norm::join(v, warp_sum[w]);
    return v;
  };
  if constexpr (sizeof(Norm) > sizeof(Square)) acc.sum = __uint_as_float(acc.bits);
  const double mine = block(acc.sum);
  if (threadIdx.x == 0) partial[done + blockIdx.x] = mine;
  if (!last_table || !rowwise::last_cta(ticket, gridDim.x, &last)) return;
  double v = 0.0;
  for (int i = threadIdx.x; i < done + static_cast<int>(gridDim.x); i += kBlock) v = Norm::join(v, __ldcg(partial + i));
  v = block(v);
  if (threadIdx.x == 0) {
    const float norm = static_cast<float>(Norm::finish(v)), c = max_norm / (norm + 1e-6f);
    result->norm = norm;
    result->factor = c < 1.f || c != c ? c : 1.f;            // (a NaN norm: every gradient becomes NaN)
    *norm_out = norm;
  }
}

// N scaled values to their place, N elements of D: 8 to 32 bytes, aligned to 16 at least
template <typename D, int N>
__device__ __forceinline__ void put(D* p, const float (&v)[N]) {
  if constexpr (sizeof(D) == 4) {
#pragma unroll
    for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N; j += 2) w[j / 2] = Pack2<D>::pack(v[j], v[j + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}
// ... a whole sector in one store (123.6M bf16 gradients into float32: 122 us, 6.1 TB/s)
__device__ __forceinline__ void put_sector(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}

template <typename S, typename D>
__device__ __forceinline__ void scale_of(const Piece& p, const uint4 (&raw)[kSteps], float c) {
  constexpr int N = 16 / sizeof(S);
  const S* src = static_cast<const S*>(p.src);
  D* dst = static_cast<D*>(p.dst);
  const uintptr_t at = reinterpret_cast<uintptr_t>(dst + p.from);
  const bool words = at % (N * sizeof(D) < 16 ? N * sizeof(D) : 16) == 0, sectors = at % 32 == 0;
  const int whole = words ? static_cast<int>((p.to - p.from) / N) : 0;     // (out lies otherwise than the gradient: one by one)
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    const int i = u * kBlock + threadIdx.x;
    alignas(16) S e[N];
    *reinterpret_cast<uint4*>(e) = raw[u];
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = value(e[j]) * c;
    if (i >= whole) continue;
    if constexpr (N == 8 && sizeof(D) == 4) {
      if (sectors) {
        put_sector(dst + p.from + N * i, v);
        continue;
      }
    }
    put(dst + p.from + N * i, v);
  }
  auto one = [&](long long i) { dst[i] = static_cast<D>(value(src[i]) * c); };
  if (p.first && static_cast<int>(threadIdx.x) < p.head) one(threadIdx.x);
  if (!words || p.last)
#pragma unroll 1
    for (long long i = p.from + static_cast<long long>(N) * whole + threadIdx.x; i < p.to; i += kBlock) one(i);
}

template <typename S>
__device__ __forceinline__ void scale_from(const Piece& p, const uint4 (&raw)[kSteps], float c) {
  if (p.out_dtype == NLFA_DTYPE_F32) scale_of<S, float>(p, raw, c);
  else if (p.out_dtype == NLFA_DTYPE_F16) scale_of<S, __half>(p, raw, c);
  else scale_of<S, __nv_bfloat16>(p, raw, c);
}

template <int K>
__global__ void __launch_bounds__(kBlock)
scale_kernel(const __grid_constant__ Table<K> t, const Result* result, int in_place) {
  grid_dep_wait();
  grid_dep_release();
  const float c = result->factor;
  if (in_place && c == 1.f) return;
  const int step = gridDim.x;
  int i = t.pieces - 1 - static_cast<int>(blockIdx.x);
  for (Piece p = piece_of(t, i), next; i >= 0; i -= step, p = next) {
    uint4 raw[kSteps];
    const bool change = c != 1.f || p.src != p.dst;
    if (change) load_words(p, raw);
    if (i >= step) next = piece_of(t, i - step);
    if (!change) continue;
    if (p.dtype == NLFA_DTYPE_F32) scale_from<float>(p, raw, c);
    else if (p.dtype == NLFA_DTYPE_F16) scale_from<__half>(p, raw, c);
    else scale_from<__nv_bfloat16>(p, raw, c);
  }
}

int checked(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

int bytes_of(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }

// Tables of up to K tensors each.
template <int K>
int run(const nlfa_grad* grads, int count, float max_norm, int norm, int scale, int in_place, float* norm_out, double* partial,
        Result* result, unsigned* own_ticket, cudaStream_t st) {
  const int most = kCtasPerSm * sm_count();
  const int tables = (count + K - 1) / K;
  const bool overlap = overlap_launches(kOverlapRowwise);
  Table<K> t;
  auto fill = [&](int which) {
    const int from = which * K, to = from + K < count ? from + K : count;
    t.count = to - from;
    long long pieces = 0;
    for (int i = from; i < to; ++i) {
      const nlfa_grad& g = grads[i];
      const int j = i - from;
      const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(g.grad) & 15u);
      long long body = g.n - (skew == 0 ? 0 : (16 - skew) / bytes_of(g.dtype));
      if (body < 1) body = 1;
      t.first[j] = static_cast<int>(pieces);
      const int size = kPieceBytes / bytes_of(g.dtype);
      pieces += (body + size - 1) / size;
      t.dtype[j] = static_cast<unsigned char>(g.dtype);
      t.out_dtype[j] = static_cast<unsigned char>(g.out != nullptr ? g.out_dtype : g.dtype);
      t.n[j] = g.n;
      t.src[j] = g.grad;
      t.dst[j] = g.out != nullptr ? g.out : const_cast<void*>(g.grad);
      if (pieces > 0x3fffffff) return false;
    }
    t.pieces = static_cast<int>(pieces);
    return true;
  };
  unsigned* ticket = nullptr;
  bool captured = false;
  int rc = launch_ticket(st, own_ticket, &ticket, &captured);
  if (rc != NLFA_OK) return rc;
  int done = 0;
  for (int i = 0; i < tables; ++i) {
    if (!fill(i)) return NLFA_ERR_BAD_SHAPE;
    const int ctas = t.pieces < most ? t.pieces : most, last = i + 1 == tables;
    auto go = [&](auto* kernel) {
      return checked(launch_kernel(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kBlock), 0, st, !captured && overlap, t, partial, done, last,
                                   max_norm, result, norm_out, ticket));
    };
    rc = norm == NLFA_NORM_INF ? go(norm_kernel<K, Largest>) : go(norm_kernel<K, Square>);
    if (rc != NLFA_OK) return rc;
    done += ctas;
  }
  for (int i = tables - 1; scale && i >= 0; --i) {
    if (tables > 1 && !fill(i)) return NLFA_ERR_BAD_SHAPE;
    const int ctas = t.pieces < most ? t.pieces : most;
    rc = checked(launch_kernel(scale_kernel<K>, dim3(static_cast<unsigned>(ctas)), dim3(kBlock), 0, st, overlap, t, result, in_place));
    if (rc != NLFA_OK) return rc;
  }
  return NLFA_OK;
}

constexpr int kSmallTable = 48, kTable = 320, kLargeTable = 1000;

}  // namespace
}  // namespace clip
}  // namespace nlfa

using namespace nlfa;
using namespace nlfa::clip;

extern "C" {

size_t nlfa_clip_scratch_bytes(void) { return 512 + static_cast<size_t>(kMostTables) * kCtasPerSm * 160 * sizeof(double); }

int nlfa_clip_grads(const nlfa_grad* grads, int count, float max_norm, int norm, int scale, float* total_norm, void* scratch,
                    size_t scratch_bytes, void* stream) {
  if (count < 0 || (norm != NLFA_NORM_2 && norm != NLFA_NORM_INF)) return NLFA_ERR_BAD_ARGUMENT;
  if (!total_norm || !scratch || (count > 0 && !grads)) return NLFA_ERR_NULL_POINTER;
  if (!rowwise::aligned16(scratch) || reinterpret_cast<uintptr_t>(total_norm) % 4 != 0) return NLFA_ERR_MISALIGNED;
  if (scratch_bytes < nlfa_clip_scratch_bytes()) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (static_cast<long long>(count) > static_cast<long long>(kMostTables) * kLargeTable || sm_count() > 160) return NLFA_ERR_BAD_SHAPE;
  int in_place = 1;
  for (int i = 0; i < count; ++i) {
    const nlfa_grad& g = grads[i];
    if (!rowwise::dtype_ok(g.dtype) || (g.out != nullptr && !rowwise::dtype_ok(g.out_dtype))) return NLFA_ERR_BAD_DTYPE;
    if (g.n < 1) return NLFA_ERR_BAD_SHAPE;
    if (!g.grad) return NLFA_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(g.grad) % bytes_of(g.dtype) != 0 ||
        (g.out != nullptr && reinterpret_cast<uintptr_t>(g.out) % bytes_of(g.out_dtype) != 0))
      return NLFA_ERR_MISALIGNED;
    if (g.out != nullptr && g.out != g.grad) in_place = 0;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (count == 0) return checked(cudaMemsetAsync(total_norm, 0, sizeof(float), st));
  uint8_t* s = static_cast<uint8_t*>(scratch);
  Result* result = reinterpret_cast<Result*>(s);
  unsigned* ticket = reinterpret_cast<unsigned*>(s + 256);
  double* partial = reinterpret_cast<double*>(s + 512);
  if (count <= kSmallTable) return run<kSmallTable>(grads, count, max_norm, norm, scale, in_place, total_norm, partial, result, ticket, st);
  if (count <= kTable) return run<kTable>(grads, count, max_norm, norm, scale, in_place, total_norm, partial, result, ticket, st);
  return run<kLargeTable>(grads, count, max_norm, norm, scale, in_place, total_norm, partial, result, ticket, st);
}

}  // extern "C"
