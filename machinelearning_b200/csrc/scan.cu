// Gated linear recurrence: for every channel of every sequence
//
//   s_t = sigmoid(z_t),  h_t = (1 - s_t) h_{t-1} + s_t f(v_t)                      f: identity, or "positive" (below)
//   G_t = dh_t + Q_{t+1},  Q_t = (1 - s_t) G_t,  dv_t = G_t s_t f'(v_t),  dz_t = G_t (f(v_t) - h_{t-1}) s_t (1 - s_t)
//
// with h_0 the state on entry, Q_{T+1} the gradient of the last state, dstate = Q_1.  A reset at t leaves h_{t-1} out; steps
// behind a sequence's length change nothing.
//
// Both directions are bound by memory: three streams of B T D elements forward, five backward.  A step is an affine map h -> a h + b, and maps
// compose, so the steps are walked in runs of kRun that start side by side: a warp has one run of 32 V channels in registers, forms its
// map, learns the maps of the runs in front of it (its CTA's through shared memory, the other CTAs' of its cluster through
// theirs), and walks the run again from the right state.  The data are read once.  CTAs of a cluster are resident together, so
// nothing waits on a CTA that has not begun; the order of all sums is fixed.
//
// Digits: the smaller of s and 1 - s, e / (1 + e) with e = exp(-|z|), is exact to a few units of 2^-24, the larger is not further than that from 1.  With
// it the step is h + s (f - h) or f + (1 - s) (h - f), whichever it belongs to: where s is 1e-6 a state that is multiplied with a rounded 1 - s
// would be off by 3% after the million steps that it lasts.
#include <cmath>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"
#include "rowwise.cuh"

namespace nlfa {
namespace scan {
namespace {

constexpr int kRun = 16;            // steps in a thread's registers; states at their starts are the backward's tape
constexpr int kWarps = 4;           // runs per CTA
constexpr int kMostClusterCtas = 8;
constexpr int kMostExtent = 1 << 30;

// V neighbouring channels as they lie in memory.
template <typename T, int V> struct Pack;
template <> struct Pack<float, 2> {
  using Raw = float2;
  __device__ static float2 get(const Raw& r) { return r; }
  __device__ static Raw put(float2 v) { return v; }
};
template <> struct Pack<float, 1> {
  using Raw = float;
  __device__ static float2 get(const Raw& r) { return make_float2(r, 0.f); }
  __device__ static Raw put(float2 v) { return v.x; }
};
template <> struct Pack<__nv_bfloat16, 2> {
  using Raw = __nv_bfloat162;
  __device__ static float2 get(const Raw& r) { return __bfloat1622float2(r); }
  __device__ static Raw put(float2 v) { return __floats2bfloat162_rn(v.x, v.y); }
};
template <> struct Pack<__nv_bfloat16, 1> {
  using Raw = __nv_bfloat16;
  __device__ static float2 get(const Raw& r) { return make_float2(__bfloat162float(r), 0.f); }
  __device__ static Raw put(float2 v) { return __float2bfloat16_rn(v.x); }
};
template <> struct Pack<__half, 2> {
  using Raw = __half2;
  __device__ static float2 get(const Raw& r) { return __half22float2(r); }
  __device__ static Raw put(float2 v) { return __floats2half2_rn(v.x, v.y); }
};
template <> struct Pack<__half, 1> {
  using Raw = __half;
  __device__ static float2 get(const Raw& r) { return make_float2(__half2float(r), 0.f); }
  __device__ static Raw put(float2 v) { return __float2half_rn(v.x); }
};

struct Params {
  const void *gate, *value;
  long long gate_b, gate_t, value_b, value_t;       // strides in elements; channels lie side by side
  const float* state;
  const uint8_t* reset;                             // [B, T]
  const void* lengths;                              // [B]
  int length_bytes;
  int B, T, D, blocks;                              // blocks: of 32 V channels
  void* h;
  float *last, *tape;
  // backward
  const void* dh;
  const float* dlast;
  void *dgate, *dvalue;
  float* dstate;
};

// exp(-|z|): 16-bit results need no more than the hardware's 2^-22; float32 ones are held to 2^-23 at every size of z
template <typename T> __device__ __forceinline__ float exp_minus(float a) { return fast_exp2(-kLog2e * a); }
template <> __device__ __forceinline__ float exp_minus<float>(float a) { return expf(-a); }

template <typename T> __device__ __forceinline__ float ratio(float a, float b) { return __fdividef(a, b); }
template <> __device__ __forceinline__ float ratio<float>(float a, float b) { return a / b; }

// The smaller of sigmoid(z) and 1 - sigmoid(z), with a minus sign where that is the latter (also a zero's).
template <typename T> __device__ __forceinline__ float lesser(float z) {
  const float e = exp_minus<T>(fabsf(z));
  return copysignf(ratio<T>(e, 1.f + e), -z);
}
__device__ __forceinline__ bool is_minus(float x) { return __float_as_int(x) < 0; }
template <typename T> __device__ __forceinline__ float sigmoid(float v) {
  const float e = exp_minus<T>(fabsf(v));
  return ratio<T>(v < 0.f ? e : 1.f, 1.f + e);
}
// f(v) and its slope.  positive: v + 1/2 from zero on, sigmoid(v) below
template <typename T, bool POSITIVE> __device__ __forceinline__ float mapped(float v) {
  if (!POSITIVE) return v;
  return v < 0.f ? sigmoid<T>(v) : v + 0.5f;
}
template <typename T, bool POSITIVE> __device__ __forceinline__ float slope(float v) {
  if (!POSITIVE) return 1.f;
  const float p = sigmoid<T>(v);
  return v < 0.f ? p * (1.f - p) : 1.f;
}

// h after a step: x from lesser()
__device__ __forceinline__ float step(float x, float f, float h) { return fmaf(x, f - h, is_minus(x) ? f : h); }
// (1 - s) q
__device__ __forceinline__ float kept(float x, float q) { return fmaf(-x, q, is_minus(x) ? 0.f : q); }

// Two channels' maps h -> a h + b of some steps, (a, b, a, b).  (a == 0: nothing of h is left, whatever it holds)
__device__ __forceinline__ float2 apply(const float4& m, float2 h) {
  return make_float2(m.x == 0.f ? m.y : fmaf(m.x, h.x, m.y), m.z == 0.f ? m.w : fmaf(m.z, h.y, m.w));
}
// m, then n
__device__ __forceinline__ float4 then(const float4& m, const float4& n) {
  const float2 b = apply(n, make_float2(m.y, m.w));
  return make_float4(m.x * n.x, b.x, m.z * n.z, b.y);
}

__device__ __forceinline__ void st_cluster_f4(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// What the runs of a stretch of steps (the cluster's CTAs x WARPS runs) tell one another.
template <int WARPS> struct Exchange {
  float4 warps[2][WARPS][32];
  float4 ctas[2][kMostClusterCtas][32];
};

// The state in front of this thread's run, given its run's map, and the state behind the stretch in `carry`.  `order`: this warp's
// place in its CTA and `rank` the CTA's place in the cluster, in the order in which the runs are walked.
template <int WARPS>
__device__ __forceinline__ float2 enter(Exchange<WARPS>& x, int buf, int order, int rank, int ctas, float4 own, float2& carry) {
  const int lane = threadIdx.x & 31;
  if (WARPS == 1 && ctas == 1) {
    const float2 in = carry;
    carry = apply(own, in);
    return in;
  }
  x.warps[buf][order][lane] = own;
  __syncthreads();
  float2 in = carry;
  if (ctas > 1) {
    float4 all = x.warps[buf][0][lane];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) all = then(all, x.warps[buf][w][lane]);
    const uint32_t slot = smem_u32(&x.ctas[buf][rank][lane]);
    for (int c = order; c < ctas; c += WARPS) st_cluster_f4(cluster_addr(slot, c), all);
    cluster_arrive();
    cluster_wait();
    for (int c = 0; c < ctas; ++c) {
      if (c == rank) in = carry;
      carry = apply(x.ctas[buf][c][lane], carry);
    }
  }
  float2 h = in;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w == order) in = h;
    h = apply(x.warps[buf][w][lane], h);
  }
  if (ctas == 1) carry = h;
  return in;
}

// Steps of a sequence that count.
__device__ __forceinline__ int live_steps(const Params& p, int b) {
  if (p.lengths == nullptr) return p.T;
  const long long n = p.length_bytes == 8 ? static_cast<const long long*>(p.lengths)[b] : static_cast<const int*>(p.lengths)[b];
  return n < 0 ? 0 : n < p.T ? static_cast<int>(n) : p.T;
}
// Resets of the steps t0 .. t0 + kRun - 1, of which the first n count.
__device__ __forceinline__ unsigned reset_bits(const Params& p, int b, int t0, int n) {
  unsigned bits = 0;
  const uint8_t* r = p.reset + static_cast<long long>(b) * p.T + t0;
#pragma unroll
  for (int i = 0; i < kRun; ++i)
    if (i < n && r[i] != 0) bits |= 1u << i;
  return bits;
}

// Where a thread works: channels c (and c + 1) of sequence b.
struct Place {
  int b, c, rank, ctas, warp;
  bool live;
  template <int V> __device__ static Place of(const Params& p, int ctas) {
    Place w;
    w.ctas = ctas;
    const unsigned cluster = blockIdx.x / ctas;
    w.rank = static_cast<int>(blockIdx.x - cluster * ctas);
    w.b = static_cast<int>(cluster / p.blocks);
    w.c = static_cast<int>(cluster - w.b * p.blocks) * 32 * V + V * (threadIdx.x & 31);
    w.warp = threadIdx.x >> 5;
    w.live = w.c < p.D;
    return w;
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_run(typename Pack<T, V>::Raw (&r)[kRun], const void* base, long long b_stride, long long t_stride, int b, int t0,
                                         int c, int n) {
  using Raw = typename Pack<T, V>::Raw;
  const T* s = static_cast<const T*>(base) + b * b_stride + t0 * t_stride + c;
#pragma unroll
  for (int i = 0; i < kRun; ++i)
    if (i < n) r[i] = __ldcs(reinterpret_cast<const Raw*>(s + i * t_stride));
}

template <typename T, int V, int WARPS, bool POSITIVE, bool RESET>
__global__ void __launch_bounds__(32 * WARPS)
scan_fwd_kernel(const Params p, int ctas) {
  using P = Pack<T, V>;
  __shared__ Exchange<WARPS> x;
  if (ctas > 1) cluster_arrive_relaxed();
  grid_dep_wait();
  grid_dep_release();
  const Place w = Place::of<V>(p, ctas);
  const long long row = static_cast<long long>(w.b) * p.D + w.c;
  float2 carry = make_float2(0.f, 0.f);
  if (w.live && p.state != nullptr) {
    carry.x = p.state[row];
    if (V == 2) carry.y = p.state[row + 1];
  }
  const int live = live_steps(p, w.b), stretch = ctas * WARPS * kRun, runs = (p.T + kRun - 1) / kRun;
  typename P::Raw z[kRun], v[kRun];
  auto load = [&](int t0) {
    const int n = w.live ? live - t0 : 0;
    load_run<T, V>(z, p.gate, p.gate_b, p.gate_t, w.b, t0, w.c, n);
    load_run<T, V>(v, p.value, p.value_b, p.value_t, w.b, t0, w.c, n);
  };
  const int first = (w.rank * WARPS + w.warp) * kRun;
  load(first);
  if (ctas > 1) cluster_wait();                                // every CTA of the cluster has begun: its shared memory may be written
  int buf = 0;
  for (int from = 0; from < p.T; from += stretch, buf ^= 1) {
    const int t0 = from + first, n = w.live ? live - t0 : 0;
    const unsigned resets = RESET && n > 0 ? reset_bits(p, w.b, t0, n) : 0u;
    float2 small[kRun], f[kRun];
    float4 map = make_float4(1.f, 0.f, 1.f, 0.f);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      small[i] = f[i] = make_float2(0.f, 0.f);               // (a step that does not count leaves h as it is)
      if (i < n) {
        const float2 zi = P::get(z[i]), vi = P::get(v[i]);
        small[i] = make_float2(lesser<T>(zi.x), V == 2 ? lesser<T>(zi.y) : 0.f);
        f[i] = make_float2(mapped<T, POSITIVE>(vi.x), V == 2 ? mapped<T, POSITIVE>(vi.y) : 0.f);
      }
      if (RESET && (resets >> i & 1u)) map = make_float4(0.f, 0.f, 0.f, 0.f);
      map.x = kept(small[i].x, map.x);
      map.y = step(small[i].x, f[i].x, map.y);
      if (V == 2) {
        map.z = kept(small[i].y, map.z);
        map.w = step(small[i].y, f[i].y, map.w);
      }
    }
    if (from + stretch < p.T) load(t0 + stretch);
    float2 h = enter<WARPS>(x, buf, w.warp, w.rank, ctas, map, carry);
    if (w.live && t0 < p.T) {
      if (p.tape != nullptr) {
        float* tape = p.tape + (static_cast<long long>(w.b) * runs + t0 / kRun) * p.D + w.c;
        tape[0] = h.x;
        if (V == 2) tape[1] = h.y;
      }
      T* out = static_cast<T*>(p.h) + (static_cast<long long>(w.b) * p.T + t0) * p.D + w.c;
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        if (t0 + i >= p.T) break;
        if (RESET && (resets >> i & 1u)) h = make_float2(0.f, 0.f);
        h.x = step(small[i].x, f[i].x, h.x);
        if (V == 2) h.y = step(small[i].y, f[i].y, h.y);
        __stcs(reinterpret_cast<typename P::Raw*>(out + static_cast<long long>(i) * p.D), P::put(i < n ? h : make_float2(0.f, 0.f)));
      }
      if (p.T - t0 <= kRun) {
        p.last[row] = h.x;
        if (V == 2) p.last[row + 1] = h.y;
      }
    }
  }
  if (p.T == 0 && w.live) {
    p.last[row] = carry.x;
    if (V == 2) p.last[row + 1] = carry.y;
  }
}

template <typename T, int V, int WARPS, bool POSITIVE, bool RESET>
__global__ void __launch_bounds__(32 * WARPS)
scan_bwd_kernel(const Params p, int ctas) {
  using P = Pack<T, V>;
  __shared__ Exchange<WARPS> x;
  if (ctas > 1) cluster_arrive_relaxed();
  grid_dep_wait();
  grid_dep_release();
  const Place w = Place::of<V>(p, ctas);
  const long long row = static_cast<long long>(w.b) * p.D + w.c;
  float2 carry = make_float2(0.f, 0.f);
  if (w.live && p.dlast != nullptr) {
    carry.x = p.dlast[row];
    if (V == 2) carry.y = p.dlast[row + 1];
  }
  const int live = live_steps(p, w.b), stretch = ctas * WARPS * kRun, runs = (p.T + kRun - 1) / kRun;
  const int first = (w.rank * WARPS + w.warp) * kRun;
  if (ctas > 1) cluster_wait();
  int buf = 0;
  for (int from = (p.T - 1) / stretch * stretch; from >= 0; from -= stretch, buf ^= 1) {
    const int t0 = from + first, n = w.live ? live - t0 : 0;
    typename P::Raw z[kRun], v[kRun], g[kRun];
    load_run<T, V>(z, p.gate, p.gate_b, p.gate_t, w.b, t0, w.c, n);
    load_run<T, V>(v, p.value, p.value_b, p.value_t, w.b, t0, w.c, n);
    if (p.dh != nullptr) load_run<T, V>(g, p.dh, static_cast<long long>(p.T) * p.D, p.D, w.b, t0, w.c, n);
    float2 h = make_float2(0.f, 0.f);
    if (n > 0) {
      const float* tape = p.tape + (static_cast<long long>(w.b) * runs + t0 / kRun) * p.D + w.c;
      h.x = tape[0];
      if (V == 2) h.y = tape[1];
    }
    const unsigned resets = RESET && n > 0 ? reset_bits(p, w.b, t0, n) : 0u;
    float2 small[kRun], rest[kRun];                            // rest: f - h of the step before
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      small[i] = rest[i] = make_float2(0.f, 0.f);
      if (i < n) {
        const float2 zi = P::get(z[i]), vi = P::get(v[i]);
        if (RESET && (resets >> i & 1u)) h = make_float2(0.f, 0.f);
        const float f0 = mapped<T, POSITIVE>(vi.x);
        small[i].x = lesser<T>(zi.x);
        rest[i].x = f0 - h.x;
        h.x = step(small[i].x, f0, h.x);
        if (V == 2) {
          const float f1 = mapped<T, POSITIVE>(vi.y);
          small[i].y = lesser<T>(zi.y);
          rest[i].y = f1 - h.y;
          h.y = step(small[i].y, f1, h.y);
        }
      }
    }
    auto grad = [&](int i) { return i < n && p.dh != nullptr ? P::get(g[i]) : make_float2(0.f, 0.f); };
    float4 map = make_float4(1.f, 0.f, 1.f, 0.f);
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const float2 d = grad(i);
      map.x = kept(small[i].x, map.x);
      map.y = kept(small[i].x, map.y + d.x);
      if (V == 2) {
        map.z = kept(small[i].y, map.z);
        map.w = kept(small[i].y, map.w + d.y);
      }
      if (RESET && (resets >> i & 1u)) map = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float2 q = enter<WARPS>(x, buf, WARPS - 1 - w.warp, ctas - 1 - w.rank, ctas, map, carry);
    if (w.live && t0 < p.T) {
      const long long at = (static_cast<long long>(w.b) * p.T + t0) * p.D + w.c;
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i) {
        if (t0 + i < p.T) {
          const float2 d = grad(i);
          float2 dz = make_float2(0.f, 0.f), dv = dz;
          if (i < n) {
            const float2 vi = P::get(v[i]);
            const float l0 = fabsf(small[i].x), s0 = is_minus(small[i].x) ? 1.f - l0 : l0, g0 = d.x + q.x;
            dv.x = g0 * s0 * slope<T, POSITIVE>(vi.x);
            dz.x = g0 * rest[i].x * (l0 * (1.f - l0));
            q.x = kept(small[i].x, g0);
            if (V == 2) {
              const float l1 = fabsf(small[i].y), s1 = is_minus(small[i].y) ? 1.f - l1 : l1, g1 = d.y + q.y;
              dv.y = g1 * s1 * slope<T, POSITIVE>(vi.y);
              dz.y = g1 * rest[i].y * (l1 * (1.f - l1));
              q.y = kept(small[i].y, g1);
            }
          }
          if (RESET && (resets >> i & 1u)) q = make_float2(0.f, 0.f);
          const long long o = at + static_cast<long long>(i) * p.D;
          if (p.dgate != nullptr) __stcs(reinterpret_cast<typename P::Raw*>(static_cast<T*>(p.dgate) + o), P::put(dz));
          if (p.dvalue != nullptr) __stcs(reinterpret_cast<typename P::Raw*>(static_cast<T*>(p.dvalue) + o), P::put(dv));
        }
      }
    }
  }
  if (w.live && w.rank == 0 && w.warp == 0 && p.dstate != nullptr) {
    p.dstate[row] = carry.x;
    if (V == 2) p.dstate[row + 1] = carry.y;
  }
}

// ------------------------------------------------------------------------------------------------ host

// CTAs per cluster: the steps of a sequence side by side.
int cluster_ctas(const Params& p) {
  const long long stretches = (p.T + kWarps * kRun - 1) / (kWarps * kRun);
  int ctas = 1;
  while (ctas < kMostClusterCtas && ctas < stretches) ctas *= 2;
  return ctas;
}

template <typename Kernel>
int launch(Kernel* kernel, int warps, int ctas, const Params& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.B) * p.blocks * ctas);
  cfg.blockDim = dim3(32u * warps);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (overlap_launches(kOverlapRowwise)) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (ctas > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, ctas);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

template <typename T, int V, int WARPS, bool POSITIVE, bool RESET>
int run_warps(const Params& p, bool backward, cudaStream_t st) {
  const int ctas = WARPS == 1 ? 1 : cluster_ctas(p);
  return backward ? launch(scan_bwd_kernel<T, V, WARPS, POSITIVE, RESET>, WARPS, ctas, p, st)
                  : launch(scan_fwd_kernel<T, V, WARPS, POSITIVE, RESET>, WARPS, ctas, p, st);
}
template <typename T, int V, bool POSITIVE, bool RESET>
int run_reset(Params p, bool backward, cudaStream_t st) {
  p.blocks = (p.D + 32 * V - 1) / (32 * V);
  if (static_cast<long long>(p.B) * p.blocks * kMostClusterCtas > 0x7fffffffll) return NLFA_ERR_BAD_SHAPE;
  return p.T <= kRun ? run_warps<T, V, 1, POSITIVE, RESET>(p, backward, st) : run_warps<T, V, kWarps, POSITIVE, RESET>(p, backward, st);
}
template <typename T, int V, bool POSITIVE>
int run_positive(const Params& p, bool backward, cudaStream_t st) {
  return p.reset != nullptr ? run_reset<T, V, POSITIVE, true>(p, backward, st) : run_reset<T, V, POSITIVE, false>(p, backward, st);
}
template <typename T, int V>
int run_width(const Params& p, int activation, bool backward, cudaStream_t st) {
  return activation == NLFA_SCAN_POSITIVE ? run_positive<T, V, true>(p, backward, st) : run_positive<T, V, false>(p, backward, st);
}
template <typename T>
int run_typed(const Params& p, int activation, bool backward, cudaStream_t st) {
  // two channels a thread where every row begins on a pair's boundary
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.h) |
                        reinterpret_cast<uintptr_t>(p.dh) | reinterpret_cast<uintptr_t>(p.dgate) | reinterpret_cast<uintptr_t>(p.dvalue);
  const long long strides = p.gate_b | p.gate_t | p.value_b | p.value_t | p.D;
  const bool pairs = strides % 2 == 0 && all % (2 * sizeof(T)) == 0;
  return pairs ? run_width<T, 2>(p, activation, backward, st) : run_width<T, 1>(p, activation, backward, st);
}
int run(const Params& p, int dtype, int activation, bool backward, cudaStream_t st) {
  if (dtype == NLFA_DTYPE_F32) return run_typed<float>(p, activation, backward, st);
  if (dtype == NLFA_DTYPE_F16) return run_typed<__half>(p, activation, backward, st);
  return run_typed<__nv_bfloat16>(p, activation, backward, st);
}

int element_bytes(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }
bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check(int dtype, int activation, int length_bytes, const void* lengths, int B, int T, int D) {
  if (B < 0 || T < 0 || D < 0 || B > kMostExtent || T > kMostExtent || D > kMostExtent) return NLFA_ERR_BAD_SHAPE;
  if (!rowwise::dtype_ok(dtype)) return NLFA_ERR_BAD_DTYPE;
  if (activation != NLFA_SCAN_NONE && activation != NLFA_SCAN_POSITIVE) return NLFA_ERR_BAD_ARGUMENT;
  if (lengths != nullptr && length_bytes != 4 && length_bytes != 8) return NLFA_ERR_BAD_ARGUMENT;
  if (lengths != nullptr && !aligned_to(lengths, length_bytes)) return NLFA_ERR_MISALIGNED;
  return NLFA_OK;
}

size_t tape_bytes(int B, int T, int D) {
  return static_cast<size_t>(B) * ((static_cast<size_t>(T) + kRun - 1) / kRun) * static_cast<size_t>(D) * sizeof(float);
}

}  // namespace
}  // namespace scan
}  // namespace nlfa

using namespace nlfa;
using namespace nlfa::scan;

extern "C" {

size_t nlfa_gated_scan_tape_bytes(int B, int T, int D) { return B < 0 || T < 0 || D < 0 ? 0 : tape_bytes(B, T, D); }

int nlfa_gated_scan_fwd(const void* gate, long long gate_b, long long gate_t, const void* value, long long value_b, long long value_t,
                        int dtype, const float* state, const unsigned char* reset, const void* lengths, int length_bytes, int activation,
                        int B, int T, int D, void* h, float* last, void* tape, size_t bytes, void* stream) {
  const int rc = check(dtype, activation, length_bytes, lengths, B, T, D);
  if (rc != NLFA_OK) return rc;
  if (B == 0 || D == 0) return NLFA_OK;
  if (!last || (T > 0 && (!gate || !value || !h))) return NLFA_ERR_NULL_POINTER;
  const int e = element_bytes(dtype);
  if (!aligned_to(gate, e) || !aligned_to(value, e) || !aligned_to(h, e) || !aligned_to(state, 4) || !aligned_to(last, 4) || !aligned_to(tape, 4))
    return NLFA_ERR_MISALIGNED;
  if (tape != nullptr && bytes < tape_bytes(B, T, D)) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  Params p{};
  p.gate = gate; p.gate_b = gate_b; p.gate_t = gate_t;
  p.value = value; p.value_b = value_b; p.value_t = value_t;
  p.state = state; p.reset = reset; p.lengths = lengths; p.length_bytes = length_bytes;
  p.B = B; p.T = T; p.D = D;
  p.h = h; p.last = last; p.tape = static_cast<float*>(tape);
  return run(p, dtype, activation, false, static_cast<cudaStream_t>(stream));
}

int nlfa_gated_scan_bwd(const void* dh, const float* dlast, const void* gate, long long gate_b, long long gate_t, const void* value,
                        long long value_b, long long value_t, int dtype, const unsigned char* reset, const void* lengths, int length_bytes,
                        int activation, int B, int T, int D, const void* tape, size_t bytes, void* dgate, void* dvalue, float* dstate,
                        void* stream) {
  const int rc = check(dtype, activation, length_bytes, lengths, B, T, D);
  if (rc != NLFA_OK) return rc;
  if (B == 0 || D == 0 || (!dgate && !dvalue && !dstate)) return NLFA_OK;
  if (T > 0 && (!gate || !value || !tape)) return NLFA_ERR_NULL_POINTER;
  const int e = element_bytes(dtype);
  if (!aligned_to(gate, e) || !aligned_to(value, e) || !aligned_to(dh, e) || !aligned_to(dgate, e) || !aligned_to(dvalue, e) ||
      !aligned_to(dlast, 4) || !aligned_to(dstate, 4) || !aligned_to(tape, 4))
    return NLFA_ERR_MISALIGNED;
  if (T > 0 && bytes < tape_bytes(B, T, D)) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  Params p{};
  p.gate = gate; p.gate_b = gate_b; p.gate_t = gate_t;
  p.value = value; p.value_b = value_b; p.value_t = value_t;
  p.reset = reset; p.lengths = lengths; p.length_bytes = length_bytes;
  p.B = B; p.T = T; p.D = D;
  p.tape = static_cast<float*>(const_cast<void*>(tape));
  p.dh = dh; p.dlast = dlast; p.dgate = dgate; p.dvalue = dvalue; p.dstate = dstate;
  return run(p, dtype, activation, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
