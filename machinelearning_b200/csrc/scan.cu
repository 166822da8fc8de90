// Gated linear recurrence: for every channel of every sequence
//
//   s_t = sigmoid(z_t),  h_t = (1 - s_t) h_{t-1} + s_t f(v_t)                      f: identity, or "positive" (below)
//   G_t = dh_t + Q_{t+1},  Q_t = (1 - s_t) G_t,  dv_t = G_t s_t f'(v_t),  dz_t = G_t (f(v_t) - h_{t-1}) s_t (1 - s_t)
//
// with h_0 the state on entry, Q_{T+1} the gradient of the last state, dstate = Q_1.  A reset at t leaves h_{t-1} out; steps
// behind a sequence's length change nothing.
//
// Both directions are bound by memory: three streams of B T D elements forward, five backward.  A step is an affine map h -> a h + b, and maps
// compose, so the steps are walked in runs that start side by side: a warp has one run of 32 V channels in registers, forms its map, learns the
// maps of its CTA's runs in front of it through shared memory, and adds to every step what is left there of the state in front of the run.  The data are read once.  Where there are too few
// channels to fill the GPU, sequences are cut into segments: a first launch forms the segments' maps (which reads the inputs once more), and
// each CTA of the second starts from the maps in front of its segment.  Nothing waits on another CTA; the order of all sums is fixed.
//
// Digits: the smaller of s and 1 - s, e / (1 + e) with e = exp(-|z|), is exact to a few units of 2^-24, the larger is not further than that from 1.  With
// it the step is h + s (f - h) or f + (1 - s) (h - f), whichever it belongs to: 1 - s itself is rounded by up to 2^-25, always the same way, which
// is 3% after the million steps that a state lasts where s is 1e-6.  A map's factor has the same two forms (Map below), or it would bring that rounding back with
// every run (2.4% measured at z = -14.1 after 2^20 steps, 1e-6 so): what is left out of a state is summed beside the factor, one multiply-add a step.
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"
#include "rowwise.cuh"

namespace nlfa {
namespace scan {
namespace {

// Steps in a thread's registers; states at their starts are the backward's tape.  (float32 with 16: 96 KB of shared memory a CTA, backward of
// 32 x 1,024 x 768 168 us; with 8 100.  bf16, 64 x 1,024 x 768, with 8: 70 and 128 us, with 16 67 and 118 then, 60 and 98 now.)
template <typename T> constexpr int kRunOf = sizeof(T) == 4 ? 8 : 16;
constexpr int kWarps = 4;           // runs side by side in a CTA (or twice as many)
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
  int segments, segment;                            // parts of a sequence, their steps
  float4* maps;                                     // of the segments but the last walked: [B][segments][blocks][lane]
  void* h;
  float *last, *tape;
  // backward
  const void* dh;
  const float* dlast;
  void *dgate, *dvalue;
  float* dstate;
};

// exp(-a), a >= 0, and a quotient: 16-bit results need no more than the hardware's 2^-22; float32 ones are held to 2^-23 at every size of a
template <typename T> __device__ __forceinline__ float exp_minus(float a) { return fast_exp2(-kLog2e * a); }
template <> __device__ __forceinline__ float exp_minus<float>(float a) { return expf(-a); }
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename T> __device__ __forceinline__ float ratio(float a, float b) { return a * reciprocal(b); }
template <> __device__ __forceinline__ float ratio<float>(float a, float b) { return a / b; }

// Arithmetic on the V channels of a thread (of one, the second component is not looked at).
template <int V> __device__ __forceinline__ float2 fma_(float2 a, float2 b, float2 c) {
  if (V == 1) return make_float2(fmaf(a.x, b.x, c.x), 0.f);
  float2 r;
  unpack_f2(ffma2(pack_f2(a.x, a.y), pack_f2(b.x, b.y), pack_f2(c.x, c.y)), r.x, r.y);
  return r;
}
template <int V> __device__ __forceinline__ float2 add_(float2 a, float2 b) {
  if (V == 1) return make_float2(a.x + b.x, 0.f);
  float2 r;
  unpack_f2(fadd2(pack_f2(a.x, a.y), pack_f2(b.x, b.y)), r.x, r.y);
  return r;
}
template <int V> __device__ __forceinline__ float2 mul_(float2 a, float2 b) {
  if (V == 1) return make_float2(a.x * b.x, 0.f);
  float2 r;
  unpack_f2(fmul2(pack_f2(a.x, a.y), pack_f2(b.x, b.y)), r.x, r.y);
  return r;
}
template <int V> __device__ __forceinline__ float2 minus_(float2 a, float2 b) { return fma_<V>(b, make_float2(-1.f, -1.f), a); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// The smaller of sigmoid(z) and 1 - sigmoid(z), with the sign of z: minus where it is sigmoid(z).
template <typename T, int V> __device__ __forceinline__ float2 lesser(float2 z) {
  const float2 e = make_float2(exp_minus<T>(fabsf(z.x)), V == 2 ? exp_minus<T>(fabsf(z.y)) : 0.f), one = add_<V>(e, both(1.f));
  float2 r;
  if (sizeof(T) == 4) r = make_float2(e.x / one.x, V == 2 ? e.y / one.y : 0.f);
  else r = mul_<V>(e, make_float2(reciprocal(one.x), V == 2 ? reciprocal(one.y) : 0.f));
  return make_float2(copysignf(r.x, z.x), copysignf(r.y, z.y));
}
__device__ __forceinline__ bool is_minus(float x) { return __float_as_int(x) < 0; }
// y's channels: a where the sign is minus, else b
__device__ __forceinline__ float2 choose(float2 y, float2 a, float2 b) { return make_float2(is_minus(y.x) ? a.x : b.x, is_minus(y.y) ? a.y : b.y); }
template <typename T> __device__ __forceinline__ float sigmoid(float v) {
  const float e = exp_minus<T>(fabsf(v));
  return ratio<T>(v < 0.f ? e : 1.f, 1.f + e);
}
// f(v) and its slope.  positive: v + 1/2 from zero on, sigmoid(v) below
template <typename T, bool POSITIVE> __device__ __forceinline__ float2 mapped(float2 v) {
  if (!POSITIVE) return v;
  return make_float2(v.x < 0.f ? sigmoid<T>(v.x) : v.x + 0.5f, v.y < 0.f ? sigmoid<T>(v.y) : v.y + 0.5f);
}
template <typename T, bool POSITIVE> __device__ __forceinline__ float slope(float v) {
  if (!POSITIVE) return 1.f;
  const float p = sigmoid<T>(v);
  return v < 0.f ? p * (1.f - p) : 1.f;
}

// h after a step, y from lesser(): h - s (h - f), or f + (1 - s) (h - f)
template <int V> __device__ __forceinline__ float2 step(float2 y, float2 f, float2 h) { return fma_<V>(y, minus_<V>(h, f), choose(y, h, f)); }
// (1 - s) q
template <int V> __device__ __forceinline__ float2 kept(float2 y, float2 q) { return fma_<V>(y, q, choose(y, q, both(0.f))); }

// Two channels' maps h -> a h + b of some steps, (y, b, y, b).  Like a step's y: a where it is at most 1/2, else minus 1 - a, so that a state of which
// little is left out keeps its digits; minus zero: all of it is left, whatever it holds.  Behind a reset nothing is, whatever it held: y is -1, which 1 - a
// (at most 1/2) is not otherwise.  A factor that underflows is +0: what is not finite goes through it as NaN.
constexpr float kNothing = -1.f;
__device__ __forceinline__ bool is_identity(float y) { return __float_as_int(y) == static_cast<int>(0x80000000u); }
template <bool RESET> __device__ __forceinline__ float apply_one(float y, float b, float h) {
  const float r = (is_identity(y) ? b : fmaf(y, h, b)) + (is_minus(y) ? h : 0.f);
  return RESET && y == kNothing ? b : r;
}
template <bool RESET> __device__ __forceinline__ float2 apply(const float4& m, float2 h) {
  return make_float2(apply_one<RESET>(m.x, m.y, h.x), apply_one<RESET>(m.z, m.w, h.y));
}
// m, then n
template <bool RESET> __device__ __forceinline__ float both_left(float m, float n) {
  const float a = is_minus(m) ? 1.f + m : m, c = a * (is_minus(n) ? 1.f + n : n), out = fmaf(n, a, m);
  const float y = is_minus(m) && is_minus(n) && out >= -0.5f ? out : c;
  return RESET && (m == kNothing || n == kNothing) ? kNothing : y;
}
template <bool RESET> __device__ __forceinline__ float4 then(const float4& m, const float4& n) {
  const float2 b = apply<RESET>(n, make_float2(m.y, m.w));
  return make_float4(both_left<RESET>(m.x, n.x), b.x, both_left<RESET>(m.z, n.z), b.y);
}
__device__ __forceinline__ float4 identity() { return make_float4(-0.f, 0.f, -0.f, 0.f); }
// The map of a run's steps, formed one by one.  What is left out is only looked at where every step leaves more than half.
template <int V> struct Map {
  float2 a, out, b;                                            // what is left of the state, minus what is left out, what is added
  __device__ __forceinline__ Map() : a(both(1.f)), out(both(-0.f)), b(both(0.f)) {}
  __device__ __forceinline__ void leave(float2 y) {            // y of lesser()
    out = fma_<V>(y, a, out);
    a = kept<V>(y, a);
  }
  // (resets: the same ones for all channels of a sequence)
  template <bool RESET> __device__ __forceinline__ float4 pack(bool resets) const {
    if (RESET && resets) return make_float4(kNothing, b.x, kNothing, b.y);
    return make_float4(a.x > 0.5f ? out.x : a.x, b.x, a.y > 0.5f ? out.y : a.y, b.y);
  }
};

// The state in front of this thread's run, given its run's map, and the state behind the CTA's runs in `carry`.  `maps`: in shared memory, [2][WARPS][lane];
// `order`: this warp's place in its CTA, in the order in which the runs are walked.
template <int WARPS> __host__ __device__ constexpr int exchange_bytes() { return WARPS > 1 ? 2 * WARPS * 32 * 16 : 0; }
template <int WARPS, bool RESET>
__device__ __forceinline__ float2 enter(float4* maps, int buf, int order, float4 own, float2& carry) {
  if (WARPS == 1) {
    const float2 in = carry;
    carry = apply<RESET>(own, in);
    return in;
  }
  float4* mine = maps + buf * WARPS * 32 + (threadIdx.x & 31);
  mine[32 * order] = own;
  __syncthreads();
  float2 in = carry;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w == order) in = carry;
    carry = apply<RESET>(mine[32 * w], carry);
  }
  return in;
}

// Steps of a sequence that count.
__device__ __forceinline__ int live_steps(const Params& p, int b) {
  if (p.lengths == nullptr) return p.T;
  const long long n = p.length_bytes == 8 ? static_cast<const long long*>(p.lengths)[b] : static_cast<const int*>(p.lengths)[b];
  return n < 0 ? 0 : n < p.T ? static_cast<int>(n) : p.T;
}
// Resets of the steps t0 .. t0 + run - 1, of which the first n count.
__device__ __forceinline__ unsigned reset_bits(int run, const Params& p, int b, int t0, int n) {
  const int i = threadIdx.x & 31;
  const bool on = i < run && i < n && p.reset[static_cast<long long>(b) * p.T + t0 + i] != 0;
  return __ballot_sync(0xffffffffu, on);
}

// Where a thread works: channels c (and c + 1) of sequence b; a lane behind the last channel (not `live`) walks along and writes nothing.
struct Place {
  int b, c, warp, segment, block;
  int t0, t1;                                         // the segment's steps
  bool live;
  template <int V> __device__ static Place of(const Params& p) {
    Place w;
    const unsigned column = blockIdx.x / p.segments;
    w.segment = static_cast<int>(blockIdx.x - column * p.segments);
    w.b = static_cast<int>(column / p.blocks);
    w.block = static_cast<int>(column - w.b * p.blocks);
    w.c = w.block * 32 * V + V * (threadIdx.x & 31);
    w.warp = threadIdx.x >> 5;
    w.live = w.c < p.D;
    w.t0 = w.segment * p.segment;
    w.t1 = p.T - w.t0 < p.segment ? p.T : w.t0 + p.segment;
    return w;
  }
  __device__ float4* map(const Params& p, int s) const {
    return p.maps + ((static_cast<long long>(b) * p.segments + s) * p.blocks + block) * 32 + (threadIdx.x & 31);
  }
};

__device__ __forceinline__ void async_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// One tensor's values of a warp's run.  Pairs (V = 2): 32 lanes' Raw by step, in two buffers of shared memory, asked for 16 bytes at a time while the run before is
// walked (4 bytes at a time, by the lane that needs them, cost as many instructions as the arithmetic: forward of 64 x 1,024 x 768 96 us).
// Single channels lie on no boundary that an asynchronous copy could start at: they wait in registers meanwhile.
template <typename T, int V> struct Stream {
  static constexpr int kRun = kRunOf<T>;
  using Raw = typename Pack<T, V>::Raw;
  static constexpr int kRow = 32 * static_cast<int>(sizeof(Raw)), kChunks = kRow / 16;      // of a step
  static_assert(kRun * kChunks % 32 == 0, "whole copies per lane");
  static constexpr int kBytes = kRun * kRow;                                                // of a buffer
  T* at;                                              // this thread's channels, first step
  long long stride;
  uint8_t* mem;                                       // this warp's buffers
  int left;                                           // channels from this thread's on
  Raw next[V == 1 ? kRun : 1];

  __device__ __forceinline__ Raw* slot(int buf, int i) const { return reinterpret_cast<Raw*>(mem + buf * kBytes + i * kRow) + (threadIdx.x & 31); }
  // the 16 bytes j of this lane: of step i0 + j kStride, from channel at + shift on
  static constexpr int kCopies = kRun * kChunks / 32, kStride = 32 / kChunks;
  template <typename F> __device__ __forceinline__ void chunks(T* from, long long step, int t0, int n, F&& f) const {
    const int lane = threadIdx.x & 31, i0 = lane / kChunks, shift = lane % kChunks * (16 / static_cast<int>(sizeof(T))) - V * lane;
    if (shift >= left) return;
    T* s = from + (t0 + i0) * step + shift;
    const long long more = kStride * step;
    if (n >= kRun) {
#pragma unroll
      for (int j = 0; j < kCopies; ++j, s += more) f(s, (lane + 32 * j) * 16);
    } else {
#pragma unroll
      for (int j = 0; j < kCopies; ++j, s += more)
        if (i0 + j * kStride < n) f(s, (lane + 32 * j) * 16);
    }
  }
  __device__ __forceinline__ void ask(int buf, int t0, int n) {
    if constexpr (V == 2) {
      const uint32_t dst = smem_u32(mem + buf * kBytes);
      chunks(at, stride, t0, n, [&](const T* s, int byte) { async_copy16(dst + byte, s); });
    } else if (left > 0) {
      const T* s = at + t0 * stride;
#pragma unroll
      for (int i = 0; i < kRun; ++i, s += stride)
        if (i < n) next[i] = *reinterpret_cast<const Raw*>(s);
    }
  }
  // (before the buffer that was asked for is read)
  __device__ __forceinline__ void settle(int buf) const {
    if constexpr (V == 1) {
#pragma unroll
      for (int i = 0; i < kRun; ++i) *slot(buf, i) = next[i];
    }
  }
  __device__ __forceinline__ float2 get(int buf, int i) const { return Pack<T, V>::get(*slot(buf, i)); }
};
// A result's values, through the buffer of an input that has been read (each lane its own places), 16 bytes at a time.
template <typename T, int V> struct Result {
  using Raw = typename Pack<T, V>::Raw;
  T* at;
  long long stride;
  __device__ __forceinline__ void put(const Stream<T, V>& through, int buf, int t0, int i, float2 v) const {
    if constexpr (V == 2) *through.slot(buf, i) = Pack<T, V>::put(v);
    else if (through.left > 0) *reinterpret_cast<Raw*>(at + (t0 + i) * stride) = Pack<T, V>::put(v);
  }
  // (after a __syncwarp)
  __device__ __forceinline__ void write(const Stream<T, V>& through, int buf, int t0, int n) const {
    if constexpr (V == 2) {
      const uint8_t* src = through.mem + buf * Stream<T, V>::kBytes;
      through.chunks(at, stride, t0, n, [&](T* to, int byte) { *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(src + byte); });
    }
  }
};

template <typename T, int V, int WARPS> constexpr int smem_bytes(int streams) {
  return exchange_bytes<WARPS>() + WARPS * streams * 2 * Stream<T, V>::kBytes;
}
template <typename T, int V, int STREAMS>
__device__ __forceinline__ Stream<T, V> stream_of(const Params& p, uint8_t* mem, int which, const void* base, long long b_stride, long long t_stride, const Place& w) {
  return {const_cast<T*>(static_cast<const T*>(base)) + w.b * b_stride + w.c, t_stride, mem + (w.warp * STREAMS + which) * 2 * Stream<T, V>::kBytes, p.D - w.c, {}};
}
template <typename T, int V> __device__ __forceinline__ Result<T, V> result_of(const Params& p, void* base, const Place& w) {
  return {static_cast<T*>(base) + static_cast<long long>(w.b) * p.T * p.D + w.c, p.D};
}
// V float32 values
template <int V> __device__ __forceinline__ float2 load_state(const float* p, bool live) {
  float2 v = make_float2(0.f, 0.f);
  if (live) {
    v.x = p[0];
    if (V == 2) v.y = p[1];
  }
  return v;
}
template <int V> __device__ __forceinline__ void store_state(float* p, float2 v) {
  p[0] = v.x;
  if (V == 2) p[1] = v.y;
}

template <typename T, int V, int WARPS, bool POSITIVE, bool RESET>
__global__ void __launch_bounds__(32 * WARPS)
scan_fwd_kernel(const Params p) {
  constexpr int kRun = kRunOf<T>, kStretch = WARPS * kRun;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* maps = reinterpret_cast<float4*>(smem);
  uint8_t* mem = smem + exchange_bytes<WARPS>();
  grid_dep_wait();
  grid_dep_release();
  const Place w = Place::of<V>(p);
  const long long row = static_cast<long long>(w.b) * p.D + w.c;
  Stream<T, V> zs = stream_of<T, V, 2>(p, mem, 0, p.gate, p.gate_b, p.gate_t, w), vs = stream_of<T, V, 2>(p, mem, 1, p.value, p.value_b, p.value_t, w);
  const Result<T, V> out = result_of<T, V>(p, p.h, w);
  const int live = live_steps(p, w.b), runs = (p.T + kRun - 1) / kRun, first = w.warp * kRun;
  auto ask = [&](int buf, int t0) {
    zs.ask(buf, t0, live - t0);
    vs.ask(buf, t0, live - t0);
    async_commit();
  };
  auto settle = [&](int buf) {
    zs.settle(buf);
    vs.settle(buf);
  };
  ask(0, w.t0 + first);
  settle(0);
  float2 carry = load_state<V>(p.state + row, w.live && p.state != nullptr);
#pragma unroll 4
  for (int s = 0; s < w.segment; ++s) carry = apply<RESET>(*w.map(p, s), carry);
  int buf = 0;
  for (int from = w.t0; from < w.t1; from += kStretch, buf ^= 1) {
    const int t0 = from + first, n = live - t0;                // (steps of this run that count: n, if it is between 0 and kRun)
    const unsigned resets = RESET ? reset_bits(kRun, p, w.b, t0, n) : 0u;
    async_wait();
    __syncwarp();
    if (from + kStretch < w.t1) ask(buf ^ 1, t0 + kStretch);
    // h from nothing, and what is left of the state in front of the run, behind every step
    float2 h[kRun], left[kRun];
    Map<V> m;
    auto walk = [&](auto whole) {
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        if (decltype(whole)::value || i < n) {                 // (a step that does not count leaves h as it is)
          if (RESET && (resets >> i & 1u)) m.b = both(0.f);
          const float2 y = lesser<T, V>(zs.get(buf, i));
          m.leave(y);
          m.b = step<V>(y, mapped<T, POSITIVE>(vs.get(buf, i)), m.b);
        }
        h[i] = m.b;
        left[i] = m.a;
      }
    };
    if (n >= kRun) walk(std::true_type{});
    else walk(std::false_type{});
    const float4 map = m.template pack<RESET>(resets != 0u);
    const float2 in = enter<WARPS, RESET>(maps, buf, w.warp, map, carry);
    if (t0 < p.T) {
      if (p.tape != nullptr && w.live) store_state<V>(p.tape + (static_cast<long long>(w.b) * runs + t0 / kRun) * p.D + w.c, in);
      // (a factor of a run's steps is rounded 16 times at most: 2^-21, forgotten at the end of the run)
      auto put = [&](auto whole) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          if (!decltype(whole)::value && t0 + i >= p.T) break;
          float2 v = h[i];
          if (!RESET || !(resets & ((2u << i) - 1u))) v = fma_<V>(left[i], in, h[i]);
          if (!decltype(whole)::value && i >= n) v = both(0.f);
          out.put(zs, buf, t0, i, v);
        }
      };
      if (n >= kRun) put(std::true_type{});
      else put(std::false_type{});
      if (p.T - t0 <= kRun) {                                  // the state behind the last step, for the next call: as the next run would get it
        const float2 state = apply<RESET>(map, in);
        if (w.live) store_state<V>(p.last + row, state);
        if (n >= p.T - t0) out.put(zs, buf, t0, p.T - 1 - t0, state);
      }
      __syncwarp();
      out.write(zs, buf, t0, p.T - t0);
    }
    settle(buf ^ 1);
  }
  if (p.T == 0 && w.live) store_state<V>(p.last + row, carry);
}

template <typename T, int V, int WARPS, bool POSITIVE, bool RESET>
__global__ void __launch_bounds__(32 * WARPS)
scan_bwd_kernel(const Params p) {
  constexpr int kRun = kRunOf<T>, kStretch = WARPS * kRun;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* maps = reinterpret_cast<float4*>(smem);
  uint8_t* mem = smem + exchange_bytes<WARPS>();
  grid_dep_wait();
  grid_dep_release();
  const Place w = Place::of<V>(p);
  const long long row = static_cast<long long>(w.b) * p.D + w.c;
  Stream<T, V> zs = stream_of<T, V, 3>(p, mem, 0, p.gate, p.gate_b, p.gate_t, w), vs = stream_of<T, V, 3>(p, mem, 1, p.value, p.value_b, p.value_t, w),
                     gs = stream_of<T, V, 3>(p, mem, 2, p.dh, static_cast<long long>(p.T) * p.D, p.D, w);
  const Result<T, V> dgate = result_of<T, V>(p, p.dgate, w), dvalue = result_of<T, V>(p, p.dvalue, w);
  const int live = live_steps(p, w.b), runs = (p.T + kRun - 1) / kRun, first = w.warp * kRun;
  auto ask = [&](int buf, int t0) {
    zs.ask(buf, t0, live - t0);
    vs.ask(buf, t0, live - t0);
    if (p.dh != nullptr) gs.ask(buf, t0, live - t0);
    async_commit();
  };
  auto state_at = [&](int t0) {
    return load_state<V>(p.tape + (static_cast<long long>(w.b) * runs + t0 / kRun) * p.D + w.c, w.live && t0 >= 0 && t0 < live);
  };
  auto settle = [&](int buf) {
    zs.settle(buf);
    vs.settle(buf);
    if (p.dh != nullptr) gs.settle(buf);
  };
  if (p.dh == nullptr) {
#pragma unroll
    for (int i = 0; i < 2 * kRun; ++i) *gs.slot(0, i) = Pack<T, V>::put(both(0.f));
  }
  const int last = w.t0 + (w.t1 - w.t0 - 1) / kStretch * kStretch;
  if (p.T > 0) ask(0, last + first);
  settle(0);
  float2 next = state_at(last + first), carry = load_state<V>(p.dlast + row, w.live && p.dlast != nullptr);
#pragma unroll 4
  for (int s = p.segments - 1; s > w.segment; --s) carry = apply<RESET>(*w.map(p, s), carry);
  int buf = 0;
  for (int from = last; from >= w.t0 && p.T > 0; from -= kStretch, buf ^= 1) {
    const int t0 = from + first, n = live - t0;
    const unsigned resets = RESET ? reset_bits(kRun, p, w.b, t0, n) : 0u;
    async_wait();
    __syncwarp();
    float2 h = next;
    if (from > w.t0) {
      ask(buf ^ 1, t0 - kStretch);
      next = state_at(t0 - kStretch);
    }
    // forward through the run: y of lesser(), and h of the step before less f; and back: the map of what comes from behind the run
    float2 y[kRun], rest[kRun];
    Map<V> m;
    auto grad = [&](int i) { return gs.get(buf, i); };         // (without dh: zeros)
    auto walk = [&](auto whole) {
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        y[i] = rest[i] = both(0.f);
        if (decltype(whole)::value || i < n) {
          if (RESET && (resets >> i & 1u)) h = both(0.f);
          const float2 f = mapped<T, POSITIVE>(vs.get(buf, i));
          y[i] = lesser<T, V>(zs.get(buf, i));
          rest[i] = minus_<V>(h, f);
          h = fma_<V>(y[i], rest[i], choose(y[i], h, f));
        }
      }
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i) {
        if (decltype(whole)::value || i < n) {
          m.leave(y[i]);
          m.b = kept<V>(y[i], add_<V>(m.b, grad(i)));
          if (RESET && (resets >> i & 1u)) m.b = both(0.f);
        }
      }
    };
    if (n >= kRun) walk(std::true_type{});
    else walk(std::false_type{});
    float2 q = enter<WARPS, RESET>(maps, buf, WARPS - 1 - w.warp, m.template pack<RESET>(resets != 0u), carry);
    if (t0 < p.T) {
      auto put = [&](auto whole) {
#pragma unroll
        for (int i = kRun - 1; i >= 0; --i) {
          if (!decltype(whole)::value && t0 + i >= p.T) continue;
          float2 dz = both(0.f), dv = both(0.f);
          if (decltype(whole)::value || i < n) {
            // l = |y|, of s and 1 - s the smaller
            const float2 g = add_<V>(grad(i), q), l = make_float2(fabsf(y[i].x), fabsf(y[i].y)), minus_l = make_float2(-l.x, -l.y);
            dv = mul_<V>(g, choose(y[i], l, add_<V>(both(1.f), minus_l)));
            if (POSITIVE) {
              const float2 v = vs.get(buf, i);
              dv = mul_<V>(dv, make_float2(slope<T, POSITIVE>(v.x), V == 2 ? slope<T, POSITIVE>(v.y) : 0.f));
            }
            dz = mul_<V>(mul_<V>(g, rest[i]), fma_<V>(y[i], y[i], minus_l));            // l (1 - l) = l - y y
            q = kept<V>(y[i], g);
          }
          if (RESET && (resets >> i & 1u)) q = both(0.f);
          if (V == 2 || p.dgate != nullptr) dgate.put(zs, buf, t0, i, dz);
          if (V == 2 || p.dvalue != nullptr) dvalue.put(vs, buf, t0, i, dv);
        }
      };
      if (n >= kRun) put(std::true_type{});
      else put(std::false_type{});
      __syncwarp();
      if (p.dgate != nullptr) dgate.write(zs, buf, t0, p.T - t0);
      if (p.dvalue != nullptr) dvalue.write(vs, buf, t0, p.T - t0);
    }
    settle(buf ^ 1);
  }
  if (w.live && w.segment == 0 && w.warp == 0 && p.dstate != nullptr) store_state<V>(p.dstate + row, carry);
}

// The maps of the segments: of h from the gates and values, or (BACKWARD) of Q from the gates and dh.  A warp walks a quarter of its segment by itself.
template <typename T, int V, bool POSITIVE, bool RESET, bool BACKWARD>
__global__ void __launch_bounds__(32 * kWarps)
scan_maps_kernel(const Params p) {
  constexpr int kRun = kRunOf<T>;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* maps = reinterpret_cast<float4*>(smem);
  uint8_t* mem = smem + exchange_bytes<kWarps>();
  grid_dep_wait();
  grid_dep_release();
  const Place w = Place::of<V>(p);
  if (w.segment == (BACKWARD ? 0 : p.segments - 1)) return;    // (nobody asks for the last one's)
  const bool with = !BACKWARD || p.dh != nullptr;
  Stream<T, V> zs = stream_of<T, V, 2>(p, mem, 0, p.gate, p.gate_b, p.gate_t, w);
  Stream<T, V> vs = BACKWARD ? stream_of<T, V, 2>(p, mem, 1, p.dh, static_cast<long long>(p.T) * p.D, p.D, w)
                                   : stream_of<T, V, 2>(p, mem, 1, p.value, p.value_b, p.value_t, w);
  const int live = live_steps(p, w.b), quarter = p.segment / kWarps, begin = w.t0 + w.warp * quarter;
  const int end = w.t1 - begin < quarter ? w.t1 : begin + quarter;
  const int runs = end > begin ? (end - begin + kRun - 1) / kRun : 0;
  auto at = [&](int r) { return begin + (BACKWARD ? runs - 1 - r : r) * kRun; };
  auto ask = [&](int buf, int t0) {
    zs.ask(buf, t0, live - t0);
    if (with) vs.ask(buf, t0, live - t0);
    async_commit();
  };
  auto settle = [&](int buf) {
    zs.settle(buf);
    if (with) vs.settle(buf);
  };
  if (runs > 0) ask(0, at(0));
  settle(0);
  float4 all = identity();
  for (int r = 0, buf = 0; r < runs; ++r, buf ^= 1) {
    const int t0 = at(r), n = live - t0;
    const unsigned resets = RESET ? reset_bits(kRun, p, w.b, t0, n) : 0u;
    async_wait();
    __syncwarp();
    if (r + 1 < runs) ask(buf ^ 1, at(r + 1));
    Map<V> m;
    auto walk = [&](auto whole) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const int i = BACKWARD ? kRun - 1 - j : j;
        if (decltype(whole)::value || i < n) {
          if (!BACKWARD && RESET && (resets >> i & 1u)) m.b = both(0.f);
          const float2 y = lesser<T, V>(zs.get(buf, i)), v = with ? vs.get(buf, i) : both(0.f);
          m.leave(y);
          m.b = BACKWARD ? kept<V>(y, add_<V>(m.b, v)) : step<V>(y, mapped<T, POSITIVE>(v), m.b);
          if (BACKWARD && RESET && (resets >> i & 1u)) m.b = both(0.f);
        }
      }
    };
    if (n >= kRun) walk(std::true_type{});
    else walk(std::false_type{});
    all = then<RESET>(all, m.template pack<RESET>(resets != 0u));
    settle(buf ^ 1);
  }
  const int lane = threadIdx.x & 31;
  maps[32 * w.warp + lane] = all;
  __syncthreads();
  if (w.warp != 0) return;
  all = maps[32 * (BACKWARD ? kWarps - 1 : 0) + lane];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) all = then<RESET>(all, maps[32 * (BACKWARD ? kWarps - 1 - i : i) + lane]);
  *w.map(p, w.segment) = all;
}

// ------------------------------------------------------------------------------------------------ host

int element_bytes(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }
int run_of(int dtype) { return dtype == NLFA_DTYPE_F32 ? kRunOf<float> : kRunOf<__half>; }

// Into how many segments the sequences are cut, and how many runs a CTA walks side by side: by the columns (of 64 channels of a sequence) there are.
//   up to a sixth of what runs at once: segments, twice as many CTAs as run at once.  1 x 131,072 x 1,024 bf16 (16 columns), forward and backward,
//     272 + 417 us, uncut with 8 warps 1,627 + 2,720; 2,048 steps of 64 columns 21 + 28, uncut 27 + 45; of 96 29 + 41, uncut 27 + 46 (float32 55 + 70, uncut 62 + 80); 16,384 of 96 197 + 283,
//     uncut 208 + 346; but 2,048 of 128 36 + 50, uncut 28 + 46: the maps read the inputs once more.
//   up to what runs at once (channels by themselves: of 32): 8 warps.  1,024 steps of 192 23 + 39, with 4 warps 24 + 38 (float32 44 + 59, 55 + 75); of 384 36 + 60, with 4 39 + 64.
//   else 4: of 768 60 + 97, with 8 65 + 110 (float32 117 + 182, 114 + 175).
constexpr int kCtasPerSm = 4;
struct Cut {
  int segments, segment;
};
Cut cut(int B, int T, int D, int dtype) {
  const long long columns = static_cast<long long>(B) * ((D + 63) / 64), stretch = kWarps * run_of(dtype);
  const long long at_once = static_cast<long long>(kCtasPerSm) * sm_count();
  if (columns > 0 && 6 * columns <= at_once && T >= 16 * stretch) {
    const long long parts = 2 * at_once / columns, length = (T + parts * stretch - 1) / (parts * stretch) * stretch;
    return {static_cast<int>((T + length - 1) / length), static_cast<int>(length)};
  }
  return {1, T > 0 ? T : 1};
}
size_t maps_bytes(int B, int T, int D, int dtype) {
  const Cut c = cut(B, T, D, dtype);
  // (a thread has one channel where pairs do not lie right: twice as many blocks)
  return c.segments > 1 ? static_cast<size_t>(B) * c.segments * ((static_cast<size_t>(D) + 31) / 32) * 32 * sizeof(float4) : 0;
}

template <typename Kernel>
int launch(Kernel* kernel, int warps, int smem, const Params& p, cudaStream_t st) {
  if (smem > 48 * 1024) {
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (rc != NLFA_OK) return rc;
  }
  const cudaError_t e = launch_kernel(kernel, dim3(static_cast<unsigned>(p.B) * p.blocks * p.segments), dim3(32u * warps), smem, st,
                                      overlap_launches(kOverlapRowwise), p);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

template <typename T, int V, int WARPS, bool POSITIVE, bool RESET>
int run_warps(const Params& p, bool backward, cudaStream_t st) {
  return backward ? launch(scan_bwd_kernel<T, V, WARPS, POSITIVE, RESET>, WARPS, smem_bytes<T, V, WARPS>(3), p, st)
                  : launch(scan_fwd_kernel<T, V, WARPS, POSITIVE, RESET>, WARPS, smem_bytes<T, V, WARPS>(2), p, st);
}
template <typename T, int V, bool POSITIVE, bool RESET>
int run_reset(Params p, bool backward, cudaStream_t st) {
  p.blocks = (p.D + 32 * V - 1) / (32 * V);
  if (static_cast<long long>(p.B) * p.blocks * p.segments > 0x7fffffffll) return NLFA_ERR_BAD_SHAPE;
  if (p.T <= kRunOf<T>) return run_warps<T, V, 1, POSITIVE, RESET>(p, backward, st);
  if (p.segments > 1) {
    const int smem = smem_bytes<T, V, kWarps>(2);
    const int rc = backward ? launch(scan_maps_kernel<T, V, false, RESET, true>, kWarps, smem, p, st)
                            : launch(scan_maps_kernel<T, V, POSITIVE, RESET, false>, kWarps, smem, p, st);
    if (rc != NLFA_OK) return rc;
  }
  const bool more = p.segments == 1 && static_cast<long long>(p.B) * p.blocks <= static_cast<long long>(kCtasPerSm) * sm_count();
  return more ? run_warps<T, V, 2 * kWarps, POSITIVE, RESET>(p, backward, st) : run_warps<T, V, kWarps, POSITIVE, RESET>(p, backward, st);
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
  // two channels a thread where every row begins on 16 bytes and ends on a whole copy; a stride that no step is taken along does not matter
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.h) |
                        reinterpret_cast<uintptr_t>(p.dh) | reinterpret_cast<uintptr_t>(p.dgate) | reinterpret_cast<uintptr_t>(p.dvalue);
  const long long strides = (p.B > 1 ? p.gate_b | p.value_b : 0) | (p.T > 1 ? p.gate_t | p.value_t : 0) | p.D;
  const bool pairs = strides % static_cast<long long>(16 / sizeof(T)) == 0 && all % 16 == 0;
  return pairs ? run_width<T, 2>(p, activation, backward, st) : run_width<T, 1>(p, activation, backward, st);
}
int run(const Params& p, int dtype, int activation, bool backward, cudaStream_t st) {
  if (dtype == NLFA_DTYPE_F32) return run_typed<float>(p, activation, backward, st);
  if (dtype == NLFA_DTYPE_F16) return run_typed<__half>(p, activation, backward, st);
  return run_typed<__nv_bfloat16>(p, activation, backward, st);
}

bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check(int dtype, int activation, int length_bytes, const void* lengths, int B, int T, int D) {
  if (B < 0 || T < 0 || D < 0 || B > kMostExtent || T > kMostExtent || D > kMostExtent) return NLFA_ERR_BAD_SHAPE;
  if (!rowwise::dtype_ok(dtype)) return NLFA_ERR_BAD_DTYPE;
  if (activation != NLFA_SCAN_NONE && activation != NLFA_SCAN_POSITIVE) return NLFA_ERR_BAD_ARGUMENT;
  if (lengths != nullptr && length_bytes != 4 && length_bytes != 8) return NLFA_ERR_BAD_ARGUMENT;
  if (lengths != nullptr && !aligned_to(lengths, length_bytes)) return NLFA_ERR_MISALIGNED;
  return NLFA_OK;
}

size_t tape_bytes(int B, int T, int D, int dtype) {
  const size_t run = run_of(dtype);
  return static_cast<size_t>(B) * ((static_cast<size_t>(T) + run - 1) / run) * static_cast<size_t>(D) * sizeof(float);
}
void set_cut(Params& p, int dtype, void* scratch) {
  const Cut c = cut(p.B, p.T, p.D, dtype);
  p.segments = c.segments;
  p.segment = c.segment;
  p.maps = static_cast<float4*>(scratch);
}

}  // namespace
}  // namespace scan
}  // namespace nlfa

using namespace nlfa;
using namespace nlfa::scan;

extern "C" {

size_t nlfa_gated_scan_tape_bytes(int B, int T, int D, int dtype) {
  return check(dtype, NLFA_SCAN_NONE, 0, nullptr, B, T, D) == NLFA_OK ? tape_bytes(B, T, D, dtype) : 0;
}
size_t nlfa_gated_scan_scratch_bytes(int B, int T, int D, int dtype) {
  return check(dtype, NLFA_SCAN_NONE, 0, nullptr, B, T, D) == NLFA_OK ? maps_bytes(B, T, D, dtype) : 0;
}

int nlfa_gated_scan_fwd(const void* gate, long long gate_b, long long gate_t, const void* value, long long value_b, long long value_t,
                        int dtype, const float* state, const unsigned char* reset, const void* lengths, int length_bytes, int activation,
                        int B, int T, int D, void* h, float* last, void* tape, size_t bytes, void* scratch, size_t scratch_bytes,
                        void* stream) {
  const int rc = check(dtype, activation, length_bytes, lengths, B, T, D);
  if (rc != NLFA_OK) return rc;
  if (B == 0 || D == 0) return NLFA_OK;
  if (!last || (T > 0 && (!gate || !value || !h))) return NLFA_ERR_NULL_POINTER;
  const int e = element_bytes(dtype);
  if (!aligned_to(gate, e) || !aligned_to(value, e) || !aligned_to(h, e) || !aligned_to(state, 4) || !aligned_to(last, 4) || !aligned_to(tape, 4))
    return NLFA_ERR_MISALIGNED;
  const size_t need = maps_bytes(B, T, D, dtype);
  if (need > 0 && !scratch) return NLFA_ERR_NULL_POINTER;
  if (!rowwise::aligned16(scratch)) return NLFA_ERR_MISALIGNED;
  if ((tape != nullptr && bytes < tape_bytes(B, T, D, dtype)) || scratch_bytes < need) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  Params p{};
  p.gate = gate; p.gate_b = gate_b; p.gate_t = gate_t;
  p.value = value; p.value_b = value_b; p.value_t = value_t;
  p.state = state; p.reset = reset; p.lengths = lengths; p.length_bytes = length_bytes;
  p.B = B; p.T = T; p.D = D;
  p.h = h; p.last = last; p.tape = static_cast<float*>(tape);
  set_cut(p, dtype, scratch);
  return run(p, dtype, activation, false, static_cast<cudaStream_t>(stream));
}

int nlfa_gated_scan_bwd(const void* dh, const float* dlast, const void* gate, long long gate_b, long long gate_t, const void* value,
                        long long value_b, long long value_t, int dtype, const unsigned char* reset, const void* lengths, int length_bytes,
                        int activation, int B, int T, int D, const void* tape, size_t bytes, void* dgate, void* dvalue, float* dstate,
                        void* scratch, size_t scratch_bytes, void* stream) {
  const int rc = check(dtype, activation, length_bytes, lengths, B, T, D);
  if (rc != NLFA_OK) return rc;
  if (B == 0 || D == 0 || (!dgate && !dvalue && !dstate)) return NLFA_OK;
  if (T > 0 && (!gate || !value || !tape)) return NLFA_ERR_NULL_POINTER;
  const int e = element_bytes(dtype);
  if (!aligned_to(gate, e) || !aligned_to(value, e) || !aligned_to(dh, e) || !aligned_to(dgate, e) || !aligned_to(dvalue, e) ||
      !aligned_to(dlast, 4) || !aligned_to(dstate, 4) || !aligned_to(tape, 4))
    return NLFA_ERR_MISALIGNED;
  const size_t need = maps_bytes(B, T, D, dtype);
  if (need > 0 && !scratch) return NLFA_ERR_NULL_POINTER;
  if (!rowwise::aligned16(scratch)) return NLFA_ERR_MISALIGNED;
  if ((T > 0 && bytes < tape_bytes(B, T, D, dtype)) || scratch_bytes < need) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  Params p{};
  p.gate = gate; p.gate_b = gate_b; p.gate_t = gate_t;
  p.value = value; p.value_b = value_b; p.value_t = value_t;
  p.reset = reset; p.lengths = lengths; p.length_bytes = length_bytes;
  p.B = B; p.T = T; p.D = D;
  p.tape = static_cast<float*>(const_cast<void*>(tape));
  p.dh = dh; p.dlast = dlast; p.dgate = dgate; p.dvalue = dvalue; p.dstate = dstate;
  set_cut(p, dtype, scratch);
  return run(p, dtype, activation, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
