// Gated feed-forward layer, forward and backward:
//
//   g = x Wg^T,  u = x Wu^T,  h = f(g) u,  y = h Wd^T                              f: silu, gelu, relu
//   dh = dy Wd,  du = dh f(g),  dg = dh u f'(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// Bound by the tensor cores: 2 N F (2 d + o) operations forward and twice that backward, in four launches of products (ffn_tc.cu).  g, u and dh exist in
// tensor memory alone (where few tiles have long sums, in float32 beside the products: apart() below); the tape keeps f(g) and u f'(g) for the
// backward.  Between the products h, dg and du are operands: 16 bits (float32: three bf16 parts), one rounding each beside that of the results.
//
// This file has what goes around the products: 16-bit copies of operands that TMA cannot read as they are, the list of tiles and
// parts, and the powers of two that hold float16's h, dg and du inside their type's range, token by token.
#include <cmath>
#include <type_traits>

#include "ffn.cuh"
#include "rowwise.cuh"

namespace nlfa {

unsigned* status_block();      // api.cu

namespace ffn {
namespace {

using rowwise::aligned16;
using rowwise::dtype_ok;

enum { kCopyX = 1, kCopyGate = 2, kCopyUp = 4, kCopyDown = 8 };

struct Call {
  int x_dtype, w_dtype, dtype;      // dtype: what the products run in
  int n, d, F, o;
  int copies;                       // operands that are converted or re-laid (otherwise the products read the caller's)
  int train;
};

size_t up(size_t v) { return (v + 255) / 256 * 256; }
int up64(int v) { return (v + 63) / 64 * 64; }
int element_bytes(int dtype) { return dtype == NLFA_DTYPE_F32 ? 4 : 2; }
bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
__host__ __device__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

constexpr int kMostRows = 1 << 30, kMostWidth = 1 << 24;
int check_call(const Call& c) {
  if (c.n < 0 || c.d < 1 || c.F < 1 || c.o < 1 || c.n > kMostRows || c.d > kMostWidth || c.F > kMostWidth || c.o > kMostWidth)
    return NLFA_ERR_BAD_SHAPE;
  if (!dtype_ok(c.x_dtype) || !dtype_ok(c.w_dtype) || !dtype_ok(c.dtype)) return NLFA_ERR_BAD_DTYPE;
  return NLFA_OK;
}

bool must_copy(const void* p, int type, int dtype, int cols) { return dtype == NLFA_DTYPE_F32 || type != dtype || cols % 64 != 0 || !aligned16(p); }

bool is_few(const void* x, const void* gate, const void* up, const void* down, int w_dtype, int dtype, int n, int d, int F, int train) {
  if (n > kFewTokens || (n > kVeryFewTokens && static_cast<long long>(n) * d * F > kFewProducts)) return false;
  return !train && few_types(w_dtype, dtype) && d % 8 == 0 && F % 8 == 0 && aligned16(x) && aligned16(gate) && aligned16(up) &&
         aligned16(down);
}

constexpr size_t kHeaderBytes = 256;          // Limits, BwdLimits

// What the forward leaves for the backward, and (inference) the forward's own workspace.
struct Layout {
  int planes, n_rows, d_pad, f_pad, o_pad;
  int parts;                        // in how many h, dg and du are held (of `planes` planes where planes is 3)
  int type;                         // of an operand
  size_t limits, x, gate, up, down, h, kept, exponents, bytes;
};
Layout layout(const Call& c) {
  Layout l{};
  l.planes = c.dtype == NLFA_DTYPE_F32 ? 3 : 1;
  l.type = c.dtype == NLFA_DTYPE_F32 ? NLFA_DTYPE_BF16 : c.dtype;
  // The roundings of h, dg and du are independent and largely cancel in sums, but results of a few tokens are few: beside their own rounding
  // the others leave 1.4 times its error on average, and up to 1.7 for a few.  A tile of rows with a backward, and as many as the kernels for a few tokens
  // would take without one, are held in two parts: their products are short.
  l.parts = l.planes == 3 ? 3 : c.n <= (c.train ? kRowTile : kFewTokens) ? 2 : 1;
  l.n_rows = (c.n + kRowTile - 1) / kRowTile * kRowTile;
  l.d_pad = up64(c.d);
  l.f_pad = up64(c.F);
  l.o_pad = up64(c.o);
  const size_t two = 2 * static_cast<size_t>(l.planes), hidden = static_cast<size_t>(l.n_rows) * l.f_pad;
  size_t at = 0;
  l.limits = at; at = up(at + kHeaderBytes + (c.dtype == NLFA_DTYPE_F16 ? 2 * sizeof(float) * c.n : 0));
  l.x = at; if (c.copies & kCopyX) at = up(at + two * c.n * l.d_pad);
  l.gate = at; if (c.copies & kCopyGate) at = up(at + two * c.F * l.d_pad);
  l.up = at; if (c.copies & kCopyUp) at = up(at + two * c.F * l.d_pad);
  l.down = at; if (c.copies & kCopyDown) at = up(at + two * c.o * l.f_pad);
  l.h = at; at = up(at + 2 * l.parts * hidden);                   // (a few tokens: float32, which takes less than a tile of 256 in 16 bits)
  if (c.train) {
    const bool wide = c.dtype != NLFA_DTYPE_BF16;
    l.kept = at; at = up(at + 2 * hidden * (wide ? 4 : 2));
    l.exponents = at; if (!wide) at = up(at + 2 * hidden / 32);
  }
  l.bytes = at;
  return l;
}

// ------------------------------------------------------------------------------------------------ tiles

// In how many parts the sums of `rest` tiles of k stages are formed: the fewest stages for the busiest pair of CTAs, with `share` more for every
// share written and added, and some for the launch that adds them.  The units are handed out in turn behind `ahead` units of `length` stages.
constexpr int kFoldStages = 1;
int choose_parts(int rest, int k, int n_pairs, int share, int ahead, int length) {
  if (rest == 0) return 1;
  int best = 1;
  long long least = -1;
  const int most = kPartsPerPair * n_pairs / rest < k ? kPartsPerPair * n_pairs / rest : k;
  for (int s = 1; s <= most;) {
    const int end = ahead + rest * s, mine = (k + s - 1) / s + (s > 1 ? share : 0);
    long long cost = 0;
    for (int i = 0; i < 3; ++i) {                          // the first pair, and the first that gets one unit less of either kind
      const int b = i == 0 ? 0 : (i == 1 ? ahead : end) % n_pairs;
      const int first = (ahead + n_pairs - 1 - b) / n_pairs, both = (end + n_pairs - 1 - b) / n_pairs;
      const long long c = static_cast<long long>(first) * length + static_cast<long long>(both - first) * mine;
      cost = c > cost ? c : cost;
    }
    cost += s > 1 ? s + kFoldStages : 0;
    if (least < 0 || cost < least) { least = cost; best = s; }
    // on to the next number of parts that makes the longest one shorter (a call is planned on the host, each time)
    const int longest = (k + s - 1) / s;
    if (longest == 1) break;
    s = (k + longest - 2) / (longest - 1);
  }
  return best;
}

// Adds a group of the segments [seg0, seg1), whose sums take k stages.
void add_group(Params& p, int seg0, int seg1, int k, int planes) {
  Group& g = p.group[p.groups];
  g = Group{};
  const int n_pairs = pairs(), share = planes == 3 ? 1 : 4;       // (a stage of three parts is three times as long)
  int tiles = 0, ahead = 0, length = 0;
  for (int i = seg0; i < seg1; ++i) tiles += p.seg[i].tiles;
  if (p.groups > 0) {
    const Group& b = p.group[p.groups - 1];
    ahead = b.rest * b.parts;
    length = ceil_div(b.k, b.parts) + (b.parts > 1 ? share : 0);
    g.first = b.end;
    g.slot = b.slot + (b.parts > 1 ? ahead : 0);
  }
  g.seg0 = seg0;
  g.seg1 = seg1;
  g.k = k;
  g.whole = tiles / n_pairs * n_pairs;
  g.rest = tiles - g.whole;
  g.parts = choose_parts(g.rest, k, n_pairs, share, ahead, length);
  g.end = g.first + g.whole + g.rest * g.parts;
  p.units = g.end;
  ++p.groups;
}
// Room for the shares of a group, however it is cut.
size_t share_room(int tiles, int k) {
  const long long odd = static_cast<long long>(tiles % pairs()) * k, most = static_cast<long long>(kPartsPerPair) * pairs();
  return static_cast<size_t>(odd < most ? odd : most) * kRowTile * kColTile * sizeof(float);
}
// A product of one sum; add() gives it more.
Segment segment(int a_map, int a_mn, int a_plane, int b_map, int b_mn, int b_plane, int k, int m, int n, void* to, int dtype, const float* scale,
                int by_row) {
  Segment s{};
  s.a_map = a_map; s.a_mn = a_mn; s.b_mn = b_mn;
  s.subs = 1; s.k_sub = k;
  s.a_plane[0] = a_plane; s.b_map[0] = b_map; s.b_plane[0] = b_plane;
  s.tiles_n = ceil_div(n, kColTile);
  s.tiles = ceil_div(m, kRowTile) * s.tiles_n;
  s.m_end = m; s.n_end = n; s.to = to; s.dtype = dtype; s.scale = scale; s.by_row = by_row;
  return s;
}
void add(Segment& s, int a_plane, int b_map, int b_plane) {
  s.a_plane[s.subs] = a_plane; s.b_map[s.subs] = b_map; s.b_plane[s.subs++] = b_plane;
}

// Stages per chain of the tensor core (ffn_tc.cu).  Operands of 16 bits leave their own roundings in a sum, 2^-9 (bf16; 2^-12 in fp16) of each summand and
// independent: over 4,096 of one sign 2^-15, under which a chain of 4,096, low by 1.1e-5, hides; in fp16 one of 2,048.
int chain(const Layout& l) { return l.planes == 3 ? 1 : l.type == NLFA_DTYPE_F16 ? 16 : 32; }

// Whether g and u, or dh, are formed apart from what is done with them: where there are so few tiles that most pairs of CTAs would watch, and their sums
// are so long that three more launches are less (80 tokens x 3,903 x 32 in float32, forward and backward 270 us with one tile's sums of 61 stages); and for parts.
// `most`: stages that are not worth it.  float32, forward: 6 stages (1,000 x 384 x 1,024) 50 us, apart 57, 12 (500 x 768 x 2,048) 69 and 73, 16 (1,000 x 1,024 x 384) 68 and 56; backward, where the
// epilogue of dh writes six planes: 1 (2,000 x 64 x 512) 60 and 55, 4 (2,000 x 256 x 512) 68 and 61, 12 (300 x 768 x 2,048) 102 and 87.  bf16, forward and backward: 24 (300 x 3,000 x 256) 35 + 35 and 34 + 33,
// 38 (300 x 4,800 x 64) 38 + 47 and 28 + 35.
bool apart(const Layout& l, int cols, int k, int most) {
  if (l.parts == 2) return true;
  return 2 * (l.n_rows / kRowTile) * ceil_div(cols, kColTile) <= pairs() && ceil_div(k, summands(l.planes)) > most;
}
bool apart_up(const Call& c, const Layout& l) { return apart(l, c.F, c.d, l.planes == 3 ? 12 : 36); }
bool apart_dh(const Call& c, const Layout& l) { return apart(l, c.F, c.o, l.planes == 3 ? 0 : 36); }

// Forward, g and u apart: maps x, Wg, Wu.
void plan_up(Params& p, const Call& c, const Layout& l, float* g, float* u) {
  const int k = ceil_div(c.d, summands(l.planes));
  p.groups = p.units = 0;
  p.seg[0] = segment(0, 0, 0, 1, 0, 0, k, c.n, c.F, g, NLFA_DTYPE_F32, nullptr, 0);
  p.seg[1] = segment(0, 0, 0, 2, 0, 0, k, c.n, c.F, u, NLFA_DTYPE_F32, nullptr, 0);
  add_group(p, 0, 2, k, l.planes);
}
// y: maps h, Wd.
void plan_fwd(Params& p, const Call& c, const Layout& l, void* y, const float* scale) {
  const int k = ceil_div(c.F, summands(l.planes));
  p.groups = p.units = 0;
  p.seg[0] = segment(0, 0, 0, 1, 0, 0, k, c.n, c.o, y, c.dtype, scale, 1);
  if (l.parts == 2) add(p.seg[0], 1, 1, 0);
  add_group(p, 0, 1, p.seg[0].subs * k, l.planes);
}
// Backward, dh apart: maps dy, Wd.
void plan_dh(Params& p, const Call& c, const Layout& l, float* dh) {
  const int k = ceil_div(c.o, summands(l.planes));
  p.groups = p.units = 0;
  p.seg[0] = segment(0, 0, 0, 1, 1, 0, k, c.n, c.F, dh, NLFA_DTYPE_F32, nullptr, 0);
  add_group(p, 0, 1, k, l.planes);
}
// The gradients; du's planes are behind dg's.
enum { kHiddenRows = 0, kHiddenColumns, kX, kDy, kH, kGateRows, kUpRows };
// `scale`: of dx's rows; of_x, of_dy: of the weights' gradients.
void plan_bwd(Params& p, const Call& c, const Layout& l, void* dx, void* dwg, void* dwu, void* dwd, const float* scale, const float* of_x, const float* of_dy) {
  const int s = summands(l.planes), kw = ceil_div(c.n, s), kf = ceil_div(c.F, s);
  int n = 0;
  p.groups = p.units = 0;
  if (dwg) p.seg[n++] = segment(kHiddenRows, 1, 0, kX, 1, 0, kw, c.F, c.d, dwg, c.w_dtype, of_x, 0);
  if (dwu) p.seg[n++] = segment(kHiddenRows, 1, l.parts, kX, 1, 0, kw, c.F, c.d, dwu, c.w_dtype, of_x, 0);
  if (dwd) p.seg[n++] = segment(kDy, 1, 0, kH, 1, 0, kw, c.o, c.F, dwd, c.w_dtype, of_dy, 0);
  if (l.parts == 2)
    for (int i = 0; i < n; ++i) {
      if (p.seg[i].a_map == kDy) add(p.seg[i], 0, kH, 1);
      else add(p.seg[i], p.seg[i].a_plane[0] + 1, kX, 0);
    }
  if (n > 0) add_group(p, 0, n, p.seg[0].subs * kw, l.planes);
  if (dx) {
    Segment& g = p.seg[n] = segment(kHiddenColumns, 0, 0, kGateRows, 1, 0, kf, c.n, c.d, dx, c.x_dtype, scale, 1);
    if (l.parts == 2) add(g, 1, kGateRows, 0);
    add(g, l.parts, kUpRows, 0);
    if (l.parts == 2) add(g, l.parts + 1, kUpRows, 0);
    add_group(p, n, n + 1, g.subs * kf, l.planes);
  }
}
bool needs_chains(const Params& p, const Layout& l) {
  for (int i = 0; i < p.groups; ++i)
    if (p.group[i].k > chain(l)) return true;
  return false;
}

// The backward's workspace.
struct BwdLayout {
  size_t limits, dy, level_x, level_dy, hidden, dh, shares, bytes;
};
BwdLayout bwd_layout(const Call& c, const Layout& l, bool copy_dy) {
  BwdLayout b{};
  const size_t two = 2 * static_cast<size_t>(l.planes);
  const bool half = c.dtype == NLFA_DTYPE_F16;
  size_t at = 0;
  b.limits = at; at = up(at + kHeaderBytes + (half ? 2 * sizeof(float) * c.n : 0));
  b.dy = at; if (copy_dy) at = up(at + two * c.n * l.o_pad);
  b.level_x = at; if (half) at = up(at + two * c.n * l.d_pad);
  b.level_dy = at; if (half) at = up(at + two * c.n * l.o_pad);
  b.hidden = at; at = up(at + 4 * static_cast<size_t>(l.parts) * l.n_rows * l.f_pad);
  b.dh = at; if (apart_dh(c, l)) at = up(at + static_cast<size_t>(c.n) * c.F * 4);
  b.shares = at;
  // enough for any choice of gradients
  at += static_cast<size_t>(kMostGroups * kPartsPerPair * pairs()) * kRowTile * kColTile * sizeof(float);
  b.bytes = at;
  return b;
}

// The forward's.
struct FwdLayout {
  size_t g, u, shares, bytes;
};
FwdLayout fwd_layout(const Call& c, const Layout& l) {
  FwdLayout f{};
  const int row_tiles = l.n_rows / kRowTile, stage = summands(l.planes);
  size_t at = 0, most = share_room(row_tiles * ceil_div(c.o, kColTile), (l.parts == 2 ? 2 : 1) * ceil_div(c.F, stage));
  if (apart_up(c, l)) {
    f.g = at; at = up(at + static_cast<size_t>(c.n) * c.F * 4);
    f.u = at; at = up(at + static_cast<size_t>(c.n) * c.F * 4);
    const size_t more = share_room(2 * row_tiles * ceil_div(c.F, kColTile), ceil_div(c.d, stage));
    most = more > most ? more : most;
  }
  f.shares = at;
  f.bytes = at + most + 256;
  return f;
}

// ------------------------------------------------------------------------------------------------ float16's range

// h, dg and du of float16 are operands of float16: of a size that nobody has seen to.  Those of a token carry a power of two that puts what they can be at
// most, by Cauchy and Schwarz from the lengths of the token's x and dy and of the weights' rows, just below 2^15.  Typical values lie some 2^10 below that, and
// 2^18 above the smallest normal number.  |f(g)| <= |g|, |f'| < 1.13.  y and dx are divided by it row by row.  (One power of two per call would take the digits
// of all other tokens' h where one x is 1,000 times as long.)
//
// A weight's gradient is a sum over tokens, so there the other operand, x or dy, carries what makes the powers alike: 2^(level - e) beside 2^e, the level being
// such that the longest row of that operand is just below 2^15 too.  What is lost is 2^-30 and less of the largest share of a token.
constexpr int kLimitCtas = 592;
struct Limits {                     // squares of the largest row lengths; of Wd the largest element
  float gate, up, down;
};
struct BwdLimits {
  int top_x, top_dy;                // the largest exponent of a row of x, of dy, less the row's own of dg and du, of h, and 1,024 (0: no row has one)
  float of_x, of_dy;                // 2^level
};
// Behind either, a float per token: the square of its row's length (x; dy), its power of two (h; dg and du).
struct Tokens {
  float *square, *scale;
};
Tokens tokens_of(void* limits, int n) {
  float* at = reinterpret_cast<float*>(static_cast<uint8_t*>(limits) + kHeaderBytes);
  return {at, at + n};
}
enum { kLongestRow = 0, kLargestElement, kEveryRow };
struct Rows {
  const void* src;
  int dtype, rows, cols, what;
  float* to;
  int vec;
};
struct RowList {
  Rows r[4];
  int n;
};

// A warp per row, of values as float16 has them; what is not finite there is left out (its results are not finite, whatever the factor).  Eight elements a load where
// rows lie on 16 bytes (element by element 65,536 x 768 takes 42 us).
template <typename S>
__device__ __forceinline__ void row_lengths(const Rows& s) {
  const S* src = static_cast<const S*>(s.src);
  const int lane = threadIdx.x & 31;
  float most = 0.f;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < s.rows; r += gridDim.x * 8) {
    const S* row = src + static_cast<size_t>(r) * s.cols;
    float sum = 0.f, top = 0.f;
    auto add = [&](float v) {
      if constexpr (!std::is_same_v<S, __half>) v = __half2float(__float2half_rn(v));
      v = fabsf(v) < INFINITY ? v : 0.f;
      sum = fmaf(v, v, sum);
      top = fmaxf(top, fabsf(v));
    };
    if (s.vec) {
#pragma unroll 4
      for (int i = 8 * lane; i < s.cols; i += 256) {
        float v[8];
        rowwise::Elem<S>::load(row + i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) add(v[j]);
      }
    } else {
#pragma unroll 4
      for (int i = lane; i < s.cols; i += 32) add(static_cast<float>(row[i]));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, off);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    if (s.what == kEveryRow && lane == 0) s.to[r] = sum;
    most = fmaxf(most, s.what == kLargestElement ? top : sum);
  }
  // (of non-negative floats the order is that of their bits: no order of these matters)
  if (s.what != kEveryRow && lane == 0 && most > 0.f) atomicMax(reinterpret_cast<int*>(s.to), __float_as_int(most));
}
__global__ void __launch_bounds__(256)
limits_kernel(const RowList list) {
  grid_dep_wait();
  grid_dep_release();
  const Rows s = list.r[blockIdx.y];
  if (s.dtype == NLFA_DTYPE_F32) row_lengths<float>(s);
  else if (s.dtype == NLFA_DTYPE_F16) row_lengths<__half>(s);
  else row_lengths<__nv_bfloat16>(s);
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }    // -127 < e < 128
// v < 2^exponent(v)
__device__ __forceinline__ int exponent(float v) {
  int b;
  frexpf(v, &b);
  return b;
}
// The exponent that a token's values carry whose largest is `bound`.  (Bounds of float16 values: below 2^113.)
__device__ __forceinline__ int carried(float bound) { return bound > 0.f && bound < INFINITY ? min(max(14 - exponent(bound), -100), 100) : 0; }

__global__ void __launch_bounds__(256)
fwd_scale_kernel(const Limits* l, Tokens x, int n) {
  grid_dep_wait();
  grid_dep_release();
  const float weights = sqrtf(l->gate) * sqrtf(l->up);
  for (int r = blockIdx.x * 256 + threadIdx.x; r < n; r += gridDim.x * 256) x.scale[r] = power_of_two(carried(x.square[r] * weights));
}
__global__ void __launch_bounds__(256)
bwd_scale_kernel(const Limits* l, Tokens x, BwdLimits* b, Tokens dy, int n, float o) {
  grid_dep_wait();
  grid_dep_release();
  const float weights = sqrtf(o) * l->down * fmaxf(sqrtf(l->gate), 1.13f * sqrtf(l->up));
  int top_x = 0, top_dy = 0;
  for (int r = blockIdx.x * 256 + threadIdx.x; r < n; r += gridDim.x * 256) {
    const float xs = sqrtf(x.square[r]), ys = sqrtf(dy.square[r]), bound = ys * weights * xs;
    const int e = carried(bound);
    dy.scale[r] = power_of_two(e);
    if (bound > 0.f) top_x = max(top_x, exponent(xs) - e + 1024);
    if (xs > 0.f && ys > 0.f) top_dy = max(top_dy, exponent(ys) - (exponent(x.scale[r]) - 1) + 1024);
  }
  top_x = __reduce_max_sync(0xffffffffu, top_x);
  top_dy = __reduce_max_sync(0xffffffffu, top_dy);
  if ((threadIdx.x & 31) == 0) {
    if (top_x > 0) atomicMax(&b->top_x, top_x);
    if (top_dy > 0) atomicMax(&b->top_dy, top_dy);
  }
}

int checked(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}

int find_limits(RowList list, void* to, size_t bytes, cudaStream_t st) {
  for (Rows& r : list.r) r.vec = r.cols % 8 == 0 && aligned16(r.src);
  const int rc = checked(cudaMemsetAsync(to, 0, bytes, st));
  if (rc != NLFA_OK) return rc;
  return checked(launch_kernel(limits_kernel, dim3(kLimitCtas, static_cast<unsigned>(list.n)), dim3(256), 0, st, false, list));
}
unsigned token_ctas(int n) { return static_cast<unsigned>((n < 256 * kLimitCtas ? n + 255 : 256 * kLimitCtas) / 256); }

// ------------------------------------------------------------------------------------------------ calls

// Copies of operands, up to four in one launch (blockIdx.y): [planes][cols padded / 64][rows][64]
struct Copy {
  const void* src;
  void* dst;
  int dtype, rows, cols, pad, vec;
};
struct CopyList {
  Copy c[4];
  int n;
};
template <typename T>
__global__ void __launch_bounds__(operands::kBlock)
copies_kernel(const CopyList list, int planes) {
  grid_dep_wait();
  grid_dep_release();
  const Copy c = list.c[blockIdx.y];
  const int chunks = c.pad / 8;
  const long long total = static_cast<long long>(c.rows) * chunks;
  T* dst = static_cast<T*>(c.dst);
  for (long long i = static_cast<long long>(blockIdx.x) * operands::kBlock + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * operands::kBlock) {
    const int r = static_cast<int>(i / chunks), col = 8 * static_cast<int>(i - static_cast<long long>(r) * chunks);
    if (c.dtype == NLFA_DTYPE_F32) operands::copy_chunk(static_cast<const float*>(c.src), dst, r, r, col, c.rows, c.cols, c.pad, planes, c.vec);
    else if (c.dtype == NLFA_DTYPE_F16) operands::copy_chunk(static_cast<const __half*>(c.src), dst, r, r, col, c.rows, c.cols, c.pad, planes, c.vec);
    else operands::copy_chunk(static_cast<const __nv_bfloat16*>(c.src), dst, r, r, col, c.rows, c.cols, c.pad, planes, c.vec);
  }
}
int make_copies(const CopyList& list, const Layout& l, cudaStream_t st) {
  if (list.n == 0) return NLFA_OK;
  long long most = 1;
  for (int i = 0; i < list.n; ++i) {
    const long long ctas = (static_cast<long long>(list.c[i].rows) * (list.c[i].pad / 8) + operands::kBlock - 1) / operands::kBlock;
    most = ctas > most ? ctas : most;
  }
  const long long limit = 16ll * sm_count();
  const dim3 grid(static_cast<unsigned>(most < limit ? most : limit), static_cast<unsigned>(list.n));
  auto* kernel = l.type == NLFA_DTYPE_F16 ? copies_kernel<__half> : copies_kernel<__nv_bfloat16>;
  return checked(launch_kernel(kernel, grid, dim3(operands::kBlock), 0, st, overlap_launches(kOverlapRowwise), list, l.planes));
}

struct Weights {
  const void *x, *gate, *up, *down;
};

// A tensor as an operand: the caller's, or its copy.
struct Operand {
  const void* at;
  long long cols, rows;
  bool blocked;
  int planes;                       // 0: as every operand's
};
Operand operand(const void* own, const void* copy, bool copied, int cols, int rows) { return {copied ? copy : own, up64(cols), rows, copied, 0}; }
// A stage of one CTA's half of it: 128 rows, the summands along the columns; or 128 columns, the summands along the rows.
int columns(CUtensorMap* m, const Operand& a, const Layout& l) {
  return operands::box_map(m, a.at, l.type, a.cols, a.rows, a.planes > 0 ? a.planes : l.planes, 128, summands(l.planes) / 64, l.planes, a.blocked);
}
int rows(CUtensorMap* m, const Operand& a, const Layout& l) {
  return operands::box_map(m, a.at, l.type, a.cols, a.rows, a.planes > 0 ? a.planes : l.planes, summands(l.planes), 2, l.planes, a.blocked);
}

// x beside dg and du, dy beside h, brought to one level (float16; above): a copy in blocks, a warp per row.  A token without a gradient, or with an x of zeros, gives zeros: its own
// level would be any.
struct Level {
  const __half* src;
  __half* dst;
  int pad, blocked;                 // columns; whether src lies in blocks too
  const float *other, *scale;       // squares of the other's row lengths; powers of two of what stands beside
  const int* top;
  float* of;
};
struct LevelList {
  Level c[2];
  int n;
};
__global__ void __launch_bounds__(operands::kBlock)
level_kernel(const LevelList list, int rows) {
  grid_dep_wait();
  grid_dep_release();
  const Level c = list.c[blockIdx.y];
  const int top = *c.top, level = top > 0 ? min(max(14 - (top - 1024), -120), 120) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *c.of = power_of_two(level);
  constexpr int kWarps = operands::kBlock / 32;
  for (int r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < rows; r += gridDim.x * kWarps) {
    // (level - e may be outside float32's exponents: two factors)
    const int k = level - (exponent(c.scale[r]) - 1), k0 = k / 2;
    const float f0 = c.other[r] > 0.f ? power_of_two(k0) : 0.f, f1 = power_of_two(k - k0);
#pragma unroll 4
    for (int col = 8 * (threadIdx.x & 31); col < c.pad; col += 256) {
      const size_t block = (static_cast<size_t>(col / 64) * rows + r) * 64 + col % 64;
      float v[8];
      rowwise::Elem<__half>::load(c.src + (c.blocked ? block : static_cast<size_t>(r) * c.pad + col), v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * f0 * f1;
      rowwise::Elem<__half>::store(c.dst + block, v);
    }
  }
}
Level level_of(const Operand& a, void* dst, const float* other, const float* scale, const int* top, float* of) {
  return {static_cast<const __half*>(a.at), static_cast<__half*>(dst), static_cast<int>(a.cols), a.blocked, other, scale, top, of};
}
int make_levels(const LevelList& list, int rows, cudaStream_t st) {
  const int need = ceil_div(rows, operands::kBlock / 32), most = 16 * sm_count();
  return checked(launch_kernel(level_kernel, dim3(static_cast<unsigned>(need < most ? need : most), static_cast<unsigned>(list.n)), dim3(operands::kBlock), 0, st,
                               overlap_launches(kOverlapRowwise), list, rows));
}

struct Operands {
  Operand x, gate, up, down, h;
};
Operands operands_of(const Call& c, const Layout& l, const Weights& w, const uint8_t* tape) {
  return {operand(w.x, tape + l.x, c.copies & kCopyX, c.d, c.n), operand(w.gate, tape + l.gate, c.copies & kCopyGate, c.d, c.F),
          operand(w.up, tape + l.up, c.copies & kCopyUp, c.d, c.F), operand(w.down, tape + l.down, c.copies & kCopyDown, c.F, c.o),
          Operand{tape + l.h, l.f_pad, l.n_rows, true, l.parts}};
}

Params params(const Call& c, const Layout& l, int activation, uint8_t* tape, unsigned* status) {
  Params p{};
  p.rows = c.n;
  p.cols = c.F;
  p.n_rows = l.n_rows;
  p.f_pad = l.f_pad;
  p.chunk = chain(l);
  p.activation = activation;
  p.kept = c.train ? tape + l.kept : nullptr;
  p.exponents = reinterpret_cast<int8_t*>(tape + l.exponents);
  p.h = tape + l.h;
  p.status = status;
  return p;
}
void fill(Maps& maps, int n) {
  for (int i = n; i < kMostMaps; ++i) maps.m[i] = maps.m[0];
}
bool long_sum(int k, const Layout& l) { return ceil_div(k, summands(l.planes)) > chain(l); }

int run_fwd(const Call& c, const Weights& w, int activation, void* y, uint8_t* tape, uint8_t* scratch, cudaStream_t st) {
  const Layout l = layout(c);
  unsigned* status = status_block();
  if (!status) return NLFA_ERR_CUDA;
  CopyList copies{};
  auto copy = [&](int flag, const void* src, int src_dtype, size_t to, int n, int cols) {
    if (c.copies & flag) copies.c[copies.n++] = {src, tape + to, src_dtype, n, cols, up64(cols), cols % 8 == 0 && aligned16(src)};
  };
  copy(kCopyX, w.x, c.x_dtype, l.x, c.n, c.d);
  copy(kCopyGate, w.gate, c.w_dtype, l.gate, c.F, c.d);
  copy(kCopyUp, w.up, c.w_dtype, l.up, c.F, c.d);
  copy(kCopyDown, w.down, c.w_dtype, l.down, c.o, c.F);
  int rc = make_copies(copies, l, st);
  Limits* limits = c.dtype == NLFA_DTYPE_F16 ? reinterpret_cast<Limits*>(tape + l.limits) : nullptr;
  const Tokens tokens = tokens_of(tape + l.limits, c.n);
  if (rc == NLFA_OK && limits != nullptr) {
    RowList list{};
    list.r[0] = {w.x, c.x_dtype, c.n, c.d, kEveryRow, tokens.square};
    list.r[1] = {w.gate, c.w_dtype, c.F, c.d, kLongestRow, &limits->gate};
    list.r[2] = {w.up, c.w_dtype, c.F, c.d, kLongestRow, &limits->up};
    list.r[3] = {w.down, c.w_dtype, c.o, c.F, kLargestElement, &limits->down};
    list.n = c.train ? 4 : 3;
    rc = find_limits(list, limits, sizeof(Limits), st);
    if (rc == NLFA_OK)
      rc = checked(launch_kernel(fwd_scale_kernel, dim3(token_ctas(c.n)), dim3(256), 0, st, overlap_launches(kOverlapRowwise), limits, tokens, c.n));
  }
  if (rc != NLFA_OK) return rc;
  const Operands a = operands_of(c, l, w, tape);
  const FwdLayout f = fwd_layout(c, l);
  Maps maps;
  rc = columns(&maps.m[0], a.x, l);
  if (rc == NLFA_OK) rc = columns(&maps.m[1], a.gate, l);
  if (rc == NLFA_OK) rc = columns(&maps.m[2], a.up, l);
  if (rc == NLFA_OK) rc = operands::box_map(&maps.m[3], tape + l.h, l.type, l.f_pad, l.n_rows, l.parts, 32, 1, 1, true);
  if (rc != NLFA_OK) return rc;
  fill(maps, 4);
  Params p = params(c, l, activation, tape, status);
  p.k = c.d;
  p.scale = limits != nullptr ? tokens.scale : nullptr;
  p.shares = reinterpret_cast<float*>(scratch + f.shares);
  if (apart_up(c, l)) {
    float *g = reinterpret_cast<float*>(scratch + f.g), *u = reinterpret_cast<float*>(scratch + f.u);
    plan_up(p, c, l, g, u);
    rc = launch_product(kProducts, l.type, l.planes, needs_chains(p, l), p, maps, st);
    if (rc == NLFA_OK) rc = launch_hidden(l.type, l.planes, l.parts, p, g, u, st);
  } else {
    rc = launch_product(kUp, l.type, l.planes, long_sum(c.d, l), p, maps, st);
  }
  if (rc != NLFA_OK) return rc;
  rc = columns(&maps.m[0], a.h, l);
  if (rc == NLFA_OK) rc = columns(&maps.m[1], a.down, l);
  if (rc != NLFA_OK) return rc;
  fill(maps, 2);
  plan_fwd(p, c, l, y, limits != nullptr ? tokens.scale : nullptr);
  return launch_product(kProducts, l.type, l.planes, needs_chains(p, l), p, maps, st);
}

int run_bwd(const Call& c, const void* dy, const Weights& w, int activation, uint8_t* tape, void* dx, void* dwg, void* dwu, void* dwd,
            uint8_t* scratch, cudaStream_t st) {
  const Layout l = layout(c);
  const bool copy_dy = must_copy(dy, c.dtype, c.dtype, c.o);
  const BwdLayout b = bwd_layout(c, l, copy_dy);
  unsigned* status = status_block();
  if (!status) return NLFA_ERR_CUDA;
  int rc = NLFA_OK;
  if (copy_dy) {
    CopyList copies{};
    copies.c[copies.n++] = {dy, scratch + b.dy, c.dtype, c.n, c.o, l.o_pad, c.o % 8 == 0 && aligned16(dy)};
    rc = make_copies(copies, l, st);
  }
  const Limits* limits = c.dtype == NLFA_DTYPE_F16 ? reinterpret_cast<const Limits*>(tape + l.limits) : nullptr;
  BwdLimits* more = reinterpret_cast<BwdLimits*>(scratch + b.limits);
  const Tokens x_tokens = tokens_of(tape + l.limits, c.n), dy_tokens = tokens_of(scratch + b.limits, c.n);
  const bool through = dx || dwg || dwu;                   // whether dg and du are needed
  if (rc == NLFA_OK && limits != nullptr) {
    RowList list{};
    list.r[0] = {dy, c.dtype, c.n, c.o, kEveryRow, dy_tokens.square};
    list.n = 1;
    rc = find_limits(list, more, sizeof(BwdLimits), st);
    if (rc == NLFA_OK)
      rc = checked(launch_kernel(bwd_scale_kernel, dim3(token_ctas(c.n)), dim3(256), 0, st, overlap_launches(kOverlapRowwise), limits, x_tokens, more,
                                 dy_tokens, c.n, static_cast<float>(c.o)));
  }
  if (rc != NLFA_OK) return rc;
  const Operands a = operands_of(c, l, w, tape);
  const Operand up_grad = operand(dy, scratch + b.dy, copy_dy, c.o, c.n), hidden{scratch + b.hidden, l.f_pad, l.n_rows, true, 2 * l.parts};
  Params p = params(c, l, activation, tape, status);
  p.dg = scratch + b.hidden;
  p.du = scratch + b.hidden + static_cast<size_t>(2 * l.parts) * l.n_rows * l.f_pad;
  p.shares = reinterpret_cast<float*>(scratch + b.shares);
  Maps maps;
  if (through) {
    rc = columns(&maps.m[0], up_grad, l);
    if (rc == NLFA_OK) rc = rows(&maps.m[1], a.down, l);
    if (rc == NLFA_OK) rc = operands::box_map(&maps.m[2], hidden.at, l.type, l.f_pad, l.n_rows, 2 * l.parts, 32, 1, 1, true);
    if (rc != NLFA_OK) return rc;
    fill(maps, 3);
    p.k = c.o;
    p.scale = limits != nullptr ? dy_tokens.scale : nullptr;
    if (apart_dh(c, l)) {
      float* dh = reinterpret_cast<float*>(scratch + b.dh);
      plan_dh(p, c, l, dh);
      rc = launch_product(kProducts, l.type, l.planes, needs_chains(p, l), p, maps, st);
      if (rc == NLFA_OK) rc = launch_grads(l.type, l.planes, l.parts, p, dh, st);
    } else {
      rc = launch_product(kDh, l.type, l.planes, long_sum(c.o, l), p, maps, st);
    }
    if (rc != NLFA_OK) return rc;
  }
  // x and dy as the weights' gradients read them
  Operand x_rows = a.x, dy_rows = up_grad;
  if (limits != nullptr) {
    LevelList list{};
    if (dwg || dwu) {
      list.c[list.n++] = level_of(a.x, scratch + b.level_x, dy_tokens.square, dy_tokens.scale, &more->top_x, &more->of_x);
      x_rows = operand(nullptr, scratch + b.level_x, true, c.d, c.n);
    }
    if (dwd) {
      list.c[list.n++] = level_of(up_grad, scratch + b.level_dy, x_tokens.square, x_tokens.scale, &more->top_dy, &more->of_dy);
      dy_rows = operand(nullptr, scratch + b.level_dy, true, c.o, c.n);
    }
    if (list.n > 0) rc = make_levels(list, c.n, st);
    if (rc != NLFA_OK) return rc;
  }
  rc = rows(&maps.m[kHiddenRows], hidden, l);
  if (rc == NLFA_OK) rc = columns(&maps.m[kHiddenColumns], hidden, l);
  if (rc == NLFA_OK) rc = rows(&maps.m[kX], x_rows, l);
  if (rc == NLFA_OK) rc = rows(&maps.m[kDy], dy_rows, l);
  if (rc == NLFA_OK) rc = rows(&maps.m[kH], a.h, l);
  if (rc == NLFA_OK) rc = rows(&maps.m[kGateRows], a.gate, l);
  if (rc == NLFA_OK) rc = rows(&maps.m[kUpRows], a.up, l);
  if (rc != NLFA_OK) return rc;
  fill(maps, kUpRows + 1);
  if (limits != nullptr) plan_bwd(p, c, l, dx, dwg, dwu, dwd, dy_tokens.scale, &more->of_x, &more->of_dy);
  else plan_bwd(p, c, l, dx, dwg, dwu, dwd, nullptr, nullptr, nullptr);
  return launch_product(kProducts, l.type, l.planes, needs_chains(p, l), p, maps, st);
}

}  // namespace
}  // namespace ffn
}  // namespace nlfa

using namespace nlfa;
using namespace nlfa::ffn;
using rowwise::aligned16;

extern "C" {

int nlfa_gated_ffn_copies(const void* x, int x_dtype, const void* w_gate, const void* w_up, const void* w_down, int w_dtype, int dtype, int n, int d,
                          int F, int train) {
  if (is_few(x, w_gate, w_up, w_down, w_dtype, dtype, n, d, F, train)) return 0;
  return (must_copy(x, x_dtype, dtype, d) ? kCopyX : 0) | (must_copy(w_gate, w_dtype, dtype, d) ? kCopyGate : 0) |
         (must_copy(w_up, w_dtype, dtype, d) ? kCopyUp : 0) | (must_copy(w_down, w_dtype, dtype, F) ? kCopyDown : 0);
}
size_t nlfa_gated_ffn_tape_bytes(int n, int d, int F, int o, int dtype, int copies, int train) {
  const Call c{dtype, dtype, dtype, n, d, F, o, copies, train};
  return check_call(c) == NLFA_OK ? layout(c).bytes : 0;
}
size_t nlfa_gated_ffn_scratch_bytes(int n, int d, int F, int o, int dtype, int copies, int train, int backward) {
  const Call c{dtype, dtype, dtype, n, d, F, o, copies, train};
  if (check_call(c) != NLFA_OK) return 0;
  const Layout l = layout(c);
  // (the gradient of y is copied where it has to be: there is room)
  if (backward) return bwd_layout(c, l, true).bytes;
  return fwd_layout(c, l).bytes;
}

int nlfa_gated_ffn_fwd(const void* x, int x_dtype, const void* w_gate, const void* w_up, const void* w_down, int w_dtype, int dtype,
                       int activation, int n, int d, int F, int o, void* y, int copies, int train, void* tape, size_t tape_bytes, void* scratch,
                       size_t scratch_bytes, void* stream) {
  const Call c{x_dtype, w_dtype, dtype, n, d, F, o, copies, train};
  const int rc = check_call(c);
  if (rc != NLFA_OK) return rc;
  if (activation < NLFA_FFN_SILU || activation > NLFA_FFN_RELU) return NLFA_ERR_BAD_ARGUMENT;
  if (!w_gate || !w_up || !w_down || !tape || !scratch || (n > 0 && (!x || !y))) return NLFA_ERR_NULL_POINTER;
  if (n == 0) return NLFA_OK;
  const int x_bytes = element_bytes(x_dtype), w_bytes = element_bytes(w_dtype);
  if (!aligned16(tape) || !aligned16(scratch) || !aligned16(y) || !aligned_to(x, x_bytes) || !aligned_to(w_gate, w_bytes) ||
      !aligned_to(w_up, w_bytes) || !aligned_to(w_down, w_bytes))
    return NLFA_ERR_MISALIGNED;
  if (nlfa_gated_ffn_copies(x, x_dtype, w_gate, w_up, w_down, w_dtype, dtype, n, d, F, train) & ~copies) return NLFA_ERR_MISALIGNED;
  if (tape_bytes < layout(c).bytes || scratch_bytes < nlfa_gated_ffn_scratch_bytes(n, d, F, o, dtype, copies, train, 0)) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (!nlfa_device_supported()) return NLFA_ERR_NOT_SM100;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  if (is_few(x, w_gate, w_up, w_down, w_dtype, dtype, n, d, F, train))
    return launch_few_tokens(x, x_dtype, w_gate, w_up, w_down, w_dtype, dtype, activation, n, d, F, o,
                             reinterpret_cast<float*>(static_cast<uint8_t*>(tape) + layout(c).h), y, static_cast<cudaStream_t>(stream));
  return run_fwd(c, {x, w_gate, w_up, w_down}, activation, y, static_cast<uint8_t*>(tape), static_cast<uint8_t*>(scratch),
                 static_cast<cudaStream_t>(stream));
}

int nlfa_gated_ffn_bwd(const void* dy, const void* x, int x_dtype, const void* w_gate, const void* w_up, const void* w_down, int w_dtype,
                       int dtype, int activation, int n, int d, int F, int o, int copies, void* tape, size_t tape_bytes, void* dx,
                       void* dw_gate, void* dw_up, void* dw_down, void* scratch, size_t scratch_bytes, void* stream) {
  const Call c{x_dtype, w_dtype, dtype, n, d, F, o, copies, 1};
  const int rc = check_call(c);
  if (rc != NLFA_OK) return rc;
  if (activation < NLFA_FFN_SILU || activation > NLFA_FFN_RELU) return NLFA_ERR_BAD_ARGUMENT;
  if (!dx && !dw_gate && !dw_up && !dw_down) return NLFA_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t w_bytes = element_bytes(w_dtype);
  if (!aligned16(dx) || !aligned16(dw_gate) || !aligned16(dw_up) || !aligned16(dw_down)) return NLFA_ERR_MISALIGNED;
  if (n == 0) {                                             // no token: gradients of zero
    for (void* t : {dw_gate, dw_up, dw_down})
      if (t != nullptr && cudaMemsetAsync(t, 0, static_cast<size_t>(F) * (t == dw_down ? o : d) * w_bytes, st) != cudaSuccess) {
        (void)cudaGetLastError();
        return NLFA_ERR_CUDA;
      }
    return NLFA_OK;
  }
  // operands that were copied are not read again
  const void* read[4] = {copies & kCopyX ? nullptr : x, copies & kCopyGate ? nullptr : w_gate, copies & kCopyUp ? nullptr : w_up,
                         copies & kCopyDown ? nullptr : w_down};
  if (!dy || !tape || !scratch) return NLFA_ERR_NULL_POINTER;
  for (int i = 0; i < 4; ++i) {
    if (!(copies >> i & 1) && !read[i]) return NLFA_ERR_NULL_POINTER;
    if (!aligned16(read[i])) return NLFA_ERR_MISALIGNED;
  }
  if (!aligned16(tape) || !aligned16(scratch) || !aligned_to(dy, element_bytes(dtype))) return NLFA_ERR_MISALIGNED;
  const Layout l = layout(c);
  if (tape_bytes < l.bytes || scratch_bytes < bwd_layout(c, l, true).bytes) return NLFA_ERR_SCRATCH_TOO_SMALL;
  if (!nlfa_device_supported()) return NLFA_ERR_NOT_SM100;
  if (nlfa_peek_status() != NLFA_OK) return NLFA_ERR_DEVICE_TIMEOUT;
  return run_bwd(c, dy, {read[0], read[1], read[2], read[3]}, activation, static_cast<uint8_t*>(tape), dx, dw_gate, dw_up, dw_down,
                 static_cast<uint8_t*>(scratch), st);
}

}  // extern "C"
