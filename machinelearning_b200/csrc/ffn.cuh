// Gated feed-forward layer (ffn.cu: layouts, copies, the C ABI; ffn_tc.cu: the products): what the two share.
#pragma once

#include "common.cuh"
#include "operands.cuh"

namespace nlfa {
namespace ffn {

using operands::kRowTile;
using operands::summands;
constexpr int kColTile = 256;       // columns of a product's tile
constexpr int kPartsPerPair = 2;    // shares of odd tiles there is room for, per pair of CTAs and group

enum { kUp = 0, kDh = 1, kProducts = 2 };

// One product of kProducts: to [m_end, n_end] = (A_0 B_0 + A_1 B_1 + ...) / scale, `subs` sums of `k_sub` stages that differ in maps and planes (dx = dg Wg + du Wu;
// hidden values in two parts).
constexpr int kMostSubs = 4;
struct Segment {
  int a_map, a_mn, b_mn;            // _mn: the sum runs along the operand's rows
  int subs, k_sub;
  int a_plane[kMostSubs], b_map[kMostSubs], b_plane[kMostSubs];
  int tiles, tiles_n, m_end, n_end;
  void* to;
  int dtype;
  const float* scale;               // powers of two, one or (by_row) each row's; NULL: 1
  int by_row;
};
// Segments whose sums have the same number of stages.  Units: whole tiles, as many as all pairs of CTAs get, then the rest, whose sums are cut
// into parts so that every pair is busy; parts of one index stand together (they read the same summands).
struct Group {
  int seg0, seg1;
  int k, whole, rest, parts;
  int first, end;                   // units
  int slot;                         // first share
};
constexpr int kMostSegments = 4, kMostGroups = 2, kMostMaps = 8;

struct Maps {
  CUtensorMap m[kMostMaps];
};

struct Params {
  int rows, cols, k;                // kUp, kDh: tokens, hidden columns, length of the sums
  int n_rows, f_pad;                // extents of h, dg, du
  int chunk;                        // stages per chain of the tensor core
  int activation;
  // kept f(g) and u f'(g): 16-bit values with a power of two per 32 values of a row, or float32 (ffn_tc.cu)
  uint8_t *kept;
  int8_t* exponents;
  void *h, *dg, *du;                // (written without TMA in float32 and by launch_hidden, launch_grads)
  const float* scale;               // powers of two of h's rows (kUp) or dg's and du's (kDh), float16 only; NULL: 1
  Segment seg[kMostSegments];
  Group group[kMostGroups];
  int groups, units;
  float* shares;
  unsigned* status;
};

int pairs();                        // of CTAs that run at once
// Maps: kUp x, Wg, Wu, h to store; kDh dy, Wd, dg and du to store; kProducts as the segments say.
int launch_product(int mode, int dtype, int planes, bool chains, const Params& p, const Maps& maps, cudaStream_t stream);

// What kUp and kDh do behind their products, from products in float32 [rows, cols]: h in `parts` parts and what is kept; dg and du in as many.
int launch_hidden(int dtype, int planes, int parts, const Params& p, const float* g, const float* u, cudaStream_t stream);
int launch_grads(int dtype, int planes, int parts, const Params& p, const float* dh, cudaStream_t stream);

// A few tokens, no backward (ffn_few.cu): operands as they lie, d and F multiples of 8, on 16 bytes.  h: n x F.
// Up to 16 tokens, and up to 64 where tokens times weights are few: the products here are not tcgen05's.  768 x 2,048, 64 tokens: 11 us in bf16, 20 in fp16, 30 in float32,
// by tiles of 256 rows 34, 45, 65; 2,048 x 4,096, 32 tokens: 29, 40, 92 and 44, 59, 129, 64 tokens 38, 80, 137 and 47, 62, 130; 4,096 x 8,192, 16 tokens: 71, 90, 182 and 81, 110, 395,
// 32 tokens 124, 160, 318 and 84, 116, 397.
constexpr int kFewTokens = 64, kVeryFewTokens = 16;
constexpr long long kFewProducts = 1ll << 28;               // n d F
bool few_types(int w_dtype, int dtype);
int launch_few_tokens(const void* x, int x_dtype, const void* gate, const void* up, const void* down, int w_dtype, int dtype, int activation, int n,
                      int d, int F, int o, float* h, void* y, cudaStream_t st);

}  // namespace ffn
}  // namespace nlfa
