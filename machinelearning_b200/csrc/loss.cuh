// Linear cross entropy (loss.cu: rows, sums, the C ABI; loss_tc.cu: the products): what the two share.
#pragma once

#include "common.cuh"
#include "operands.cuh"

namespace nlfa {
namespace loss {

using operands::kRowTile;
constexpr int kColTile = 256;       // columns of a tile
using operands::summands;
// dl is held in 16 bits.  Its roundings (half a step, 2^-8 in bf16) are independent and largely cancel in sums over many rows or words:
// gradients of 513 rows are off by 2.2e-3 as a whole, 1.7e-3 of that by their own rounding.  A row's own target has most of its dl,
// though, and in a sum of a few rows one such rounding shows (3.3e-3 for one row): up to a tile of rows with a target dl is held in two
// parts, and up to kTwoParts where the rows' gradients differ, so that a few of them can be most of the sum (2.5e-3 for 160 rows).
constexpr int kTwoParts = 1024;
__device__ __forceinline__ int dl_parts(int planes, int per_row, int rows) {
  return planes == 3 ? 3 : rows <= (per_row ? kTwoParts : kRowTile) ? 2 : 1;
}
constexpr int kPartsPerPair = 2;    // shares of dW's, and of dx's, odd tiles there is room for, per pair of CTAs

// The forward leaves its tape in one buffer; counts and places, known on the device only, stand first.
struct Head {
  int count;                        // rows with a target
  int splits;                       // parts of the vocabulary in the forward's units
};
// In how many parts the sums of dW's and dx's odd tiles are formed, in all pieces of the vocabulary but the last, and in the last.
struct Parts {
  int dw[2], dx[2];
};

// Tape and scratch, laid out for n rows.  Rows without a target are left out on the way in (`row_of` names the source
// of each row that stays), so they cost no products and whatever stands in them reaches nothing.
struct Layout {
  int n_rows;                       // rows a call can hold, up to a multiple of kRowTile
  int d_pad;                        // row length of the 16-bit copies, a multiple of 64
  int x_planes;                     // 16-bit parts of an operand: 1, or 3 for float32
  bool copy_w;                      // the weight is converted or re-laid (otherwise the products read the caller's)
  size_t row_of, target, lse, lse_rest, own, x, w, tape_bytes;
  int max_splits;
  size_t partial, at_target, sums, ticket, fwd_bytes;
  int max_parts;                    // (maximum, sum) pairs per row
};

// One product's launch.
struct Params {
  const Head* head;
  int V, d, d_pad;
  int planes;                       // parts of an operand: 1 or 3
  int per_row;                      // a gradient for each row (dl_parts)
  int dl_second;                    // rows between the first and the second part of dl
  int chunk;                        // stages per chain of the tensor core (0: the whole sum; kProducts: of dl in one part, or three)
  int v0, v1;                       // piece of the vocabulary
  int n_rows;
  int w_stands;                     // kFew: w is the caller's, not a copy made by the launch before
  // forward: (max, sum) of every part of a row, logit of the target
  float2* partial;
  float* at_target;
  const int* target;
  // gradient of the logits
  const float *lse, *lse_rest;      // lse + lse_rest: to better than float32
  const float* own;                 // p - 1 of the row's target
  const float* row_scale;
  // products with it: dx [N, d] by row_of, dw [V, d]
  const int* row_of;
  const float* alpha;
  void *dx, *dw;
  float* dx_sum;                    // float32 sums of dx over the pieces
  const Parts* parts;
  float* shares;                    // of tiles formed in parts
  int dx_dtype, dw_dtype;
  int first, last;                  // piece is the first / last one
  int want_dx, want_dw;
  unsigned* status;
};

int most_pairs();                   // of CTAs that run at once
size_t share_bytes();
enum { kLse = 0, kGrad = 1, kProducts = 2, kFew = 3 };
constexpr int kFewRows = 64;        // rows of a call that kFew takes
// Maps: kLse, kFew and kGrad: x and w as operands along the columns, kGrad: ds_out to store dl; kProducts: x and w as operands along the rows,
// dl along the columns (ds) and along the rows (ds_out).
int launch_product(int mode, int dtype, const Params& p, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& ds,
                   const CUtensorMap& ds_out, cudaStream_t stream);

}  // namespace loss
}  // namespace nlfa
