// Operands of products on pairs of CTAs (loss_tc.cu, ffn_tc.cu): 16-bit copies of tensors that TMA cannot read as they are (float32: sums
// of three bf16 parts, exact to 2^-24), and the tensor maps of copies and of tensors read where they lie.
#pragma once

#include "common.cuh"
#include "rowwise.cuh"

namespace nlfa {
namespace operands {

constexpr int kRowTile = 256;       // rows of a product's tile: two CTAs of 128
constexpr int kBlock = 256;         // threads of a copy
// Summands per stage of a product's pipeline: 128, or 64 of operands in three parts.
__host__ __device__ constexpr int summands(int planes) { return planes == 3 ? 64 : 128; }

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

// Rows from row_of (*count of them), or r itself, zeros behind the last one up to a whole tile and behind column d.
template <typename S, typename T>
__global__ void __launch_bounds__(kBlock)
copy_rows_kernel(const S* __restrict__ src, T* __restrict__ dst, const int* count, const int* __restrict__ row_of, int n_src,
                 int n_rows, int d, int d_pad, int planes, int vec) {
  grid_dep_wait();
  grid_dep_release();
  int end = n_src;
  if (row_of != nullptr) {
    const int all = *count;
    end = all < kRowTile ? kRowTile : (all + kRowTile - 1) / kRowTile * kRowTile;
  }
  const int chunks = d_pad / 8;
  const long long total = static_cast<long long>(end) * chunks;
  for (long long i = static_cast<long long>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kBlock) {
    const int r = static_cast<int>(i / chunks), c = 8 * static_cast<int>(i - static_cast<long long>(r) * chunks);
    copy_chunk(src, dst, row_of != nullptr ? row_of[r] : r, r, c, n_rows, d, d_pad, planes, vec);
  }
}

template <typename S, typename T>
int copy_rows_typed(const void* src, void* dst, const int* count, const int* row_of, int n_src, int n_rows, int d, int d_pad,
                    int planes, cudaStream_t st) {
  const int vec = d % 8 == 0 && rowwise::aligned16(src) ? 1 : 0;
  const long long work = static_cast<long long>(row_of != nullptr ? n_rows : n_src) * (d_pad / 8);
  const long long most = 16ll * sm_count();
  const long long need = (work + kBlock - 1) / kBlock;
  const cudaError_t e = launch_kernel(copy_rows_kernel<S, T>, dim3(static_cast<unsigned>(need < most ? need : most)), dim3(kBlock), 0, st,
                               overlap_launches(kOverlapRowwise), static_cast<const S*>(src), static_cast<T*>(dst), count, row_of,
                               n_src, n_rows, d, d_pad, planes, vec);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? NLFA_OK : NLFA_ERR_CUDA;
}
inline int copy_rows(const void* src, int src_dtype, void* dst, int dtype, const int* count, const int* row_of, int n_src, int n_rows,
              int d, int d_pad, int planes, cudaStream_t st) {
#define NLFA_TO(S) (dtype == NLFA_DTYPE_F16 ? copy_rows_typed<S, __half>(src, dst, count, row_of, n_src, n_rows, d, d_pad, planes, st) \
                                            : copy_rows_typed<S, __nv_bfloat16>(src, dst, count, row_of, n_src, n_rows, d, d_pad, planes, st))
  if (src_dtype == NLFA_DTYPE_F32) return NLFA_TO(float);
  if (src_dtype == NLFA_DTYPE_F16) return NLFA_TO(__half);
  return NLFA_TO(__nv_bfloat16);
#undef NLFA_TO
}

// What lies in a tape or scratch lies in blocks, [planes][blocks of 64 columns][rows][64], so that a box is contiguous; a caller's tensor is
// [rows][cols].  Either as (64 columns, rows, blocks of 64 columns, planes), cols a multiple of 64.
inline int box_map(CUtensorMap* map, const void* base, int dtype, long long cols, long long rows, int planes, int box_rows, int box_blocks,
            int box_planes, bool blocked) {
  const unsigned long long pitch = static_cast<unsigned long long>(cols) * 2, r = static_cast<unsigned long long>(rows);
  const unsigned long long dims[4] = {64ull, r, pitch / 128, static_cast<unsigned long long>(planes)};
  const unsigned long long strides[3] = {blocked ? 128ull : pitch, blocked ? 128ull * r : 128ull, pitch * r};
  const unsigned box[4] = {64u, static_cast<unsigned>(box_rows), static_cast<unsigned>(box_blocks), static_cast<unsigned>(box_planes)};
  return make_map(map, base, dtype, dims, strides, box);
}
// One CTA's half of an operand, a stage of it, in all its parts: 128 rows, the summands along the columns ...
inline int column_map(CUtensorMap* map, const void* base, int dtype, long long cols, long long rows, int planes, bool blocked = true) {
  return box_map(map, base, dtype, cols, rows, planes, 128, summands(planes) / 64, planes == 3 ? 3 : 1, blocked);
}
// ... or 128 columns, the summands along the rows.
inline int row_map(CUtensorMap* map, const void* base, int dtype, long long cols, long long rows, int planes, bool blocked = true) {
  return box_map(map, base, dtype, cols, rows, planes, summands(planes), 2, planes == 3 ? 3 : 1, blocked);
}


}  // namespace operands
}  // namespace nlfa
