// Internal interface of the 8-bit products (moe_int8.hip, moe_gemm_int8.hip).
#pragma once

#include "moe_gemm.h"

namespace astrai_moe {

// Rows of 8-bit codes take whole 16-byte units: the kernels read 16 bytes at a
// time. What lies in a weight row behind its last column does not matter, since
// the activations' codes there are 0.
inline int64_t int8_row_bytes(int64_t k) { return ceil_div(k, 16) * 16; }
// Longest row whose products of codes, at most 127 * 128 each, add up below 2^31.
constexpr int64_t kInt8MaxK = 131072;

// C[r, n] = a_scale[r] w_scale[e, n] sum_k a[src, k] w[e, n, k] over the rows r of the
// tile list (src = row_src[r], or r without row_src; e = the tile's expert),
// rounded to dtype: one product and bias, or (w1 set) silu(g) * u of the products
// g with w0 and u with w1.
struct Int8Gemm {
  RowCounts rows;         // the rows as far as the host knows them
  int64_t a_bytes = 0;    // of a, where gathered
  const int8_t* a;        // [*, kp]
  const float* a_scale;   // by row r
  const int32_t* row_src;
  const int32_t* tiles;   // null: one expert's n_rows rows, in tiles of block_m
  int64_t capacity;       // tiles the list holds (without a list: ceil(n_rows / block_m))
  const int8_t *w0, *w1;  // [experts, n, kp]
  const float *s0, *s1;   // [experts, n]
  const void* bias;       // [n] dtype, or null
  int64_t kp, n;
  int dtype;
  void* c;                // [*, n] dtype
  int64_t n_rows;
  int block_m;
  // of the 256-row tiles, as the bf16 products'; its first int32, the counter of the
  // run-time claims, is 0 (the quantiser of a clears it)
  GemmWorkspace ws;
};

// silu(g) u of the sums of two products. An fp32 h is taken in 64 bits and rounded
// once: in 32 bits its last bits would move values across the border between two
// of the codes it is quantised to next (a code in 1e5, an output off by 1e-4 of
// its size). A bf16 h is a step of 2^-8 wide; 32 bits move it to the next one in a
// value of 1e4.
template <typename T>
__device__ __forceinline__ float swiglu(int g, int u, float sa, float sg, float su);
template <>
__device__ __forceinline__ float swiglu<float>(int g, int u, float sa, float sg, float su) {
  const double gd = (double)g * ((double)sa * (double)sg), ud = (double)u * ((double)sa * (double)su);
  return (float)(gd / (1.0 + exp(-gd)) * ud);
}
template <>
__device__ __forceinline__ float swiglu<bf16_t>(int g, int u, float sa, float sg, float su) {
  const float gf = (float)g * (sa * sg);
  const float ex = __builtin_amdgcn_exp2f(gf * -1.4426950408889634f);
  return gf * __builtin_amdgcn_rcpf(1.0f + ex) * ((float)u * (sa * su));
}

int launch_int8_gemm(const Int8Gemm& g, hipStream_t s);

// On the matrix cores (moe_gemm_int8.hip); gate/up products are gathered (row_src),
// the others not. a under 4 GiB where gathered. ragged: rows of a partial K step, or
// outputs whose rows are no whole number of 16 bytes.
int launch_int8_mfma(const Int8Gemm& g, hipStream_t s);
namespace ragged {
int launch_int8_mfma(const Int8Gemm& g, hipStream_t s);
int launch_int8_few(const Int8Gemm& g, hipStream_t s);  // few rows (few_rows), every shape; c aligned
}

}  // namespace astrai_moe
