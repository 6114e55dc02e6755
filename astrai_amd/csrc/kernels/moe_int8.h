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
  const int8_t* a;        // [*, kp]; null: the kernel quantises the rows of x itself
  const float* a_scale;   // by row r
  const void* x;          // [*, k] dtype
  int64_t k;
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

// round-half-even of 127 x / most, |x| <= most, exactly: n = the nearest integer to
// the product with a rounded reciprocal is off by one at most, and the remainder 127
// x - n most decides. C holds it exactly: 127 x and n most have 7 more bits than x
// and most, and where n is not 0 their exponents are within 8 of each other (bf16
// in 32 bits, fp32 in 64).
template <typename C>
__device__ __forceinline__ int code_of(C x, C most, C inv) {
  C n = __builtin_elementwise_rint(x * inv);
  const C d = __builtin_elementwise_fma(-n, most, x * (C)127), twice = (C)2 * __builtin_elementwise_abs(d);
  const int i = (int)n;
  const bool away = twice > most || (twice == most && (i & 1) != 0);
  return away ? i + (d > (C)0 ? 1 : -1) : i;
}

template <typename T>
struct CodeType {
  typedef float type;  // of bf16
};
template <>
struct CodeType<float> {
  typedef double type;
};

// A power of two that brings a row's maximum away from the ends of the range, where
// 127 x or 127 / most would leave it. (Values that vanish by it have code 0.)
__device__ __forceinline__ float range_shift(float most) {
  return most >= 0x1p100f ? 0x1p-64f : most < 0x1p-60f ? 0x1p64f : 1.0f;
}

__device__ __forceinline__ uint32_t word_of(bf16_t v) { return v; }
__device__ __forceinline__ uint32_t word_of(float v) { return __float_as_uint(v); }

// Eight consecutive values of a row in registers, two bf16 a word.
template <typename T>
struct Unit {
  static constexpr int WORDS = 2 * sizeof(T);
  uint32_t w[WORDS];
  // from column c on, zeros from column k on; kVec: 16-byte loads (rows of whole 16-byte
  // pieces on 16-byte boundaries), without a branch, so that several are in flight
  template <bool kVec>
  __device__ __forceinline__ void load(const T* row, int64_t c, int64_t k) {
    if (kVec) {
#pragma unroll
      for (int j = 0; j < WORDS; j += 4) {
        const int64_t at = c + j * (4 / (int)sizeof(T));
        const bool in = at < k;
        const uint4 v = *reinterpret_cast<const uint4*>(row + (in ? at : 0));
        w[j] = in ? v.x : 0, w[j + 1] = in ? v.y : 0, w[j + 2] = in ? v.z : 0, w[j + 3] = in ? v.w : 0;
      }
    } else {
      T in[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) in[j] = c + j < k ? row[c + j] : (T)0;
#pragma unroll
      for (int j = 0; j < WORDS; ++j)
        w[j] = sizeof(T) == 2 ? word_of(in[(2 * j) & 7]) | word_of(in[(2 * j + 1) & 7]) << 16 : word_of(in[j & 7]);
    }
  }
  // the j-th value as a float's bits
  __device__ __forceinline__ uint32_t bits(int j) const {
    if constexpr (sizeof(T) == 2)
      return (j & 1) != 0 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16;
    else
      return w[j];
  }
  // the codes for a row's shifted maximum `most`, 127 / most = inv
  template <typename C>
  __device__ __forceinline__ uint2 codes(float shift, C most, C inv) const {
    union {
      int8_t b[8];
      uint2 u;
    } o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.b[j] = (int8_t)code_of<C>((C)__uint_as_float(bits(j)) * (C)shift, most, inv);
    return o.u;
  }
};

// On the matrix cores (moe_gemm_int8.hip); gate/up products are gathered (row_src),
// the others not. a under 4 GiB where gathered. ragged: rows of a partial K step, or
// outputs whose rows are no whole number of 16 bytes.
int launch_int8_mfma(const Int8Gemm& g, hipStream_t s);
namespace ragged {
int launch_int8_mfma(const Int8Gemm& g, hipStream_t s);
int launch_int8_few(const Int8Gemm& g, hipStream_t s);  // few rows, every shape; c aligned
int launch_int8_quant(const Int8Gemm& g, hipStream_t s);
}
// Whether a product runs on the few-row kernels.
bool int8_few_rows(const RowCounts& rows, int block_m, int64_t kp, int64_t n, bool gate_up);
// Whether a product of row_tiles row tiles of at most most_rows rows of k values is to
// quantise them itself (launch_int8_quant).
bool int8_quantises(int64_t most_rows, int64_t k, int64_t row_tiles, int64_t n, bool gate_up);

}  // namespace astrai_moe
