// Products in 8-bit integers with a scale for each token and each output channel:
// quantisation of rows, the general product, the layer's weighted sum, and the
// entry points of the dense product (a Linear's) and of the experts' forward.
//
// A row x of k values has max = max |x|, scale = max / 127 and the codes
// q = round(127 x / max), halves to even, in [-127, 127]; a row of zeros has scale 0
// and zero codes, one with an infinity or a NaN scale NaN and zero codes, so that
// every product with it is NaN. Then
//   x . w = scale_x scale_w sum_k q_x q_w
// up to the codes' rounding, the sum in 32-bit integers: exact, in any order.
//
// The codes are those of the exact quotient 127 x / max (not of a rounded one), so
// that they do not depend on how the division is carried out: a value in the
// middle between two codes, as x = max / 2 always is, must not turn on a last bit.
#include "moe_common.h"
#include "moe_int8.h"
#include "wave_lanes.h"

namespace astrai_moe {
namespace {

// Where a row's scale goes: scale[r], or the places of its token's rows in the
// permuted order.
struct ScaleOut {
  float* scale;
  const int32_t* token_pos;  // [n_rows, slots], or null
  int slots;
  __device__ void put(int64_t r, float v, int lane) const {
    if (token_pos == nullptr) {
      if (lane == 0) scale[r] = v;
    } else if (lane < slots) {
      scale[token_pos[r * slots + lane]] = v;
    }
  }
};

// One row per WAVES waves, held in registers between its maximum and its codes: a
// thread has NV units of 8 columns, WAVES * 512 columns apart. kVec: rows start on
// 16-byte boundaries. clear: a counter of the product that follows, set to 0. One read
// of x and one write of the codes, bound by these: bf16, 8192 rows of 4096 25 to 28 us
// (3.8 TB/s), 32768 of 14336 255 to 282 us (5.0 to 5.5 TB/s; a large copy reaches 5.2).
template <typename T, int WAVES, int NV, bool kVec>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t n_rows, int64_t k,
                                                            int64_t kp, int8_t* __restrict__ q, const ScaleOut out,
                                                            int32_t* clear) {
  using C = typename CodeType<T>::type;
  constexpr int ROWS = 4 / WAVES;
  __shared__ float s_most[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * ROWS + (WAVES == 1 ? wave : 0);
  const bool on = r < n_rows;
  const T* const row = x + (on ? r : 0) * k;
  const int c0 = (WAVES == 1 ? lane : (int)threadIdx.x) * 8;
  if (clear != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *clear = 0;
  Unit<T> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i].template load<kVec>(row, c0 + i * WAVES * 512, on ? k : 0);
  // (as integers, which order the magnitudes of floats, NaN above infinity)
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, v[i].bits(j) & 0x7fffffffu);
  top = lanes_max<64>(top);
  if constexpr (WAVES > 1) {
    if (lane == 0) s_most[wave] = __uint_as_float(top);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, __float_as_uint(s_most[w]));
  }
  if (!on) return;
  const float most = __uint_as_float(top);
  const bool bad = top >= 0x7f800000u;
  if (WAVES == 1 || wave == 0) out.put(r, bad ? NAN : most / 127.0f, lane);
  const float shift = range_shift(most);
  const C m = (C)most * (C)shift, inv = (C)127 / m;
  const bool zero = bad || most == 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * WAVES * 512;
    if (c >= kp) continue;
    *reinterpret_cast<uint2*>(q + r * kp + c) = zero ? make_uint2(0, 0) : v[i].template codes<C>(shift, m, inv);
  }
}

// Rows longer than the registers of a workgroup (16384 columns): read twice.
template <typename T>
__global__ __launch_bounds__(256) void quantize_long_rows_kernel(const T* __restrict__ x, int64_t n_rows, int64_t k,
                                                                 int64_t kp, int8_t* __restrict__ q,
                                                                 const ScaleOut out, int32_t* clear) {
  using C = typename CodeType<T>::type;
  __shared__ uint32_t s_top[4];
  if (clear != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *clear = 0;
  const int64_t r = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const T* const row = x + r * k;
  uint32_t top = 0;
  for (int64_t c = threadIdx.x; c < k; c += 256) top = max(top, __float_as_uint(Elem<T>::to_f32(row[c])) & 0x7fffffffu);
  top = lanes_max<64>(top);
  if (lane == 0) s_top[wave] = top;
  __syncthreads();
  top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
  const float most = __uint_as_float(top);
  const bool bad = top >= 0x7f800000u, zero = bad || most == 0.0f;
  if (wave == 0) out.put(r, bad ? NAN : most / 127.0f, lane);
  const float shift = range_shift(most);
  const C m = (C)most * (C)shift, inv = (C)127 / m;
  for (int64_t c0 = threadIdx.x * 8; c0 < kp; c0 += 256 * 8) {
    union {
      int8_t b[8];
      uint2 u;
    } o;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o.b[j] = zero || c0 + j >= k ? (int8_t)0 : (int8_t)code_of<C>((C)Elem<T>::to_f32(row[c0 + j]) * (C)shift, m, inv);
    *reinterpret_cast<uint2*>(q + r * kp + c0) = o.u;
  }
}

template <typename T, int WAVES, int NV>
void launch_quantize_cfg(const void* x, bool vec, int64_t n_rows, int64_t k, int8_t* q, const ScaleOut& out,
                         int32_t* clear, hipStream_t s) {
  hipLaunchKernelGGL((vec ? quantize_rows_kernel<T, WAVES, NV, true> : quantize_rows_kernel<T, WAVES, NV, false>),
                     dim3((unsigned)ceil_div(n_rows, 4 / WAVES)), dim3(256), 0, s, static_cast<const T*>(x), n_rows, k,
                     int8_row_bytes(k), q, out, clear);
}

// A wave per row up to 1024 columns, a workgroup beyond.
template <typename T>
int launch_quantize(const void* x, int64_t n_rows, int64_t k, int8_t* q, const ScaleOut& out, int32_t* clear,
                    hipStream_t s) {
  const bool vec = k * (int64_t)sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  if (k <= 512)
    launch_quantize_cfg<T, 1, 1>(x, vec, n_rows, k, q, out, clear, s);
  else if (k <= 1024)
    launch_quantize_cfg<T, 1, 2>(x, vec, n_rows, k, q, out, clear, s);
  else if (k <= 2048)
    launch_quantize_cfg<T, 4, 1>(x, vec, n_rows, k, q, out, clear, s);
  else if (k <= 4096)
    launch_quantize_cfg<T, 4, 2>(x, vec, n_rows, k, q, out, clear, s);
  else if (k <= 8192)
    launch_quantize_cfg<T, 4, 4>(x, vec, n_rows, k, q, out, clear, s);
  else if (k <= 16384)
    launch_quantize_cfg<T, 4, 8>(x, vec, n_rows, k, q, out, clear, s);
  else
    hipLaunchKernelGGL(quantize_long_rows_kernel<T>, dim3((unsigned)n_rows), dim3(256), 0, s,
                       static_cast<const T*>(x), n_rows, k, int8_row_bytes(k), q, out, clear);
  return check_launch("quantize_rows_kernel");
}

int launch_quantize_rows(const void* x, int dtype, int64_t n_rows, int64_t k, int8_t* q, const ScaleOut& out,
                         int32_t* clear, hipStream_t s) {
  if (n_rows == 0) return ASTRAI_MOE_OK;
  return dtype == ASTRAI_MOE_BF16 ? launch_quantize<bf16_t>(x, n_rows, k, q, out, clear, s)
                                  : launch_quantize<float>(x, n_rows, k, q, out, clear, s);
}

// The gate/up product without matrix cores, for what those kernels leave: gathered codes
// of 4 GiB and more, whose rows 32-bit offsets do not reach. 64 x 64 tiles, 64 bytes of
// K staged at a time, four codes a multiply-add (v_dot4), which bounds it.
constexpr int kTile = 64, kStep = 64, kPad = 16;

template <typename T>
__global__ __launch_bounds__(256) void gate_up_dot4_kernel(const Int8Gemm p) {
  const int tile = blockIdx.x;
  if (tile >= min(p.tiles[0], (int)min((int64_t)p.tiles[2], p.capacity))) return;
  const int32_t* const ti = p.tiles + ASTRAI_MOE_TILE_HEADER + (int64_t)tile * ASTRAI_MOE_TILE_STRIDE;
  const int64_t e = ti[0], row0 = ti[1], rows = min(p.tiles[1], ti[2] - ti[1]);
  const int64_t n0 = (int64_t)blockIdx.y * kTile;
  const int8_t* const w0 = p.w0 + e * p.n * p.kp;
  const int8_t* const w1 = p.w1 + e * p.n * p.kp;
  __shared__ __attribute__((aligned(16))) int8_t As[kTile][kStep + kPad];
  __shared__ __attribute__((aligned(16))) int8_t B0[kTile][kStep + kPad];
  __shared__ __attribute__((aligned(16))) int8_t B1[kTile][kStep + kPad];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int lr = threadIdx.x / 4, lc = threadIdx.x % 4 * 16;  // staged row and byte
  for (int64_t rs = 0; rs < rows; rs += kTile) {
    int acc0[4][4] = {}, acc1[4][4] = {};
    const bool row_in = rs + lr < rows, col_in = n0 + lr < p.n;
    const int64_t src = row_in ? p.row_src[row0 + rs + lr] : 0;
    for (int64_t k0 = 0; k0 < p.kp; k0 += kStep) {
      const bool k_in = k0 + lc < p.kp;
      const uint4 none = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(&As[lr][lc]) =
          row_in && k_in ? *reinterpret_cast<const uint4*>(p.a + src * p.kp + k0 + lc) : none;
      *reinterpret_cast<uint4*>(&B0[lr][lc]) =
          col_in && k_in ? *reinterpret_cast<const uint4*>(w0 + (n0 + lr) * p.kp + k0 + lc) : none;
      *reinterpret_cast<uint4*>(&B1[lr][lc]) =
          col_in && k_in ? *reinterpret_cast<const uint4*>(w1 + (n0 + lr) * p.kp + k0 + lc) : none;
      __syncthreads();
      for (int kk = 0; kk < kStep; kk += 4) {
        int a[4], b0[4], b1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const int*>(&As[ty + 16 * i][kk]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          b0[j] = *reinterpret_cast<const int*>(&B0[tx + 16 * j][kk]);
          b1[j] = *reinterpret_cast<const int*>(&B1[tx + 16 * j][kk]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc0[i][j] = __builtin_amdgcn_sdot4(a[i], b0[j], acc0[i][j], false);
            acc1[i][j] = __builtin_amdgcn_sdot4(a[i], b1[j], acc1[i][j], false);
          }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t in = rs + ty + 16 * i;
      if (in >= rows) continue;
      const int64_t row = row0 + in;
      const float sa = p.a_scale[row];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + tx + 16 * j;
        if (n >= p.n) continue;
        const float v = swiglu<T>(acc0[i][j], acc1[i][j], sa, p.s0[e * p.n + n], p.s1[e * p.n + n]);
        static_cast<T*>(p.c)[row * p.n + n] = Elem<T>::from_f32(v);
      }
    }
  }
}

template <typename T>
int launch_gate_up_dot4(const Int8Gemm& g, hipStream_t s) {
  const int64_t cols = ceil_div(g.n, kTile);
  ASTRAI_REQUIRE(g.capacity < (1ll << 31) && cols < 65536, "int8 product: too many tiles");
  if (g.capacity == 0) return ASTRAI_MOE_OK;
  hipLaunchKernelGGL((gate_up_dot4_kernel<T>), dim3((unsigned)g.capacity, (unsigned)cols), dim3(256), 0, s, g);
  return check_launch("gate_up_dot4_kernel");
}

// out[t] = sum over the routed slots of w y + (sum over the shared ones of y) /
// n_shared: 32-bit sums in the order of the slots, rounded once. A slot of weight 0
// adds nothing, whatever its row holds (padding tokens have only such).
// One workgroup per token (and 2048 columns), a thread per VW columns; the rows' loads
// of up to 8 slots in flight at a time. Bound by reading y and writing out: 16384 tokens
// of 2 rows of 4096 bf16 values 96 us (4.2 TB/s).
template <typename T, int VW>
__global__ __launch_bounds__(256) void sum_slots_kernel(const T* __restrict__ y, const int32_t* __restrict__ token_pos,
                                                        const T* __restrict__ row_w, int64_t n_tokens, int top_k,
                                                        int n_shared, int64_t dim, T* __restrict__ out) {
  struct alignas(VW * sizeof(T)) Vec {
    T v[VW];
  };
  const int64_t t = blockIdx.x;
  const int slots = top_k + n_shared;
  const float part = n_shared > 0 ? 1.0f / (float)n_shared : 0.0f;
  for (int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * VW; c < dim; c += (int64_t)gridDim.y * 256 * VW) {
    float sum[VW] = {};
    for (int k0 = 0; k0 < slots; k0 += 8) {
      Vec in[8];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = 0.0f;
        if (k0 + j < slots) {
          const int row = token_pos[t * slots + k0 + j];
          w[j] = k0 + j < top_k ? Elem<T>::to_f32(row_w[row]) : part;
          in[j] = *reinterpret_cast<const Vec*>(y + (int64_t)row * dim + c);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w[j] != 0.0f)
#pragma unroll
          for (int i = 0; i < VW; ++i) sum[i] = fmaf(w[j], Elem<T>::to_f32(in[j].v[i]), sum[i]);
    }
    Vec o;
#pragma unroll
    for (int i = 0; i < VW; ++i) o.v[i] = Elem<T>::from_f32(sum[i]);
    *reinterpret_cast<Vec*>(out + t * dim + c) = o;
  }
}

template <typename T>
int launch_sum_typed(const void* y, const int32_t* token_pos, const void* row_w, int64_t n_tokens, int top_k,
                     int n_shared, int64_t dim, void* out, hipStream_t s) {
  constexpr int kVW = 16 / sizeof(T);
  const bool vec = dim % kVW == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;  // (y is the workspace's)
  const dim3 grid((unsigned)n_tokens, (unsigned)std::min<int64_t>(ceil_div(dim, 256 * (vec ? kVW : 1)), 64));
  hipLaunchKernelGGL((vec ? sum_slots_kernel<T, kVW> : sum_slots_kernel<T, 1>), grid, dim3(256), 0, s,
                     static_cast<const T*>(y), token_pos, static_cast<const T*>(row_w), n_tokens, top_k, n_shared, dim,
                     static_cast<T*>(out));
  return check_launch("sum_slots_kernel");
}

int launch_sum_slots(const void* y, const int32_t* token_pos, const void* row_w, int dtype, int64_t n_tokens,
                     int top_k, int n_shared, int64_t dim, void* out, hipStream_t s) {
  return dtype == ASTRAI_MOE_BF16
             ? launch_sum_typed<bf16_t>(y, token_pos, row_w, n_tokens, top_k, n_shared, dim, out, s)
             : launch_sum_typed<float>(y, token_pos, row_w, n_tokens, top_k, n_shared, dim, out, s);
}

int check_int8(const char* who, int dtype, int64_t k, int64_t n) {
  ASTRAI_REQUIRE(dtype == ASTRAI_MOE_BF16 || dtype == ASTRAI_MOE_F32, "%s: unsupported dtype %d", who, dtype);
  ASTRAI_REQUIRE(k >= 1 && k <= kInt8MaxK && n >= 1 && n <= (1ll << 22),
                 "%s: inner size must be in [1, %lld] and outputs in [1, 2^22] (got %lld, %lld)", who,
                 (long long)kInt8MaxK, (long long)k, (long long)n);
  return ASTRAI_MOE_OK;
}

// Row-tile heights: those of the bf16 products (astrai_moe_select_block_m), whose
// tiles take the same time a step.
int layer_block_m(int64_t rows_per_expert) {
  return rows_per_expert < 24    ? kMfmaSmallBM
         : rows_per_expert < 48  ? kMfmaMidBM
         : rows_per_expert < 128 ? kMfmaMid2BM
                                 : kMfmaBigBM;
}
int linear_block_m(int64_t n_rows, int64_t kp, int64_t n) {
  if (n_rows <= 32 || (n_rows < 96 && int8_few_rows(RowCounts(n_rows, 1), kMfmaSmallBM, kp, n, false)))
    return kMfmaSmallBM;
  return dense_gemm_block_m(n_rows, kp / 2, n, false);
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct Parts {  // of a workspace, 256-byte aligned
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t here = bytes;
    bytes += (n + 255) / 256 * 256;
    return here;
  }
};

struct LinearPlan {
  int block_m;
  int64_t q, scale, gemm_ws, gemm_ws_bytes = 0, bytes;
  LinearPlan(int64_t m, int64_t k, int64_t n) {
    const int64_t kp = int8_row_bytes(k);
    block_m = linear_block_m(m, kp, n);
    if (block_m == kMfmaBigBM)
      gemm_ws_bytes = gemm_workspace_bytes(down_splits(RowCounts(m, 1), block_m, kp / 2, n, false));
    Parts p;
    q = p.take(m * kp);
    scale = p.take(m * 4);
    gemm_ws = p.take(gemm_ws_bytes);
    bytes = p.bytes;
  }
};

struct LayerSizes {
  int64_t n_tokens;
  int n_experts, top_k, n_shared;
  int64_t dim, dim_ffn;
  int dtype;
};

int check_layer(const LayerSizes& z) {
  if (int rc = check_int8("int8_forward", z.dtype, z.dim, z.dim_ffn)) return rc;
  if (int rc = check_int8("int8_forward", z.dtype, z.dim_ffn, z.dim)) return rc;
  ASTRAI_REQUIRE(z.n_shared >= 0 && z.n_shared <= ASTRAI_MOE_MAX_TOPK, "int8_forward: bad n_shared %d", z.n_shared);
  ASTRAI_REQUIRE(z.n_experts >= 1 && z.n_experts + z.n_shared <= ASTRAI_MOE_MAX_EXPERTS,
                 "int8_forward: n_experts + n_shared must be in [1, %d] (got %d + %d)", ASTRAI_MOE_MAX_EXPERTS,
                 z.n_experts, z.n_shared);
  ASTRAI_REQUIRE(z.top_k >= 1 && z.top_k <= z.n_experts && z.top_k + z.n_shared <= ASTRAI_MOE_MAX_TOPK,
                 "int8_forward: top_k must be in [1, n_experts] and top_k + n_shared at most %d (got %d + %d)",
                 ASTRAI_MOE_MAX_TOPK, z.top_k, z.n_shared);
  ASTRAI_REQUIRE(z.n_tokens >= 0 && z.n_tokens * (int64_t)(z.top_k + z.n_shared) < (1ll << 31),
                 "int8_forward: n_tokens * (top_k + n_shared) must be in [0, 2^31)");
  return ASTRAI_MOE_OK;
}

RowCounts row_counts(const LayerSizes& z) { return {z.n_tokens * z.top_k, z.n_experts, z.n_shared, z.n_tokens}; }

struct LayerPlan {
  int experts, slots, block_m;
  bool quant_up, quant_down;  // the products quantise their rows themselves
  int64_t rows, tiles_len, dp, fp;
  int64_t topk_idx, topk_w, chunk_hist, chunk_base, offsets, sorted_token, sorted_w, token_pos, tiles, xq, xs, h, hq, hs,
      y, gemm_ws, gemm_ws_bytes = 0, bytes;
  explicit LayerPlan(const LayerSizes& z) {
    const int64_t size = z.dtype == ASTRAI_MOE_BF16 ? 2 : 4, T = z.n_tokens;
    experts = z.n_experts + z.n_shared;
    slots = z.top_k + z.n_shared;
    rows = T * slots;
    block_m = layer_block_m(T * z.top_k / z.n_experts);
    tiles_len = astrai_moe_tile_list_len(T, experts, slots, block_m);
    dp = int8_row_bytes(z.dim);
    fp = int8_row_bytes(z.dim_ffn);
    Parts p;
    topk_idx = p.take(rows * 4);
    topk_w = p.take(rows * size);
    chunk_hist = p.take(n_chunks(T) * experts * 4);
    chunk_base = p.take(n_chunks(T) * experts * 4);
    offsets = p.take((experts + 1) * 4);
    sorted_token = p.take(rows * 4);
    sorted_w = p.take(rows * size);
    token_pos = p.take(rows * 4);
    tiles = p.take(tiles_len * 4);
    xq = p.take(T * dp);
    xs = p.take(rows * 4);  // by permuted row
    // h is read once, to be quantised, before the down product writes y (which a product
    // that quantises it itself does meanwhile)
    h = p.take(rows * std::max(z.dim_ffn, z.dim) * size);
    // An expert meets a token once: its rows are at most the tokens.
    const int64_t tiles_most = (tiles_len - ASTRAI_MOE_TILE_HEADER) / ASTRAI_MOE_TILE_STRIDE;
    quant_up = int8_quantises(T, z.dim, tiles_most, z.dim_ffn, true);
    quant_down = int8_quantises(T, z.dim_ffn, tiles_most, z.dim, false);
    y = quant_down ? p.take(rows * z.dim * size) : h;
    hq = p.take(rows * fp);
    hs = p.take(rows * 4);
    if (block_m == kMfmaBigBM)
      gemm_ws_bytes = gemm_workspace_bytes(down_splits(row_counts(z), block_m, fp / 2, z.dim, false));
    gemm_ws = p.take(gemm_ws_bytes);
    bytes = p.bytes;
  }
};

}  // namespace

// (gate/up products gather their rows, the others do not)
int launch_int8_gemm(const Int8Gemm& g, hipStream_t s) {
  if (g.a == nullptr || g.row_src == nullptr || g.a_bytes < (1ll << 32)) return launch_int8_mfma(g, s);
  return g.dtype == ASTRAI_MOE_BF16 ? launch_gate_up_dot4<bf16_t>(g, s) : launch_gate_up_dot4<float>(g, s);
}

}  // namespace astrai_moe

using namespace astrai_moe;

extern "C" int64_t astrai_moe_int8_row_bytes(int64_t k) { return k < 0 ? -1 : int8_row_bytes(k); }

extern "C" int astrai_moe_quantize_rows(const void* x, int dtype, int64_t n_rows, int64_t k, int8_t* q, float* scale,
                                        void* stream) {
  clear_error();
  if (int rc = check_int8("quantize_rows", dtype, k, 1)) return rc;
  ASTRAI_REQUIRE(n_rows >= 0 && n_rows < (1ll << 31), "quantize_rows: n_rows must be in [0, 2^31)");
  if (n_rows == 0) return ASTRAI_MOE_OK;
  ASTRAI_REQUIRE(x && q && scale, "quantize_rows: null buffer");
  ASTRAI_REQUIRE(on16(q), "quantize_rows: q must start on a 16-byte boundary");
  return launch_quantize_rows(x, dtype, n_rows, k, q, ScaleOut{scale, nullptr, 0}, nullptr,
                              static_cast<hipStream_t>(stream));
}

extern "C" int64_t astrai_moe_int8_linear_workspace_bytes(int64_t n_rows, int64_t k, int64_t n, int dtype) {
  clear_error();
  if (int rc = check_int8("int8_linear", dtype, k, n)) return rc;
  ASTRAI_REQUIRE(n_rows >= 0 && n_rows < (1ll << 31), "int8_linear: n_rows must be in [0, 2^31)");
  return LinearPlan(n_rows, k, n).bytes;
}

extern "C" int astrai_moe_int8_linear(const void* x, int dtype, const int8_t* w, const float* w_scale,
                                      const void* bias, int64_t n_rows, int64_t k, int64_t n, void* workspace,
                                      int64_t workspace_bytes, void* out, void* stream) {
  clear_error();
  if (int rc = check_int8("int8_linear", dtype, k, n)) return rc;
  ASTRAI_REQUIRE(n_rows >= 0 && n_rows < (1ll << 31), "int8_linear: n_rows must be in [0, 2^31)");
  if (n_rows == 0) return ASTRAI_MOE_OK;
  ASTRAI_REQUIRE(x && w && w_scale && workspace && out, "int8_linear: null buffer");
  ASTRAI_REQUIRE(on16(w), "int8_linear: the weight must start on a 16-byte boundary");
  ASTRAI_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "int8_linear: workspace must be 256-byte aligned");
  const LinearPlan p(n_rows, k, n);
  ASTRAI_REQUIRE(workspace_bytes >= p.bytes, "int8_linear: workspace holds %lld bytes, needs %lld",
                 (long long)workspace_bytes, (long long)p.bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const base = static_cast<char*>(workspace);
  int8_t* const q = reinterpret_cast<int8_t*>(base + p.q);
  float* const scale = reinterpret_cast<float*>(base + p.scale);
  int32_t* const claims = p.gemm_ws_bytes > 0 ? reinterpret_cast<int32_t*>(base + p.gemm_ws) : nullptr;
  Int8Gemm g{RowCounts(n_rows, 1)};
  if (int8_quantises(n_rows, k, 1, n, false) && on16(out)) {
    g.x = x, g.k = k;
  } else {
    if (int rc = launch_quantize_rows(x, dtype, n_rows, k, q, ScaleOut{scale, nullptr, 0}, claims, s)) return rc;
    g.a = q, g.a_scale = scale;
  }
  g.w0 = w, g.s0 = w_scale, g.bias = bias;
  g.kp = int8_row_bytes(k), g.n = n, g.dtype = dtype, g.c = out;
  g.n_rows = n_rows, g.block_m = p.block_m, g.capacity = ceil_div(n_rows, g.block_m);
  if (p.gemm_ws_bytes > 0) g.ws = {base + p.gemm_ws, p.gemm_ws_bytes};
  return launch_int8_gemm(g, s);
}

extern "C" int64_t astrai_moe_int8_forward_workspace_bytes(int64_t n_tokens, int n_experts, int top_k, int n_shared,
                                                           int64_t dim, int64_t dim_ffn, int dtype) {
  clear_error();
  const LayerSizes z{n_tokens, n_experts, top_k, n_shared, dim, dim_ffn, dtype};
  if (int rc = check_layer(z)) return rc;
  return LayerPlan(z).bytes;
}

extern "C" int astrai_moe_int8_forward(const void* x, int dtype, const void* logits, int logits_dtype,
                                       const float* bias, const astrai_moe_routing* routing, const int8_t* w_gate,
                                       const int8_t* w_up, const int8_t* w_down, const float* gate_scale,
                                       const float* up_scale, const float* down_scale, int64_t n_tokens, int n_experts,
                                       int top_k, int n_shared, int64_t dim, int64_t dim_ffn, void* workspace,
                                       int64_t workspace_bytes, void* out, void* stream) {
  clear_error();
  const LayerSizes z{n_tokens, n_experts, top_k, n_shared, dim, dim_ffn, dtype};
  int rc = check_layer(z);
  if (rc) return rc;
  if (routing != nullptr) {
    if ((rc = check_routing("int8_forward", routing, logits_dtype, dtype, n_tokens, n_experts, top_k))) return rc;
  } else {
    ASTRAI_REQUIRE(logits_dtype == dtype && bias == nullptr,
                   "int8_forward: without a routing the logits have x's dtype and no bias");
  }
  if (n_tokens == 0) return ASTRAI_MOE_OK;
  ASTRAI_REQUIRE(x && logits && w_gate && w_up && w_down && gate_scale && up_scale && down_scale && workspace && out,
                 "int8_forward: null buffer");
  ASTRAI_REQUIRE(on16(w_gate) && on16(w_up) && on16(w_down), "int8_forward: weights must start on 16-byte boundaries");
  ASTRAI_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "int8_forward: workspace must be 256-byte aligned");
  const LayerPlan p(z);
  ASTRAI_REQUIRE(workspace_bytes >= p.bytes, "int8_forward: workspace holds %lld bytes, needs %lld",
                 (long long)workspace_bytes, (long long)p.bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const base = static_cast<char*>(workspace);
  auto i32 = [&](int64_t off) { return reinterpret_cast<int32_t*>(base + off); };
  auto i8 = [&](int64_t off) { return reinterpret_cast<int8_t*>(base + off); };
  auto f32 = [&](int64_t off) { return reinterpret_cast<float*>(base + off); };
  int32_t *const topk_idx = i32(p.topk_idx), *const hist = i32(p.chunk_hist), *const tiles = i32(p.tiles);
  int32_t* const claims = p.gemm_ws_bytes > 0 ? i32(p.gemm_ws) : nullptr;
  // One chunk of tokens: routing and permutation in one workgroup.
  if (n_tokens <= ASTRAI_MOE_CHUNK_TOKENS) {
    const RouteList list{i32(p.sorted_token), base + p.sorted_w, i32(p.token_pos), tiles,
                         (p.tiles_len - ASTRAI_MOE_TILE_HEADER) / ASTRAI_MOE_TILE_STRIDE, p.block_m};
    rc = routing != nullptr ? launch_route_scores_list(logits, logits_dtype, bias, *routing, n_tokens, n_experts, top_k,
                                                       n_shared, dtype, list, s)
                            : launch_route_list(logits, dtype, n_tokens, n_experts, top_k, n_shared, list, s);
    if (rc) return rc;
  } else {
    rc = routing != nullptr
             ? launch_route_scores(logits, logits_dtype, bias, *routing, n_tokens, n_experts, top_k, n_shared, dtype,
                                   topk_idx, base + p.topk_w, hist, s)
             : launch_route(logits, dtype, n_tokens, n_experts, top_k, n_shared, topk_idx, base + p.topk_w, hist, s);
    if (rc) return rc;
    if ((rc = astrai_moe_permute(topk_idx, base + p.topk_w, hist, nullptr, dtype, n_tokens, p.experts, p.slots, p.dp / 2,
                                 p.block_m, i32(p.offsets), i32(p.sorted_token), base + p.sorted_w, i32(p.token_pos),
                                 nullptr, tiles, p.tiles_len, i32(p.chunk_base), stream)))
      return rc;
  }
  Int8Gemm g{row_counts(z)};
  if (p.gemm_ws_bytes > 0) g.ws = {base + p.gemm_ws, p.gemm_ws_bytes};
  if (p.quant_up) {
    g.x = x, g.k = dim;
  } else {
    if ((rc = launch_quantize_rows(x, dtype, n_tokens, dim, i8(p.xq), ScaleOut{f32(p.xs), i32(p.token_pos), p.slots},
                                   claims, s)))
      return rc;
    g.a = i8(p.xq), g.a_scale = f32(p.xs), g.a_bytes = n_tokens * p.dp;
  }
  g.row_src = i32(p.sorted_token);
  g.tiles = tiles, g.capacity = (p.tiles_len - ASTRAI_MOE_TILE_HEADER) / ASTRAI_MOE_TILE_STRIDE;
  g.w0 = w_gate, g.w1 = w_up, g.s0 = gate_scale, g.s1 = up_scale;
  g.kp = p.dp, g.n = dim_ffn, g.dtype = dtype, g.c = base + p.h, g.block_m = p.block_m;
  if ((rc = launch_int8_gemm(g, s))) return rc;
  if (p.quant_down) {
    g.a = nullptr, g.x = base + p.h, g.k = dim_ffn;
  } else {
    if ((rc = launch_quantize_rows(base + p.h, dtype, p.rows, dim_ffn, i8(p.hq), ScaleOut{f32(p.hs), nullptr, 0}, claims,
                                   s)))
      return rc;
    g.a = i8(p.hq), g.a_scale = f32(p.hs);
  }
  g.row_src = nullptr;
  g.w0 = w_down, g.w1 = nullptr, g.s0 = down_scale, g.s1 = nullptr;
  g.kp = p.fp, g.n = dim, g.c = base + p.y;
  if ((rc = launch_int8_gemm(g, s))) return rc;
  return launch_sum_slots(base + p.y, i32(p.token_pos), base + p.sorted_w, dtype, n_tokens, top_k, n_shared, dim, out, s);
}
