// Routing by scores: softmax or sigmoid scores, a bias for balance, groups of
// experts, top-k and renormalised weights; the gradient of its weights; the
// experts' loads and the step of the bias that evens them out.
//
// For a token with logits l over E experts in G groups of E / G consecutive ones:
//   s = softmax(l) or sigmoid(l)
//   c_e = s_e + b_e, -inf where l_e = -inf (an expert switched off)
//   a group's value is the sum of its group_top (1 or 2) largest c; the
//   topk_groups best groups stay (ties: the lower group)
//   chosen: the top_k largest c of these, descending (ties: the lower expert);
//   slots for which no c above -inf is left take the lowest experts not chosen
//   yet, with weight 0
//   w_k = scale s_k / S, S = sum of the chosen s (0 where S = 0), or, not
//   renormalised, scale s_k: one rounding to the weights' type.
// A row with a NaN among its logits (softmax: or +inf) has experts 0 .. top_k - 1
// and NaN weights, and NaN gradients at these (softmax: at all). A bias of -inf or
// NaN turns its expert off.
//
// The decisions are made in 64 bits: c in 32 bits takes two experts whose scores
// differ by less than a rounding for equal, or swaps them.
#include "moe_common.h"
#include "moe_gemm.h"

#include <math.h>

namespace astrai_moe {
namespace {

constexpr int kScoreWaves = 8;  // tokens of a chunk in flight at a time

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// A 64-bit float as an integer that orders alike; every float's is above 0, which
// stands for what is taken or does not exist. NaN counts as -inf.
constexpr uint64_t kNone = 0, kOff = 0x000fffffffffffffull;  // kOff: -inf's
__device__ __forceinline__ uint64_t order_of(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);  // (-0 as 0)
  return v != v ? kOff : (u >> 63) != 0 ? ~u : u | 1ull << 63;
}

__device__ __forceinline__ double value_of(uint64_t o) {
  return __builtin_bit_cast(double, (o >> 63) != 0 ? o & ~(1ull << 63) : ~o);
}

// The largest of the lanes' (value, index) pairs, ties to the lower index.
__device__ __forceinline__ void wave_best(uint64_t& v, int& at) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off, 64);
    const int oi = __shfl_xor(at, off, 64);
    if (o > v || (o == v && oi < at)) v = o, at = oi;
  }
}

// The best of the lanes' N pairs, taken out of them: its value, and its index in `at`.
template <int N>
__device__ __forceinline__ uint64_t take_best(uint64_t (&v)[N], const int (&index)[N], int& at) {
  uint64_t best = v[0];
  at = index[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (v[i] > best) best = v[i], at = index[i];  // (a lane's indices ascend)
  wave_best(best, at);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (index[i] == at) v[i] = kNone;
  return best;
}

template <typename T, typename W, int ITER>
__global__ __launch_bounds__(kScoreWaves * 64) void route_scores_kernel(
    const T* __restrict__ logits, const float* __restrict__ bias, const astrai_moe_routing opt, int64_t n_tokens,
    int n_experts, int top_k, int n_shared, int32_t* __restrict__ topk_idx, W* __restrict__ topk_w,
    int32_t* __restrict__ chunk_hist) {
  __shared__ int hist[ASTRAI_MOE_MAX_EXPERTS];
  __shared__ uint64_t s_key[kScoreWaves][ITER * 64];
  __shared__ uint32_t s_kept[kScoreWaves][ASTRAI_MOE_MAX_EXPERTS / 32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t_begin = (int64_t)blockIdx.x * ASTRAI_MOE_CHUNK_TOKENS;
  const int64_t t_end = min(t_begin + (int64_t)ASTRAI_MOE_CHUNK_TOKENS, n_tokens);
  const int slots = top_k + n_shared, columns = n_experts + n_shared;
  for (int e = threadIdx.x; e < n_experts; e += kScoreWaves * 64) hist[e] = 0;
  for (int i = threadIdx.x; i < (int)(t_end - t_begin) * n_shared; i += kScoreWaves * 64) {
    const int64_t at = (t_begin + i / n_shared) * slots + top_k + i % n_shared;
    topk_idx[at] = n_experts + i % n_shared;
    topk_w[at] = Elem<W>::from_f32(1.0f);
  }
  __syncthreads();
  uint64_t* const keys = s_key[wave];
  uint32_t* const kept = s_kept[wave];
  // (every wave takes the same number of turns: the barriers inside are the workgroup's)
  for (int64_t t0 = t_begin; t0 < t_end; t0 += kScoreWaves) {
    const int64_t t = t0 + wave;
    const bool on = t < t_end;
    double s[ITER];
    uint64_t key[ITER];
    int col[ITER];
    bool poison = false, off[ITER];
    double mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      col[i] = lane + 64 * i;
      s[i] = on && col[i] < n_experts ? (double)Elem<T>::to_f32(logits[t * n_experts + col[i]]) : -INFINITY;
      poison |= s[i] != s[i] || (opt.score == ASTRAI_MOE_SCORE_SOFTMAX && s[i] == INFINITY);
      off[i] = s[i] == -INFINITY;
      mx = s[i] > mx ? s[i] : mx;
    }
    poison = __any(poison);
    if (opt.score == ASTRAI_MOE_SCORE_SOFTMAX) {
#pragma unroll
      for (int off_ = 32; off_ > 0; off_ >>= 1) {
        const double o = __shfl_xor(mx, off_, 64);
        mx = o > mx ? o : mx;
      }
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        s[i] = off[i] ? 0.0 : exp(s[i] - mx);
        sum += s[i];
      }
#pragma unroll
      for (int off_ = 32; off_ > 0; off_ >>= 1) sum += __shfl_xor(sum, off_, 64);
#pragma unroll
      for (int i = 0; i < ITER; ++i) s[i] = off[i] ? 0.0 : s[i] / sum;
    } else {
#pragma unroll
      for (int i = 0; i < ITER; ++i) s[i] = 1.0 / (1.0 + exp(-s[i]));
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      if (col[i] >= n_experts)
        key[i] = kNone;
      else if (poison || off[i])
        key[i] = kOff;
      else
        key[i] = order_of(s[i] + (bias != nullptr ? (double)bias[col[i]] : 0.0));
    }
    if (opt.n_groups > 1) {
      const int per = n_experts / opt.n_groups;
#pragma unroll
      for (int i = 0; i < ITER; ++i) keys[col[i]] = key[i];
      if (lane < ASTRAI_MOE_MAX_EXPERTS / 32) kept[lane] = 0;
      __syncthreads();
      uint64_t value[ITER];
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        value[i] = kNone;
        if (col[i] >= opt.n_groups) continue;
        uint64_t a = kNone, b = kNone;
        for (int j = 0; j < per; ++j) {
          const uint64_t v = keys[col[i] * per + j];
          b = v > a ? a : v > b ? v : b;
          a = v > a ? v : a;
        }
        value[i] = opt.group_top == 2 ? order_of(value_of(a) + value_of(b)) : a;
      }
      for (int k = 0; k < opt.topk_groups; ++k) {
        int at;
        take_best(value, col, at);
        if (lane == 0) kept[at >> 5] |= 1u << (at & 31);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int g = min(col[i], n_experts - 1) / per;
        if (key[i] != kNone && (kept[g >> 5] >> (g & 31) & 1) == 0) key[i] = kOff;
      }
    }
    double my_s = 0.0, total = 0.0;
    int my_e = 0;
    for (int k = 0; k < top_k; ++k) {
      int at;
      const uint64_t best = take_best(key, col, at);
      double own = 0.0;  // its score, in the lane that holds it
#pragma unroll
      for (int i = 0; i < ITER; ++i)
        if (col[i] == at) own = s[i];
      const double score = __shfl(own, at & 63, 64);
      const double counted = best > kOff ? score : 0.0;
      total += counted;
      if (lane == k) my_s = counted, my_e = at;
    }
    if (on && lane < top_k) {
      double w = opt.renormalise ? (total > 0.0 ? my_s / total : 0.0) : my_s;
      w = poison ? (double)NAN : w * (double)opt.scale;
      topk_idx[t * slots + lane] = my_e;
      topk_w[t * slots + lane] = Elem<W>::from_f32((float)w);
      atomicAdd(&hist[my_e], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < columns; e += kScoreWaves * 64)
    chunk_hist[(int64_t)blockIdx.x * columns + e] = e < n_experts ? hist[e] : (int)(t_end - t_begin);
}

// dlogits of a token from dw, the gradient of its weights, at the chosen experts
// (a slot of weight 0 has no part: it was filled without a live expert, or its
// score is below every float):
//   ds_k = scale (dw_k - sum_j dw_j s_j / S) / S, or scale dw_k
//   sigmoid: dl = ds s (1 - s);  softmax: dl_e = s_e (ds_e - sum_j ds_j s_j).
template <typename T, typename W, int ITER>
__global__ __launch_bounds__(256) void route_scores_grad_kernel(
    const T* __restrict__ logits, const int32_t* __restrict__ topk_idx, const W* __restrict__ topk_w,
    const W* __restrict__ dw, const astrai_moe_routing opt, int64_t n_tokens, int n_experts, int top_k,
    T* __restrict__ dlogits) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (t >= n_tokens) return;
  const bool mine = lane < top_k;
  const int idx = mine ? topk_idx[t * top_k + lane] : -1;
  const float wk = mine ? Elem<W>::to_f32(topk_w[t * top_k + lane]) : 0.0f;
  const float g = mine && wk != 0.0f ? Elem<W>::to_f32(dw[t * top_k + lane]) : 0.0f;
  const T* const row = logits + t * n_experts;
  const bool softmax = opt.score == ASTRAI_MOE_SCORE_SOFTMAX;
  const float chosen = idx >= 0 && idx < n_experts && wk != 0.0f ? Elem<T>::to_f32(row[idx]) : -INFINITY;
  float p[ITER], s = 0.0f, slope = 0.0f;
  if (softmax) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = lane + i * 64;
      p[i] = c < n_experts ? Elem<T>::to_f32(row[c]) : -INFINITY;
      mx = fmaxf(mx, p[i]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if (mx == -INFINITY) mx = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      p[i] = expf(p[i] - mx);
      sum += p[i];
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < ITER; ++i) p[i] *= inv;
    s = expf(chosen - mx) * inv;
  } else {
    // s (1 - s) = s(l) s(-l), without the cancellation of 1 - s
    const float e = expf(-fabsf(chosen)), d = 1.0f / (1.0f + e);
    s = chosen >= 0.0f ? d : e * d;
    slope = e * d * d;
  }
  const float S = wave_sum(s);
  float ds = g * opt.scale;
  if (opt.renormalise) {
    const float inv = S == 0.0f ? 0.0f : 1.0f / S;
    const float dot = wave_sum(ds * s) * inv;
    ds = wk != 0.0f ? (ds - dot) * inv : 0.0f;
  }
  if (wk != wk) ds = wk;
  const float at_chosen = softmax ? ds : ds * slope;
  const float dot = softmax ? wave_sum(ds * s) : 0.0f;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = lane + i * 64;
    float d = 0.0f;
    for (int k = 0; k < top_k; ++k) {
      const int e = __shfl(idx, k, 64);
      const float v = __shfl(at_chosen, k, 64);
      if (e == c) d = v;
    }
    if (c < n_experts) dlogits[t * n_experts + c] = Elem<T>::from_f32(softmax ? p[i] * (d - dot) : d);
  }
}

// Tokens routed to each expert: the sum of the chunks' histograms.
__global__ __launch_bounds__(256) void expert_load_kernel(const int32_t* __restrict__ chunk_hist, int64_t n_chunks_,
                                                          int n_experts, int32_t* __restrict__ load) {
  __shared__ int part[256];
  const int e = blockIdx.x;
  int sum = 0;
  for (int64_t c = threadIdx.x; c < n_chunks_; c += 256) sum += chunk_hist[c * n_experts + e];
  part[threadIdx.x] = sum;
  for (int half = 128; half > 0; half >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < half) part[threadIdx.x] += part[threadIdx.x + half];
  }
  if (threadIdx.x == 0) load[e] = part[0];
}

// bias + rate * sign(mean load - load), the sign from sum(load) - E load in 64-bit integers.
__global__ __launch_bounds__(ASTRAI_MOE_MAX_EXPERTS) void balance_bias_kernel(const float* __restrict__ bias,
                                                                              const int32_t* __restrict__ load,
                                                                              int n_experts, float rate,
                                                                              float* __restrict__ out) {
  __shared__ int64_t part[ASTRAI_MOE_MAX_EXPERTS];
  const int e = threadIdx.x;
  part[e] = e < n_experts ? load[e] : 0;
  for (int half = ASTRAI_MOE_MAX_EXPERTS / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (e < half) part[e] += part[e + half];
  }
  __syncthreads();
  if (e >= n_experts) return;
  const int64_t d = part[0] - (int64_t)n_experts * load[e];
  out[e] = bias[e] + (d > 0 ? rate : d < 0 ? -rate : 0.0f);
}

template <typename T, typename W>
int launch_scores(const void* logits, const float* bias, const astrai_moe_routing& opt, int64_t n_tokens,
                  int n_experts, int top_k, int n_shared, int32_t* topk_idx, void* topk_w, int32_t* chunk_hist,
                  hipStream_t s) {
  auto kernel = n_experts <= 64    ? &route_scores_kernel<T, W, 1>
                : n_experts <= 128 ? &route_scores_kernel<T, W, 2>
                : n_experts <= 256 ? &route_scores_kernel<T, W, 4>
                : n_experts <= 512 ? &route_scores_kernel<T, W, 8>
                                   : &route_scores_kernel<T, W, ASTRAI_MOE_MAX_EXPERTS / 64>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)n_chunks(n_tokens)), dim3(kScoreWaves * 64), 0, s,
                     static_cast<const T*>(logits), bias, opt, n_tokens, n_experts, top_k, n_shared, topk_idx,
                     static_cast<W*>(topk_w), chunk_hist);
  return check_launch("route_scores_kernel");
}

template <typename T, typename W>
int launch_scores_grad(const void* logits, const int32_t* topk_idx, const void* topk_w, const void* dw,
                       const astrai_moe_routing& opt, int64_t n_tokens, int n_experts, int top_k, void* dlogits,
                       hipStream_t s) {
  auto kernel = n_experts <= 64    ? &route_scores_grad_kernel<T, W, 1>
                : n_experts <= 128 ? &route_scores_grad_kernel<T, W, 2>
                : n_experts <= 256 ? &route_scores_grad_kernel<T, W, 4>
                : n_experts <= 512 ? &route_scores_grad_kernel<T, W, 8>
                                   : &route_scores_grad_kernel<T, W, ASTRAI_MOE_MAX_EXPERTS / 64>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(n_tokens, 4)), dim3(256), 0, s, static_cast<const T*>(logits),
                     topk_idx, static_cast<const W*>(topk_w), static_cast<const W*>(dw), opt, n_tokens, n_experts,
                     top_k, static_cast<T*>(dlogits));
  return check_launch("route_scores_grad_kernel");
}

// (the four pairs of the logits' and the weights' types)
#define BY_TYPES(dtype, weight_dtype, fn, ...)                                                          \
  (dtype) == ASTRAI_MOE_BF16                                                                            \
      ? ((weight_dtype) == ASTRAI_MOE_BF16 ? fn<bf16_t, bf16_t>(__VA_ARGS__) : fn<bf16_t, float>(__VA_ARGS__)) \
      : ((weight_dtype) == ASTRAI_MOE_BF16 ? fn<float, bf16_t>(__VA_ARGS__) : fn<float, float>(__VA_ARGS__))

}  // namespace

int check_routing(const char* who, const astrai_moe_routing* opt, int dtype, int weight_dtype, int64_t n_tokens,
                  int n_experts, int top_k) {
  ASTRAI_REQUIRE(opt != nullptr, "%s: null routing", who);
  ASTRAI_REQUIRE(n_tokens >= 0 && n_tokens < (1ll << 31), "%s: n_tokens must be in [0, 2^31)", who);
  ASTRAI_REQUIRE(n_experts >= 1 && n_experts <= ASTRAI_MOE_MAX_EXPERTS, "%s: n_experts must be in [1, %d] (got %d)",
                 who, ASTRAI_MOE_MAX_EXPERTS, n_experts);
  ASTRAI_REQUIRE(top_k >= 1 && top_k <= n_experts && top_k <= ASTRAI_MOE_MAX_TOPK,
                 "%s: top_k must be in [1, min(n_experts, %d)] (got %d)", who, ASTRAI_MOE_MAX_TOPK, top_k);
  ASTRAI_REQUIRE(opt->score == ASTRAI_MOE_SCORE_SOFTMAX || opt->score == ASTRAI_MOE_SCORE_SIGMOID,
                 "%s: unknown score %d", who, opt->score);
  ASTRAI_REQUIRE(opt->n_groups >= 1 && n_experts % opt->n_groups == 0,
                 "%s: n_groups must divide n_experts (got %d of %d)", who, opt->n_groups, n_experts);
  ASTRAI_REQUIRE(opt->topk_groups >= 1 && opt->topk_groups <= opt->n_groups,
                 "%s: topk_groups must be in [1, n_groups] (got %d)", who, opt->topk_groups);
  ASTRAI_REQUIRE(top_k <= opt->topk_groups * (n_experts / opt->n_groups),
                 "%s: %d groups of %d experts hold fewer than top_k = %d", who, opt->topk_groups,
                 n_experts / opt->n_groups, top_k);
  ASTRAI_REQUIRE((opt->group_top == 1 || opt->group_top == 2) && opt->group_top <= n_experts / opt->n_groups,
                 "%s: group_top must be 1 or 2 and at most a group's experts (got %d)", who, opt->group_top);
  ASTRAI_REQUIRE(isfinite(opt->scale), "%s: scale must be finite", who);
  ASTRAI_REQUIRE((dtype == ASTRAI_MOE_BF16 || dtype == ASTRAI_MOE_F32) &&
                     (weight_dtype == ASTRAI_MOE_BF16 || weight_dtype == ASTRAI_MOE_F32),
                 "%s: unsupported dtype %d / %d", who, dtype, weight_dtype);
  return ASTRAI_MOE_OK;
}

int launch_route_scores(const void* logits, int dtype, const float* bias, const astrai_moe_routing& opt,
                        int64_t n_tokens, int n_experts, int top_k, int n_shared, int weight_dtype, int32_t* topk_idx,
                        void* topk_w, int32_t* chunk_hist, hipStream_t s) {
  return BY_TYPES(dtype, weight_dtype, launch_scores, logits, bias, opt, n_tokens, n_experts, top_k, n_shared,
                  topk_idx, topk_w, chunk_hist, s);
}

}  // namespace astrai_moe

using namespace astrai_moe;

extern "C" int astrai_moe_route_scores(const void* logits, int dtype, const float* bias,
                                       const astrai_moe_routing* routing, int64_t n_tokens, int n_experts, int top_k,
                                       int weight_dtype, int32_t* topk_idx, void* topk_w, int32_t* chunk_hist,
                                       void* stream) {
  clear_error();
  if (int rc = check_routing("route_scores", routing, dtype, weight_dtype, n_tokens, n_experts, top_k)) return rc;
  if (n_tokens == 0) return ASTRAI_MOE_OK;
  ASTRAI_REQUIRE(logits && topk_idx && topk_w && chunk_hist, "route_scores: null buffer");
  return launch_route_scores(logits, dtype, bias, *routing, n_tokens, n_experts, top_k, 0, weight_dtype, topk_idx,
                             topk_w, chunk_hist, static_cast<hipStream_t>(stream));
}

extern "C" int astrai_moe_route_scores_grad(const void* logits, int dtype, const int32_t* topk_idx,
                                            const void* topk_w, const void* dw, int weight_dtype,
                                            const astrai_moe_routing* routing, int64_t n_tokens, int n_experts,
                                            int top_k, void* dlogits, void* stream) {
  clear_error();
  if (int rc = check_routing("route_scores_grad", routing, dtype, weight_dtype, n_tokens, n_experts, top_k)) return rc;
  if (n_tokens == 0) return ASTRAI_MOE_OK;
  ASTRAI_REQUIRE(logits && topk_idx && topk_w && dw && dlogits, "route_scores_grad: null buffer");
  return BY_TYPES(dtype, weight_dtype, launch_scores_grad, logits, topk_idx, topk_w, dw, *routing, n_tokens, n_experts,
                  top_k, dlogits, static_cast<hipStream_t>(stream));
}

extern "C" int astrai_moe_expert_load(const int32_t* chunk_hist, int64_t n_chunks, int n_experts, int32_t* load,
                                      void* stream) {
  clear_error();
  ASTRAI_REQUIRE(n_chunks >= 0 && n_experts >= 1 && n_experts <= ASTRAI_MOE_MAX_EXPERTS,
                 "expert_load: n_chunks must be >= 0 and n_experts in [1, %d]", ASTRAI_MOE_MAX_EXPERTS);
  ASTRAI_REQUIRE(load && (chunk_hist || n_chunks == 0), "expert_load: null buffer");
  hipLaunchKernelGGL(expert_load_kernel, dim3((unsigned)n_experts), dim3(256), 0, static_cast<hipStream_t>(stream),
                     chunk_hist, n_chunks, n_experts, load);
  return check_launch("expert_load_kernel");
}

extern "C" int astrai_moe_balance_bias(const float* bias, const int32_t* load, int n_experts, float rate, float* out,
                                       void* stream) {
  clear_error();
  ASTRAI_REQUIRE(n_experts >= 1 && n_experts <= ASTRAI_MOE_MAX_EXPERTS, "balance_bias: n_experts must be in [1, %d]",
                 ASTRAI_MOE_MAX_EXPERTS);
  ASTRAI_REQUIRE(isfinite(rate), "balance_bias: rate must be finite");
  ASTRAI_REQUIRE(bias && load && out, "balance_bias: null buffer");
  hipLaunchKernelGGL(balance_bias_kernel, dim3(1), dim3(ASTRAI_MOE_MAX_EXPERTS), 0, static_cast<hipStream_t>(stream),
                     bias, load, n_experts, rate, out);
  return check_launch("balance_bias_kernel");
}
