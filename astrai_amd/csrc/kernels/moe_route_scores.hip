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
// The choice is that of exact scores as far as 64 bits tell them apart. Without a
// bias it goes by the logits, of which every score is a rising function. With one it
// is made in 32 bits, and again in 64 where two neighbours of the order, or the two
// groups at the border, are closer than the scores' errors in 32 (kTol), or a row
// holds what is no number or too few live experts (choose_slowly).
//
// A workgroup takes a chunk of 32 tokens, L lanes a token (32, so that a chunk is in
// flight at once; 64 from 513 experts on), each with C consecutive experts. A pick
// is a maximum over the lanes (DPP and a lane swap, no LDS) and the first lane that
// has it; that lane puts expert and score into LDS and looks for its next best.
// Bound by the instructions of the picks, not by the logits' bytes.
#include "moe_common.h"
#include "moe_gemm.h"
#include "route_list.h"

#include <math.h>

namespace astrai_moe {
namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}

// op over the L lanes of a token, in every one of them: lanes 1 and 2 apart (quad
// permutations), the halves of 8 and of 16 mirrored, then 16-lane rows and 32-lane
// halves swapped. Needs the whole wave.
template <int L, typename Op>
__device__ __forceinline__ float reduce(float v, Op op) {
  v = op(v, dpp<0xB1>(v));
  v = op(v, dpp<0x4E>(v));
  v = op(v, dpp<0x141>(v));
  v = op(v, dpp<0x140>(v));
  auto i = __builtin_bit_cast(unsigned, v);
  const auto a = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  v = op(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1]));
  if constexpr (L == 64) {
    i = __builtin_bit_cast(unsigned, v);
    const auto b = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    v = op(__builtin_bit_cast(float, (unsigned)b[0]), __builtin_bit_cast(float, (unsigned)b[1]));
  }
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
  return reduce<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  return reduce<L>(v, [](float a, float b) { return a + b; });
}

// The first lane of the token for which `yes` holds (lanes counted from the token's first; 32 or 64: none).
template <int L>
__device__ __forceinline__ int first_lane(bool yes) {
  const uint64_t m = __ballot(yes);
  if constexpr (L == 64) return m != 0 ? __builtin_ctzll(m) : 64;
  const uint32_t half = (__lane_id() & 32) != 0 ? (uint32_t)(m >> 32) : (uint32_t)m;
  return half != 0 ? __builtin_ctz(half) : 32;
}

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
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

// The best of the wave's (value, index) pairs, ties to the lower index.
__device__ __forceinline__ void wave_best(uint64_t& v, int& at) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off, 64);
    const int oi = __shfl_xor(at, off, 64);
    if (o > v || (o == v && oi < at)) v = o, at = oi;
  }
}

// LDS of a token: the picks, the experts' values (as floats, or as 64-bit keys) and
// the groups kept.
template <int E>
struct TokenLds {
  int pick[ASTRAI_MOE_MAX_TOPK];
  float score[ASTRAI_MOE_MAX_TOPK];
  uint64_t key[E];
  uint32_t kept[(E + 31) / 32];
};

// Score of one expert in 64 bits (softmax: with the row's maximum and sum).
__device__ __forceinline__ double score_of(double l, bool softmax, double mx, double sum) {
  if (l == -INFINITY) return 0.0;
  return softmax ? exp(l - mx) / sum : 1.0 / (1.0 + exp(-l));
}

// The choice of one token by a whole wave in 64 bits, for any logits and biases:
// fills m.pick and, in m.score, 1, 0 where no live expert was left, or NaN in a row
// that holds no number. A call that keeps everything in LDS, so that its registers do not cost
// the waves that never come here their places.
template <typename T, typename Lds>
__device__ __attribute__((noinline)) void choose_slowly(const T* row, const float* bias,
                                                        const astrai_moe_routing* opt, int n_experts, int top_k,
                                                        Lds* lds) {
  Lds& m = *lds;
  const int sub = threadIdx.x & 63;
  const bool softmax = opt->score == ASTRAI_MOE_SCORE_SOFTMAX;
  double mx = -INFINITY, sum = 0.0;
  bool poison = false;
#pragma unroll 1
  for (int c = sub; c < n_experts; c += 64) {
    const double l = Elem<T>::to_f32(row[c]);
    poison |= l != l || (softmax && l == INFINITY);
    mx = l > mx ? l : mx;
  }
  poison = __any(poison);
  if (softmax) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const double o = __shfl_xor(mx, off, 64);
      mx = o > mx ? o : mx;
    }
#pragma unroll 1
    for (int c = sub; c < n_experts; c += 64) {
      const double l = Elem<T>::to_f32(row[c]);
      if (l != -INFINITY) sum += exp(l - mx);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  }
#pragma unroll 1
  for (int c = sub; c < n_experts; c += 64) {
    const double l = Elem<T>::to_f32(row[c]);
    m.key[c] = poison || l == -INFINITY
                   ? kOff
                   : order_of(score_of(l, softmax, mx, sum) + (bias != nullptr ? (double)bias[c] : 0.0));
    if (c < (n_experts + 31) / 32) m.kept[c] = 0;
  }
  wave_sync();
  const int groups = opt->n_groups;
  if (groups > 1) {
    const int per = n_experts / groups;
    auto value_of_group = [&](int g) {
      uint64_t a = kNone, b = kNone;
#pragma unroll 1
      for (int j = 0; j < per; ++j) {
        const uint64_t v = m.key[g * per + j];
        b = v > a ? a : v > b ? v : b;
        a = v > a ? v : a;
      }
      return opt->group_top == 2 ? order_of(value_of(a) + value_of(b)) : a;
    };
    const uint64_t first = sub < groups ? value_of_group(sub) : kNone;
#pragma unroll 1
    for (int k = 0; k < opt->topk_groups; ++k) {
      uint64_t best = kNone;
      int at = INT32_MAX;
#pragma unroll 1
      for (int g = sub; g < groups; g += 64)
        if ((m.kept[g >> 5] >> (g & 31) & 1) == 0) {
          const uint64_t v = g == sub ? first : value_of_group(g);
          if (v > best) best = v, at = g;
        }
      wave_best(best, at);
      wave_sync();
      if (sub == 0) m.kept[at >> 5] |= 1u << (at & 31);
      wave_sync();
    }
#pragma unroll 1
    for (int c = sub; c < n_experts; c += 64) {
      const int g = c / per;
      if ((m.kept[g >> 5] >> (g & 31) & 1) == 0) m.key[c] = kOff;
    }
    wave_sync();
  }
#pragma unroll 1
  for (int k = 0; k < top_k; ++k) {
    uint64_t best = kNone;
    int at = INT32_MAX;
#pragma unroll 1
    for (int c = sub; c < n_experts; c += 64)
      if (m.key[c] > best) best = m.key[c], at = c;
    wave_best(best, at);
    if (sub == (at & 63)) {
      m.key[at] = kNone;
      m.pick[k] = at;
      m.score[k] = poison ? NAN : best > kOff ? 1.0f : 0.0f;
    }
  }
  wave_sync();
}

// Bounds of the error of a difference of two scores (at most 1, each off by 4
// roundings; softmax: by the sum's too, up to 21) plus biases, times two.
constexpr float kTolSigmoid = 0x1p-20f, kTolSoftmax = 0x1p-18f, kTolBias = 0x1p-21f;

template <typename T, typename W, int L, int C, bool kGroups, bool kList>
__global__ __launch_bounds__(kRouteThreads, L * C <= 256 ? 8 : 4) void route_scores_kernel(
    const T* __restrict__ logits, const float* __restrict__ bias, const astrai_moe_routing opt, int64_t n_tokens,
    int n_experts, int top_k, int n_shared, int32_t* __restrict__ topk_idx, W* __restrict__ topk_w,
    int32_t* __restrict__ chunk_hist, const RouteList list) {
  constexpr int TOKENS = kRouteThreads / L;  // in flight
  __shared__ int hist[ASTRAI_MOE_MAX_EXPERTS];  // kList: the experts' first rows
  __shared__ TokenLds<L * C> lds[TOKENS];
  constexpr int kEntries = kList ? ASTRAI_MOE_CHUNK_TOKENS * ASTRAI_MOE_MAX_TOPK : 1;
  __shared__ uint32_t mask[kList ? ASTRAI_MOE_MAX_EXPERTS : 1];
  __shared__ int s_e[kEntries];
  __shared__ W s_w[kEntries];
  const int sub = threadIdx.x % L, in_flight = threadIdx.x / L;
  const int64_t t_begin = (int64_t)blockIdx.x * ASTRAI_MOE_CHUNK_TOKENS;
  const int64_t t_end = min(t_begin + (int64_t)ASTRAI_MOE_CHUNK_TOKENS, n_tokens);
  const int slots = top_k + n_shared, columns = n_experts + n_shared;
  if constexpr (kList) {
    const uint32_t all = n_tokens < 32 ? (1u << (int)n_tokens) - 1u : ~0u;
    for (int e = threadIdx.x; e < columns; e += kRouteThreads) mask[e] = e < n_experts ? 0u : all;
  } else {
    for (int e = threadIdx.x; e < n_experts; e += kRouteThreads) hist[e] = 0;
  }
  for (int i = threadIdx.x; i < (int)(t_end - t_begin) * n_shared; i += kRouteThreads) {
    const int64_t at = (t_begin + i / n_shared) * slots + top_k + i % n_shared;
    (kList ? s_e : topk_idx)[at] = n_experts + i % n_shared;
    (kList ? s_w : topk_w)[at] = Elem<W>::from_f32(1.0f);
  }
  __syncthreads();
  auto& m = lds[in_flight];
  const bool softmax = opt.score == ASTRAI_MOE_SCORE_SOFTMAX;
  float b[C];
#pragma unroll
  for (int i = 0; i < C; ++i) b[i] = bias != nullptr && sub * C + i < n_experts ? bias[sub * C + i] : 0.0f;
  for (int64_t t0 = t_begin; t0 < t_end; t0 += TOKENS) {
    const int64_t t = t0 + in_flight;
    const bool on = t < t_end;
    float l[C], s[C], key[C];
    bool slow = false;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = sub * C + i;
      l[i] = c < n_experts ? (on ? Elem<T>::to_f32(logits[t * n_experts + c]) : 0.0f) : -INFINITY;
      slow |= !(l[i] < INFINITY);
    }
    float mx = l[0], inv = 1.0f;
    if (softmax) {
#pragma unroll
      for (int i = 1; i < C; ++i) mx = fmaxf(mx, l[i]);
      mx = lanes_max<L>(mx);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        s[i] = expf(l[i] - mx);
        sum += s[i];
      }
      inv = 1.0f / lanes_sum<L>(sum);
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] = 1.0f / (1.0f + expf(-l[i]));
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      key[i] = bias == nullptr || l[i] == -INFINITY ? l[i] : s[i] + b[i];
      slow |= !(key[i] < INFINITY);  // (NaN or +inf)
    }
    const float tol = softmax ? kTolSoftmax : kTolSigmoid;
    if constexpr (kGroups) {
      // P lanes share a group's experts; more groups than lanes go the other way
      const int per = n_experts / opt.n_groups;
      const bool by_score = bias == nullptr && opt.group_top == 2;
      slow |= opt.n_groups > L;
      float* const value_of_expert = reinterpret_cast<float*>(m.key);
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (sub * C + i < n_experts) value_of_expert[sub * C + i] = by_score && l[i] != -INFINITY ? s[i] : key[i];
      wave_sync();
      int p = 1;
      while (2 * p * opt.n_groups <= L) p *= 2;
      const int g = sub / p;
      float a1 = -INFINITY, a2 = -INFINITY;
      if (g < opt.n_groups)
        for (int j = sub % p; j < per; j += p) {
          const float v = value_of_expert[g * per + j];
          a2 = fmaxf(a2, fminf(a1, v));
          a1 = fmaxf(a1, v);
        }
      for (int off = 1; off < p; off *= 2) {
        const float o1 = __shfl_xor(a1, off, L), o2 = __shfl_xor(a2, off, L);
        a2 = fmaxf(fminf(a1, o1), fmaxf(a2, o2));
        a1 = fmaxf(a1, o1);
      }
      float value = opt.group_top == 2 ? a1 + a2 : a1, last = 0.0f;
      uint64_t kept = 0;
      for (int k = 0; k < opt.topk_groups; ++k) {
        last = lanes_max<L>(value);
        const int at = first_lane<L>(value == last) / p;
        kept |= 1ull << at;
        if (g == at) value = -INFINITY;
      }
      const float next = lanes_max<L>(value);
      slow |= !(last > -INFINITY);
      // (one live expert of two, or the first of the groups left out as good as the last taken)
      if (bias != nullptr || by_score) slow |= last - next <= 2.0f * (tol + kTolBias * (fabsf(last) + fabsf(next)));
      int gi = sub * C / per, left = per - (sub * C - gi * per);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if ((kept >> gi & 1) == 0) key[i] = -INFINITY;
        if (--left == 0) left = per, ++gi;
      }
    }
    // the picks: every lane's best, the lanes' best
    float best = -INFINITY, best_s = 0.0f;
    int best_i = 0;
    auto look = [&]() {
      best = key[0], best_s = s[0], best_i = 0;
#pragma unroll
      for (int i = 1; i < C; ++i)
        if (key[i] > best) best = key[i], best_s = s[i], best_i = i;
    };
    look();
    float before = 0.0f;
    const int rounds = bias != nullptr && top_k < n_experts ? top_k + 1 : top_k;  // (the first one left out too)
    for (int k = 0; k < rounds; ++k) {
      const float top = lanes_max<L>(best);
      if (bias != nullptr && k > 0)
        slow |= before - top <= tol + kTolBias * (fabsf(before) + fabsf(top)) && top > -INFINITY;
      if (k == top_k) break;
      slow |= !(top > -INFINITY);
      before = top;
      if (sub == first_lane<L>(best == top)) {
        m.pick[k] = sub * C + best_i;
        m.score[k] = best_s;
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (i == best_i) key[i] = -INFINITY;
        look();
      }
    }
    const uint64_t again = __ballot(slow && on);
    wave_sync();
    if (again != 0) {
      const int first = (threadIdx.x & ~63) / L;  // the wave's first token in flight
#pragma unroll 1
      for (int h = 0; h < 64 / L; ++h)
        if (L == 64 || (uint32_t)(again >> (32 * h)) != 0)
          choose_slowly<T>(logits + (t0 + first + h) * n_experts, bias, &opt, n_experts,
                                                      top_k, &lds[first + h]);
    }
    float v = sub < top_k && on ? m.score[sub] : 0.0f;
    if ((L == 64 ? again != 0 : (uint32_t)(again >> (threadIdx.x & 32)) != 0) && v == 1.0f) {
      // a live pick's score in 32 bits, as the quick choice takes it
      const float at = Elem<T>::to_f32(logits[t * n_experts + m.pick[sub]]);
      v = softmax ? expf(at - mx) * inv : 1.0f / (1.0f + expf(-at));
    }
    const float total = lanes_sum<L>(v);
    if (on && sub < top_k) {
      const int e = m.pick[sub];
      float w = opt.renormalise ? (total == 0.0f ? 0.0f : v / total) : v;
      w *= opt.scale;
      (kList ? s_e : topk_idx)[t * slots + sub] = e;
      (kList ? s_w : topk_w)[t * slots + sub] = Elem<W>::from_f32(w);
      if constexpr (kList)
        atomicOr(&mask[e], 1u << (int)t);
      else
        atomicAdd(&hist[e], 1);
    }
  }
  __syncthreads();
  if constexpr (kList) {
    write_chunk_list<W>(mask, hist, s_e, s_w, (int)n_tokens, columns, slots, list);
    return;
  }
  for (int e = threadIdx.x; e < columns; e += kRouteThreads)
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

template <typename T, typename W, int L, int C>
void launch_scores_cfg(const void* logits, const float* bias, const astrai_moe_routing& opt, int64_t n_tokens,
                       int n_experts, int top_k, int n_shared, int32_t* topk_idx, void* topk_w, int32_t* chunk_hist,
                       const RouteList* list, hipStream_t s) {
  const dim3 grid(list != nullptr ? 1u : (unsigned)n_chunks(n_tokens));
  auto kernel = opt.n_groups > 1
                    ? (list != nullptr ? &route_scores_kernel<T, W, L, C, true, true> : &route_scores_kernel<T, W, L, C, true, false>)
                    : (list != nullptr ? &route_scores_kernel<T, W, L, C, false, true> : &route_scores_kernel<T, W, L, C, false, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(kRouteThreads), 0, s, static_cast<const T*>(logits), bias, opt, n_tokens,
                     n_experts, top_k, n_shared, topk_idx, static_cast<W*>(topk_w), chunk_hist,
                     list != nullptr ? *list : RouteList{});
}

template <typename T, typename W>
int launch_scores(const void* logits, const float* bias, const astrai_moe_routing& opt, int64_t n_tokens,
                  int n_experts, int top_k, int n_shared, int32_t* topk_idx, void* topk_w, int32_t* chunk_hist,
                  const RouteList* list, hipStream_t s) {
#define ROUTE_CASE(L, C)                                                                                       \
  launch_scores_cfg<T, W, L, C>(logits, bias, opt, n_tokens, n_experts, top_k, n_shared, topk_idx, topk_w,      \
                                chunk_hist, list, s)
  if (n_experts <= 32)
    ROUTE_CASE(32, 1);
  else if (n_experts <= 64)
    ROUTE_CASE(32, 2);
  else if (n_experts <= 128)
    ROUTE_CASE(32, 4);
  else if (n_experts <= 256)
    ROUTE_CASE(32, 8);
  else if (n_experts <= 512)
    ROUTE_CASE(32, 16);
  else
    ROUTE_CASE(64, ASTRAI_MOE_MAX_EXPERTS / 64);
#undef ROUTE_CASE
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
                  topk_idx, topk_w, chunk_hist, nullptr, s);
}

int launch_route_scores_list(const void* logits, int dtype, const float* bias, const astrai_moe_routing& opt,
                             int64_t n_tokens, int n_experts, int top_k, int n_shared, int weight_dtype,
                             const RouteList& list, hipStream_t s) {
  if (n_tokens > ASTRAI_MOE_CHUNK_TOKENS || n_experts + n_shared > ASTRAI_MOE_MAX_EXPERTS ||
      top_k + n_shared > ASTRAI_MOE_MAX_TOPK || list.block_m < ASTRAI_MOE_CHUNK_TOKENS)
    return fail(ASTRAI_MOE_EINVAL, "route: more than one chunk of tokens, too many experts or slots, or short tiles");
  return BY_TYPES(dtype, weight_dtype, launch_scores, logits, bias, opt, n_tokens, n_experts, top_k, n_shared, nullptr,
                  nullptr, nullptr, &list, s);
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
