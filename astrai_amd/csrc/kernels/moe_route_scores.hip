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
// bias it goes by the logits, of which every score is a rising function. With one, and
// for groups valued by two scores, it is made in 32 bits, and again in 64, from the few
// experts that may be chosen, where two neighbours of the order, or the two groups at
// the border, are closer than the scores' errors in 32 (kTol...): one token in a
// thousand. Equal logits with equal biases are in order as they are. Rows that hold what
// is no number go through choose_slowly.
//
// A workgroup takes a chunk of 32 tokens, L lanes a token (16 up to 256 experts), each
// with C consecutive experts, sorted by a network in its registers: the experts' values
// as integers whose low 4 bits are their places in the lane, so that a comparator is a
// maximum and a minimum. A pick is a maximum over the lanes' first ones (DPP, no LDS)
// and the first lane that has it; that lane notes the expert and moves its list up.
// Groups of whole lanes are valued and picked in registers alike.
// Bound by the instructions (1380 of the vector units a wave of four tokens), not by the
// logits' bytes: 16384 tokens of 256 experts in 8 groups, sigmoid scores with a bias, 17
// to 20 us (the logits' 17 MB: 3.3), 12 of them without the near ties, which a wave
// settles while the others are done; softmax without groups and bias 10.
#include "moe_common.h"
#include "moe_gemm.h"
#include "route_list.h"
#include "wave_lanes.h"

#include <math.h>

namespace astrai_moe {
namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// The token's lanes for which `yes` holds, from bit 0 on.
template <int L>
__device__ __forceinline__ uint64_t lanes_of(bool yes) {
  const uint64_t m = __ballot(yes);
  return L == 64 ? m : m >> (__lane_id() & (64 - L)) & ((1ull << (L & 63)) - 1);
}
// The first of them, or L.
template <int L>
__device__ __forceinline__ int first_lane(bool yes) {
  const uint64_t m = lanes_of<L>(yes);
  if constexpr (L == 64) return m != 0 ? __builtin_ctzll(m) : 64;
  return __builtin_ctz((uint32_t)m | (L < 32 ? 1u << (L & 31) : 0u)) + (L == 32 && (uint32_t)m == 0 ? 32 : 0);
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

// exp in 64 bits, a call: where it is needed few waves come, and inlined its registers
// and its code would cost the others theirs.
__device__ __attribute__((noinline)) double exp64(double x) { return exp(x); }

// Score of one expert in 64 bits (softmax: with the row's maximum and sum).
__device__ __forceinline__ double score_of(double l, bool softmax, double mx, double sum) {
  if (l == -INFINITY) return 0.0;
  const double t = exp64(softmax ? l - mx : -l);
  return (softmax ? t : 1.0) / (softmax ? sum : 1.0 + t);
}

// The choice of one token by a whole wave in 64 bits, for any logits and biases:
// fills m.pick and, in m.score, 0, -inf where no live expert was left, or NaN in a row
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
      m.score[k] = poison ? NAN : best > kOff ? 0.0f : -INFINITY;
    }
  }
  wave_sync();
}

// Bounds of the error of a difference of two scores: a sigmoid s from exp_near is off
// by s (1 - s) (|l| 2^-24 + 2^-23) + s (2^-23 + 2^-24) < 2^-22, a softmax by up to 40
// roundings of its sum and of 1 / sum more, relative to the row's largest score (the
// largest 1 / sum). The addition of a bias: half a step (kTolAdd: doubled). A value that
// went through a key is off by 16 units in the last place, 2^-19 of it, and that (kTolKey).
constexpr float kTolSigmoid = 0x1p-21f, kTolSoftmax = 0x1p-18f, kTolAdd = 0x1p-23f, kTolKey = 0x1.1p-19f;

// Whether two values that went through keys, a and b <= a, may be the other way round.
__device__ __forceinline__ bool near(float a, float b, float tol) {
  return b > -INFINITY && a - b <= tol + kTolKey * (fabsf(a) + fabsf(b));
}

// How the groups lie: `per` experts each; where a group is 2^shift whole lanes, shift,
// otherwise -1.
struct GroupShape {
  int per, shift;
};

// The two largest of two pairs a1 >= a2, b1 >= b2.
template <typename F>
__device__ __forceinline__ void merge_two(F& a1, F& a2, F b1, F b2) {
  const F low = b1 < a1 ? b1 : a1, high2 = b2 > a2 ? b2 : a2;
  a2 = low > high2 ? low : high2;
  a1 = b1 > a1 ? b1 : a1;
}

// The best topk_groups of the groups' values (p lanes a group; -inf: no live expert) as
// bits; `last` is the least of them and `next` the best of the others.
template <int L, typename F>
__device__ __forceinline__ uint64_t best_groups(F mine, int g, int p, int topk_groups, F& last, F& next) {
  constexpr F kDead = (F)-INFINITY;
  uint64_t kept = 0;
  for (int k = 0; k < topk_groups; ++k) {
    last = lanes_max<L>(mine);
    // (groups without live experts: the lowest not kept yet)
    const int at = last > kDead ? first_lane<L>(mine == last) / p : __builtin_ctzll(~kept);
    kept |= 1ull << (at & 63);
    if (g == at) mine = kDead;
  }
  next = lanes_max<L>(mine);
  return kept;
}

// The groups that stay (as bits; at most 64) from the experts' values (-inf: off),
// however they lie. Where the border of a token of the wave lies between two that are
// near, again from exact(expert, sum64()), of each group's experts that may be its best.
template <int L, int C, typename Lds, typename Sum, typename Exact>
__device__ __forceinline__ uint64_t groups_kept(const float (&value)[C], float tol, int sub,
                                                const astrai_moe_routing& opt, int per, int n_experts, bool on, Lds& m,
                                                Sum sum64, Exact exact) {
  float* const values = reinterpret_cast<float*>(m.key);
  const auto store = [&] {
    wave_sync();
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (sub * C + i < n_experts) values[sub * C + i] = value[i];
    wave_sync();
  };
  store();
  int p = 1;  // lanes of a group
  while (2 * p * opt.n_groups <= L) p *= 2;
  const int g = sub / p, begin = g < opt.n_groups ? sub & (p - 1) : per;
  const bool two = opt.group_top == 2;
  float a1 = -INFINITY, a2 = -INFINITY;
  for (int j = begin; j < per; j += p) merge_two(a1, a2, values[g * per + j], -INFINITY);
  for (int off = 1; off < p; off *= 2) merge_two(a1, a2, __shfl_xor(a1, off, L), __shfl_xor(a2, off, L));
  const float mine = two ? a1 + a2 : a1;
  float last, next;
  const uint64_t kept = best_groups<L>(mine, g, p, opt.topk_groups, last, next);
  if (tol == 0.0f) return kept;
  const float size = lanes_max<L>(mine > -INFINITY ? fabsf(a1) + (two ? fabsf(a2) : 0.0f) : 0.0f);
  const bool close = on && next > -INFINITY && last - next <= 2.0f * tol + 4.0f * kTolAdd * size;
  if (__ballot(close) == 0) return kept;
  const double sum = sum64();
  store();
  const float least = two ? a2 : a1;
  double d1 = -INFINITY, d2 = -INFINITY;
  for (int j = close ? begin : per;;) {
    for (; j < per; j += p) {
      const float v = values[g * per + j];
      if (v > -INFINITY && least - v <= tol + kTolAdd * (fabsf(v) + fabsf(least))) break;
    }
    if (__ballot(j < per) == 0) break;
    if (j < per) {
      merge_two(d1, d2, exact(g * per + j, sum), (double)-INFINITY);
      j += p;
    }
  }
  for (int off = 1; off < p; off *= 2) merge_two(d1, d2, __shfl_xor(d1, off, L), __shfl_xor(d2, off, L));
  double last64, next64;
  const uint64_t exactly = best_groups<L>(two ? d1 + d2 : d1, g, p, opt.topk_groups, last64, next64);
  return close ? exactly : kept;
}

// Which of the lane's C experts are in a group that stays, as bits.
template <int C>
__device__ __forceinline__ uint32_t in_kept(uint64_t kept, int sub, int per) {
  int g = sub * C / per, left = per - (sub * C - g * per);
  uint32_t in = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    in |= (uint32_t)(kept >> (g & 63) & 1) << i;
    if (--left == 0) left = per, ++g;
  }
  return in;
}

// A float as an unsigned integer that orders alike; 0, below every float's, stands for
// what is taken or does not exist.
__device__ __forceinline__ uint32_t bits_of(float v) {
  const int b = __float_as_int(v + 0.0f);  // (-0 as 0)
  return (uint32_t)(b ^ (b >> 31 | INT32_MIN));
}
__device__ __forceinline__ float float_of(uint32_t o) {
  return __int_as_float((int)(o ^ (~(uint32_t)((int)o >> 31) | 0x80000000u)));
}
// A key orders like a value without its 4 lowest bits, and among equals by the
// expert's place i in its lane, lower first: these bits hold 15 - i. Exact for logits that
// were bf16.
constexpr uint32_t kValueBits = ~15u;
constexpr uint32_t kOffKey = 0x007ffff0u;  // -inf's
__device__ __forceinline__ uint32_t key_of(float v, int i) { return (bits_of(v) & kValueBits) | (uint32_t)(15 - i); }
__device__ __forceinline__ float value_of(uint32_t key) {
  return (key & kValueBits) <= kOffKey ? -INFINITY : float_of(key & kValueBits);
}

// Sorts a lane's C keys downwards: odd-even merges.
template <int C>
__device__ __forceinline__ void sort_down(uint32_t (&v)[C]) {
#pragma unroll
  for (int p = 1; p < C; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < C; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < C && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t a = v[i + j], b = v[i + j + k];
            v[i + j] = max(a, b);
            v[i + j + k] = min(a, b);
          }
}

// Whether the lane's group stays, where groups are 2^shift whole lanes, from what the
// experts go by (-inf: off): logits, whose `score` groups of two go by, or scores with
// their biases (scored). Where the border of a token lies between two groups that are
// near, from exact(expert, sum64()) of the experts that may be a group's best.
template <int L, int C, typename Lds, typename Score, typename Sum, typename Exact>
__device__ __forceinline__ bool group_stays(const float (&value)[C], float tol, bool scored, int sub,
                                            const astrai_moe_routing& opt, int shift, bool on, Lds& m, Score score,
                                            Sum sum64, Exact exact) {
  const bool two = opt.group_top == 2;
  float a1 = value[0], a2 = -INFINITY;
#pragma unroll
  for (int i = 1; i < C; ++i) {
    a2 = __builtin_amdgcn_fmed3f(a1, a2, value[i]);
    a1 = fmaxf(a1, value[i]);
  }
  if (shift > 0) merge_two(a1, a2, other<0>(a1), other<0>(a2));
  if (shift > 1) merge_two(a1, a2, other<1>(a1), other<1>(a2));
  if (shift > 2) merge_two(a1, a2, other<2>(a1), other<2>(a2));
  if (shift > 3) merge_two(a1, a2, other<3>(a1), other<3>(a2));
  if constexpr (L >= 64)
    if (shift > 4) merge_two(a1, a2, other<4>(a1), other<4>(a2));
  const float least = two ? a2 : a1;
  float size = fabsf(a1);  // (what the sums' roundings are relative to)
  if (two) {
    const float s1 = scored || a1 == -INFINITY ? a1 : score(a1), s2 = scored || a2 == -INFINITY ? a2 : score(a2);
    size = fabsf(s1) + fabsf(s2);
    a1 = s1 + s2;
  }
  uint32_t mine = bits_of(a1), last = 0;
  if (a1 == -INFINITY) size = 0.0f;
  bool stays = false;
  for (int k = 0; k < opt.topk_groups; ++k) {
    last = lanes_max<L>(mine);
    const int at = first_lane<L>(mine == last);
    if (sub >> shift == at >> shift) mine = 0, stays = true;
  }
  if (tol == 0.0f) return stays;
  const float next = float_of(max(lanes_max<L>(mine), bits_of(-INFINITY)));
  const float sizes = lanes_max<L>(size);
  const bool close = on && next > -INFINITY && float_of(last) - next <= 2.0f * tol + 4.0f * kTolAdd * sizes;
  if (__ballot(close) == 0) return stays;
  const double sum = sum64();
  uint32_t open = 0;  // (logits are exact)
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (value[i] > -INFINITY && least - value[i] <= (scored ? tol + kTolAdd * (fabsf(value[i]) + fabsf(least)) : 0.0f))
      open |= 1u << i;
  if (!close) open = 0;
  double d1 = -INFINITY, d2 = -INFINITY;
#pragma unroll 1
  for (; __ballot(open != 0) != 0; open &= open - 1)
    if (open != 0) merge_two(d1, d2, exact(sub * C + __builtin_ctz(open), sum), (double)-INFINITY);
#pragma unroll 1
  for (int off = 1; off < 1 << shift; off *= 2) merge_two(d1, d2, __shfl_xor(d1, off, L), __shfl_xor(d2, off, L));
  const uint64_t v = order_of(two ? d1 + d2 : d1);
  const int g = sub >> shift;
  wave_sync();
  if (g << shift == sub) m.key[g] = v;
  wave_sync();
  int better = 0;
#pragma unroll 1
  for (int i = 0; i < opt.n_groups; ++i) better += m.key[i] > v || (m.key[i] == v && i < g);
  wave_sync();
  return close ? better < opt.topk_groups : stays;
}

// The top_k experts of the largest keys (0: none) into m.pick, their values into
// m.score; dead ones (-inf) come last, by their index. Returns the largest value left.
template <int L, int C, typename Lds>
__device__ __forceinline__ float pick(uint32_t (&v)[C], int sub, int top_k, Lds& m) {
  for (int k = 0; k < top_k; ++k) {
    const uint32_t mine = v[0] & kValueBits;
    const uint32_t top = lanes_max<L>(mine);
    if (sub == first_lane<L>(mine == top)) {
      m.pick[k] = sub * C + 15 - (int)(v[0] & 15);
      m.score[k] = value_of(top);
#pragma unroll
      for (int i = 0; i + 1 < C; ++i) v[i] = v[i + 1];
      v[C - 1] = 0;
    }
  }
  return value_of(lanes_max<L>(v[0]));
}

// The same from the exact values of the experts that may be chosen (`open`, bits of the
// lane's; none of tokens whose choice stands): each takes the place that the number of
// better ones gives it. False for a token of more than the list holds.
template <int L, int C, typename Lds, typename Exact>
__device__ __forceinline__ bool pick_exact(uint32_t open, int sub, int top_k, Lds& m, Exact exact) {
  constexpr int kMost = ASTRAI_MOE_MAX_TOPK, MINE = kMost > L ? kMost / L : 1;
  int& count = *reinterpret_cast<int*>(m.kept);
  if (sub == 0) count = 0;
  wave_sync();
#pragma unroll 1
  for (; __ballot(open != 0) != 0; open &= open - 1)
    if (open != 0) {
      const int e = sub * C + __builtin_ctz(open), at = atomicAdd(&count, 1);
      const uint64_t v = order_of(exact(e));
      if (at < kMost) m.key[at] = v, m.pick[at] = e;
    }
  wave_sync();
  const int n = count;
  uint64_t v[MINE];
  int e[MINE], better[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int c = min(sub + i * L, kMost - 1);
    v[i] = m.key[c], e[i] = m.pick[c], better[i] = 0;
  }
#pragma unroll 1
  for (int j = 0; j < min(n, kMost); ++j) {
    const uint64_t vj = m.key[j];
    const int ej = m.pick[j];
#pragma unroll
    for (int i = 0; i < MINE; ++i) better[i] += vj > v[i] || (vj == v[i] && ej < e[i]);
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < MINE; ++i)
    if (sub + i * L < n && n <= kMost && better[i] < top_k) {
      m.pick[better[i]] = e[i];
      m.score[better[i]] = (float)value_of(v[i]);
    }
  return n <= kMost;
}

// The lane's C of a row of n values from column c0 on, `none` behind its end. vec: rows
// are whole 16-byte units on 16-byte boundaries.
template <typename T, int C>
__device__ __forceinline__ void load_run(const T* row, int c0, int n, bool vec, float none, float (&out)[C]) {
  constexpr int V = C * sizeof(T) < 16 ? C : 16 / (int)sizeof(T);
  struct alignas(V * sizeof(T)) Unit {
    T v[V];
  };
  if (vec) {
#pragma unroll
    for (int i = 0; i < C; i += V) {
      Unit u{};
      const bool in = c0 + i < n;
      if (in) u = *reinterpret_cast<const Unit*>(row + c0 + i);
#pragma unroll
      for (int j = 0; j < V; ++j) out[i + j] = in ? Elem<T>::to_f32(u.v[j]) : none;
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) out[i] = c0 + i < n ? Elem<T>::to_f32(row[c0 + i]) : none;
  }
}

constexpr float kLog2e = 1.4426950408889634f;
// exp on the hardware's exponential: off by |x| 2^-24 + 2^-23 of its value.
__device__ __forceinline__ float exp_near(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// Score of an expert in 32 bits over e^base (a softmax's without 1 / sum; a sigmoid's base
// is at most 0): renormalised weights take the largest chosen logit, so that scores below
// every float still have their share. What 64 bits hold as 0 is 0.
constexpr float kLeastLog = -708.0f;
__device__ __forceinline__ float score32(float l, bool softmax, float base, float mx) {
  if (softmax) return l - mx < kLeastLog ? 0.0f : expf(l - base);
  const float d = 1.0f / (1.0f + expf(-fabsf(l)));
  return l >= 0.0f ? d : l < kLeastLog ? 0.0f : expf(l - base) * d;
}

template <int L, bool kList>
constexpr int score_threads() {  // a chunk at once where 32 L threads allow it
  return kList || L > 32 ? kRouteThreads : ASTRAI_MOE_CHUNK_TOKENS * L;
}

template <typename T, typename W, int L, int C, bool kGroups, bool kList>
__global__ __launch_bounds__((score_threads<L, kList>()), 4) void route_scores_kernel(
    const T* __restrict__ logits, const float* __restrict__ bias, const astrai_moe_routing opt, int64_t n_tokens,
    int n_experts, int top_k, int n_shared, int32_t* __restrict__ topk_idx, W* __restrict__ topk_w,
    int32_t* __restrict__ chunk_hist, const RouteList list, const GroupShape shape, bool vec, bool vec_bias) {
  constexpr int THREADS = score_threads<L, kList>();
  constexpr int TOKENS = THREADS / L < ASTRAI_MOE_CHUNK_TOKENS ? THREADS / L : ASTRAI_MOE_CHUNK_TOKENS;  // in flight
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
    for (int e = threadIdx.x; e < columns; e += THREADS) mask[e] = e < n_experts ? 0u : all;
  } else {
    for (int e = threadIdx.x; e < n_experts; e += THREADS) hist[e] = 0;
  }
  for (int i = threadIdx.x; i < (int)(t_end - t_begin) * n_shared; i += THREADS) {
    const int64_t at = (t_begin + i / n_shared) * slots + top_k + i % n_shared;
    (kList ? s_e : topk_idx)[at] = n_experts + i % n_shared;
    (kList ? s_w : topk_w)[at] = Elem<W>::from_f32(1.0f);
  }
  __syncthreads();
  const bool softmax = opt.score == ASTRAI_MOE_SCORE_SOFTMAX;
  const bool by_score = bias != nullptr || (kGroups && opt.group_top == 2);  // (otherwise the logits decide)
  for (int64_t t0 = t_begin; t0 < t_end; t0 += TOKENS) {
    const int64_t t = t0 + in_flight;
    const bool on = t < t_end && in_flight < TOKENS;
    if (__ballot(on) == 0) break;  // (none of the wave's tokens)
    auto& m = lds[min(in_flight, TOKENS - 1)];
    float l[C], b[C];
    bool odd = kGroups && opt.n_groups > L;  // what is no finite number, or more groups than lanes
    load_run<T, C>(logits + (on ? t : t_begin) * n_experts, sub * C, n_experts, vec, -INFINITY, l);
    if (bias != nullptr)
      load_run<float, C>(bias, sub * C, n_experts, vec_bias, 0.0f, b);
    else
#pragma unroll
      for (int i = 0; i < C; ++i) b[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) odd |= !(l[i] < INFINITY) || !(b[i] < INFINITY);
    float mx = l[0], inv = 1.0f;
    if (softmax) {
#pragma unroll
      for (int i = 1; i < C; ++i) mx = fmaxf(mx, l[i]);
      mx = lanes_max<L>(mx);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i) sum += l[i] == -INFINITY ? 0.0f : exp_near(l[i] - mx);
      inv = 1.0f / lanes_sum<L>(sum);
    }
    const auto score = [&](float x) {
      return softmax ? exp_near(x - mx) * inv : __builtin_amdgcn_rcpf(1.0f + exp_near(-x));
    };
    const float tol = !by_score ? 0.0f : softmax ? kTolSoftmax * inv : kTolSigmoid;
    float value[C];  // what the experts go by
#pragma unroll
    for (int i = 0; i < C; ++i) value[i] = l[i];
    if (bias != nullptr)
#pragma unroll
      for (int i = 0; i < C; ++i) value[i] = l[i] == -INFINITY ? l[i] : score(l[i]) + b[i];
    const T* const row = logits + (on ? t : t_begin) * n_experts;
    // what decides near ties: a softmax's sum and the value of an expert in 64 bits
    const auto sum64 = [&] {
      double sum = 0.0;
      if (softmax) {
        float* const values = reinterpret_cast<float*>(m.key);
        float again[C];  // (the row's logits: kept, they would cost the main path registers)
        load_run<T, C>(row, sub * C, n_experts, vec, -INFINITY, again);
        wave_sync();
#pragma unroll
        for (int i = 0; i < C; ++i) values[sub * C + i] = again[i];
        wave_sync();
#pragma unroll 1
        for (int i = 0; i < C; ++i) {
          const float x = values[sub * C + i];
          if (x != -INFINITY) sum += exp64((double)x - (double)mx);
        }
        sum = lanes_sum<L>(sum);
        wave_sync();
      }
      return sum;
    };
    const auto exact = [&](int e, double sum) {
      const double x = Elem<T>::to_f32(row[e]);
      return x == -INFINITY ? x : score_of(x, softmax, mx, sum) + (bias != nullptr ? (double)bias[e] : 0.0);
    };
    uint32_t key[C];
#pragma unroll
    for (int i = 0; i < C; ++i) key[i] = sub * C + i >= n_experts ? 0 : key_of(value[i], i);
    uint32_t in = ~0u;  // the lane's experts in groups that stay
    if constexpr (kGroups) {
      if (shape.shift >= 0) {
        in = group_stays<L, C>(value, tol, bias != nullptr, sub, opt, shape.shift, on, m, score, sum64, exact) ? ~0u : 0u;
      } else if (opt.n_groups <= L) {
        float worth[C];  // what the groups go by
#pragma unroll
        for (int i = 0; i < C; ++i)
          worth[i] = by_score && bias == nullptr && l[i] != -INFINITY ? score(l[i]) : value[i];
        in = in_kept<C>(groups_kept<L, C>(worth, tol, sub, opt, shape.per, n_experts, on, m, sum64, exact), sub,
                        shape.per);
      }
#pragma unroll
      for (int i = 0; i < C; ++i) key[i] = key[i] != 0 && (in >> i & 1) == 0 ? kOffKey | (15 - i) : key[i];
    }
    sort_down(key);
    const float left_out = pick<L, C>(key, sub, top_k, m);
    wave_sync();
    if (bias != nullptr || sizeof(T) == 4) {
      // (logits alone: only what their keys leave out)
      const auto apart = [&](float a, float b) { return bias != nullptr ? near(a, b, tol) : b > -INFINITY && a == b; };
      const float a = m.score[top_k - 1];
      bool seen = apart(a, left_out), close = false;
      for (int k = sub; k + 1 < top_k; k += L) seen |= apart(m.score[k], m.score[k + 1]);
      if (__ballot(seen && on) != 0) {
        // on the values themselves (their keys may have them in the wrong order); two alike
        // in logit and bias are in order
        const auto swapped = [&](float v0, float v1) {
          return bias == nullptr || v0 - v1 <= tol + kTolAdd * (fabsf(v0) + fabsf(v1));
        };
        const auto look = [&](int k, float& l0, float& b0) {
          const int e = min(m.pick[k], n_experts - 1);  // (odd rows hold anything)
          l0 = Elem<T>::to_f32(row[e]), b0 = bias != nullptr ? bias[e] : 0.0f;
          return e;
        };
        float l0, b0, l1, b1;
        for (int k = sub; k + 1 < top_k; k += L)
          if (apart(m.score[k], m.score[k + 1])) {
            look(k, l0, b0), look(k + 1, l1, b1);
            close |= (l0 != l1 || b0 != b1) && swapped(score(l0) + b0, score(l1) + b1);
          }
        const int e0 = look(top_k - 1, l0, b0);
        const float v0 = score(l0) + b0;
        const uint32_t k0 = key_of(a, 15);
        float ls[C], bs[C];
        load_run<T, C>(row, sub * C, n_experts, vec, -INFINITY, ls);
        if (bias != nullptr)
          load_run<float, C>(bias, sub * C, n_experts, vec_bias, 0.0f, bs);
        else
#pragma unroll
          for (int i = 0; i < C; ++i) bs[i] = 0.0f;
        uint32_t open = 0;  // the lane's experts that may be among the chosen
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const bool stays = (in >> i & 1) != 0;
          const uint32_t ki = stays ? key_of(value[i], 15) : kOffKey;
          const bool beside = apart(a, value_of(ki)), left = ki < k0 || (ki == k0 && sub * C + i > e0);
          if (sub * C + i < n_experts && (ki >= k0 || beside)) open |= 1u << i;
          close |= beside && left && (ls[i] != l0 || bs[i] != b0) && swapped(v0, value[i]);
        }
        const bool again = lanes_of<L>(close && on) != 0;
        if (__ballot(again) != 0) {
          const double sum = bias != nullptr ? sum64() : 0.0;
          odd |= !pick_exact<L, C>(again ? open : 0u, sub, top_k, m, [&](int e) {
            return (in >> (e - sub * C) & 1) == 0 ? -INFINITY
                   : bias != nullptr              ? exact(e, sum)
                                                  : (double)Elem<T>::to_f32(row[e]);
          });
          wave_sync();
        }
      }
    }
    const uint64_t odd_lanes = __ballot(odd && on);
    if (odd_lanes != 0) {
      const int first = (threadIdx.x & ~63) / L;  // the wave's first token in flight
#pragma unroll 1
      for (int h = 0; h < 64 / L; ++h)
        if ((odd_lanes >> (h * (L & 63)) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) != 0)
          choose_slowly<T>(logits + (t0 + first + h) * n_experts, bias, &opt, n_experts, top_k, &lds[first + h]);
    }
    // the weights, slots k = sub, sub + L, ...
    constexpr int SLOTS = ASTRAI_MOE_MAX_TOPK > L ? ASTRAI_MOE_MAX_TOPK / L : 1;
    float v[SLOTS], total = 0.0f, best = -INFINITY;
    int e[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int k = sub + i * L;
      v[i] = -INFINITY, e[i] = 0;
      if (on && k < top_k) {
        e[i] = m.pick[k];
        v[i] = m.score[k];  // NaN: the row holds no number; -inf: no live expert
        if (v[i] > -INFINITY) v[i] = Elem<T>::to_f32(logits[t * n_experts + e[i]]);
      }
      best = fmaxf(best, v[i]);
    }
    best = lanes_max<L>(best);
    const float base = opt.renormalise ? (softmax ? best : fminf(best, 0.0f)) : softmax ? mx : 0.0f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const float s = score32(v[i], softmax, base, mx);
      v[i] = v[i] == -INFINITY ? 0.0f : v[i] != v[i] ? v[i] : softmax && !opt.renormalise ? s * inv : s;
      total += v[i];
    }
    total = lanes_sum<L>(total);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int k = sub + i * L;
      if (!on || k >= top_k) continue;
      const float w = (opt.renormalise ? (total == 0.0f ? 0.0f : v[i] / total) : v[i]) * opt.scale;
      (kList ? s_e : topk_idx)[t * slots + k] = e[i];
      (kList ? s_w : topk_w)[t * slots + k] = Elem<W>::from_f32(w);
      if constexpr (kList)
        atomicOr(&mask[e[i]], 1u << (int)t);
      else
        atomicAdd(&hist[e[i]], 1);
    }
  }
  __syncthreads();
  if constexpr (kList) {
    write_chunk_list<W>(mask, hist, s_e, s_w, (int)n_tokens, columns, slots, list);
    return;
  }
  for (int e = threadIdx.x; e < columns; e += THREADS)
    chunk_hist[(int64_t)blockIdx.x * columns + e] = e < n_experts ? hist[e] : (int)(t_end - t_begin);
}

// dlogits of a token from dw, the gradient of its weights, at the chosen experts
// (a slot of weight 0 has no part: it was filled without a live expert, or its
// score is below every float), g_k = scale dw_k:
//   renormalised, r_k = s_k / S:  dl_k = r_k sum_j r_j (g_k - g_j), sigmoid times 1 - s_k,
//     and 0 at the others (a softmax over the row and S cancel); of differences, so that
//     one expert alone, or one that has nearly all the weight, loses no digits
//   otherwise:  sigmoid dl_k = g_k s_k (1 - s_k), softmax dl_e = s_e (g_e - sum_j g_j s_j).
// A wave per token, slot k in lane k; columns lane, lane + 64, ... of the row.
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
  const float g = mine && wk != 0.0f ? Elem<W>::to_f32(dw[t * top_k + lane]) * opt.scale : 0.0f;
  const T* const row = logits + t * n_experts;
  const bool softmax = opt.score == ASTRAI_MOE_SCORE_SOFTMAX, renorm = opt.renormalise != 0;
  const float chosen = idx >= 0 && idx < n_experts && wk != 0.0f ? Elem<T>::to_f32(row[idx]) : -INFINITY;
  float p[ITER], s = 0.0f, against = 1.0f;  // (against: 1 - s of a sigmoid)
  if (softmax) {
    float mx = chosen;
    if (!renorm)
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int c = lane + i * 64;
        p[i] = c < n_experts ? Elem<T>::to_f32(row[c]) : -INFINITY;
        mx = fmaxf(mx, p[i]);
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if (mx == -INFINITY) mx = 0.0f;
    s = expf(chosen - mx);
    if (!renorm) {
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
      s *= inv;
    }
  } else {
    // 1 - s(l) = s(-l), without the cancellation
    // (over e^base, as the weights)
    float base = renorm ? chosen : 0.0f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) base = fmaxf(base, __shfl_xor(base, off, 64));
    base = fminf(base, 0.0f);
    const float e = expf(-fabsf(chosen)), d = 1.0f / (1.0f + e);
    s = chosen >= 0.0f ? d : chosen == -INFINITY ? 0.0f : expf(chosen - base) * d;
    against = chosen >= 0.0f ? e * d : d;
  }
  float at_chosen, dot = 0.0f;
  if (renorm) {
    const float S = wave_sum(s), r = S == 0.0f ? 0.0f : s / S;
    float sum = 0.0f;
    for (int k = 0; k < top_k; ++k) sum += __shfl(r, k, 64) * (g - __shfl(g, k, 64));
    at_chosen = r * sum * against;
  } else {
    at_chosen = softmax ? g : g * s * against;
    if (softmax) dot = wave_sum(g * s);
  }
  if (wk != wk) at_chosen = wk;  // (the row holds no number)
  const bool poison = softmax && __any(wk != wk);
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = lane + i * 64;
    float d = 0.0f;
    for (int k = 0; k < top_k; ++k) {
      const int e = __shfl(idx, k, 64);
      const float v = __shfl(at_chosen, k, 64);
      if (e == c) d += v;
    }
    if (softmax && !renorm) d = p[i] * (d - dot);
    if (c < n_experts) dlogits[t * n_experts + c] = Elem<T>::from_f32(poison ? NAN : d);
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
  const int threads = list != nullptr ? score_threads<L, true>() : score_threads<L, false>();
  GroupShape shape{n_experts / opt.n_groups, -1};
  if (shape.per % C == 0 && (shape.per / C & (shape.per / C - 1)) == 0) shape.shift = __builtin_ctz(shape.per / C);
  hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, static_cast<const T*>(logits), bias, opt, n_tokens, n_experts,
                     top_k, n_shared, topk_idx, static_cast<W*>(topk_w), chunk_hist,
                     list != nullptr ? *list : RouteList{}, shape,
                     n_experts * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0,
                     n_experts % 4 == 0 && reinterpret_cast<uintptr_t>(bias) % 16 == 0);
}

template <typename T, typename W>
int launch_scores(const void* logits, const float* bias, const astrai_moe_routing& opt, int64_t n_tokens,
                  int n_experts, int top_k, int n_shared, int32_t* topk_idx, void* topk_w, int32_t* chunk_hist,
                  const RouteList* list, hipStream_t s) {
#define ROUTE_CASE(L, C)                                                                                       \
  launch_scores_cfg<T, W, L, C>(logits, bias, opt, n_tokens, n_experts, top_k, n_shared, topk_idx, topk_w,      \
                                chunk_hist, list, s)
  // As many lanes as groups, more than 64 of which are for choose_slowly. (16384 tokens, us,
  // 128 experts in 32 groups by 16 lanes, so choose_slowly, 82, by 32 lanes 31; 256 in 64
  // groups by 16 lanes 126, by 64 lanes 92.)
  const bool few = opt.n_groups <= 16;
  if (n_experts <= 32 && few)
    ROUTE_CASE(16, 2);
  else if (n_experts <= 64 && few)
    ROUTE_CASE(16, 4);
  else if (n_experts <= 128 && few)
    ROUTE_CASE(16, 8);
  else if (n_experts <= 256 && few)
    ROUTE_CASE(16, 16);
  else if (n_experts <= 512 && opt.n_groups <= 32)
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
