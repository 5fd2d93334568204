// Choice of experts from a router's logits, and its gradient.
//
//   s   = sigmoid(x) or softmax(x)           (32-bit values; see below)
//   sel = s + bias                           (bias: for balance, in the choice only)
//   groups: the n_group blocks of E / n_group experts are scored by the sum of their two highest
//           sel (or the highest); the topk_group best stay
//   the top_k highest sel of what stays, equal ones from the lowest index up (groups likewise)
//   w_k = s_k, divided by (sum of the chosen s + 1e-20) if renormalised, times scale
//
// A logit of -inf or of its type's lowest value switches an expert off: it is never chosen, and
// slots for which no expert is left hold id -1 and weight 0.  A row with a NaN score chooses
// nothing and has NaN weights.
//
// Scores are 32-bit by definition, with the exponential (sigmoid: 1 / (1 + fl(exp(-x))), the
// routing kernel's own form; softmax: the quotient) rounded to 32 bits once from a double
// evaluation, so a choice depends on no order of summation and on no approximation.
//
// One warp per token; lane l holds experts V l .. V l + V - 1.  A double exponential per logit would
// be most of the work, so a token is first chosen for with 32-bit scores whose error is bounded,
// and the choice stands if every decision (the last group kept against the best one dropped, the
// last expert chosen against the best one left) is further apart than that allows for; otherwise,
// which for continuous logits is one token in some hundreds, the scores
// are computed as defined and the choice is made again from those.
//
// Bound by the warps' instructions, about 850 per token of 256 experts in 8 groups (scores, a sort of
// eight keys per lane, rounds of maxima), not by HBM: 16384 tokens 20.7 us with counts (17.9 without
// groups, 18.0 softmax) where the logits alone would take 2.7; 512 experts 41 us, 64 experts 11.  Few
// tokens are bound by the one token's chain of operations: 16 tokens 4.6 us.
#include <type_traits>

#include "exp64.cuh"
#include "op_common.cuh"

namespace moe {

constexpr int kSelMaxE = 512;
constexpr int kSelMaxK = 32;
constexpr int kSelWarps = 8;

struct SelectArgs {
  const void* logits;
  const void* bias;
  int* idx;
  float* w;
  int* counts;
  int64_t ld;
  int T, E, K, type, bias_type, n_group, topk_group, top2, renorm;
  int vec;       // rows start on 16 (32-bit logits) or 8 bytes
  int cluster;   // the grid is one cluster, which adds up the counts by itself
  float scale;
};

struct SelectBwdArgs {
  const void* logits;
  const int* idx;
  const float* dw;
  void* dlogits;
  int64_t ld, dld;
  int T, E, K, type, renorm;
  int vec, dvec;   // rows start on 16 (32-bit logits) or 8 bytes
  float scale;
};

__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A logit at or below this switches its expert off.
__device__ __forceinline__ float lowest_of(int type) {
  return type == MOE_B200_BF16 ? __uint_as_float(0xff7f0000u) : type == MOE_B200_FP16 ? -65504.f : -3.4028234663852886e38f;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// Sorts v[0..N-1] descending (odd-even merge network).
template <int N>
__device__ __forceinline__ void sort_desc(float (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const float hi = fmaxf(v[i + j], v[i + j + k]), lo = fminf(v[i + j], v[i + j + k]);
            v[i + j] = hi;
            v[i + j + k] = lo;
          }
}

__device__ __forceinline__ float redux_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ float redux_min(float v) {
  float m;
  asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Loads this lane's V logits (experts first.. of E; the rest as -inf).
template <int V>
__device__ __forceinline__ void load_logits(const void* p, int type, int64_t off, int first, int E, bool vec, float* x) {
  if (V >= 4 && vec && first + V <= E) {
    if (type == MOE_B200_FP32) {
#pragma unroll
      for (int i = 0; i + 4 <= V; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + off + first + i);
        x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i + 4 <= V; i += 4) {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + off + first + i);
        if (type == MOE_B200_BF16) {
          unpack2(u.x, x + i, bf16{});
          unpack2(u.y, x + i + 2, bf16{});
        } else {
          unpack2(u.x, x + i, fp16{});
          unpack2(u.y, x + i + 2, fp16{});
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = first + i < E ? load1_dyn(p, type, off + first + i) : -INFINITY;
  }
}

template <int V>
__device__ __forceinline__ void store_logits(void* p, int type, int64_t off, int first, int E, bool vec, const float* x) {
  if (V >= 4 && vec && first + V <= E) {
#pragma unroll
    for (int i = 0; i + 4 <= V; i += 4) {
      if (type == MOE_B200_FP32)
        *reinterpret_cast<float4*>(static_cast<float*>(p) + off + first + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      else if (type == MOE_B200_BF16)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + off + first + i) =
            make_uint2(pack2(x[i], x[i + 1], bf16{}), pack2(x[i + 2], x[i + 3], bf16{}));
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + off + first + i) =
            make_uint2(pack2(x[i], x[i + 1], fp16{}), pack2(x[i + 2], x[i + 3], fp16{}));
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (first + i < E) store1_dyn(p, type, off + first + i, x[i]);
  }
}

// exp(d) for d <= 0, in double (a score's numerator).
__device__ __forceinline__ double exp_below(double d) { return d != d ? d : d < -700.0 ? 0.0 : exp_series(d); }

// The scores as defined (EXACT), or 32-bit ones.  Returns the largest score of the row that is
// known without looking (sigmoid: 1; softmax: that of the largest logit): the size that errors
// are measured by.  A 32-bit score is off by less than 20 * 2^-23 of it, __expf(-d) being off by
// (2 + 1.2 d) 2^-23 of itself:
//   sigmoid: that moves s by s (1 - s) times as much, at most 2^-23; the sum and the quotient add 3.
//   softmax: d e^-d is at most 0.37, so its own exponential moves a score by 2.5.  The row's sum moves
//     with the exponentials of all, up to 6 (512 experts alike, each ln 511 below the first), and by 10
//     for its roundings, 15 in a lane and 5 over the lanes.  The quotient and the product add 1.
// *top: softmax: the row's largest logit.
template <int V, bool SOFTMAX, bool EXACT>
__device__ __forceinline__ float scores(const float* x, float lowest, float* s, float* top) {
  if constexpr (!SOFTMAX) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (EXACT) s[i] = x[i] <= lowest ? 0.f : __frcp_rn(1.0f + exp_to_f32(-static_cast<double>(x[i])));
      else s[i] = x[i] <= lowest ? 0.f : __fdividef(1.0f, 1.0f + __expf(-max_nan(x[i], -80.f)));
    }
    return 1.f;
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);   // (switched off ones do no harm)
    m = redux_max(m);
    *top = m;
    if constexpr (EXACT) {
      double ex[V], sum = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = static_cast<double>(x[i]) - static_cast<double>(m);
        ex[i] = x[i] <= lowest ? 0.0 : exp_below(d);
        sum += ex[i];
      }
      const double inv = 1.0 / warp_sum_d(sum);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = x[i] <= lowest ? 0.f : static_cast<float>(ex[i] * inv);
      return static_cast<float>(inv);
    } else {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] = x[i] <= lowest ? 0.f : __expf(x[i] - m);
        sum += s[i];
      }
      const float inv = 1.f / max_nan(warp_sum(sum), 1e-30f);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] *= inv;
      return inv;
    }
  }
}

// exp(d) in double for -700 < d <= 0, within 2^-32 of itself: the series of exp_series to degree 8 (.3466^9 /
// 9! = 2^-32.2), ln 2 in one part, k by adding 1.5 * 2^52 in place of conversions, which run at a quarter of
// the rate.
__device__ __forceinline__ double exp_to_33_bits(double d) {
  const double shifted = fma(d, 1.4426950408889634074, 0x1.8p52);
  const double r = fma(shifted - 0x1.8p52, -6.93147180559945309417e-01, d);
  double p = 1.0 / 40320.0;
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(shifted) << 20), __double2loint(p));
}

// The sum of the row's exp(x - top) within 2^-32 of itself (if an expert is on), in all lanes.
template <int V>
__device__ __forceinline__ double softmax_sum(const float* x, float top) {
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {   // (e^-60 is next to nothing beside the largest's 1)
    const double e = exp_to_33_bits(static_cast<double>(x[i]) - static_cast<double>(top));
    sum += x[i] - top > -60.f ? e : 0.0;
  }
  return warp_sum_d(sum);
}

// The scores from those exponentials, each rounded once; returns that of the largest logit (*top).
template <int V>
__device__ __forceinline__ float softmax_scores(const float* x, float lowest, float* s, float* top) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
  *top = m = redux_max(m);
  double e[V], sum = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float d = x[i] - m;
    e[i] = x[i] <= lowest ? 0.0 : d > -690.f ? exp_to_33_bits(static_cast<double>(x[i]) - static_cast<double>(m)) : d != d ? d : 0.0;
    sum += e[i];
  }
  sum = warp_sum_d(sum);
  const double inv = sum > 0.0 ? 1.0 / sum : sum;   // (NaN stays)
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = static_cast<float>(e[i] * inv);
  return static_cast<float>(inv);
}

// Two sides of a decision are told apart by the 32-bit scores if they differ by more than this
// share of the sizes involved, M = max(size, both sides).  In units of 2^-18: an expert's score is off by
// 5/8 of the row's size and its key by 1 of itself (the lane in the low five bits); for two experts that
// is at most 3.25 M.  A group's score is the sum of two such keys, and its own key is off by 1 once more:
// 1.25 size + |m1| + |m2| + |m1 + m2| a side.  Where m1 and m2 have opposite signs, |m1| + |m2| is up to
// |m1 + m2| + 2 B, B = the lowest bias's distance below 0 (scores are not negative), so for sums of two M
// counts 2 B as well (group_size): 2.5 size + 4 M + 4 B <= 6.5 M.  Sums round by 2^-6 each.  The margin is 8.
constexpr float kMargin = 3.0517578125e-05f;

// Whether `in` (the weakest taken) is above `out` (the strongest left) for certain.  -inf for
// either: nothing was taken or left, no decision.
__device__ __forceinline__ bool apart(float in, float out, float size) {
  return out == -INFINITY || in == -INFINITY || in - out > kMargin * fmaxf(size, fmaxf(fabsf(in), fabsf(out)));
}

// Keys of the fast choice: sel (below kHuge in size) with the lane in its low 5 bits, so that no two
// lanes have equal ones; at most kNone: not to be chosen.
constexpr float kNone = -3.39e38f, kFloor = -3.38e38f, kHuge = 1e30f;
__device__ __forceinline__ float lane_key(float sel, int lane) {
  return __uint_as_float((__float_as_uint(fmaxf(sel, -3.4e38f)) & ~31u) | lane);
}
__device__ __forceinline__ float or_none(float v) { return v <= kNone ? -INFINITY : v; }

// Group scores from shared memory: lane g < n_group scans group g.
__device__ __forceinline__ void scan_group(const float* sel, int lane, int n_group, int gs, float* m1, float* m2) {
  *m1 = *m2 = -INFINITY;
  if (lane < n_group)
    for (int j = 0; j < gs; ++j) {
      // each lane starts elsewhere in its group, so that they do not meet in one bank
      const int k = j + lane;
      const float v = sel[lane * gs + (k < gs ? k : k % gs)];
      *m2 = fmaxf(*m2, fminf(*m1, v));
      *m1 = fmaxf(*m1, v);
    }
}
__device__ __forceinline__ float group_score(const SelectArgs& a, float m1, float m2) {
  return a.top2 ? m1 + (m2 == -INFINITY ? 0.f : m2) : m1;
}

// Whether group g (its score in each of its lanes, lane h * lanes first) is among the topk_group
// best, equal ones from the first up.
__device__ __forceinline__ bool keep_group(const SelectArgs& a, float score, int g, int lanes) {
  int rank = 0;
  for (int h = 0; h < a.n_group; ++h) {
    const float o = __shfl_sync(0xffffffffu, score, h * lanes);
    rank += (o > score || (o == score && h < g)) ? 1 : 0;
  }
  return g < a.n_group && rank < a.topk_group;
}
// The same by 32-bit scores: rounds of the highest score left, the group in its low 5 bits; *sure:
// the last one kept is apart from the best one dropped.
__device__ __forceinline__ bool keep_group_fast(const SelectArgs& a, float score, int g, float size, bool* sure) {
  const float key = g < a.n_group ? lane_key(score, g) : -3.4e38f;
  float left = key, last = 0.f;
#pragma unroll 4
  for (int r = 0; r < a.topk_group; ++r) {
    last = redux_max(left);   // (kNone or below where nothing is left)
    left = left == last ? -3.4e38f : left;
  }
  *sure = apart(or_none(last), or_none(redux_max(left)), size);
  return key >= fmaxf(last, kFloor);
}

// Whether a group is a power of two of neighbouring lanes (*lanes); otherwise groups are scored
// through shared memory.
template <int V>
__device__ __forceinline__ bool groups_by_lane(const SelectArgs& a, int* lanes) {
  const int gs = a.E / a.n_group;
  *lanes = gs / V;
  return gs % V == 0 && (*lanes & (*lanes - 1)) == 0;
}
// The score of a lane's group, m1 >= m2 being the two highest of the lane's own part of it.
__device__ __forceinline__ float score_by_lane(const SelectArgs& a, float m1, float m2, int lanes) {
  for (int d = 1; d < lanes; d <<= 1) {
    const float o1 = __shfl_xor_sync(0xffffffffu, m1, d), o2 = __shfl_xor_sync(0xffffffffu, m2, d);
    m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
    m1 = fmaxf(m1, o1);
  }
  return group_score(a, m1, m2);
}

// Drops what is not in a kept group from sel, through shared memory: groups of any size.
template <int V>
__device__ __forceinline__ void drop_groups(const SelectArgs& a, float* sel, float* s_sel, int lane, bool fast, float size,
                                            bool* sure) {
  const int first = lane * V, gs = a.E / a.n_group;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (first + i < a.E) s_sel[first + i] = sel[i];
  __syncwarp();
  float m1, m2;
  scan_group(s_sel, lane, a.n_group, gs, &m1, &m2);
  const float score = group_score(a, m1, m2);
  const uint32_t kept =
      __ballot_sync(0xffffffffu, fast ? keep_group_fast(a, score, lane, size, sure) : keep_group(a, score, lane, 1));
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (first + i < a.E && !((kept >> ((first + i) / gs)) & 1u)) sel[i] = -INFINITY;
  __syncwarp();
}

// The choice by the defined scores: bit i of the result says that this lane's expert i is chosen.
template <int V>
__device__ __forceinline__ uint32_t choose_exact(const SelectArgs& a, float* sel, float* s_sel, int lane) {
  bool kept = true;
  int lanes;
  if (a.n_group > 1) {
    if (groups_by_lane<V>(a, &lanes)) {
      float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        m2 = fmaxf(m2, fminf(m1, sel[i]));
        m1 = fmaxf(m1, sel[i]);
      }
      kept = keep_group(a, score_by_lane(a, m1, m2, lanes), lane / lanes, lanes);
    } else {
      drop_groups<V>(a, sel, s_sel, lane, false, 0.f, nullptr);
    }
  }
  uint32_t key[V], taken = 0;   // key 0: not to be chosen
#pragma unroll
  for (int i = 0; i < V; ++i) key[i] = !kept || sel[i] == -INFINITY ? 0u : order_key(sel[i]);
  for (int r = 0; r < a.K; ++r) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = V - 1; i >= 0; --i)
      if (key[i] >= best) {
        best = key[i];
        at = i;
      }
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    if (m == 0) break;
    if (lane == __ffs(__ballot_sync(0xffffffffu, best == m)) - 1) {
      taken |= 1u << at;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i == at) key[i] = 0;
    }
  }
  return taken;
}

// K rounds of the highest key left in the warp, each a maximum over the lanes' first keys and a
// shift of the list that held it; returns the last one's (kNone or below where there are fewer).
// Up to eight rounds are unrolled, so that a list is shifted only as far as later rounds may reach.
template <int V>
__device__ __forceinline__ float last_of_rounds(float (&list)[V + 1], int K) {
  float last = 0.f;
  if (K <= 8) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r >= K) break;
      last = redux_max(list[0]);
      const bool mine = list[0] == last;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i <= 7 - r) list[i] = mine ? list[i + 1] : list[i];
    }
  } else {
    for (int r = 0; r < K; ++r) {
      last = redux_max(list[0]);
      const bool mine = list[0] == last;
#pragma unroll
      for (int i = 0; i < V; ++i) list[i] = mine ? list[i + 1] : list[i];
    }
  }
  return last;
}

// The choice by 32-bit scores; *sure tells whether they decide it.  Each lane sorts its keys; what
// is chosen is what reaches the last round's maximum.
template <int V>
__device__ __forceinline__ uint32_t choose_fast(const SelectArgs& a, float* sel, float* s_sel, int lane, float size,
                                                float group_size, bool* sure) {
  *sure = true;
  int lanes = 0;
  const bool by_lane = a.n_group > 1 && groups_by_lane<V>(a, &lanes);
  if (a.n_group > 1 && !by_lane) drop_groups<V>(a, sel, s_sel, lane, true, group_size, sure);
  float key[V], list[V + 1];
#pragma unroll
  for (int i = 0; i < V; ++i) key[i] = lane_key(sel[i], lane);
  {
    float sorted[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sorted[i] = key[i];
    sort_desc(sorted);
#pragma unroll
    for (int i = 0; i < V; ++i) list[i] = sorted[i];
    list[V] = -3.4e38f;
  }
  bool kept = true;
  if (by_lane) {
    const float score = score_by_lane(a, or_none(list[0]), V > 1 ? or_none(list[V > 1 ? 1 : 0]) : -INFINITY, lanes);
    kept = keep_group_fast(a, score, lane / lanes, group_size, sure);
#pragma unroll
    for (int i = 0; i < V; ++i) list[i] = kept ? list[i] : -3.4e38f;
  }
  const float last = last_of_rounds<V>(list, a.K);
  // (equal keys of one lane on both sides of the end are not apart)
  *sure = *sure && apart(or_none(last), or_none(redux_max(list[0])), size);
  const float least = kept ? fmaxf(last, kFloor) : INFINITY;
  uint32_t taken = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) taken |= key[i] >= least ? 1u << i : 0u;
  return taken;
}

// The chosen experts' weights are computed by the lanes that store them, one expert each.  A sigmoid is the
// score as defined.  A softmax's exponentials are taken in double and rounded once; renormalised, the row's
// sum stands beside the chosen ones' only in the 1e-20, which counts for less than 2^-28 where the best of
// them is within e^-20 of the row's first: a share of e^-20 / 512 of the sum at least.  (Weights of the 32-bit
// scores were off by |x - m| units, on average 5.8e-8.)  16384 x 256 softmax 18.0 us renormalised; 21.3 not,
// for which every exponential is taken in double for the row's sum, and is then the score as well (22.4
// when the sum was taken beside 32-bit scores).
constexpr float kNoneBeside = 20.f;

// Registers: 64 a thread for up to 256 experts (more CTAs on an SM with less gain nothing: 16384 x 256
// 21.3 us with five, 22.0 with six), 80 for 512, where three CTAs fit an SM (16384 x 512: sigmoid 42.1 us
// against 48.5 with as many as it would take, two CTAs; softmax 42.2 against 47.9).  No form spills.
template <int V, bool SOFTMAX>
__global__ void __launch_bounds__(kSelWarps * 32, V == 16 ? 3 : 4) select_kernel(SelectArgs a) {
  extern __shared__ __align__(16) float s_dyn[];   // [warps][32 V] values of a token, then [E] counts
  __shared__ int s_id[kSelWarps][kSelMaxK];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* s_row = s_dyn + warp * 32 * V;
  int* s_cnt = reinterpret_cast<int*>(s_dyn + kSelWarps * 32 * V);
  if (a.counts) {
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) s_cnt[e] = 0;
    __syncthreads();
  }
  const float lowest = lowest_of(a.type);
  const int first = lane * V;
  float bias[V], below = 0.f;
  bool wild = false;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && first + i < a.E ? load1_dyn(a.bias, a.bias_type, first + i) : 0.f;
    wild |= fabsf(bias[i]) >= kHuge && bias[i] != -INFINITY;
    below = bias[i] == -INFINITY ? below : fminf(below, bias[i]);
  }
  // biases so large that sums of two overflow: every choice by the defined scores
  wild = __any_sync(0xffffffffu, wild);
  const float cancel = a.n_group > 1 && a.top2 ? -2.f * redux_min(below) : 0.f;   // 2 B of the margin
  const int step = gridDim.x * kSelWarps;
  for (int t = blockIdx.x * kSelWarps + warp; t < a.T; t += step) {
    float x[V], s[V], sel[V];
    load_logits<V>(a.logits, a.type, t * a.ld, first, a.E, a.vec, x);
    if (t < a.T - step && first < a.E)   // the next token's, toward L2
      prefetch_l2(static_cast<const uint8_t*>(a.logits) + ((t + step) * a.ld + first) * (a.type == MOE_B200_FP32 ? 4 : 2));
    float top = 0.f;
    // weights that are a softmax's scores themselves are computed with them (512 experts leave no registers for it)
    const bool ready = SOFTMAX && V <= 8 && !a.renorm;
    float size;
    if (ready) size = softmax_scores<V <= 8 ? V : 1>(x, lowest, s, &top);
    else size = scores<V, SOFTMAX, false>(x, lowest, s, &top);
    float nan = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sel[i] = x[i] <= lowest ? -INFINITY : s[i] + bias[i];
      nan = max_nan(nan, sel[i]);
    }
    const bool bad = __any_sync(0xffffffffu, nan != nan);
    uint32_t taken = 0;
    bool sure = bad || !wild;
    if (!bad && sure) taken = choose_fast<V>(a, sel, s_row, lane, size, size + cancel, &sure);
    if (!sure) {
      scores<V, SOFTMAX, true>(x, lowest, s, &top);
#pragma unroll
      for (int i = 0; i < V; ++i) sel[i] = x[i] <= lowest ? -INFINITY : s[i] + bias[i];
      taken = choose_exact<V>(a, sel, s_row, lane);
    }
    // the chosen, by ascending id, to one lane each: those compute and store the weights
#pragma unroll
    for (int i = 0; i < V; ++i) s_row[first + i] = ready ? s[i] : x[i];
    const int mine = __popc(taken);
    int pos = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, pos, d);
      if (lane >= d) pos += o;
    }
    const int total = __shfl_sync(0xffffffffu, pos, 31);
    for (pos -= mine; taken; taken &= taken - 1) s_id[warp][pos++] = first + __ffs(taken) - 1;
    __syncwarp();
    const bool have = lane < total;
    const int id = have ? s_id[warp][lane] : -1;
    const float logit = have ? s_row[id] : SOFTMAX ? -INFINITY : 0.f;
    __syncwarp();
    float w = 0.f, denom = 1.f;   // (the division is left to the lanes that have an expert)
    if constexpr (!SOFTMAX) {
      w = have ? __frcp_rn(1.0f + exp_to_f32(-static_cast<double>(logit))) : 0.f;
      denom = warp_sum(w) + 1e-20f;
    } else if (ready) {
      w = have ? logit : 0.f;   // the score
    } else if (total > 0) {
      const float best = redux_max(logit);
      if (a.renorm && top - best <= kNoneBeside) {
        w = logit - best > -110.f ? static_cast<float>(exp_to_33_bits(static_cast<double>(logit) - static_cast<double>(best))) : 0.f;
        denom = warp_sum(w);
      } else {
        const double e = logit - top > -690.f ? exp_to_33_bits(static_cast<double>(logit) - static_cast<double>(top)) : 0.0;
        double sum = softmax_sum<V>(x, top);
        if (a.renorm) sum = warp_sum_d(e) + 1e-20 * sum;
        w = static_cast<float>(e / sum);
      }
    }
    if (lane < a.K) {
      const int64_t o = static_cast<int64_t>(t) * a.K + lane;
      a.idx[o] = id;
      a.w[o] = bad ? __uint_as_float(0x7fc00000u) : (a.renorm ? w / denom : w) * a.scale;
    }
    if (a.counts && have) atomicAdd(s_cnt + id, 1);
  }
  if (!a.counts) return;
  if (a.cluster) {   // the CTAs of one cluster are the whole grid: the first adds up their counts
    cluster_sync();
    if (blockIdx.x == 0)
      for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        int n = 0;
        for (uint32_t c = 0; c < gridDim.x; ++c) n += ld_cluster_s32(cluster_addr(smem_u32(s_cnt + e), c));
        a.counts[e] = n;
      }
    cluster_sync();
  } else {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x)
      if (s_cnt[e]) atomicAdd(a.counts + e, s_cnt[e]);   // integers: the order does not matter
  }
}

__global__ void __launch_bounds__(kSelMaxE) select_zero_kernel(int* counts, int E) {
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < E) counts[threadIdx.x] = 0;
}

// dlogits of a token, from the gradients dw of its chosen weights (ids distinct, -1: no expert).
//   renormalised, S = sum of the chosen s + 1e-20:  ds_k = scale * (dw_k - sum_j dw_j s_j / S) / S
//   softmax: dx_e = s_e (ds_e - sum_j ds_j s_j);  sigmoid: dx_e = ds_e s_e (1 - s_e)
// The scores go to shared memory, where a lane per chosen expert finds its own; those lanes work out
// the sums and put their own results among what every lane stores.  16384 x 256 softmax 10.4 us (3.3
// TB/s: about half by memory, half by the exponentials and sums), sigmoid 9.6, 512 experts 33.5 and 32.3.
template <int V, bool SOFTMAX>
__global__ void __launch_bounds__(kSelWarps * 32) select_bwd_kernel(SelectBwdArgs a) {
  __shared__ __align__(16) float s_row[kSelWarps][32 * V];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float lowest = lowest_of(a.type);
  const int first = lane * V;
  float* row = s_row[warp];
  // a token's logits, ids and gradients are loaded while the one before it is computed
  float next_x[V], next_d = 0.f;
  int next_id = -1;
  auto load = [&](int t) {
    load_logits<V>(a.logits, a.type, t * a.ld, first, a.E, a.vec, next_x);
    const int64_t at = static_cast<int64_t>(t) * a.K + lane;
    next_id = lane < a.K ? a.idx[at] : -1;
    next_d = lane < a.K ? a.dw[at] : 0.f;
  };
  int t = blockIdx.x * kSelWarps + warp;
  if (t < a.T) load(t);
  for (const int step = gridDim.x * kSelWarps; t < a.T; t += step) {
    float x[V], s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = next_x[i];
    const int id = next_id;
    const bool have = id >= 0 && id < a.E;
    float d = have ? next_d * a.scale : 0.f;
    if (t < a.T - step) load(t + step);
    if constexpr (SOFTMAX) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
      m = redux_max(m);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] = x[i] <= lowest ? 0.f : expf(x[i] - m);
        sum += s[i];
      }
      const float inv = 1.f / max_nan(warp_sum(sum), 1e-30f);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = x[i];
    }
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      row[first + i] = s[i];
      all = max_nan(all, s[i]);
    }
    const bool bad = __any_sync(0xffffffffu, all != all);   // a NaN logit, or an infinite one of a softmax
    __syncwarp();
    float sk = have ? row[id] : 0.f;
    // sigmoid: from the logit that was put there (one that is switched off gives 0).  With h =
    // exp(-|x| / 2) and r = 1 / (1 + h h), s (1 - s) = (h r)^2: nothing cancels where s is near 1, and nothing
    // overflows or loses its bits where it is next to 0.
    float root = 0.f;
    if constexpr (!SOFTMAX) {
      const float h = expf(-0.5f * fabsf(sk)), r = 1.f / fmaf(h, h, 1.f);
      root = h * r;
      sk = have ? (sk < 0.f ? h * root : r) : 0.f;
    }
    float dot = d * sk;
    if (a.renorm) {
      const float S = warp_sum(sk) + 1e-20f;
      const float mean = warp_sum(dot) / S;
      d = have ? (d - mean) / S : 0.f;
      dot = d * sk;
    }
    float mine;   // this lane's chosen expert's gradient
    if constexpr (SOFTMAX) {
      dot = warp_sum(dot);
      mine = sk * (d - dot);
    } else {
      mine = d * root * root;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i) row[first + i] = SOFTMAX ? -s[i] * dot : 0.f;
    __syncwarp();
    if (have) row[id] = mine;
    __syncwarp();
    float g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = bad ? __uint_as_float(0x7fc00000u) : row[first + i];
    store_logits<V>(a.dlogits, a.type, t * a.dld, first, a.E, a.dvec, g);
    __syncwarp();
  }
}

namespace {

// f(values per lane): the smallest power of two that holds E experts
template <class F>
void dispatch_select(int E, F&& f) {
  if (E <= 32) f(std::integral_constant<int, 1>{});
  else if (E <= 64) f(std::integral_constant<int, 2>{});
  else if (E <= 128) f(std::integral_constant<int, 4>{});
  else if (E <= 256) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}

// Eight CTAs of eight warps for every SM, which are all its warps; registers leave the forward four at a
// time.  With four the backward of 16384 x 256 takes 15.7 us instead of 10.4, the forward 21.1 instead of
// 20.7.
int select_grid(int T, int sms) {
  const int need = (T + kSelWarps - 1) / kSelWarps;
  return need < 8 * sms ? need : 8 * sms;
}

}  // namespace
}  // namespace moe

extern "C" {

MOE_B200_API int moe_b200_select_experts(const moe_b200_select_args* a, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->num_tokens < 0 || a->num_tokens > kOpMaxRows || a->num_experts < 1 || a->num_experts > kSelMaxE)
    return report_error(MOE_B200_ERR_ARG, "select_experts: num_tokens must be in [0, 2^30] and num_experts in [1, 512]");
  if (a->n_group < 1 || a->n_group > 32 || a->num_experts % a->n_group)
    return report_error(MOE_B200_ERR_ARG, "select_experts: n_group must be in [1, 32] and divide num_experts");
  const int gs = a->num_experts / a->n_group;
  if (a->topk_group < 1 || a->topk_group > a->n_group)
    return report_error(MOE_B200_ERR_ARG, "select_experts: topk_group must be in [1, n_group]");
  if (a->top_k < 1 || a->top_k > kSelMaxK || a->top_k > a->topk_group * gs)
    return report_error(MOE_B200_ERR_ARG, "select_experts: top_k must be in [1, 32] and at most the experts of topk_group groups");
  if (a->group_score != MOE_B200_GROUP_TOP2 && a->group_score != MOE_B200_GROUP_MAX)
    return report_error(MOE_B200_ERR_ARG, "select_experts: bad group_score");
  if (a->n_group > 1 && a->group_score == MOE_B200_GROUP_TOP2 && gs < 2)
    return report_error(MOE_B200_ERR_ARG, "select_experts: groups scored by their top 2 need two experts or more");
  if (a->score != MOE_B200_SCORE_SIGMOID && a->score != MOE_B200_SCORE_SOFTMAX)
    return report_error(MOE_B200_ERR_ARG, "select_experts: bad score");
  if (!is_float_type(a->logits_type) || (a->bias && !is_float_type(a->bias_type)))
    return report_error(MOE_B200_ERR_ARG, "select_experts: logits and bias are bf16, fp16 or fp32");
  if (a->num_tokens > 0 && (!a->logits || !a->idx || !a->weight))
    return report_error(MOE_B200_ERR_ARG, "null tensor pointer");
  int sms = 0;
  if (int rc = op_device(&sms)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  // Counts: up to 64 tokens are one cluster's, which adds up its CTAs' histograms; beyond that
  // the CTAs add theirs to counts zeroed first.  On the device the two are alike (1 token 3.7 us
  // against 4.2, 16 tokens 4.6 against 4.4, 64 tokens 4.6 against 5.3), but the cluster is one launch,
  // 2.5 us of the caller's time less.
  const int ctas = select_grid(a->num_tokens, sms);
  const bool cluster = a->counts && a->num_tokens > 0 && ctas <= 8;
  if (a->counts && !cluster) {
    e = launch_pdl(select_zero_kernel, dim3(1), dim3(kSelMaxE), 0, st, a->counts, a->num_experts);
    if (e != cudaSuccess) return report_cuda(e, "select_experts launch");
  }
  if (a->num_tokens == 0) return MOE_B200_OK;
  SelectArgs s{};
  s.logits = a->logits;
  s.bias = a->bias;
  s.idx = a->idx;
  s.w = a->weight;
  s.counts = a->counts;
  s.ld = a->logits_stride;
  s.T = a->num_tokens;
  s.E = a->num_experts;
  s.K = a->top_k;
  s.type = a->logits_type;
  s.bias_type = a->bias_type;
  s.n_group = a->topk_group < a->n_group ? a->n_group : 1;   // keeping every group is no limit
  s.topk_group = a->topk_group;
  s.top2 = a->group_score == MOE_B200_GROUP_TOP2;
  s.renorm = a->renormalize;
  s.scale = a->scale;
  const int bytes = 4 * type_bytes(s.type);
  s.vec = reinterpret_cast<uintptr_t>(s.logits) % bytes == 0 && (s.T == 1 || s.ld % 4 == 0);
  s.cluster = cluster;
  const dim3 grid(ctas), block(kSelWarps * 32);
  dispatch_select(s.E, [&](auto v) {
    constexpr int V = decltype(v)::value;
    const size_t smem = (kSelWarps * 32 * V + (s.counts ? s.E : 0)) * sizeof(float);
    auto kernel = a->score == MOE_B200_SCORE_SOFTMAX ? select_kernel<V, true> : select_kernel<V, false>;
    e = cluster ? launch_cluster_pdl(kernel, grid, block, smem, ctas, st, s) : launch_pdl(kernel, grid, block, smem, st, s);
  });
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "select_experts launch");
}

MOE_B200_API int moe_b200_select_experts_backward(const moe_b200_select_backward_args* a, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->num_tokens < 0 || a->num_tokens > kOpMaxRows || a->num_experts < 1 || a->num_experts > kSelMaxE)
    return report_error(MOE_B200_ERR_ARG, "select_experts_backward: num_tokens must be in [0, 2^30] and num_experts in [1, 512]");
  if (a->top_k < 1 || a->top_k > kSelMaxK || a->top_k > a->num_experts)
    return report_error(MOE_B200_ERR_ARG, "select_experts_backward: top_k must be in [1, 32] and at most num_experts");
  if (a->score != MOE_B200_SCORE_SIGMOID && a->score != MOE_B200_SCORE_SOFTMAX)
    return report_error(MOE_B200_ERR_ARG, "select_experts_backward: bad score");
  if (!is_float_type(a->logits_type))
    return report_error(MOE_B200_ERR_ARG, "select_experts_backward: logits are bf16, fp16 or fp32");
  if (a->num_tokens == 0) return MOE_B200_OK;
  if (!a->logits || !a->idx || !a->dweight || !a->dlogits) return report_error(MOE_B200_ERR_ARG, "null tensor pointer");
  int sms = 0;
  if (int rc = op_device(&sms)) return rc;
  SelectBwdArgs s{};
  s.logits = a->logits;
  s.idx = a->idx;
  s.dw = a->dweight;
  s.dlogits = a->dlogits;
  s.ld = a->logits_stride;
  s.dld = a->dlogits_stride;
  s.T = a->num_tokens;
  s.E = a->num_experts;
  s.K = a->top_k;
  s.type = a->logits_type;
  s.renorm = a->renormalize;
  s.scale = a->scale;
  const int bytes = 4 * type_bytes(s.type);
  s.vec = reinterpret_cast<uintptr_t>(s.logits) % bytes == 0 && (s.T == 1 || s.ld % 4 == 0);
  s.dvec = reinterpret_cast<uintptr_t>(s.dlogits) % bytes == 0 && (s.T == 1 || s.dld % 4 == 0);
  cudaError_t e = cudaSuccess;
  const dim3 grid(select_grid(s.T, sms)), block(kSelWarps * 32);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  dispatch_select(s.E, [&](auto v) {
    constexpr int V = decltype(v)::value;
    e = a->score == MOE_B200_SCORE_SOFTMAX ? launch_pdl(select_bwd_kernel<V, true>, grid, block, 0, st, s)
                                           : launch_pdl(select_bwd_kernel<V, false>, grid, block, 0, st, s);
  });
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "select_experts_backward launch");
}

}  // extern "C"
