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
// One warp per token; lane l holds experts l, l + 32, ...
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
  float scale;
};

struct SelectBwdArgs {
  const void* logits;
  const int* idx;
  const float* dw;
  void* dlogits;
  int64_t ld, dld;
  int T, E, K, type, renorm;
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
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

template <int V, bool SOFTMAX>
__global__ void __launch_bounds__(kSelWarps * 32) select_kernel(SelectArgs a) {
  extern __shared__ float s_dyn[];   // [warps][E] sel of a token (groups only), then [E] counts
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* s_sel = s_dyn + warp * a.E;
  int* s_cnt = reinterpret_cast<int*>(s_dyn + (a.n_group > 1 ? kSelWarps * a.E : 0));
  if (a.counts) {
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) s_cnt[e] = 0;
    __syncthreads();
  }
  const float lowest = lowest_of(a.type);
  const int gs = a.E / a.n_group;
  float bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    bias[i] = a.bias && e < a.E ? load1_dyn(a.bias, a.bias_type, e) : 0.f;
  }
  for (int t = blockIdx.x * kSelWarps + warp; t < a.T; t += gridDim.x * kSelWarps) {
    float x[V], s[V], sel[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * 32 + lane;
      x[i] = e < a.E ? load1_dyn(a.logits, a.type, t * a.ld + e) : -INFINITY;
    }
    if constexpr (SOFTMAX) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[i] <= lowest ? -INFINITY : x[i]);
      m = warp_max(m);
      double ex[V], sum = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = static_cast<double>(x[i]) - static_cast<double>(m);
        ex[i] = x[i] <= lowest ? 0.0 : d != d ? d : d < -700.0 ? 0.0 : exp_series(d);
        sum += ex[i];
      }
      sum = warp_sum_d(sum);
      const double inv = 1.0 / sum;
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = x[i] <= lowest ? 0.f : static_cast<float>(ex[i] * inv);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        s[i] = x[i] <= lowest ? 0.f : __frcp_rn(1.0f + exp_to_f32(-static_cast<double>(x[i])));
    }
    bool bad = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sel[i] = x[i] <= lowest ? -INFINITY : s[i] + bias[i];
      bad |= sel[i] != sel[i];
    }
    bad = __any_sync(0xffffffffu, bad);
    if (a.n_group > 1) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i * 32 + lane < a.E) s_sel[i * 32 + lane] = sel[i];
      __syncwarp();
      float m1 = -INFINITY, m2 = -INFINITY;
      if (lane < a.n_group)
        for (int j = 0; j < gs; ++j) {
          const float v = s_sel[lane * gs + j];
          m2 = fmaxf(m2, fminf(m1, v));
          m1 = fmaxf(m1, v);
        }
      const float score = a.top2 ? m1 + (m2 == -INFINITY ? 0.f : m2) : m1;
      int rank = 0;
      for (int h = 0; h < a.n_group; ++h) {
        const float o = __shfl_sync(0xffffffffu, score, h);
        rank += (o > score || (o == score && h < lane)) ? 1 : 0;
      }
      const uint32_t kept = __ballot_sync(0xffffffffu, lane < a.n_group && rank < a.topk_group);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = i * 32 + lane;
        if (e < a.E && !((kept >> (e / gs)) & 1u)) sel[i] = -INFINITY;
      }
      __syncwarp();
    }
    // key 0: not to be chosen (order_key(-inf) is above it, so -inf is mapped here)
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = bad || sel[i] == -INFINITY ? 0u : order_key(sel[i]);
    uint32_t taken = 0;
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
      const uint32_t e = __reduce_min_sync(0xffffffffu, best == m ? static_cast<uint32_t>(at * 32 + lane) : ~0u);
      if ((e & 31u) == static_cast<uint32_t>(lane)) {
        taken |= 1u << (e >> 5);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == static_cast<int>(e >> 5)) key[i] = 0;
      }
    }
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if ((taken >> i) & 1u) part += s[i];
    const float denom = warp_sum(part) + 1e-20f;
    int pos = 0;
    const int64_t base = static_cast<int64_t>(t) * a.K;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool mine = (taken >> i) & 1u;
      const uint32_t b = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        const int p = pos + __popc(b & ((1u << lane) - 1u));
        a.idx[base + p] = i * 32 + lane;
        a.w[base + p] = (a.renorm ? s[i] / denom : s[i]) * a.scale;
        if (a.counts) atomicAdd(s_cnt + i * 32 + lane, 1);
      }
      pos += __popc(b);
    }
    if (lane >= pos && lane < a.K) {
      a.idx[base + lane] = -1;
      a.w[base + lane] = bad ? __uint_as_float(0x7fc00000u) : 0.f;
    }
  }
  if (a.counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x)
      if (s_cnt[e]) atomicAdd(a.counts + e, s_cnt[e]);   // integers: the order does not matter
  }
}

// dlogits of a token, from the gradients dw of its chosen weights (ids distinct, -1: no expert).
//   renormalised, S = sum of the chosen s + 1e-20:  ds_k = scale * (dw_k - sum_j dw_j s_j / S) / S
//   softmax: dx_e = s_e (ds_e - sum_j ds_j s_j);  sigmoid: dx_e = ds_e s_e (1 - s_e)
template <int V, bool SOFTMAX>
__global__ void __launch_bounds__(kSelWarps * 32) select_bwd_kernel(SelectBwdArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float lowest = lowest_of(a.type);
  for (int t = blockIdx.x * kSelWarps + warp; t < a.T; t += gridDim.x * kSelWarps) {
    float x[V], s[V], d[V] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * 32 + lane;
      x[i] = e < a.E ? load1_dyn(a.logits, a.type, t * a.ld + e) : -INFINITY;
    }
    const int64_t base = static_cast<int64_t>(t) * a.K;
    const int my_id = lane < a.K ? a.idx[base + lane] : -1;
    const float my_dw = lane < a.K ? a.dw[base + lane] * a.scale : 0.f;
    if constexpr (SOFTMAX) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[i] <= lowest ? -INFINITY : x[i]);
      m = warp_max(m);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] = x[i] <= lowest ? 0.f : expf(x[i] - m);
        sum += s[i];
      }
      const float inv = 1.f / fmaxf(warp_sum(sum), 1e-30f);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = x[i] <= lowest ? 0.f : 1.f / (1.f + expf(-x[i]));
    }
    bool bad = false;
#pragma unroll
    for (int i = 0; i < V; ++i) bad |= x[i] != x[i] || s[i] != s[i];
    bad = __any_sync(0xffffffffu, bad);
    uint32_t taken = 0;
    for (int k = 0; k < a.K; ++k) {
      const int id = __shfl_sync(0xffffffffu, my_id, k);
      const float dw = __shfl_sync(0xffffffffu, my_dw, k);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (id == i * 32 + lane) {
          d[i] = dw;
          taken |= 1u << i;
        }
    }
    float chosen = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if ((taken >> i) & 1u) chosen += s[i];
      dot += d[i] * s[i];
    }
    if (a.renorm) {
      const float S = warp_sum(chosen) + 1e-20f;
      const float mean = warp_sum(dot) / S;
      dot = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = (taken >> i) & 1u ? (d[i] - mean) / S : 0.f;
        dot += d[i] * s[i];
      }
    }
    if constexpr (SOFTMAX) {
      dot = warp_sum(dot);
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = s[i] * (d[i] - dot);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] *= s[i] * (1.f - s[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * 32 + lane;
      if (e >= a.E) continue;
      const float v = bad ? __uint_as_float(0x7fc00000u) : d[i];
      const int64_t o = t * a.dld + e;
      if (a.type == MOE_B200_BF16) static_cast<bf16*>(a.dlogits)[o] = from_f<bf16>(v);
      else if (a.type == MOE_B200_FP16) static_cast<fp16*>(a.dlogits)[o] = from_f<fp16>(v);
      else static_cast<float*>(a.dlogits)[o] = v;
    }
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
  if (a->num_tokens < 0 || a->num_experts < 1 || a->num_experts > kSelMaxE)
    return report_error(MOE_B200_ERR_ARG, "select_experts: num_tokens must be >= 0 and num_experts in [1, 512]");
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
  if (a->counts) {
    e = cudaMemsetAsync(a->counts, 0, sizeof(int) * a->num_experts, st);
    if (e != cudaSuccess) return report_cuda(e, "cudaMemsetAsync");
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
  const size_t smem = ((s.n_group > 1 ? kSelWarps * s.E : 0) + (s.counts ? s.E : 0)) * sizeof(float);
  const dim3 grid(select_grid(s.T, sms)), block(kSelWarps * 32);
  dispatch_select(s.E, [&](auto v) {
    constexpr int V = decltype(v)::value;
    e = a->score == MOE_B200_SCORE_SOFTMAX ? launch_pdl(select_kernel<V, true>, grid, block, smem, st, s)
                                           : launch_pdl(select_kernel<V, false>, grid, block, smem, st, s);
  });
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "select_experts launch");
}

MOE_B200_API int moe_b200_select_experts_backward(const moe_b200_select_backward_args* a, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->num_tokens < 0 || a->num_experts < 1 || a->num_experts > kSelMaxE)
    return report_error(MOE_B200_ERR_ARG, "select_experts_backward: num_tokens must be >= 0 and num_experts in [1, 512]");
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
