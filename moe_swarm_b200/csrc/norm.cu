// The norms around a block, fused with its gate and residual sum (forward).
//
//   n  = y                                  or, with post_weight,  y * s(y) * (post_weight + off)
//   r' = residual + scale * gate * n                               (stored in the residual's type)
//   x  = r' * s(r') * (pre_weight + off)                           (bf16, fp16, fp32 or e4m3 blocks)
//   s(v) = 1 / sqrt(mean(v^2) + eps)
//
// gate is broadcast over rows, over columns or over neither.  x is computed from the unrounded
// 32-bit r'.  In e4m3, x is quantised per row and 128 columns, scale = max(amax, 1e-12) / 448,
// which is the expert layer's hidden_states / hidden_states_scale pair.
//
// One row is held in the registers of a group of warps (16 elements per thread), so each tensor
// crosses HBM once; all sums are 32-bit in a fixed order.
#include "norm_common.cuh"

namespace moe {

struct NormArgs {
  const void *y, *residual, *post_w, *pre_w, *gate;
  void *residual_out, *x;
  float* x_scale;
  int64_t y_ld, r_ld, ro_ld, x_ld, g_ld;
  int rows, cols, warps;
  int post_type, pre_type, gate_type, gate_cols, x_type;   // gate_cols: the gate varies along a row
  float scale, eps, off;
};

// e4m3 codes are those of the 32-bit quotients v / scale.  v times the scale's rounded reciprocal alone falls
// on the other side of some rounding boundaries (of 235 million codes 1920 differ from those of 64-bit
// arithmetic throughout, of the quotients' 1839), so the product is corrected once by its exact remainder,
// which gives the rounded quotient (Markstein, Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990): 4096 x 7168 36.3 us against 35.2 without.  An infinite scale takes no
// remainder: what is finite becomes 0, an infinity NaN.
struct BlockScale {
  float inv, minus;   // reciprocal, negative divisor
};
__device__ __forceinline__ BlockScale block_scale(float sc) {
  return {__frcp_rn(sc), isinf(sc) ? 0.f : -sc};
}
// max(m, 1e-12) / 448, rounded (every mantissa checked against the division), and infinities and NaN as they are.
__device__ __forceinline__ float scale_of_block(float m) {
  m = max_nan(m, 1e-12f);
  const float p = m * (1.f / 448.f);
  return m < INFINITY ? fmaf(fmaf(p, -448.f, m), 1.f / 448.f, p) : m;
}
__device__ __forceinline__ float2 quotient2(float2 v, BlockScale s) {
  const float2 inv = dup2(s.inv), p = mul2(v, inv);
  return fma2(fma2(p, dup2(s.minus), v), inv, p);
}

// x = r * rstd * w of this thread's elements, stored in the type asked for.  Whole warps call it
// (kPacked, which has no e4m3, aside): a 128-column block's maximum is a shuffle over its half warp (eight
// elements each, two blocks in a thread) or warp (four each, four blocks).
template <int LAY>
__device__ __forceinline__ void store_x(const NormArgs& a, int row, int cols, Row16& r, const Row16& w, float rstd) {
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = mul2(mul2(r.v[i], dup2(rstd)), w.v[i]);
  if (a.x_type != MOE_B200_E4M3) {
    store_row_dyn<LAY>(a.x, a.x_type, row * a.x_ld, cols, r);
    return;
  }
  uint8_t* dst = static_cast<uint8_t*>(a.x) + row * a.x_ld;
  if constexpr (!is_vec(LAY)) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      float m = 0.f;
#pragma unroll
      for (int j = i; j < i + 4; ++j)
        if (exists<LAY>(j, cols)) m = max_nan(m, fabsf(r[j]));
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float sc = scale_of_block(m);
      const BlockScale by = block_scale(sc);
      const int e0 = col_of<LAY>(i) & ~127;
      if ((threadIdx.x & 31) == 0 && e0 < cols) a.x_scale[static_cast<int64_t>(e0 >> 7) * a.rows + row] = sc;
#pragma unroll
      for (int j = i; j < i + 4; j += 2) {
        const float2 q = quotient2(r.v[j >> 1], by);
        if (exists<LAY>(j, cols)) dst[col_of<LAY>(j)] = static_cast<uint8_t>(cvt_e4m3x2(q.x, 0.f));
        if (exists<LAY>(j + 1, cols)) dst[col_of<LAY>(j + 1)] = static_cast<uint8_t>(cvt_e4m3x2(q.y, 0.f));
      }
    }
  } else {
    float m[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = fabsf(r[8 * i]);
#pragma unroll
      for (int j = 1; j < 8; ++j) m[i] = max_nan(m[i], fabsf(r[8 * i + j]));
      if (!exists<LAY>(8 * i, cols)) m[i] = 0.f;
    }
    // both maxima in one butterfly: the lower eight lanes of a half warp go on with the first
    // block's, the upper with the second's
    const bool upper = threadIdx.x & 8;
    const float mine = upper ? m[1] : m[0];
    float v = max_nan(mine, __shfl_xor_sync(0xffffffffu, upper ? m[0] : m[1], 8));
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
    const float sc = scale_of_block(v);
    const BlockScale mine_by = block_scale(sc);
    const BlockScale other_by = {__shfl_xor_sync(0xffffffffu, mine_by.inv, 8), __shfl_xor_sync(0xffffffffu, mine_by.minus, 8)};
    const int block = col_of<LAY>(upper ? 8 : 0) >> 7;   // lane 0 or 8 of the half warp writes it
    if ((threadIdx.x & 7) == 0 && block * 128 < cols) a.x_scale[static_cast<int64_t>(block) * a.rows + row] = sc;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const BlockScale by = (i == 1) == upper ? mine_by : other_by;
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 p = quotient2(r.v[4 * i + j], by);
        q[j] = cvt_e4m3x2(p.x, p.y);
      }
      if (exists<LAY>(8 * i, cols))
        *reinterpret_cast<uint2*>(dst + col_of<LAY>(8 * i)) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
    }
  }
}

// One row per group of warps.  blockDim = (32 * warps, rows per CTA), or less than a warp per row
// (kPacked).  Rows beyond the last are the last one again, without a store: what a layout promises of
// its elements (exists()) holds for rows that exist only.  Bound by latency where rows are few (one row
// of 7168: 2.6 us), by HBM where many: 592 rows 6.4 us, 16384 x 512 11.6 us (5.8 TB/s), 901 x 5001
// with both norms and a 32-bit residual 15.4 to 16.9 us (3.2 to 3.5 TB/s: odd rows are read and written two
// bytes at a time, and their threads spill).  Beyond 8192 columns, where no ring is: 2048 x 16384 60.0 us to
// 16 bits (4.5 TB/s), 61.6 to e4m3, 74.4 with a 32-bit residual (5.4).
template <class YT, class RT, int LAY, int MAXT>
__global__ void __launch_bounds__(MAXT, 1024 / MAXT) norm_fwd_kernel(NormArgs a) {
  __shared__ float buf[2][8 * 32];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int cols = a.cols;
  const bool live = row < a.rows;
  const int from = min(row, a.rows - 1);   // a row that exists
  Row16 r, w;
  if (a.residual) {
    load_row<RT, LAY>(static_cast<const RT*>(a.residual) + from * a.r_ld, cols, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = dup2(0.f);
  }
  if (a.y) {
    Row16 y;
    load_row<YT, LAY>(static_cast<const YT*>(a.y) + from * a.y_ld, cols, y);
    float k = a.scale;
    if (a.post_w) {
      load_weight<LAY>(a.post_w, a.post_type, a.off, cols, w);
      float ss[1] = {dot16<LAY>(y, y)};
      if constexpr (LAY == kPacked) packed_sum(ss);
      else row_sum(ss, a.warps, buf[0]);
      k *= rsqrtf(ss[0] / a.cols + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] = mul2(y.v[i], w.v[i]);
    }
    if (a.gate && a.gate_cols) {
      load_row_dyn<LAY>(a.gate, a.gate_type, from * a.g_ld, cols, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] = mul2(y.v[i], w.v[i]);
    } else if (a.gate) {
      k *= load1_dyn(a.gate, a.gate_type, from * a.g_ld);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = fma2(dup2(k), y.v[i], r.v[i]);
    if (a.residual_out && live) store_row<RT, LAY>(static_cast<RT*>(a.residual_out) + row * a.ro_ld, cols, r);
  }
  if (!a.pre_w) return;
  load_weight<LAY>(a.pre_w, a.pre_type, a.off, cols, w);
  float ss[1] = {squares_existing<LAY>(r, cols)};
  if constexpr (LAY == kPacked) packed_sum(ss);
  else row_sum(ss, a.warps, buf[1]);
  if (live) store_x<LAY>(a, row, cols, r, w, rsqrtf(ss[0] / a.cols + a.eps));   // (the same in all of a warp but kPacked's)
}

// Many rows: persistent CTAs, whose next rows (y, residual, gate per element) are on their way
// to shared memory as bulk copies while a row is computed, so that the row's barriers and latencies
// leave the memory busy.  Weights and a gate per column come from L1.  A stage is refilled after
// the row's last barrier, when every thread holds its part.  1024 threads of an SM, whose rows in flight
// are about 200 KB; 4096 x 7168 from bf16 to e4m3 36.3 us (5.7 TB/s, HBM), to bf16 40.3, with both
// norms and a gate per element 54 (5.4 TB/s).
// POST: 0, 1: without and with post_weight; kNoBlock: there is no y.
constexpr int kNoBlock = 2;
template <class YT, class RT, int POST, int LAY>
__global__ void __launch_bounds__(512, 2) norm_ring_kernel(NormArgs a, RingPlan g) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float buf[3][32];   // sums of y^2; of r'^2 of even and odd rows
  __shared__ uint64_t full[kRingMaxStages];
  __shared__ int abort;
  if (threadIdx.x == 0) {
    abort = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int step = gridDim.x, cols = a.cols;
  if (threadIdx.x == 0)
    for (int i = 0; i < g.stages; ++i) {
      const int64_t row = blockIdx.x + static_cast<int64_t>(i) * step;
      if (row < a.rows) ring_fetch(g, static_cast<int>(row), ring + i * g.stage_bytes, &full[i]);
    }
  const bool g_element = a.gate && a.gate_cols && a.g_ld;   // the ring's last tensor
  const float inv_cols = 1.f / cols;
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  bool ok = true;
  float g_next = a.gate && !a.gate_cols ? load1_dyn(a.gate, a.gate_type, blockIdx.x * a.g_ld) : 0.f;
  for (int row = blockIdx.x; row < a.rows; row += step) {
    // after a wait that ran out the CTA still goes through its rows, without their contents
    if (ok) ok = mbar_wait(&full[stage], phase, &abort, &g_op_status, kStWaitProducer);
    uint8_t* src = ring + stage * g.stage_bytes;
    Row16 r, w;
    if constexpr (POST == kNoBlock) {
      load_row<RT, LAY>(reinterpret_cast<const RT*>(src + g.t[0].at), cols, r);
    } else {
      Row16 y;
      load_row<YT, LAY>(reinterpret_cast<const YT*>(src + g.t[0].at), cols, y);
      if (a.residual) {
        load_row<RT, LAY>(reinterpret_cast<const RT*>(src + g.t[1].at), cols, r);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = dup2(0.f);
      }
      float k = a.scale;
      if constexpr (POST == 1) {
        load_weight<LAY>(a.post_w, a.post_type, a.off, cols, w);
        float ss[1] = {dot16<LAY>(y, y)};
        row_sum(ss, a.warps, buf[0]);
        k *= rsqrtf(ss[0] * inv_cols + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) y.v[i] = mul2(y.v[i], w.v[i]);
      }
      if (a.gate && !a.gate_cols) {
        k *= g_next;   // loaded a row ahead
        if (row + static_cast<int64_t>(step) < a.rows) g_next = load1_dyn(a.gate, a.gate_type, (row + step) * a.g_ld);
      } else if (a.gate) {
        load_row_dyn<LAY>(g_element ? static_cast<const void*>(src + g.t[a.residual ? 2 : 1].at) : a.gate, a.gate_type, 0, cols, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) y.v[i] = mul2(y.v[i], w.v[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = fma2(dup2(k), y.v[i], r.v[i]);
      store_row<RT, LAY>(static_cast<RT*>(a.residual_out) + row * a.ro_ld, cols, r);
    }
    float ss[1] = {squares_existing<LAY>(r, cols)};
    if (a.pre_w) load_weight<LAY>(a.pre_w, a.pre_type, a.off, cols, w);
    row_sum(ss, a.warps, buf[1 + parity]);
    parity ^= 1;
    // every thread has its part of the stage (row_sum's barrier)
    const int64_t next = row + static_cast<int64_t>(g.stages) * step;
    if (threadIdx.x == 0 && ok && next < a.rows) ring_fetch(g, static_cast<int>(next), src, &full[stage]);
    if (ok && ++stage == g.stages) {
      stage = 0;
      phase ^= 1u;
    }
    if (a.pre_w) store_x<LAY>(a, row, cols, r, w, rsqrtf(ss[0] * inv_cols + a.eps));
  }
  if (!ok && threadIdx.x == 0)   // given up: the loads in flight land first
    for (int i = 0; i < g.stages; ++i) {
      int none = 0;
      if (blockIdx.x + static_cast<int64_t>(i) * step < a.rows)
        mbar_wait(&full[i], i >= stage ? phase : phase ^ 1u, &none, &g_op_status, kStWaitDrain);
    }
}

cudaError_t norm_status(cudaStream_t st, bool clear, int* v) {
  int f = 0, b = 0;
  cudaError_t e = take_status(st, clear, &f);
  if (e == cudaSuccess) e = norm_bwd_status(st, clear, &b);
  *v = f ? f : b;
  return e;
}

}  // namespace moe

extern "C" {

MOE_B200_API int moe_b200_block_norm(const moe_b200_norm_args* a, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->rows < 0 || a->rows > kOpMaxRows || a->cols < 1 || a->cols > kNormMaxCols)
    return report_error(MOE_B200_ERR_ARG, "block_norm: rows must be in [0, 2^30] and cols in [1, 16384]");
  if (!type_pair_ok(a->y_type, a->residual_type))
    return report_error(MOE_B200_ERR_ARG, "block_norm: with a y of fp32 the residual is fp32 too (types bf16, fp16, fp32)");
  if (a->rows == 0) return MOE_B200_OK;
  if (!a->y && !a->residual) return report_error(MOE_B200_ERR_ARG, "block_norm: y or residual is required");
  if (a->y && !a->residual_out) return report_error(MOE_B200_ERR_ARG, "block_norm: residual_out is required with y");
  if (!a->y && (a->post_weight || a->gate || !a->pre_weight))
    return report_error(MOE_B200_ERR_ARG, "block_norm: without y only the norm of the residual can be asked for");
  if (a->pre_weight && !a->x) return report_error(MOE_B200_ERR_ARG, "block_norm: x is required with pre_weight");
  if (a->pre_weight && !is_float_type(a->x_type) && a->x_type != MOE_B200_E4M3)
    return report_error(MOE_B200_ERR_ARG, "block_norm: bad x type");
  if (a->pre_weight && a->x_type == MOE_B200_E4M3 && !a->x_scale)
    return report_error(MOE_B200_ERR_ARG, "block_norm: x_scale is required for an e4m3 x");
  if ((a->pre_weight && !is_float_type(a->pre_weight_type)) || (a->post_weight && !is_float_type(a->post_weight_type)) ||
      (a->gate && !is_float_type(a->gate_type)))
    return report_error(MOE_B200_ERR_ARG, "block_norm: weights and gate are bf16, fp16 or fp32");
  int sms = 0;
  if (int rc = op_device(&sms)) return rc;
  NormArgs n{};
  n.y = a->y;
  n.residual = a->residual;
  n.post_w = a->post_weight;
  n.pre_w = a->pre_weight;
  n.gate = a->gate;
  n.residual_out = a->residual_out;
  n.x = a->x;
  n.x_scale = a->x_scale;
  n.y_ld = a->y_stride;
  n.r_ld = a->residual_stride;
  n.ro_ld = a->residual_out_stride;
  n.x_ld = a->x_stride;
  n.g_ld = a->gate_row_stride;
  if (a->rows == 1) n.y_ld = n.r_ld = n.ro_ld = n.x_ld = n.g_ld = 0;   // a single row has no pitch
  n.rows = a->rows;
  n.cols = a->cols;
  n.post_type = a->post_weight_type;
  n.pre_type = a->pre_weight_type;
  n.gate_type = a->gate_type;
  n.gate_cols = a->gate_per_column;
  n.x_type = a->x_type;
  n.scale = a->scale;
  n.eps = a->eps;
  n.off = a->weight_offset;
  int rpc;
  norm_shape(a->cols, &n.warps, &rpc);
  // whole 16-byte accesses need every row of every tensor on a 16-byte boundary (8 for e4m3)
  const bool vec = a->cols % 8 == 0 && rows_aligned(a->y, n.y_ld, a->y_type) &&
                   rows_aligned(a->residual, n.r_ld, a->residual_type) &&
                   rows_aligned(a->residual_out, n.ro_ld, a->residual_type) && aligned16(a->post_weight) &&
                   aligned16(a->pre_weight) &&
                   (!a->gate_per_column || rows_aligned(a->gate, n.g_ld, a->gate_type)) &&
                   (a->x_type == MOE_B200_E4M3 ? (reinterpret_cast<uintptr_t>(a->x) & 7u) == 0 && n.x_ld % 8 == 0
                                               : rows_aligned(a->x, n.x_ld, a->x_type));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  // Rows of up to 256 columns: several to a warp (65536 x 128: 11.7 us, 5.7 TB/s, against 31.5 with
  // one).  An e4m3 block's maximum wants a half warp.
  const bool packed = vec && a->cols <= 256 && !(a->pre_weight && a->x_type == MOE_B200_E4M3);
  // The ring: aligned rows of two warps or more, at least four per SM, and two or more of them in
  // a CTA's share of shared memory.  7168 columns, bf16 in, e4m3 out, ring against direct: 592 rows
  // 6.0 us against 6.4, 4096 rows 36.3 (5.7 TB/s) against 51.9; at 148 and 296 rows the ring is 0.1
  // to 0.2 us behind.  The norm alone of 4096 x 7168 in 16 bits: 24.8 us against 33.7.
  // A 32-bit residual with nothing but the sum and its norm to compute has wide loads that keep the memory
  // busy without a ring.  In us, ring against direct:
  //   sum without a norm: direct (4096 x 7168 49.9 against 43.6; 1184 rows 13.2 against 13.4)
  //   norm without a sum: the ring from 13 warps on (4096 x 7168 30.0 against 33.4, 4096 x 2048 10.4 against 9.2)
  //   both, up to 8 warps: the ring while no CTA has two rows (1184 x 2048 4.9 against 5.3, 2368 x 2048 10.3
  //     against 10.0, 8192 x 2048 35.4 against 31.8)
  //   both, longer rows: the ring below 2^24 elements (1184 x 7168 16.5 against 18.3, 4096 x 7168 63.2 against
  //     55.7), and with 13 warps beyond that for an x of another width than 16 bits (to e4m3 54.6 against 57.1)
  RingPlan g{};
  ring_add(&g, a->y, n.y_ld, a->cols, a->y_type);
  ring_add(&g, a->residual, n.r_ld, a->cols, a->residual_type);
  if (a->gate_per_column && n.g_ld) ring_add(&g, a->gate, n.g_ld, a->cols, a->gate_type);
  const int ctas = n.warps >= 2 && n.warps <= 16 ? 32 / n.warps : 0;   // 1024 threads of an SM
  g.stages = ctas ? kRingSmem / ctas / g.stage_bytes : 0;
  if (g.stages > kRingMaxStages) g.stages = kRingMaxStages;
  bool direct = false;
  if (a->residual_type == MOE_B200_FP32 && !a->post_weight && !a->gate) {
    const bool large = static_cast<int64_t>(a->rows) * a->cols >= 1 << 24, wide = n.warps > 12;
    const bool x16 = a->x_type == MOE_B200_BF16 || a->x_type == MOE_B200_FP16;
    direct = !a->pre_weight    ? true
             : !a->y           ? !wide
             : n.warps <= 8    ? a->rows > ctas * sms
                               : large && (x16 || !wide);
  }
  if (vec && !packed && a->rows >= 4 * sms && g.stages >= 2 && !direct) {
    const dim3 grid(a->rows < ctas * sms ? a->rows : ctas * sms), block(n.warps * 32);
    const size_t smem = static_cast<size_t>(g.stages) * g.stage_bytes;
    dispatch_types(a->y_type, a->residual_type, [&](auto yt, auto rt) {
      using YT = decltype(yt);
      using RT = decltype(rt);
      auto laid = [&](auto post) {
        constexpr int P = decltype(post)::value;
        return a->cols == n.warps * 32 * kNormPerThread ? norm_ring_kernel<YT, RT, P, kFull>
                                                        : norm_ring_kernel<YT, RT, P, kHalf>;
      };
      auto kernel = !a->y            ? laid(std::integral_constant<int, kNoBlock>{})
                    : a->post_weight ? laid(std::integral_constant<int, 1>{})
                                     : laid(std::integral_constant<int, 0>{});
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
      if (e == cudaSuccess) e = launch_pdl(kernel, grid, block, smem, st, n, g);
    });
    return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "block_norm launch");
  }
  const int lanes = packed ? packed_lanes(a->cols) : n.warps * 32;
  if (packed) rpc = 256 / lanes;
  const dim3 block(lanes, rpc), grid((a->rows + rpc - 1) / rpc);
  dispatch_types(a->y_type, a->residual_type, [&](auto yt, auto rt) {
    using YT = decltype(yt);
    using RT = decltype(rt);
    // rows of up to 8192 columns take at most 512 threads, so that two CTAs fit an SM; a thread has 64 registers
    // either way, which odd rows exceed by some (kTail and kScattered spill 108 and 80 bytes).  Odd rows of up
    // to 256 columns have no loads for elements that they do not hold (30000 x 99: 10.4 us against 33.8)
    auto sized = [&](auto t) {
      constexpr int MAXT = decltype(t)::value;
      if constexpr (MAXT == 1024) return vec ? norm_fwd_kernel<YT, RT, kVec, MAXT> : norm_fwd_kernel<YT, RT, kTail, MAXT>;
      else
        return packed                     ? norm_fwd_kernel<YT, RT, kPacked, MAXT>
               : vec                      ? norm_fwd_kernel<YT, RT, kVec, MAXT>
               : a->cols <= 128           ? norm_fwd_kernel<YT, RT, kShort, MAXT>
               : a->cols <= 256           ? norm_fwd_kernel<YT, RT, kThin, MAXT>
               : a->cols >= 384 * n.warps ? norm_fwd_kernel<YT, RT, kTail, MAXT>
                                          : norm_fwd_kernel<YT, RT, kScattered, MAXT>;
    };
    auto kernel = block.x * block.y <= 512 ? sized(std::integral_constant<int, 512>{})
                                           : sized(std::integral_constant<int, 1024>{});
    e = launch_pdl(kernel, grid, block, 0, st, n);
  });
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "block_norm launch");
}

}  // extern "C"
