// The norms around a block, fused with its gate and residual sum, forward and backward.
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
#include <type_traits>

#include "op_common.cuh"

namespace moe {

constexpr int kNormPerThread = 16;            // two 8-element chunks
constexpr int kNormMaxCols = 1024 * kNormPerThread;

struct NormArgs {
  const void *y, *residual, *post_w, *pre_w, *gate;
  void *residual_out, *x;
  float* x_scale;
  int64_t y_ld, r_ld, ro_ld, x_ld, g_ld;
  int rows, cols, warps;
  int post_type, pre_type, gate_type, gate_cols, x_type;   // gate_cols: the gate varies along a row
  float scale, eps, off;
};

struct NormBwdArgs {
  const void *dx, *dr, *r, *y, *post_w, *pre_w, *gate;
  void *dres, *dy, *dgate;          // dgate: per element (gate type) or per row (fp32); null: none
  float* partial;                   // [n_sums][parts][cols]: pre, post, gate column sums
  int64_t dx_ld, dr_ld, r_ld, y_ld, g_ld, dres_ld, dy_ld, dg_ld;
  int rows, cols, warps, parts;
  int post_type, pre_type, gate_type, gate_cols;
  int gate_grad;                    // 0 none, 1 per column, 2 per row, 3 per element
  int post_slot, gate_slot;         // index of that column sum in `partial`
  float scale, eps, off;
};

template <bool VEC>
__device__ __forceinline__ void load_gate(const void* g, int type, int cols_vary, int64_t row_off, int e0, int n,
                                          float* v) {
  if (!g) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 1.f;
  } else if (cols_vary) {
    load8_dyn<VEC>(g, type, row_off + e0, n, v);
  } else {
    const float s = n > 0 ? load1_dyn(g, type, row_off) : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s;
  }
}

// x = r * rstd * w of this thread's two chunks (w already holds pre_weight + off), stored in the
// type asked for.  Whole half warps call it: a 128-column block is the 16 chunks of one.
template <bool VEC>
__device__ __forceinline__ void store_x(const NormArgs& a, int row, const int* e0, const int* n, float (&r)[2][8],
                                        const float (&w)[2][8], float rstd) {
#pragma unroll
  for (int j = 0; j < 16; ++j) r[j >> 3][j & 7] *= rstd * w[j >> 3][j & 7];
  if (a.x_type != MOE_B200_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) store8_dyn<VEC>(a.x, a.x_type, row * a.x_ld + e0[i], n[i], r[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n[i]) m = max_nan(m, fabsf(r[i][j]));
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float sc = max_nan(m, 1e-12f) / 448.f;
    const float inv = 1.f / sc;
    if (n[i] <= 0) continue;
    if ((threadIdx.x & 15) == 0) a.x_scale[static_cast<int64_t>(e0[i] >> 7) * a.rows + row] = sc;
    uint8_t* dst = static_cast<uint8_t*>(a.x) + row * a.x_ld + e0[i];
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = cvt_e4m3x2(r[i][2 * j] * inv, r[i][2 * j + 1] * inv);
    if constexpr (VEC) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n[i]) dst[j] = static_cast<uint8_t>(q[j >> 1] >> (8 * (j & 1)));
    }
  }
}

// One row per group of warps.  blockDim = (32 * warps, rows per CTA); a thread holds chunks
// threadIdx.x and threadIdx.x + blockDim.x of its row.  Rows beyond the last run with no elements.
template <class YT, class RT, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) norm_fwd_kernel(NormArgs a) {
  __shared__ float buf[2][8 * 32];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int cols = row < a.rows ? a.cols : 0;
  float r[2][8], w[2][8];
  int n[2], e0[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e0[i] = (threadIdx.x + i * blockDim.x) * 8;
    n[i] = min(8, cols - e0[i]);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < 2; ++i) load8<RT, VEC>(static_cast<const RT*>(a.residual) + row * a.r_ld + e0[i], n[i], r[i]);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j >> 3][j & 7] = 0.f;
  }
  if (a.y) {
    float y[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i) load8<YT, VEC>(static_cast<const YT*>(a.y) + row * a.y_ld + e0[i], n[i], y[i]);
    if (a.post_w) {
#pragma unroll
      for (int i = 0; i < 2; ++i) load8_dyn<VEC>(a.post_w, a.post_type, e0[i], n[i], w[i]);
      float ss[1] = {0.f};
#pragma unroll
      for (int j = 0; j < 16; ++j) ss[0] += y[j >> 3][j & 7] * y[j >> 3][j & 7];
      row_sum(ss, a.warps, buf[0]);
      const float rstd = rsqrtf(ss[0] / a.cols + a.eps);
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j >> 3][j & 7] *= rstd * (w[j >> 3][j & 7] + a.off);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float g[8];
      load_gate<VEC>(a.gate, a.gate_type, a.gate_cols, row * a.g_ld, e0[i], n[i], g);
#pragma unroll
      for (int j = 0; j < 8; ++j) r[i][j] += a.scale * (g[j] * y[i][j]);
    }
    if (a.residual_out) {
#pragma unroll
      for (int i = 0; i < 2; ++i) store8<RT, VEC>(static_cast<RT*>(a.residual_out) + row * a.ro_ld + e0[i], n[i], r[i]);
    }
  }
  if (!a.pre_w) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) load8_dyn<VEC>(a.pre_w, a.pre_type, e0[i], n[i], w[i]);
  float ss[1] = {0.f};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    ss[0] += n[j >> 3] > (j & 7) ? r[j >> 3][j & 7] * r[j >> 3][j & 7] : 0.f;
    w[j >> 3][j & 7] += a.off;
  }
  row_sum(ss, a.warps, buf[1]);
  store_x<VEC>(a, row, e0, n, r, w, rsqrtf(ss[0] / a.cols + a.eps));
}

// Many rows: persistent CTAs, whose next rows (y | residual | gate per element) are on their way
// to shared memory as bulk copies while a row is computed, so that the row's barriers and latencies
// leave the memory busy.  Row tensors are 16-byte aligned; weights and a gate per column come
// from L1.  A stage is refilled after the row's first barrier, when every thread holds its part.
struct RingArgs {
  int stages, y_bytes, r_bytes, g_bytes;   // bytes of a row of each tensor in a stage (0: not read)
};
constexpr int kRingMaxStages = 8;
constexpr int kRingSmem = 200 * 1024;   // of an SM, shared by its CTAs

template <class YT, class RT, bool POST>
__global__ void __launch_bounds__(512, 2) norm_ring_kernel(NormArgs a, RingArgs g) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float buf[3][32];   // sums of y^2; of r'^2 of even and odd rows
  __shared__ uint64_t full[kRingMaxStages];
  __shared__ int abort;
  const int stage_bytes = g.y_bytes + g.r_bytes + g.g_bytes;
  if (threadIdx.x == 0) {
    abort = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  auto fetch = [&](int row, int stage) {   // one thread
    uint8_t* dst = ring + stage * stage_bytes;
    mbar_arrive_expect_tx(&full[stage], stage_bytes);
    bulk_load(dst, static_cast<const YT*>(a.y) + row * a.y_ld, g.y_bytes, &full[stage]);
    if (g.r_bytes)
      bulk_load(dst + g.y_bytes, static_cast<const RT*>(a.residual) + row * a.r_ld, g.r_bytes, &full[stage]);
    if (g.g_bytes)
      bulk_load(dst + g.y_bytes + g.r_bytes,
                static_cast<const uint8_t*>(a.gate) + row * a.g_ld * (g.g_bytes / a.cols), g.g_bytes, &full[stage]);
  };
  const int step = gridDim.x;
  if (threadIdx.x == 0)
    for (int i = 0; i < g.stages; ++i) {
      const int64_t row = blockIdx.x + static_cast<int64_t>(i) * step;
      if (row < a.rows) fetch(static_cast<int>(row), i);
    }
  int n[2], e0[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e0[i] = (threadIdx.x + i * blockDim.x) * 8;
    n[i] = min(8, a.cols - e0[i]);
  }
  const float inv_cols = 1.f / a.cols;
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int row = blockIdx.x; row < a.rows; row += step) {
    // after a wait that ran out the CTA still goes through its rows, without their contents
    if (ok) ok = mbar_wait(&full[stage], phase, &abort, &g_op_status, kStWaitProducer);
    const uint8_t* src = ring + stage * stage_bytes;
    float r[2][8], y[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load8<YT, true>(reinterpret_cast<const YT*>(src) + e0[i], n[i], y[i]);
      if (g.r_bytes) load8<RT, true>(reinterpret_cast<const RT*>(src + g.y_bytes) + e0[i], n[i], r[i]);
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[i][j] = 0.f;
      }
    }
    float k = a.scale;
    if (POST) {
      float ss[1] = {0.f};
#pragma unroll
      for (int j = 0; j < 16; ++j) ss[0] += y[j >> 3][j & 7] * y[j >> 3][j & 7];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float pw[8];
        load8_dyn<true>(a.post_w, a.post_type, e0[i], n[i], pw);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[i][j] *= pw[j] + a.off;
      }
      row_sum(ss, a.warps, buf[0]);
      k *= rsqrtf(ss[0] * inv_cols + a.eps);
    }
    if (a.gate && !a.gate_cols) {
      k *= load1_dyn(a.gate, a.gate_type, row * a.g_ld);
    } else if (a.gate) {
      const void* ge = g.g_bytes ? static_cast<const void*>(src + g.y_bytes + g.r_bytes) : a.gate;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[8];
        load8_dyn<true>(ge, a.gate_type, e0[i], n[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[i][j] *= v[j];
      }
    }
    float ss[1] = {0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float p = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[i][j] = fmaf(k, y[i][j], r[i][j]);
        p = fmaf(r[i][j], r[i][j], p);
      }
      if (n[i] > 0) ss[0] += p;   // (k may be infinite)
      store8<RT, true>(static_cast<RT*>(a.residual_out) + row * a.ro_ld + e0[i], n[i], r[i]);
    }
    float w[2][8];
    if (a.pre_w) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load8_dyn<true>(a.pre_w, a.pre_type, e0[i], n[i], w[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] += a.off;
      }
    }
    row_sum(ss, a.warps, buf[1 + parity]);
    parity ^= 1;
    // every thread has its part of the stage (row_sum's barrier)
    const int64_t next = row + static_cast<int64_t>(g.stages) * step;
    if (threadIdx.x == 0 && ok && next < a.rows) fetch(static_cast<int>(next), stage);
    if (ok && ++stage == g.stages) {
      stage = 0;
      phase ^= 1u;
    }
    if (a.pre_w) store_x<true>(a, row, e0, n, r, w, rsqrtf(ss[0] * inv_cols + a.eps));
  }
  if (!ok && threadIdx.x == 0)   // given up: the loads in flight land first
    for (int i = 0; i < g.stages; ++i) {
      int none = 0;
      if (blockIdx.x + static_cast<int64_t>(i) * step < a.rows)
        mbar_wait(&full[i], i >= stage ? phase : phase ^ 1u, &none, &g_op_status, kStWaitDrain);
    }
}

// Persistent over rows; per-column sums stay in registers and go to `partial`, one slice per
// (CTA, row of the CTA), summed in a fixed order by norm_sum_kernel.
template <class YT, class RT, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) norm_bwd_kernel(NormBwdArgs a) {
  __shared__ float buf[2][3 * 8 * 32];
  pdl_wait();
  pdl_launch_dependents();
  float pre[2][8] = {}, post[2][8] = {}, gsum[2][8] = {};
  int parity = 0;
  const float inv_cols = 1.f / a.cols;
  const int step = gridDim.x * blockDim.y;
  for (int row0 = blockIdx.x * blockDim.y; row0 < a.rows; row0 += step) {
    const int row = row0 + threadIdx.y;
    const int cols = row < a.rows ? a.cols : 0;
    float dx[2][8] = {}, r[2][8] = {}, y[2][8] = {}, G[2][8] = {};
    int n[2], e0[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e0[i] = (threadIdx.x + i * blockDim.x) * 8;
      n[i] = min(8, cols - e0[i]);
      if (a.r) load8<RT, VEC>(static_cast<const RT*>(a.r) + row * a.r_ld + e0[i], n[i], r[i]);
      if (a.dr) load8<RT, VEC>(static_cast<const RT*>(a.dr) + row * a.dr_ld + e0[i], n[i], G[i]);
      if (a.dx) load8<YT, VEC>(static_cast<const YT*>(a.dx) + row * a.dx_ld + e0[i], n[i], dx[i]);
      if (a.y) load8<YT, VEC>(static_cast<const YT*>(a.y) + row * a.y_ld + e0[i], n[i], y[i]);
    }
    float s[3] = {0.f, 0.f, 0.f};   // sum r^2, sum w dx r, sum y^2
    float w[2][8];
    if (a.dx) {
#pragma unroll
      for (int i = 0; i < 2; ++i) load8_dyn<VEC>(a.pre_w, a.pre_type, e0[i], n[i], w[i]);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float rv = r[j >> 3][j & 7];
        s[0] += rv * rv;
        w[j >> 3][j & 7] = (w[j >> 3][j & 7] + a.off) * dx[j >> 3][j & 7];
        s[1] += w[j >> 3][j & 7] * rv;
      }
    }
    if (a.y && a.post_w) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[2] += y[j >> 3][j & 7] * y[j >> 3][j & 7];
    }
    row_sum(s, a.warps, buf[parity]);
    parity ^= 1;
    if (a.dx) {
      const float rstd = row < a.rows ? rsqrtf(s[0] * inv_cols + a.eps) : 0.f;
      const float k = s[1] * inv_cols * rstd * rstd;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float rv = r[j >> 3][j & 7];
        pre[j >> 3][j & 7] += dx[j >> 3][j & 7] * (rv * rstd);
        G[j >> 3][j & 7] += rstd * (w[j >> 3][j & 7] - rv * k);
      }
    }
    if (a.dres) {
#pragma unroll
      for (int i = 0; i < 2; ++i) store8<RT, VEC>(static_cast<RT*>(a.dres) + row * a.dres_ld + e0[i], n[i], G[i]);
    }
    if (!a.y) continue;
    const float ystd = row < a.rows ? rsqrtf(s[2] * inv_cols + a.eps) : 0.f;
    float t[2] = {0.f, 0.f};   // sum wp dn y, sum of the row's gate gradient
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float wp[8], g[8];
      if (a.post_w) load8_dyn<VEC>(a.post_w, a.post_type, e0[i], n[i], wp);
      load_gate<VEC>(a.gate, a.gate_type, a.gate_cols, row * a.g_ld, e0[i], n[i], g);
      float dg[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float dn0 = a.scale * G[i][j];
        const float yh = a.post_w ? y[i][j] * ystd : y[i][j];
        const float wv = a.post_w ? wp[j] + a.off : 1.f;
        dg[j] = j < n[i] ? dn0 * (yh * wv) : 0.f;
        const float dn = dn0 * g[j];
        post[i][j] += dn * yh;
        gsum[i][j] += dg[j];
        t[1] += dg[j];
        G[i][j] = wv * dn;
        t[0] += j < n[i] ? G[i][j] * y[i][j] : 0.f;
      }
      if (a.gate_grad == 3) store8_dyn<VEC>(a.dgate, a.gate_type, row * a.dg_ld + e0[i], n[i], dg);
    }
    if (a.post_w || a.gate_grad == 2) {
      row_sum(t, a.warps, buf[parity]);
      parity ^= 1;
      if (a.gate_grad == 2 && threadIdx.x == 0 && row < a.rows) static_cast<float*>(a.dgate)[row] = t[1];
    }
    if (a.dy) {
      if (a.post_w) {
        const float k = t[0] * inv_cols * ystd * ystd;
#pragma unroll
        for (int j = 0; j < 16; ++j) G[j >> 3][j & 7] = ystd * (G[j >> 3][j & 7] - y[j >> 3][j & 7] * k);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) store8<YT, VEC>(static_cast<YT*>(a.dy) + row * a.dy_ld + e0[i], n[i], G[i]);
    }
  }
  const int64_t slice = static_cast<int64_t>(a.parts) * a.cols;
  float* dst = a.partial + (static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y) * a.cols;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e0 = (threadIdx.x + i * blockDim.x) * 8, n = min(8, a.cols - e0);
    if (a.dx) store8<float, VEC>(dst + e0, n, pre[i]);
    if (a.post_slot >= 0) store8<float, VEC>(dst + a.post_slot * slice + e0, n, post[i]);
    if (a.gate_slot >= 0) store8<float, VEC>(dst + a.gate_slot * slice + e0, n, gsum[i]);
  }
}

// out[c] = sum over p of partial[p][c]: 32 columns per CTA, eight warps over the parts, their
// sums added in warp order.  blockIdx.y selects the sum.
struct NormSumArgs {
  const float* partial;
  float* out[3];
  int parts, cols;
};
__global__ void __launch_bounds__(256) norm_sum_kernel(NormSumArgs a) {
  __shared__ float buf[8][32];
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* p = a.partial + static_cast<int64_t>(blockIdx.y) * a.parts * a.cols + c;
  float s = 0.f;
  if (c < a.cols)
    for (int i = threadIdx.y; i < a.parts; i += 8) s += p[static_cast<int64_t>(i) * a.cols];
  buf[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < a.cols) {
#pragma unroll
    for (int w = 1; w < 8; ++w) s += buf[w][threadIdx.x];
    a.out[blockIdx.y][c] = s;
  }
}

// One value from `rows` of them (the gradient of a gate that is one number).
__global__ void __launch_bounds__(1024) norm_total_kernel(const float* v, int rows, float* out) {
  __shared__ float buf[32];
  pdl_wait();
  pdl_launch_dependents();
  float s[1] = {0.f};
  for (int i = threadIdx.x; i < rows; i += 1024) s[0] += v[i];
  row_sum(s, 32, buf);
  if (threadIdx.x == 0) *out = s[0];
}

namespace {

// Warps of a row and rows of a CTA: a row takes as few warps as hold it; short rows share a CTA
// of up to eight warps.
void norm_shape(int cols, int* warps, int* rows_per_cta) {
  *warps = (cols + 32 * kNormPerThread - 1) / (32 * kNormPerThread);
  *rows_per_cta = *warps >= 8 ? 1 : 8 / *warps;
}

int bwd_parts(int rows, int cols) {
  int warps, rpc;
  norm_shape(cols, &warps, &rpc);
  const int need = (rows + rpc - 1) / rpc;
  const int per_sm = warps >= 8 ? 1 : 2;
  const int grid = need < 148 * per_sm ? need : 148 * per_sm;
  return grid * rpc;
}

// f(y type, residual type, vector accesses, most threads of a CTA): rows of up to 8192 columns
// take at most 512 threads, which may then use twice the registers.
template <class F>
void dispatch_norm(int y_type, int r_type, bool vec, int threads, F&& f) {
  auto sized = [&](auto yt, auto rt, auto v) {
    if (threads <= 512) f(yt, rt, v, std::integral_constant<int, 512>{});
    else f(yt, rt, v, std::integral_constant<int, 1024>{});
  };
  auto with = [&](auto yt, auto rt) {
    if (vec) sized(yt, rt, std::true_type{});
    else sized(yt, rt, std::false_type{});
  };
  if (y_type == MOE_B200_BF16) r_type == MOE_B200_FP32 ? with(bf16{}, float{}) : with(bf16{}, bf16{});
  else if (y_type == MOE_B200_FP16) r_type == MOE_B200_FP32 ? with(fp16{}, float{}) : with(fp16{}, fp16{});
  else with(float{}, float{});
}

bool type_pair_ok(int y, int r) { return is_float_type(y) && is_float_type(r) && (r == y || r == MOE_B200_FP32); }

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

cudaError_t norm_status(cudaStream_t st, bool clear, int* v) { return take_status(st, clear, v); }

}  // namespace moe

extern "C" {

MOE_B200_API int moe_b200_block_norm(const moe_b200_norm_args* a, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->rows < 0 || a->cols < 1 || a->cols > kNormMaxCols)
    return report_error(MOE_B200_ERR_ARG, "block_norm: rows must be >= 0 and cols in [1, 16384]");
  if (!type_pair_ok(a->y_type, a->residual_type))
    return report_error(MOE_B200_ERR_ARG, "block_norm: the residual has y's type or fp32");
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
  // The ring: rows of two warps or more whose row tensors are 16-byte aligned, at least four per
  // SM, and two or more of them in a CTA's share of shared memory.
  RingArgs g{};
  g.y_bytes = a->cols * type_bytes(a->y_type);
  g.r_bytes = a->residual ? a->cols * type_bytes(a->residual_type) : 0;
  g.g_bytes = a->gate && n.gate_cols && n.g_ld ? a->cols * type_bytes(a->gate_type) : 0;
  const int stage_bytes = g.y_bytes + g.r_bytes + g.g_bytes;
  const int ctas = n.warps >= 2 && n.warps <= 16 ? 32 / n.warps : 0;   // 1024 threads of an SM
  g.stages = ctas ? kRingSmem / ctas / stage_bytes : 0;
  if (g.stages > kRingMaxStages) g.stages = kRingMaxStages;
  if (vec && a->y && a->rows >= 4 * sms && g.stages >= 2) {
    const dim3 grid(a->rows < ctas * sms ? a->rows : ctas * sms), block(n.warps * 32);
    const size_t smem = static_cast<size_t>(g.stages) * stage_bytes;
    dispatch_norm(a->y_type, a->residual_type, true, 0, [&](auto yt, auto rt, auto, auto) {
      auto kernel = a->post_weight ? norm_ring_kernel<decltype(yt), decltype(rt), true>
                                   : norm_ring_kernel<decltype(yt), decltype(rt), false>;
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
      if (e == cudaSuccess) e = launch_pdl(kernel, grid, block, smem, st, n, g);
    });
    return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "block_norm launch");
  }
  const dim3 block(n.warps * 32, rpc), grid((a->rows + rpc - 1) / rpc);
  dispatch_norm(a->y_type, a->residual_type, vec, block.x * block.y, [&](auto yt, auto rt, auto v, auto t) {
    e = launch_pdl(norm_fwd_kernel<decltype(yt), decltype(rt), decltype(v)::value, decltype(t)::value>, grid, block, 0,
                   st, n);
  });
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "block_norm launch");
}

MOE_B200_API size_t moe_b200_block_norm_backward_workspace_size(int32_t rows, int32_t cols) {
  using namespace moe;
  if (rows < 0 || cols < 1 || cols > kNormMaxCols) return 0;
  return static_cast<size_t>(align256(static_cast<int64_t>(3) * bwd_parts(rows, cols) * cols * 4) +
                             align256(static_cast<int64_t>(rows) * 4) + 256);
}

MOE_B200_API int moe_b200_block_norm_backward(const moe_b200_norm_backward_args* a, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->rows < 0 || a->cols < 1 || a->cols > kNormMaxCols)
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: rows must be >= 0 and cols in [1, 16384]");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // what the gate varies over: columns only, rows only, both, neither
  const bool g_rows = a->gate_row_stride != 0, g_cols = a->gate_per_column;
  cudaError_t e = cudaSuccess;
  if (a->rows == 0) {   // sums over no rows
    if (a->dpre_weight) e = cudaMemsetAsync(a->dpre_weight, 0, sizeof(float) * a->cols, st);
    if (e == cudaSuccess && a->dpost_weight) e = cudaMemsetAsync(a->dpost_weight, 0, sizeof(float) * a->cols, st);
    if (e == cudaSuccess && a->dgate && !g_rows)
      e = cudaMemsetAsync(a->dgate, 0, sizeof(float) * (g_cols ? a->cols : 1), st);
    return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "cudaMemsetAsync");
  }
  if (!type_pair_ok(a->y_type, a->residual_type))
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: the residual has y's type or fp32");
  if (!a->dx && !a->dresidual) return report_error(MOE_B200_ERR_ARG, "block_norm_backward: dx or dresidual is required");
  if (a->dx && (!a->residual || !a->pre_weight || !a->dpre_weight || !is_float_type(a->pre_weight_type)))
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: dx needs residual, pre_weight and dpre_weight");
  if (!a->y && (a->post_weight || a->gate || a->dy))
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: post_weight, gate and dy need y");
  if (a->post_weight && (!a->dpost_weight || !is_float_type(a->post_weight_type)))
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: post_weight needs dpost_weight");
  if (a->gate && (!a->dgate || !is_float_type(a->gate_type)))
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: gate needs dgate");
  if (!workspace || workspace_bytes < moe_b200_block_norm_backward_workspace_size(a->rows, a->cols))
    return report_error(MOE_B200_ERR_WORKSPACE, "block_norm_backward: workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return report_error(MOE_B200_ERR_ARG, "workspace must be 256-byte aligned");
  int sms = 0;
  if (int rc = op_device(&sms)) return rc;
  NormBwdArgs n{};
  n.dx = a->dx;
  n.dr = a->dresidual;
  n.r = a->dx ? a->residual : nullptr;
  n.y = a->y;
  n.post_w = a->post_weight;
  n.pre_w = a->pre_weight;
  n.gate = a->gate;
  n.dres = a->dresidual_in;
  n.dy = a->dy;
  n.dx_ld = a->dx_stride;
  n.dr_ld = a->dresidual_stride;
  n.r_ld = a->residual_stride;
  n.y_ld = a->y_stride;
  n.g_ld = a->gate_row_stride;
  n.dres_ld = a->dresidual_in_stride;
  n.dy_ld = a->dy_stride;
  n.dg_ld = a->dgate_stride;
  if (a->rows == 1) n.dx_ld = n.dr_ld = n.r_ld = n.y_ld = n.g_ld = n.dres_ld = n.dy_ld = n.dg_ld = 0;
  n.rows = a->rows;
  n.cols = a->cols;
  n.post_type = a->post_weight_type;
  n.pre_type = a->pre_weight_type;
  n.gate_type = a->gate_type;
  n.gate_cols = a->gate_per_column;
  n.scale = a->scale;
  n.eps = a->eps;
  n.off = a->weight_offset;
  n.partial = static_cast<float*>(workspace);
  n.parts = bwd_parts(a->rows, a->cols);
  float* row_dots = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                             align256(static_cast<int64_t>(3) * n.parts * a->cols * 4));
  NormSumArgs s{};
  int sums = 0;
  if (a->dx) s.out[sums++] = a->dpre_weight;   // slot 0 when present
  n.post_slot = n.gate_slot = -1;
  if (a->post_weight) {
    n.post_slot = sums;
    s.out[sums++] = a->dpost_weight;
  }
  n.gate_grad = !a->gate ? 0 : g_rows && g_cols ? 3 : g_cols ? 1 : 2;
  if (n.gate_grad == 1) {
    n.gate_slot = sums;
    s.out[sums++] = static_cast<float*>(a->dgate);
  }
  n.dgate = n.gate_grad == 3 ? a->dgate : n.gate_grad == 2 ? (g_rows ? a->dgate : row_dots) : nullptr;
  int rpc;
  norm_shape(a->cols, &n.warps, &rpc);
  const bool vec = a->cols % 8 == 0 && rows_aligned(a->y, n.y_ld, a->y_type) &&
                   rows_aligned(a->dx, n.dx_ld, a->y_type) && rows_aligned(a->dresidual, n.dr_ld, a->residual_type) &&
                   rows_aligned(n.r, n.r_ld, a->residual_type) &&
                   rows_aligned(a->dresidual_in, n.dres_ld, a->residual_type) &&
                   rows_aligned(a->dy, n.dy_ld, a->y_type) && aligned16(a->post_weight) && aligned16(a->pre_weight) &&
                   (!g_cols || rows_aligned(a->gate, n.g_ld, a->gate_type)) &&
                   (n.gate_grad != 3 || rows_aligned(a->dgate, n.dg_ld, a->gate_type));
  const dim3 block(n.warps * 32, rpc), grid(n.parts / rpc);
  dispatch_norm(a->y_type, a->residual_type, vec, block.x * block.y, [&](auto yt, auto rt, auto v, auto t) {
    e = launch_pdl(norm_bwd_kernel<decltype(yt), decltype(rt), decltype(v)::value, decltype(t)::value>, grid, block, 0,
                   st, n);
  });
  if (e != cudaSuccess) return report_cuda(e, "block_norm_backward launch");
  if (sums) {
    s.partial = n.partial;
    s.parts = n.parts;
    s.cols = a->cols;
    e = launch_pdl(norm_sum_kernel, dim3((a->cols + 31) / 32, sums), dim3(32, 8), 0, st, s);
    if (e != cudaSuccess) return report_cuda(e, "block_norm_backward sum launch");
  }
  if (n.gate_grad == 2 && !g_rows) {
    e = launch_pdl(norm_total_kernel, dim3(1), dim3(1024), 0, st, static_cast<const float*>(row_dots), a->rows,
                   static_cast<float*>(a->dgate));
    if (e != cudaSuccess) return report_cuda(e, "block_norm_backward total launch");
  }
  return MOE_B200_OK;
}

}  // extern "C"
