// Linear layer in 8-bit integers with one scale per token and one per output channel.
//
//   q[t][k] = rint(v[t][k] / sx[t]) in [-127, 127],  sx[t] = max(max_k |v[t][k]| / 127, 2^-126)
//   y[t][n] = sx[t] * sw[n] * sum_k q[t][k] * w[n][k]  (+ bias[n])
//
// v is x, or silu(x2) * x1 of x = [x1 | x2] (the expert layer's order).  The codes of x are those of
// 64-bit arithmetic with max |x| * (1 / 127) for a scale; sx is that in 32 bits.  Sums of products are
// exact 32-bit integers (|sum| <= K * 2^14, so K <= 131056 cannot overflow).  A row holding a NaN
// or an infinity gets a NaN scale, so its outputs are NaN.
#include <type_traits>

#include "int8_gemm.cuh"
#include "norm_common.cuh"

namespace moe {

constexpr int kQuantMaxCols = 2 * kNormMaxCols;
constexpr int kInt8MaxK = 131056;

constexpr float kQuantMinScale = 1.17549435082228751e-38f;   // 2^-126

struct QuantArgs {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t x_ld, q_ld;
  int rows, cols, warps, type, swiglu;
};

// silu(gate) * up.  The fast exponential is off by (|gate| + 4) 2^-24 of itself: a share of the
// product that only counts where gate is far below 0 and the product next to nothing, and that is
// small beside half a code, 2^-8 of the row's largest.
__device__ __forceinline__ void swiglu16(Row16& up, const Row16& gate) {
#pragma unroll
  for (int j = 0; j < 16; ++j) up[j] *= silu_fast(gate[j]);
}

__device__ __forceinline__ float row_amax(const Row16& v) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < 16; ++j) m = max_nan(m, fabsf(v[j]));
  return m;
}
// Magnitudes are ordered as their bits are, NaN above all.
__device__ __forceinline__ float warp_amax(float m) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
}
// Maximum over a row's warps (blockDim = (32 * warps, rows)); `buf` [rows][32] is free again after
// the next CTA barrier.
__device__ __forceinline__ float row_max(float m, int warps, float* buf) {
  m = warp_amax(m);
  if (warps == 1) return m;
  const int lane = threadIdx.x & 31;
  float* b = buf + threadIdx.y * 32;
  if (lane == 0) b[threadIdx.x >> 5] = m;
  __syncthreads();
  return warp_amax(lane < warps ? b[lane] : 0.f);
}

// A row's scale and its reciprocal; a row with a NaN or an infinity: NaN, and 0 for zero codes.
__device__ __forceinline__ float quant_scale(float m, float* inv) {
  const bool finite = m <= 3.4028234663852886e38f;
  const float sc = finite ? fmaxf(m / 127.f, kQuantMinScale) : __uint_as_float(0x7fc00000u);
  *inv = finite ? 1.f / sc : 0.f;
  return sc;
}

// Codes: v * inv lies in [-127, 127] to 2 units, so adding 1.5 * 2^23 rounds it to an integer (ties
// to even) whose two's complement is the sum's low byte; four bytes are picked out of four sums.
// (Conversions run at an eighth of the rate.)
__device__ __forceinline__ uint32_t codes4(float2 a, float2 b, float2 inv) {
  const float2 magic = dup2(12582912.f);
  a = fma2(a, inv, magic);
  b = fma2(b, inv, magic);
  const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// Of given 16-bit values, one in some hundreds lies on a tie of v / s (one half of the row's largest
// always does), where 32-bit arithmetic would take either side; a whole code is much beside the
// result's other errors.  With integer mantissas a of v and b of m, v / s = 127 a 2^z / b is either a tie or
// away from one by 1 / (254 * 2047) > 2^-19 of itself.  So the codes of inv (1 - 2^-21) and inv (1 + 2^-21)
// differ where there is a tie and nowhere else, and are the two sides of it.
//
// Which side: s = m * fl(1 / 127) in 64 bits is m / 127 (1 + e) with |e| of about 2^-53.  The quotient,
// t (1 - e) of a tie t = k + 1/2, is rounded back to t, and then to even, if t |e| is at most half the
// spacing of 64-bit numbers at t, that is if mantissa(t) |e| 2^53 <= 1; otherwise it goes the way of -e.
// With d = 127 s - m (exact) and |e| = |d| / m that is the same for a whole row where 2^54 |d| <= m or
// 2^53 |d| > m.
//
// (d is a multiple of the last place of s, of which there are 64 at most: seven bits, and mantissa(t) has
// eight, so their product is exact in 32 bits.)
enum : int { kTieEven, kTieDown, kTieUp, kTieMixed };
struct TieRule {
  float d53, m;   // 2^53 |d| and m, both by 2^-4
  int mode;
  bool down;
};
__device__ __forceinline__ double scale64(float m) { return fmax(m * (1.0 / 127.0), static_cast<double>(kQuantMinScale)); }
__device__ __forceinline__ TieRule tie_rule(float m) {
  TieRule r;
  const double s = m * (1.0 / 127.0);
  const float d = m < 127.f * kQuantMinScale ? 0.f   // the scale is a power of two
                                             : static_cast<float>(fma(s, 127.0, -static_cast<double>(m)) * 0x1p49);
  r.m = m * 0x1p-4f;
  r.down = d > 0.f;
  r.d53 = fabsf(d);
  r.mode = 2.f * r.d53 <= r.m ? kTieEven : r.d53 <= r.m ? kTieMixed : r.down ? kTieDown : kTieUp;
  return r;
}
// lo, hi: four codes on the sides of their ties towards 0 and away from it.
__device__ __forceinline__ uint32_t even4(uint32_t lo, uint32_t hi) {
  const uint32_t odd = (hi & 0x01010101u) * 255u;
  return (lo & odd) | (hi & ~odd);
}
__device__ __forceinline__ uint32_t mixed4(const TieRule& r, uint32_t lo, uint32_t hi) {
  uint32_t c = even4(lo, hi);
  for (uint32_t diff = lo ^ hi; diff != 0;) {
    const int shift = (__ffs(diff) - 1) & 24;
    const uint32_t byte = 255u << shift;
    diff &= ~byte;
    const float t = fabsf(static_cast<float>(static_cast<int8_t>(lo >> shift))) + 0.5f;
    // 1 to 2; below t = 1/2 numbers are twice as dense
    const float mantissa = t == 0.5f && r.down ? 2.f : __uint_as_float((__float_as_uint(t) & 0x7fffffu) | 0x3f800000u);
    const float part = mantissa * r.d53;
    if (part > r.m || (part == r.m && !r.down)) c = (c & ~byte) | ((r.down ? lo : hi) & byte);
  }
  return c;
}
// 32-bit values may be near a tie without being on it: where the two codes differ, 64 bits decide.
__device__ __forceinline__ uint32_t near4(double s, uint32_t lo, uint32_t hi, float2 a, float2 b) {
  const float v[4] = {a.x, a.y, b.x, b.y};
  uint32_t c = lo;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t byte = 255u << (8 * j);
    if (((lo ^ hi) & byte) == 0) continue;
    const int q = static_cast<int>(fmin(fmax(rint(v[j] / s), -127.0), 127.0));
    c = (c & ~byte) | ((static_cast<uint32_t>(q) << (8 * j)) & byte);
  }
  return c;
}
// The codes of 4 N given values, as 64-bit arithmetic has them; v: pairs.
template <class XT, int N>
__device__ __forceinline__ void given_codes(const float2* v, float m, float inv, uint32_t (&c)[N]) {
  const float2 down = dup2(inv * (1.f - 0x1p-21f)), up = dup2(inv * (1.f + 0x1p-21f));
  uint32_t hi[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c[i] = codes4(v[2 * i], v[2 * i + 1], down);
    hi[i] = codes4(v[2 * i], v[2 * i + 1], up);
  }
  if constexpr (sizeof(XT) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c[i] != hi[i]) c[i] = near4(scale64(m), c[i], hi[i], v[2 * i], v[2 * i + 1]);
  } else {
    const TieRule r = tie_rule(m);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (r.mode == kTieMixed && c[i] != hi[i]) c[i] = mixed4(r, c[i], hi[i]);
      else if (r.mode != kTieDown) c[i] = r.mode == kTieUp ? hi[i] : even4(c[i], hi[i]);
    }
  }
}

template <class XT, int LAY>
__device__ __forceinline__ void store_codes(int8_t* row, int cols, const Row16& v, float m, float inv, bool given) {
  uint32_t c[4] = {0, 0, 0, 0};
  if (inv != 0.f && given) {
    given_codes<XT>(v.v, m, inv, c);
  } else if (inv != 0.f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = codes4(v.v[2 * i], v.v[2 * i + 1], dup2(inv));
  }
  if constexpr (is_vec(LAY)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (exists<LAY>(8 * i, cols)) *reinterpret_cast<uint2*>(row + col_of<LAY>(8 * i)) = make_uint2(c[2 * i], c[2 * i + 1]);
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (exists<LAY>(q, cols)) row[col_of<LAY>(q)] = static_cast<int8_t>(c[q >> 2] >> (8 * (q & 3)));
  }
}

// One row in the registers of a group of warps, N times 16 elements per thread (N = 2: the second
// 16 are those of the row's second half of threads x 16 columns).  Few rows: bound by latency (80 x 2048
// with the activation 1.9 us).
template <class XT, int LAY, int N>
__global__ void __launch_bounds__(N == 1 ? 512 : 1024, 1) quant_kernel(QuantArgs a) {
  __shared__ float buf[8 * 32];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const XT* src = static_cast<const XT*>(a.x) + min(row, a.rows - 1) * a.x_ld;
  Row16 v[N];
  float m = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int at = n * 16 * blockDim.x, cols = row < a.rows ? max(0, a.cols - at) : 0;
    load_row<XT, LAY>(src + (cols ? at : 0), cols, v[n]);
    if (a.swiglu) {
      Row16 g;
      load_row<XT, LAY>(src + (cols ? a.cols + at : 0), cols, g);
      swiglu16(v[n], g);
    }
    m = max_nan(m, row_amax(v[n]));
  }
  m = row_max(m, a.warps, buf);
  if (row >= a.rows) return;
  float inv;
  const float sc = quant_scale(m, &inv);
  if (threadIdx.x == 0) a.scale[row] = sc;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int at = n * 16 * blockDim.x;
    if (at < a.cols) store_codes<XT, LAY>(a.q + row * a.q_ld + at, a.cols - at, v[n], m, inv, !a.swiglu);
  }
}

// Many aligned rows: persistent CTAs with their next rows on the way to shared memory, as the norm's.
// 8192 x 7168 from bf16 39.7 us (4.4 TB/s): 250 instructions per warp and row, a third of them for the
// ties (without which 30.8, but for 16-bit values on the tie of their scale the codes are then chance);
// with the activation, 8192 x 2048, 15.8 us (5.3 TB/s), bound by HBM.
template <class XT, int LAY>
__global__ void __launch_bounds__(512, 2) quant_ring_kernel(QuantArgs a, RingPlan g) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float buf[2][32];   // of even and odd rows
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
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int row = blockIdx.x; row < a.rows; row += step) {
    // after a wait that ran out the CTA still goes through its rows, without their contents
    if (ok) ok = mbar_wait(&full[stage], phase, &abort, &g_op_status, kStWaitProducer);
    uint8_t* src = ring + stage * g.stage_bytes;
    Row16 v;
    load_row<XT, LAY>(reinterpret_cast<const XT*>(src), cols, v);
    if (a.swiglu) {
      Row16 gate;
      load_row<XT, LAY>(reinterpret_cast<const XT*>(src + g.t[1].at), cols, gate);
      swiglu16(v, gate);
    }
    const float m = row_max(row_amax(v), a.warps, buf[parity]);
    parity ^= 1;
    // every thread has its part of the stage (row_max's barrier)
    const int64_t next = row + static_cast<int64_t>(g.stages) * step;
    if (threadIdx.x == 0 && ok && next < a.rows) ring_fetch(g, static_cast<int>(next), src, &full[stage]);
    if (ok && ++stage == g.stages) {
      stage = 0;
      phase ^= 1u;
    }
    float inv;
    const float sc = quant_scale(m, &inv);
    if (threadIdx.x == 0) a.scale[row] = sc;
    store_codes<XT, LAY>(a.q + row * a.q_ld, cols, v, m, inv, !a.swiglu);
  }
  if (!ok && threadIdx.x == 0)   // given up: the loads in flight land first
    for (int i = 0; i < g.stages; ++i) {
      int none = 0;
      if (blockIdx.x + static_cast<int64_t>(i) * step < a.rows)
        mbar_wait(&full[i], i >= stage ? phase : phase ^ 1u, &none, &g_op_status, kStWaitDrain);
    }
}

// ---------------------------------------------------------------- one or two tokens
// The whole layer in one launch: every CTA quantises the tokens for itself into shared memory (they
// come from L2; 14 KB each at 7168), then each warp takes whole weight rows, 4 KB of them in
// flight, and adds up four products per instruction (dp4a).  The weights cross HBM once; the warps
// per SM are chosen so that the rows come out even.  One token 7168 -> 4096 from bf16: 5.6 us, 5.2
// TB/s (the streaming kernel and its quantisation: 9.2).  From three tokens on the products take
// longer than the weights: 11 us against 9.2.
constexpr int kGemvMaxT = 2;

struct GemvArgs {
  const void* x;
  const float* sx;
  const int8_t* w;
  const float* sw;
  const void* bias;
  void* y;
  int64_t x_ld, w_ld, y_ld;
  int T, N, K, vec, swiglu, y_type, bias_type;
};

// Eight elements of a row from column e on (what is quantised), as the row kernels compute them.
template <class XT>
__device__ __forceinline__ void gemv_load8(const GemvArgs& a, const XT* row, int e, float* v) {
  auto load = [&](const XT* p, float* out) {
    if (a.vec) load8<XT, true>(p, out);
    else load8<XT, false>(p, out);
  };
  load(row + e, v);
  if (!a.swiglu) return;
  float g[8];
  load(row + a.K + e, g);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= silu_fast(g[j]);
}

template <class XT, int TT>
__global__ void __launch_bounds__(1024, 1) int8_gemv_kernel(GemvArgs a) {
  extern __shared__ int4 xs[];   // [TT][K / 16] codes
  __shared__ float s_max[TT][32], s_scale[TT];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int units = a.K / 16;
  int n = blockIdx.x * warps + warp;
  int4 w[8];
  auto load_w = [&](int row, int u0) {
    const int4* p = reinterpret_cast<const int4*>(a.w + row * a.w_ld) + u0 + lane;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[j] = u0 + lane + 32 * j < units ? p[32 * j] : make_int4(0, 0, 0, 0);
  };
  if (n < a.N) load_w(n, 0);   // on its way while the tokens are quantised
  if constexpr (std::is_same<XT, int8_t>::value) {
    for (int t = 0; t < TT; ++t)
      for (int u = threadIdx.x; u < units; u += blockDim.x)
        xs[t * units + u] = t < a.T ? reinterpret_cast<const int4*>(static_cast<const int8_t*>(a.x) + t * a.x_ld)[u]
                                    : make_int4(0, 0, 0, 0);
    if (threadIdx.x < TT) s_scale[threadIdx.x] = static_cast<int>(threadIdx.x) < a.T ? a.sx[threadIdx.x] : 0.f;
  } else {
    const XT* x = static_cast<const XT*>(a.x);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float m = 0.f;
      if (t < a.T)
        for (int e = threadIdx.x * 8; e < a.K; e += blockDim.x * 8) {
          float v[8];
          gemv_load8(a, x + t * a.x_ld, e, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
        }
      m = warp_amax(m);
      if (lane == 0) s_max[t][warp] = m;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const float m = warp_amax(lane < warps ? s_max[t][lane] : 0.f);
      float inv;
      const float sc = quant_scale(m, &inv);
      if (threadIdx.x == 0) s_scale[t] = sc;
      uint2* dst = reinterpret_cast<uint2*>(xs + t * units);
      for (int e = threadIdx.x * 8; e < a.K; e += blockDim.x * 8) {
        uint2 c = make_uint2(0, 0);
        if (t < a.T && inv != 0.f) {
          float v[8];
          gemv_load8(a, x + t * a.x_ld, e, v);
          const float2 p[4] = {make_float2(v[0], v[1]), make_float2(v[2], v[3]), make_float2(v[4], v[5]),
                               make_float2(v[6], v[7])};
          uint32_t q[2];
          if (a.swiglu) {
            q[0] = codes4(p[0], p[1], dup2(inv));
            q[1] = codes4(p[2], p[3], dup2(inv));
          } else {
            given_codes<XT>(p, m, inv, q);
          }
          c = make_uint2(q[0], q[1]);
        }
        dst[e / 8] = c;
      }
    }
  }
  __syncthreads();
  for (; n < a.N; n += gridDim.x * warps) {
    int acc[TT] = {};
    for (int u0 = 0; u0 < units; u0 += 256) {
      if (u0) load_w(n, u0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int u = u0 + lane + 32 * j;
        if (u >= units) break;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          const int4 q = xs[t * units + u];
          acc[t] = __dp4a(w[j].x, q.x, acc[t]);
          acc[t] = __dp4a(w[j].y, q.y, acc[t]);
          acc[t] = __dp4a(w[j].z, q.z, acc[t]);
          acc[t] = __dp4a(w[j].w, q.w, acc[t]);
        }
      }
    }
    const int next = n + gridDim.x * warps;
    if (next < a.N) load_w(next, 0);
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = __reduce_add_sync(0xffffffffu, acc[t]);
    // lane t stores token t's output
    int mine = acc[0];
#pragma unroll
    for (int t = 1; t < TT; ++t) mine = lane == t ? acc[t] : mine;
    if (lane < a.T) {
      const float b = a.bias ? load1_dyn(a.bias, a.bias_type, n) : 0.f;
      const float v = fmaf(static_cast<float>(mine), s_scale[lane] * a.sw[n], b);
      store1_dyn(a.y, a.y_type, lane * a.y_ld + n, v);
    }
  }
}

cudaError_t quant_status(cudaStream_t st, bool clear, int* v) { return take_status(st, clear, v); }

namespace {

cudaError_t quant_launch(const QuantArgs& q0, int sms, cudaStream_t st) {
  QuantArgs q = q0;
  if (q.rows == 1) q.x_ld = q.q_ld = 0;   // a single row has no pitch
  int rpc;
  const bool twice = q.cols > kNormMaxCols / 2;   // 32 elements per thread
  norm_shape(twice ? (q.cols + 1) / 2 : q.cols, &q.warps, &rpc);
  const bool vec = q.cols % 8 == 0 && rows_aligned(q.x, q.x_ld, q.type) &&
                   (reinterpret_cast<uintptr_t>(q.q) & 7u) == 0 && q.q_ld % 8 == 0;
  cudaError_t e = cudaSuccess;
  auto go = [&](auto t) {
    using XT = decltype(t);
    // The ring: aligned rows of two warps or more, at least four per SM (7168 columns, ring against
    // direct: 148 rows 1.9 us against 1.8, 592 rows 3.2 against 3.3, 8192 rows 30.8 against 51.5, before the rule for ties).
    RingPlan g{};
    ring_add(&g, q.x, q.x_ld, q.cols, q.type);
    if (q.swiglu) ring_add(&g, static_cast<const XT*>(q.x) + q.cols, q.x_ld, q.cols, q.type);
    const int ctas = q.warps >= 2 ? 32 / q.warps : 0;   // 1024 threads of an SM
    g.stages = ctas ? kRingSmem / ctas / g.stage_bytes : 0;
    if (g.stages > kRingMaxStages) g.stages = kRingMaxStages;
    if (vec && !twice && q.rows >= 4 * sms && g.stages >= 2) {
      const dim3 grid(q.rows < ctas * sms ? q.rows : ctas * sms), block(q.warps * 32);
      auto kernel = q.cols == q.warps * 32 * kNormPerThread ? quant_ring_kernel<XT, kFull> : quant_ring_kernel<XT, kHalf>;
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
      if (e == cudaSuccess) e = launch_pdl(kernel, grid, block, static_cast<size_t>(g.stages) * g.stage_bytes, st, q, g);
      return;
    }
    const dim3 block(q.warps * 32, rpc), grid((q.rows + rpc - 1) / rpc);
    auto kernel = twice ? (vec ? quant_kernel<XT, kVec, 2> : quant_kernel<XT, kScattered, 2>)
                        : (vec ? quant_kernel<XT, kVec, 1> : quant_kernel<XT, kScattered, 1>);
    e = launch_pdl(kernel, grid, block, 0, st, q);
  };
  if (q.type == MOE_B200_BF16) go(bf16{});
  else if (q.type == MOE_B200_FP16) go(fp16{});
  else go(float{});
  return e;
}

cudaError_t gemv_launch(const GemvArgs& g, int x_type, int sms, cudaStream_t st) {
  // rows per SM in as few rounds of at most 32 warps as it takes; the same number in each
  const int rows = (g.N + sms - 1) / sms, rounds = (rows + 31) / 32;
  int warps = (rows + rounds - 1) / rounds;
  if (warps < 8) warps = 8;
  const int need = (g.N + warps - 1) / warps;
  const dim3 grid(need < sms ? need : sms), block(warps * 32);
  auto sized = [&](auto t, auto tt) {
    using XT = decltype(t);
    constexpr int TT = decltype(tt)::value;
    auto kernel = int8_gemv_kernel<XT, TT>;
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), TT * kQuantMaxCols);
    return e == cudaSuccess ? launch_pdl(kernel, grid, block, static_cast<size_t>(TT) * g.K, st, g) : e;
  };
  auto go = [&](auto t) {
    return g.T == 1 ? sized(t, std::integral_constant<int, 1>{}) : sized(t, std::integral_constant<int, 2>{});
  };
  return x_type == MOE_B200_BF16 ? go(bf16{}) : x_type == MOE_B200_FP16 ? go(fp16{}) : x_type == MOE_B200_FP32 ? go(0.f) : go(int8_t{});
}

int quant_check(const void* x, int type, int rows, int cols, const char** why) {
  if (rows < 0 || rows > kOpMaxRows || cols < 1 || cols > kQuantMaxCols)
    *why = "int8 quantisation: rows must be in [0, 2^30] and cols in [1, 32768]";
  else if (!is_float_type(type)) *why = "int8 quantisation: x is bf16, fp16 or fp32";
  else if (rows > 0 && !x) *why = "null tensor pointer";
  else return 0;
  return 1;
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace
}  // namespace moe

extern "C" {

MOE_B200_API int moe_b200_quantize_int8(const moe_b200_quantize_args* a, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  const char* why = nullptr;
  if (quant_check(a->x, a->x_type, a->rows, a->cols, &why)) return report_error(MOE_B200_ERR_ARG, why);
  if (a->rows == 0) return MOE_B200_OK;
  if (!a->q || !a->scale) return report_error(MOE_B200_ERR_ARG, "null tensor pointer");
  int sms = 0;
  if (int rc = op_device(&sms)) return rc;
  QuantArgs q{};
  q.x = a->x;
  q.q = a->q;
  q.scale = a->scale;
  q.x_ld = a->x_stride;
  q.q_ld = a->q_stride;
  q.rows = a->rows;
  q.cols = a->cols;
  q.type = a->x_type;
  q.swiglu = a->swiglu;
  const cudaError_t e = quant_launch(q, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "quantize_int8 launch");
}

MOE_B200_API size_t moe_b200_int8_linear_workspace_size(int32_t num_tokens, int32_t out_features, int32_t in_features,
                                                        int32_t x_type) {
  using namespace moe;
  if (num_tokens < 0 || num_tokens > kOpMaxRows || out_features < 1 || in_features < 1 || in_features > kInt8MaxK) return 0;
  const size_t T = num_tokens;
  return 256 + (x_type == MOE_B200_INT8 ? 0 : align256(T * in_features) + align256(T * sizeof(float)));
}

MOE_B200_API int moe_b200_int8_linear(const moe_b200_linear_args* a, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->num_tokens < 0 || a->num_tokens > kOpMaxRows || a->out_features < 1 || a->out_features > kOpMaxRows ||
      a->in_features < 16 || a->in_features > kInt8MaxK || a->in_features % 16)
    return report_error(MOE_B200_ERR_ARG, "int8_linear: num_tokens must be in [0, 2^30], out_features in [1, 2^30] and in_features a multiple of 16 up to 131056");
  const bool quantise = a->x_type != MOE_B200_INT8;
  const char* why = nullptr;
  if (quantise && quant_check(a->x, a->x_type, a->num_tokens, a->in_features, &why))
    return report_error(MOE_B200_ERR_ARG, why);
  if (!quantise && a->swiglu) return report_error(MOE_B200_ERR_ARG, "int8_linear: swiglu needs a floating-point x");
  if (!is_float_type(a->y_type) || (a->bias && !is_float_type(a->bias_type)))
    return report_error(MOE_B200_ERR_ARG, "int8_linear: y and bias are bf16, fp16 or fp32");
  if (a->num_tokens == 0) return MOE_B200_OK;
  if (!a->x || !a->weight || !a->weight_scale || !a->y || (!quantise && !a->x_scale))
    return report_error(MOE_B200_ERR_ARG, "null tensor pointer");
  // a single row has no pitch
  const int64_t w_ld = a->out_features == 1 ? a->in_features : a->weight_stride;
  const int64_t x_ld = a->num_tokens == 1 && !quantise ? a->in_features : a->x_stride;
  if (!aligned16(a->weight) || w_ld % 16 || w_ld < a->in_features)
    return report_error(MOE_B200_ERR_ARG, "int8_linear: weight rows must start on 16-byte boundaries");
  if (!quantise && (!aligned16(a->x) || x_ld % 16 || x_ld < a->in_features))
    return report_error(MOE_B200_ERR_ARG, "int8_linear: int8 x rows must start on 16-byte boundaries");
  const size_t need = moe_b200_int8_linear_workspace_size(a->num_tokens, a->out_features, a->in_features, a->x_type);
  if (!workspace || workspace_bytes < need)
    return report_error(MOE_B200_ERR_WORKSPACE, "int8_linear: workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return report_error(MOE_B200_ERR_ARG, "workspace must be 256-byte aligned");
  int sms = 0;
  if (int rc = op_device(&sms)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->num_tokens <= kGemvMaxT && a->in_features <= kQuantMaxCols) {
    GemvArgs g{};
    g.x = a->x;
    g.sx = a->x_scale;
    g.w = a->weight;
    g.sw = a->weight_scale;
    g.bias = a->bias;
    g.y = a->y;
    g.x_ld = a->num_tokens == 1 ? 0 : a->x_stride;
    g.w_ld = w_ld;
    g.y_ld = a->y_stride;
    g.T = a->num_tokens;
    g.N = a->out_features;
    g.K = a->in_features;
    g.vec = quantise && rows_aligned(a->x, g.x_ld, a->x_type);
    g.swiglu = a->swiglu;
    g.y_type = a->y_type;
    g.bias_type = a->bias_type;
    const cudaError_t e = gemv_launch(g, a->x_type, sms, st);
    return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "int8_linear launch");
  }
  const int8_t* q_rows = static_cast<const int8_t*>(a->x);
  int64_t q_ld = x_ld;
  LinearArgs l{};
  l.sx = a->x_scale;
  cudaError_t e = cudaSuccess;
  if (quantise) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    QuantArgs q{};
    q.x = a->x;
    q.q = reinterpret_cast<int8_t*>(ws);
    q.scale = reinterpret_cast<float*>(ws + align256(static_cast<size_t>(a->num_tokens) * a->in_features));
    q.x_ld = a->x_stride;
    q.q_ld = a->in_features;
    q.rows = a->num_tokens;
    q.cols = a->in_features;
    q.type = a->x_type;
    q.swiglu = a->swiglu;
    e = quant_launch(q, sms, st);
    if (e != cudaSuccess) return report_cuda(e, "int8_linear quantisation launch");
    q_rows = q.q;
    q_ld = q.q_ld;
    l.sx = q.scale;
    l.early_w = 1;   // the quantisation waited for everything before it, and writes no weights
  }
  l.sw = a->weight_scale;
  l.bias = a->bias;
  l.y = a->y;
  l.y_ld = a->num_tokens == 1 ? 0 : a->y_stride;
  l.T = a->num_tokens;
  l.N = a->out_features;
  l.K = a->in_features;
  l.y_type = a->y_type;
  l.bias_type = a->bias_type;
  e = int8_gemm_launch(q_rows, q_ld, a->weight, w_ld, l, sms, st);
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "int8_linear launch");
}

}  // extern "C"
