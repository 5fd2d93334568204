// Gradients of the norms around a block (norm.cu), from dx of x and dr of r'.
//
//   G   = dr + s(r') (w dx - r^ mean(w dx r^)),  r^ = r' s(r')      gradient of the residual
//   dw  = sum over rows of dx r^
//   b   = (post_weight + off) * gate per column (1 where absent)
//   dy  = scale gate s(y) (b G - y^ mean(b G y^)),  y^ = y s(y)     (scale gate b G without post_weight)
//   dpost = scale gate sum over rows of G y^;  dgate = scale G y^ (post_weight + off), summed over what
//   the gate is broadcast over.  A gate per column is a constant of the sum over rows, so one sum
//   P = sum of G y^ serves dpost and dgate.
//
// s(r') and s(y) are computed again from the rows, whose elements stay in registers between the
// row's sums.  Per-column sums are held in registers over a persistent CTA's rows (32-bit, fixed
// order), written once per CTA and added up by norm_sum_kernel.
#include "norm_common.cuh"

namespace moe {

constexpr int kBwdSide = 8;   // rows of several warps side by side in a CTA
constexpr int kFactorBytes = 2 * kNormPerThread * 4;   // per thread of a row
constexpr int kNoBlock = 3;
enum : int { kGateNone = 0, kGateColumn = 1, kGateRow = 2, kGateElement = 3 };

struct NormBwdArgs {
  const void *dx, *dr, *r, *y, *post_w, *pre_w, *gate;
  void *dres, *dy, *dgate;          // dgate: per element (gate type) or per row (fp32); null: none
  float* partial;                   // [slots][parts][cols]: sums of dx r^ and of G y^
  int64_t dx_ld, dr_ld, r_ld, y_ld, g_ld, dres_ld, dy_ld, dg_ld;
  int rows, cols, warps, parts;
  int post_type, pre_type, gate_type;
  int gate_grad, pre_slot, post_slot;
  float scale, eps, off;
};

// What a row's computation keeps from row to row.
struct NormBwdSums {
  Row16 pre, post;
};

// Factors per column: w = pre_weight + off, b = (post_weight + off) * gate per column.
template <int LAY>
__device__ __forceinline__ void factor_w(const NormBwdArgs& a, Row16& w) {
  load_weight<LAY>(a.pre_w, a.pre_type, a.off, a.cols, w);
}
template <int LAY>
__device__ __forceinline__ void factor_b(const NormBwdArgs& a, Row16& b) {
  if (a.post_w) {
    load_weight<LAY>(a.post_w, a.post_type, a.off, a.cols, b);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) b.v[i] = dup2(1.f);
  }
  if (a.gate_grad != kGateColumn) return;
  Row16 g;
  load_row_dyn<LAY>(a.gate, a.gate_type, 0, a.cols, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) b.v[i] = mul2(b.v[i], g.v[i]);
}

// One row.  load(which, v): which = 0 dx, 1 r', 2 y, 3 dr, 4 the gate per element, 5 w, 6 b; done()
// is called when everything is loaded.  A row with no columns (one that is missing) adds nothing to the
// column sums: its 1 / sqrt(0 + eps) may be infinite.  POST, GATE (0 none or per column, 1 per row, 2 per
// element, kNoBlock: there is no y): -1 = known at run time only.
template <class YT, class RT, int LAY, int POST, int GATE, class Load, class Done>
__device__ __forceinline__ void bwd_row(const NormBwdArgs& a, int row, int cols, float inv_cols, float* buf0, float* buf1,
                                        NormBwdSums& sum, float g_of_row, Load&& load, Done&& done) {
  const bool post = POST < 0 ? a.post_w != nullptr : POST == 1;
  const int gate = GATE < 0 ? (a.gate_grad == kGateElement ? 2 : a.gate_grad == kGateRow ? 1 : 0) : GATE;
  const bool has_dx = GATE < 0 ? a.dx != nullptr : true, has_y = GATE < 0 ? a.y != nullptr : GATE != kNoBlock;
  const bool live = LAY == kPacked || LAY == kShort || LAY == kThin ? cols > 0 : true;
  Row16 r, dx, y, G;
  float s[3] = {0.f, 0.f, 0.f};   // sum r'^2, sum w dx r', sum y^2
  if (has_dx) {
    load(1, r);
    load(0, dx);
    load(5, G);
#pragma unroll
    for (int i = 0; i < 8; ++i) G.v[i] = mul2(G.v[i], dx.v[i]);
    s[0] = dot16<LAY>(r, r);
    s[1] = dot16<LAY>(G, r);
  }
  if (has_y) {
    load(2, y);
    if (post) s[2] = dot16<LAY>(y, y);
  }
  if constexpr (LAY == kPacked) packed_sum(s);
  else if (LAY == kFull || a.warps <= 16) row_sum3(s, a.warps, buf0);
  else row_sum(s, a.warps, buf0);
  const float rstd = rsqrtf(s[0] * inv_cols + a.eps);
  {
    Row16 d;
    if (a.dr) {
      load(3, d);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) d.v[i] = dup2(0.f);
    }
    if (has_dx) {
      const float k = -s[1] * inv_cols * rstd * rstd;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (live) sum.pre.v[i] = fma2(mul2(dx.v[i], r.v[i]), dup2(rstd), sum.pre.v[i]);
        G.v[i] = fma2(dup2(rstd), fma2(r.v[i], dup2(k), G.v[i]), d.v[i]);
      }
    } else {
      G = d;
    }
  }
  if (a.dres) store_row<RT, LAY>(static_cast<RT*>(a.dres) + row * a.dres_ld, cols, G);
  if (!has_y) {
    done();
    return;
  }
  const float ystd = post ? rsqrtf(s[2] * inv_cols + a.eps) : 1.f;
  const float g_row = gate == 1 ? g_of_row : 1.f;
  const float q = g_row * ystd;
  const bool has_b = post || a.gate_grad == kGateColumn;
  Row16 b;
  if (has_b) load(6, b);
  if (gate == 2) {
    Row16 ge, dg;
    load(4, ge);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 gy = mul2(G.v[i], y.v[i]);
      if (live) sum.post.v[i] = fma2(mul2(gy, ge.v[i]), dup2(q), sum.post.v[i]);
      dg.v[i] = mul2(has_b ? mul2(gy, b.v[i]) : gy, dup2(a.scale * ystd));
      G.v[i] = mul2(G.v[i], ge.v[i]);
    }
    store_row_dyn<LAY>(a.dgate, a.gate_type, row * a.dg_ld, cols, dg);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (live) sum.post.v[i] = fma2(mul2(G.v[i], y.v[i]), dup2(q), sum.post.v[i]);
  }
  if (has_b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) G.v[i] = mul2(G.v[i], b.v[i]);
  }
  float k = 0.f;
  if (post || gate == 1) {
    float t[1] = {dot16<LAY>(G, y)};   // sum of b G y
    if constexpr (LAY == kPacked) packed_sum(t);
    else row_sum(t, a.warps, buf1);
    done();
    if (gate == 1 && threadIdx.x == 0 && cols > 0) static_cast<float*>(a.dgate)[row] = a.scale * ystd * t[0];
    if (post) k = -t[0] * inv_cols * ystd * ystd;
  } else {
    done();
  }
  if (!a.dy) return;
  const float m = a.scale * q;
#pragma unroll
  for (int i = 0; i < 8; ++i) G.v[i] = mul2(post ? fma2(y.v[i], dup2(k), G.v[i]) : G.v[i], dup2(m));
  store_row<YT, LAY>(static_cast<YT*>(a.dy) + row * a.dy_ld, cols, G);
}

// Writes a CTA's part of the column sums.  Rows side by side in a CTA (threadIdx.y) are added up
// first, in their order, through `shared` ([rows][cols] floats; null with one row).
template <int LAY>
__device__ __forceinline__ void bwd_store_sums(const NormBwdArgs& a, const NormBwdSums& sum, float* shared) {
  float* dst = a.partial + static_cast<int64_t>(blockIdx.x) * a.cols;
  const int64_t slot = static_cast<int64_t>(a.parts) * a.cols;
  auto put = [&](float* out, const Row16& v) {
    if (blockDim.y == 1) {
      store_row<float, LAY>(out, a.cols, v);
      return;
    }
    __syncthreads();
    store_row<float, LAY>(shared + threadIdx.y * a.cols, a.cols, v);
    __syncthreads();
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < a.cols; c += blockDim.x * blockDim.y) {
      float s = shared[c];
      for (int y = 1; y < static_cast<int>(blockDim.y); ++y) s += shared[y * a.cols + c];
      out[c] = s;
    }
  };
  if (a.pre_slot >= 0) put(dst + a.pre_slot * slot, sum.pre);
  if (a.post_slot >= 0) put(dst + a.post_slot * slot, sum.post);
}

// Any alignment, any set of tensors: rows straight from global memory, one per CTA at a time, or
// blockDim.y side by side, of which those beyond the last run with no elements.
// kPacked: 65536 x 128 40 us (2.5 TB/s) against 98 with a warp per row.
// kShort, kThin: rows on odd boundaries, whose 2-byte loads, stores and checks make many instructions.  Four
// elements a thread (eight beyond 4096 columns) let two to four times the warps share them, and the factors
// per column are put into shared memory once: 16384 x 301 44.6 us against 65 with eight and factors
// in place, 16384 x 99 14.8 against 41 with all sixteen, 4096 x 5001 with a 32-bit residual 193 against
// 304.  What bounds it is still that chain of instructions, not memory: bulk copies of the rows
// ahead (their ends by plain loads) left 901 x 5001 at 55 us against 53, prefetching them to L2 at 52.
template <class YT, class RT, int LAY>
__device__ __forceinline__ void bwd_direct(const NormBwdArgs& a, float (*buf)[kBwdSide * 3 * 32], float4* shared) {
  constexpr bool kMany = LAY == kPacked || LAY == kShort || LAY == kThin;
  constexpr int kQuads = slots(LAY) / 4;
  // w and b as this thread reads them, then the sums of rows side by side
  float4* sums_of_rows = shared + 2 * kQuads * blockDim.x;
  if (threadIdx.y == 0) {
    Row16 f;
    auto put = [&](int at) {
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
        shared[(at + i) * blockDim.x + threadIdx.x] = make_float4(f.v[2 * i].x, f.v[2 * i].y, f.v[2 * i + 1].x, f.v[2 * i + 1].y);
    };
    if (a.dx) {
      factor_w<LAY>(a, f);
      put(0);
    }
    if (a.y) {
      factor_b<LAY>(a, f);
      put(kQuads);
    }
  }
  if (blockDim.y > 1) __syncthreads();   // (a row's threads read what they wrote themselves)
  NormBwdSums sum;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum.pre.v[i] = sum.post.v[i] = dup2(0.f);
  // a row without a second sum alternates the first one's buffer by itself
  const bool two = a.y && (a.post_w || a.gate_grad == kGateRow);
  int first = 0;
  const int many = kMany ? blockDim.y : 1;
  for (int row0 = blockIdx.x * many; row0 < a.rows; row0 += gridDim.x * many) {
    const int row = kMany ? row0 + threadIdx.y : row0, cols = kMany && row >= a.rows ? 0 : a.cols;
    const int from = kMany ? min(row, a.rows - 1) : row;   // a row that exists
    const float g_row = a.gate_grad == kGateRow && cols ? load1_dyn(a.gate, a.gate_type, row * a.g_ld) : 0.f;
    bwd_row<YT, RT, LAY, -1, -1>(a, row, cols, 1.f / a.cols, buf[first], buf[1], sum, g_row, [&](int which, Row16& v) {
      if (which >= 5) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 f = i < kQuads ? shared[((which - 5) * kQuads + i) * blockDim.x + threadIdx.x] : make_float4(0.f, 0.f, 0.f, 0.f);
          v.v[2 * i] = make_float2(f.x, f.y);
          v.v[2 * i + 1] = make_float2(f.z, f.w);
        }
      } else if (which == 0) load_row<YT, LAY>(static_cast<const YT*>(a.dx) + from * a.dx_ld, cols, v);
      else if (which == 1) load_row<RT, LAY>(static_cast<const RT*>(a.r) + from * a.r_ld, cols, v);
      else if (which == 2) load_row<YT, LAY>(static_cast<const YT*>(a.y) + from * a.y_ld, cols, v);
      else if (which == 3) load_row<RT, LAY>(static_cast<const RT*>(a.dr) + from * a.dr_ld, cols, v);
      else load_row_dyn<LAY>(a.gate, a.gate_type, from * a.g_ld, cols, v);
    }, [] {});
    if (!two) first ^= 1;
  }
  bwd_store_sums<LAY>(a, sum, reinterpret_cast<float*>(sums_of_rows));
}

template <class YT, class RT, int LAY, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) norm_bwd_kernel(NormBwdArgs a) {
  extern __shared__ float4 shared[];   // factors per column, sums of rows side by side
  __shared__ float buf[2][kBwdSide * 3 * 32];
  pdl_wait();
  pdl_launch_dependents();
  bwd_direct<YT, RT, LAY>(a, buf, shared);
}

// Aligned rows with dx and r': the next rows (dx, r', y, dr, gate per element) are on their
// way to shared memory as bulk copies while a row is computed.  The factors per column are put
// into shared memory once, 32-bit, as each thread reads them, beside a 16-bit residual; a 32-bit one
// leaves its ring too little room, and they are read in place.  Rows of one warp go eight to a CTA,
// each warp with a ring of its own and no CTA barrier until the sums are written.  4096 x 7168 with
// both norms and a gate per column: 66.5 us with its column sums (5.3 TB/s) against 176 straight from
// memory; 64 rows 9.0 against 10.1, so there is no lower limit of rows.  With a 32-bit residual 4096 x 7168
// 111 us (4.8 TB/s), 8192 x 4096 116 (5.2).
template <class YT, class RT, int LAY, int POST, int GATE>
__global__ void __launch_bounds__(512, 1) norm_bwd_ring_kernel(NormBwdArgs a, RingPlan g) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float buf[2][3 * 32];
  __shared__ uint64_t bars[8][kRingMaxStages];
  __shared__ int abort;
  constexpr bool kShared = sizeof(RT) == 2;
  const int factor_bytes = kShared ? kFactorBytes * blockDim.x : 0;
  float4* factors = reinterpret_cast<float4*>(ring);   // [w | b][4][threads of a row]
  uint8_t* my_ring = ring + factor_bytes + threadIdx.y * g.stages * g.stage_bytes;
  uint64_t* full = bars[threadIdx.y];
  if (threadIdx.x == 0) {
    if (threadIdx.y == 0) abort = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int step = gridDim.x * blockDim.y, cols = a.cols;
  const int row0 = blockIdx.x * blockDim.y + threadIdx.y;
  if (threadIdx.x == 0)
    for (int i = 0; i < g.stages; ++i) {
      const int64_t row = row0 + static_cast<int64_t>(i) * step;
      if (row < a.rows) ring_fetch(g, static_cast<int>(row), my_ring + i * g.stage_bytes, &full[i]);
    }
  if (kShared && threadIdx.y == 0) {
    Row16 f;
    auto put = [&](int at) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        factors[(at + i) * blockDim.x + threadIdx.x] =
            make_float4(f.v[2 * i].x, f.v[2 * i].y, f.v[2 * i + 1].x, f.v[2 * i + 1].y);
    };
    factor_w<LAY>(a, f);
    put(0);
    factor_b<LAY>(a, f);
    put(4);
  }
  if (blockDim.y > 1) __syncthreads();   // (a row's threads read what they wrote themselves)
  NormBwdSums sum;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum.pre.v[i] = sum.post.v[i] = dup2(0.f);
  const float inv_cols = 1.f / cols;
  const bool two = (POST < 0 ? a.post_w != nullptr : POST == 1) ||   // a second sum over the row
                   (GATE < 0 ? a.gate_grad == kGateRow : GATE == 1);
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  bool ok = true;
  float g_next = a.gate_grad == kGateRow && row0 < a.rows ? load1_dyn(a.gate, a.gate_type, row0 * a.g_ld) : 0.f;
  for (int row = row0; row < a.rows; row += step) {
    // after a wait that ran out the CTA still goes through its rows, without their contents
    if (ok) ok = mbar_wait(&full[stage], phase, &abort, &g_op_status, kStWaitProducer);
    uint8_t* src = my_ring + stage * g.stage_bytes;
    const float g_row = g_next;   // the gate per row, loaded a row ahead
    if (a.gate_grad == kGateRow && row + static_cast<int64_t>(step) < a.rows)
      g_next = load1_dyn(a.gate, a.gate_type, (row + step) * a.g_ld);
    bwd_row<YT, RT, LAY, POST, GATE>(
        a, row, cols, inv_cols, buf[two ? 0 : parity], buf[1], sum, g_row, [&](int which, Row16& v) {
          if (which >= 5 && !kShared) {
            if (which == 5) factor_w<LAY>(a, v);
            else factor_b<LAY>(a, v);
            return;
          }
          if (which >= 5) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 f = factors[((which - 5) * 4 + i) * blockDim.x + threadIdx.x];
              v.v[2 * i] = make_float2(f.x, f.y);
              v.v[2 * i + 1] = make_float2(f.z, f.w);
            }
            return;
          }
          // the ring's order: dx, r', y (if any), dr (if any), gate (if per element)
          const uint8_t* p = src + g.t[which == 4 && !a.dr ? 3 : which == 3 && GATE == kNoBlock ? 2 : which].at;
          if (which == 0 || which == 2) load_row<YT, LAY>(reinterpret_cast<const YT*>(p), cols, v);
          else if (which != 4) load_row<RT, LAY>(reinterpret_cast<const RT*>(p), cols, v);
          else load_row_dyn<LAY>(p, a.gate_type, 0, cols, v);
        },
        [&] {
          // every thread has read the stage: the second sum's barrier, or one more
          if (a.warps == 1) __syncwarp();
          else if (!two) __syncthreads();
          const int64_t next = row + static_cast<int64_t>(g.stages) * step;
          if (threadIdx.x == 0 && ok && next < a.rows) ring_fetch(g, static_cast<int>(next), src, &full[stage]);
        });
    parity ^= 1;
    if (ok && ++stage == g.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (!ok && threadIdx.x == 0)   // given up: the loads in flight land first
    for (int i = 0; i < g.stages; ++i) {
      int none = 0;
      if (row0 + static_cast<int64_t>(i) * step < a.rows)
        mbar_wait(&full[i], i >= stage ? phase : phase ^ 1u, &none, &g_op_status, kStWaitDrain);
    }
  bwd_store_sums<LAY>(a, sum, reinterpret_cast<float*>(ring + factor_bytes));
}

// Adds up the parts of a column, 32 columns per CTA: eight parts per warp in flight together, the
// warps' sums in their order.  blockIdx.y selects the sum: that of dx r^ is dpre_weight; that of G y^
// gives dpost_weight and the gradient of a gate per column.  Bound by the loads' latency: 148 parts
// of 7168 columns about 4 us behind the rows; 1184 parts of 700 took 22 us with eight warps and one load at a time.
struct NormSumArgs {
  const float* partial;
  float *pre, *post, *gate;
  const void *post_w, *chan;   // chan: the gate per column
  int parts, cols, pre_slot, post_type, chan_type;
  float scale, off;
};
__global__ void __launch_bounds__(1024) norm_sum_kernel(NormSumArgs a) {
  __shared__ float buf[32][32];
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x * 32 + threadIdx.x, warps = blockDim.y;
  const float* p = a.partial + static_cast<int64_t>(blockIdx.y) * a.parts * a.cols + c;
  float s = 0.f;
  if (c < a.cols)
    for (int i = threadIdx.y; i < a.parts; i += 8 * warps) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = i + j * warps < a.parts ? p[static_cast<int64_t>(i + j * warps) * a.cols] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
  buf[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || c >= a.cols) return;
  for (int w = 1; w < warps; ++w) s += buf[w][threadIdx.x];
  if (static_cast<int>(blockIdx.y) == a.pre_slot) {
    a.pre[c] = s;
    return;
  }
  const float k = a.scale * s;
  if (a.post) a.post[c] = a.chan ? k * load1_dyn(a.chan, a.chan_type, c) : k;
  if (a.gate) a.gate[c] = a.post_w ? k * (load1_dyn(a.post_w, a.post_type, c) + a.off) : k;
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

// CTAs and with them the parts of the column sums, from the sizes alone (the workspace's size
// goes by them): 148 SMs, each with 512 threads' worth of registers.
struct NormBwdShape {
  int warps, direct_parts, ring_ctas, ring_rows, ring_parts;   // ring_rows: rows side by side in a CTA
  int lanes, packed_rows, packed_parts;
  int thin_warps, thin_rows, thin_parts;   // 0: too long
};
NormBwdShape bwd_shape(int rows, int cols) {
  NormBwdShape s{};
  if (rows < 1) rows = 1;
  int rpc;
  norm_shape(cols, &s.warps, &rpc);
  const int per_sm = s.warps > 16 ? 1 : 16 / s.warps;
  s.direct_parts = rows < 148 * per_sm ? rows : 148 * per_sm;
  if (s.warps <= 16) {
    s.ring_rows = 1;
    s.ring_ctas = per_sm;
    if (s.warps == 1) {   // few rows spread over the SMs, many share a CTA's final sum
      s.ring_ctas = 2;
      const int even = (rows + 148 * 2 - 1) / (148 * 2);
      s.ring_rows = even < 8 ? even : 8;
    }
    const int need = (rows + s.ring_rows - 1) / s.ring_rows;
    s.ring_parts = need < 148 * s.ring_ctas ? need : 148 * s.ring_ctas;
  }
  s.lanes = packed_lanes(cols);
  const int of_warp = s.lanes < 32 ? 32 / s.lanes : 1;   // whole warps, few rows spread over the SMs
  const int even = ((rows + 147) / 148 + of_warp - 1) / of_warp * of_warp;
  s.packed_rows = even < 16 * of_warp ? even : 16 * of_warp;
  const int need = (rows + s.packed_rows - 1) / s.packed_rows;
  s.packed_parts = need < 148 ? need : 148;
  if (cols <= 32 * 256) {   // 1024 threads of an SM, four or eight elements each
    s.thin_warps = cols <= 32 * 128 ? (cols + 127) / 128 : (cols + 255) / 256;
    // rows of one warp need no barrier, 32 of them make a CTA; 16 warps of longer ones
    const int side = s.thin_warps == 1 ? 32 : s.thin_warps <= 8 ? 16 / s.thin_warps : 1;
    const int per_sm = 32 / (side * s.thin_warps), each = (rows + 148 * per_sm - 1) / (148 * per_sm);
    s.thin_rows = each < side ? each : side;
    const int ctas = 148 * per_sm;
    const int wanted = (rows + s.thin_rows - 1) / s.thin_rows;
    s.thin_parts = wanted < ctas ? wanted : ctas;
  }
  return s;
}

bool shared_factors(int residual_type) { return type_bytes(residual_type) == 2; }   // as the ring kernel has them

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

cudaError_t norm_bwd_status(cudaStream_t st, bool clear, int* v) { return take_status(st, clear, v); }

}  // namespace moe

extern "C" {

MOE_B200_API size_t moe_b200_block_norm_backward_workspace_size(int32_t rows, int32_t cols) {
  using namespace moe;
  if (rows < 0 || rows > kOpMaxRows || cols < 1 || cols > kNormMaxCols) return 0;
  const NormBwdShape shape = bwd_shape(rows, cols);
  int parts = shape.direct_parts > shape.ring_parts ? shape.direct_parts : shape.ring_parts;
  if (parts < shape.packed_parts) parts = shape.packed_parts;
  if (parts < shape.thin_parts) parts = shape.thin_parts;
  return static_cast<size_t>(align256(static_cast<int64_t>(2) * parts * cols * 4) + align256(static_cast<int64_t>(rows) * 4) +
                             256);
}

MOE_B200_API int moe_b200_block_norm_backward(const moe_b200_norm_backward_args* a, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->rows < 0 || a->rows > kOpMaxRows || a->cols < 1 || a->cols > kNormMaxCols)
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: rows must be in [0, 2^30] and cols in [1, 16384]");
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
    return report_error(MOE_B200_ERR_ARG, "block_norm_backward: with a y of fp32 the residual is fp32 too (types bf16, fp16, fp32)");
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
  n.scale = a->scale;
  n.eps = a->eps;
  n.off = a->weight_offset;
  n.partial = static_cast<float*>(workspace);
  n.gate_grad = !a->gate ? kGateNone : g_rows && g_cols ? kGateElement : g_cols ? kGateColumn : kGateRow;
  NormSumArgs s{};
  int sums = 0;
  n.pre_slot = n.post_slot = -1;
  if (a->dx) {
    n.pre_slot = sums;
    s.pre = a->dpre_weight;
    ++sums;
  }
  if (a->post_weight || n.gate_grad == kGateColumn) {
    n.post_slot = sums;
    s.post = a->post_weight ? a->dpost_weight : nullptr;
    s.gate = n.gate_grad == kGateColumn ? static_cast<float*>(a->dgate) : nullptr;
    ++sums;
  }
  const bool vec = a->cols % 8 == 0 && rows_aligned(a->y, n.y_ld, a->y_type) &&
                   rows_aligned(a->dx, n.dx_ld, a->y_type) && rows_aligned(a->dresidual, n.dr_ld, a->residual_type) &&
                   rows_aligned(n.r, n.r_ld, a->residual_type) &&
                   rows_aligned(a->dresidual_in, n.dres_ld, a->residual_type) &&
                   rows_aligned(a->dy, n.dy_ld, a->y_type) && aligned16(a->post_weight) && aligned16(a->pre_weight) &&
                   (!g_cols || rows_aligned(a->gate, n.g_ld, a->gate_type)) &&
                   (n.gate_grad != kGateElement || rows_aligned(a->dgate, n.dg_ld, a->gate_type));
  const NormBwdShape shape = bwd_shape(a->rows, a->cols);
  n.warps = shape.warps;
  RingPlan g{};
  ring_add(&g, a->dx, n.dx_ld, a->cols, a->y_type);
  ring_add(&g, n.r, n.r_ld, a->cols, a->residual_type);
  ring_add(&g, a->y, n.y_ld, a->cols, a->y_type);
  ring_add(&g, a->dresidual, n.dr_ld, a->cols, a->residual_type);
  if (n.gate_grad == kGateElement) ring_add(&g, a->gate, n.g_ld, a->cols, a->gate_type);
  const int factors = shared_factors(a->residual_type) ? kFactorBytes * n.warps * 32 : 0;
  g.stages = shape.ring_ctas ? (kRingSmem / shape.ring_ctas - factors) / shape.ring_rows / g.stage_bytes : 0;
  if (g.stages > kRingMaxStages) g.stages = kRingMaxStages;
  // rows of up to 256 columns: several to a warp; odd ones: kThin; the ring takes the others that have dx
  const bool packed = vec && a->cols <= 256;
  const bool ring = vec && !packed && a->dx && g.stages >= 1;
  const bool thin = !vec && shape.thin_warps > 0;
  n.parts = packed ? shape.packed_parts : thin ? shape.thin_parts : ring ? shape.ring_parts : shape.direct_parts;
  // the row sums of a gate that is one number go through the workspace
  float* row_dots = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                             align256(static_cast<int64_t>(2) * n.parts * a->cols * 4));
  n.dgate = n.gate_grad == kGateElement ? a->dgate : n.gate_grad == kGateRow ? (g_rows ? a->dgate : row_dots) : nullptr;
  dispatch_types(a->y_type, a->residual_type, [&](auto yt, auto rt) {
    using YT = decltype(yt);
    using RT = decltype(rt);
    if (ring) {
      auto of_gate = [&](auto lay, auto post) {
        constexpr int L = decltype(lay)::value, P = decltype(post)::value;
        return n.gate_grad == kGateElement ? norm_bwd_ring_kernel<YT, RT, L, P, 2>
               : n.gate_grad == kGateRow   ? norm_bwd_ring_kernel<YT, RT, L, P, 1>
                                           : norm_bwd_ring_kernel<YT, RT, L, P, 0>;
      };
      auto of_post = [&](auto lay) {
        return !a->y            ? norm_bwd_ring_kernel<YT, RT, decltype(lay)::value, 0, kNoBlock>
               : a->post_weight ? of_gate(lay, std::integral_constant<int, 1>{}) : of_gate(lay, std::integral_constant<int, 0>{});
      };
      auto kernel = a->cols == n.warps * 32 * kNormPerThread ? of_post(std::integral_constant<int, kFull>{})
                                                             : of_post(std::integral_constant<int, kHalf>{});
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
      if (e == cudaSuccess)
        e = launch_pdl(kernel, dim3(n.parts), dim3(n.warps * 32, shape.ring_rows),
                       factors + static_cast<size_t>(g.stages) * g.stage_bytes * shape.ring_rows, st, n, g);
    } else {
      if (thin) n.warps = shape.thin_warps;
      auto kernel = packed          ? norm_bwd_kernel<YT, RT, kPacked, 512>
                    : thin          ? (a->cols <= 32 * 128 ? norm_bwd_kernel<YT, RT, kShort, 1024>
                                                      : norm_bwd_kernel<YT, RT, kThin, 1024>)
                    : !vec          ? norm_bwd_kernel<YT, RT, kTail, 1024>
                    : n.warps <= 16 ? norm_bwd_kernel<YT, RT, kVec, 512>
                                    : norm_bwd_kernel<YT, RT, kVec, 1024>;
      const int side = packed ? shape.packed_rows : thin ? shape.thin_rows : 1;   // rows of a CTA
      const dim3 block(packed ? shape.lanes : n.warps * 32, side);
      const int quads = !thin ? 8 : a->cols <= 32 * 128 ? 2 : 4;   // factors of a thread
      const size_t smem = sizeof(float4) * quads * block.x + (side > 1 ? sizeof(float) * side * a->cols : 0);
      // 48 KB are what a launch may have unasked, the 6 KB of the kernel's own buffers among them
      if (smem + sizeof(float) * 2 * kBwdSide * 3 * 32 > 48 * 1024)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
      if (e == cudaSuccess) e = launch_pdl(kernel, dim3(n.parts), block, smem, st, n);
    }
  });
  if (e != cudaSuccess) return report_cuda(e, "block_norm_backward launch");
  if (sums) {
    s.partial = n.partial;
    s.parts = n.parts;
    s.cols = a->cols;
    s.pre_slot = n.pre_slot;
    s.post_w = a->post_weight;
    s.post_type = a->post_weight_type;
    s.chan = n.gate_grad == kGateColumn ? a->gate : nullptr;
    s.chan_type = a->gate_type;
    s.scale = a->scale;
    s.off = a->weight_offset;
    const int sum_warps = n.parts < 8 * 32 ? (n.parts + 7) / 8 : 32;   // eight parts each, then rounds
    e = launch_pdl(norm_sum_kernel, dim3((a->cols + 31) / 32, sums), dim3(32, sum_warps), 0, st, s);
    if (e != cudaSuccess) return report_cuda(e, "block_norm_backward sum launch");
  }
  if (n.gate_grad == kGateRow && !g_rows) {
    e = launch_pdl(norm_total_kernel, dim3(1), dim3(1024), 0, st, static_cast<const float*>(row_dots), a->rows,
                   static_cast<float*>(a->dgate));
    if (e != cudaSuccess) return report_cuda(e, "block_norm_backward total launch");
  }
  return MOE_B200_OK;
}

}  // extern "C"
