// Products of 8-bit integers with one scale per token and one per output channel, on tcgen05
// (kind::i8: exact 32-bit integer sums in TMEM).
//
//   y[t][n] = (sx[t] * sw[n]) * sum_k q[t][k] * w[n][k]  (+ bias[n])
//
// stream: few tokens, bound by reading the weights once.  The weights are the MMA's M side (128
//   rows), up to 256 tokens its N side; K is split over the CTAs of a cluster, whose integer
//   partial sums meet in distributed shared memory (exact in any order).  16 x 4096 x
//   7168 7.9 us (the weights' 29 MB alone 4.5), 64 tokens 10.1, 256 14.4, 512 19.0; from bf16, with the
//   quantisation, 9.6, 12.1, 16.9 and 22.6; 80 x 7168 x 2048 with the activation 9.1.  The launches,
//   the filling of the pipeline and the joining of the partial sums are the rest.
// wide: many tokens, bound by the tensor cores.  Persistent pairs of CTAs, each pair one 256 x 256
//   output tile at a time (cta_group::2: each CTA loads half of either operand, 32 KB per 128
//   bytes of K for 256 x 256 x 128 products), two TMEM accumulators so that one tile's epilogue
//   runs under the next tile's products.  8192 x 4096 x 7168: 146 to 151 us, 3.2 to 3.3 POP/s (the
//   measured 16-bit rate of the card doubled is 3.34); 8192 x 4095 x 7168, whose outputs go through
//   shared memory, 160.
//
// Every wait is bounded (2 s); one that runs out is recorded in g_op_status.
#include "int8_gemm.cuh"

namespace moe {

// 32 consecutive outputs of a row, n of which exist.  align: bytes that every such address is a
// multiple of (32 or 16: whole vectors).
template <class YT>
__device__ __forceinline__ void store_cols32(YT* dst, int n, int align, const float* v) {
  if (n >= 32) {
#pragma unroll
    for (int i = 0; i < 32; i += 32 / static_cast<int>(sizeof(YT))) {
      uint32_t p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(YT) == 4) p[j] = __float_as_uint(v[i + j]);
        else p[j] = pack2(v[i + 2 * j], v[i + 2 * j + 1], YT{});
      }
      if (align == 32) {
        st_global_v8_b32(dst + i, p);
      } else {
        reinterpret_cast<uint4*>(dst + i)[0] = make_uint4(p[0], p[1], p[2], p[3]);
        reinterpret_cast<uint4*>(dst + i)[1] = make_uint4(p[4], p[5], p[6], p[7]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) dst[i] = from_f<YT>(v[i]);
  }
}

// 32 lanes x 32 consecutive columns, complete on return.
__device__ __forceinline__ void tmem_ld32_wait(uint32_t ta, int* v) {
  uint32_t r[32];
  tmem_ld16x2_issue(ta, ta + 16, r);
  tmem_wait_ld32(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = static_cast<int>(r[i]);
}

// ---------------------------------------------------------------- wide
constexpr int kIWStages = 6;
constexpr int kIWStageBytes = 32768;     // 128 token rows | 128 weight rows of 128 bytes
// Rows of one bulk copy.  A box's loads go through the copy unit one after another; two per operand
// half keep it busier than one (8192 x 4096 x 7168: 152 us with 128 rows, 146 with 64), smaller ones
// cost more in their number (176 with 32, 263 with 16).
constexpr int kIWBox = 64;
constexpr int kIWThreads = 320;          // producer, MMA, 8 epilogue warps
constexpr int kIWEpiThreads = 256;
constexpr int kIWGroup = 8;              // token tiles whose weight tiles run together (L2 reuse)

// Beside the stages, which are dynamic shared memory at a 1024-byte boundary.
struct IntWideSmem {
  uint64_t full[kIWStages], empty[kIWStages];
  uint64_t tfull[2], tempty[2];
  alignas(16) float sw[2][256];
  float bias[2][256];
  float turn[8][32][17];   // unaligned outputs: 16 columns of a warp's 32 rows, turned to whole rows
  uint32_t tmem_base;
  int abort;
};
constexpr size_t kIWSmemBytes = kIWStages * kIWStageBytes + 1024;
static_assert(kIWSmemBytes + sizeof(IntWideSmem) <= 232448, "wide int8 kernel shared memory");

// Tile order: blocks of kIWGroup token tiles, all weight tiles of a block before the next, token
// tiles fastest, so that the tiles in flight share few rows of either operand.
__device__ __forceinline__ void iw_tile(int tile, int mt, int nt, int* m, int* n) {
  const int per = kIWGroup * nt, g = tile / per, r = tile - g * per;
  const int rows = min(kIWGroup, mt - g * kIWGroup);
  *n = r / rows;
  *m = g * kIWGroup + r - *n * rows;
}

template <class YT>
__global__ void __launch_bounds__(kIWThreads, 1)
    int8_wide_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmW, LinearArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ IntWideSmem sm;
  const uint32_t stages = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int mt = (a.T + 255) / 256, nt = (a.N + 255) / 256, tiles = mt * nt, kbs = (a.K + 127) / 128;
  if (threadIdx.x == 0) {
    sm.abort = 0;
    for (int i = 0; i < kIWStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.tfull[i], 1);
      mbar_init(&sm.tempty[i], 16);   // 8 epilogue warps of each CTA
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&sm.tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers and TMEM exist before either touches the other's
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  pdl_launch_dependents();

  if (warp == 0) {
    // producer: this CTA's 128 rows of either operand; the bytes of both CTAs complete on the
    // even CTA's barrier, whose thread issues the pair's products
    uint32_t stage = 0, phase = 0, last = 0;   // last: bit s = parity of stage s's latest load
    int issued = 0;
    bool waited = false, ok = true;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      int m, n;
      iw_tile(tile, mt, nt, &m, &n);
      const int y0 = m * 256 + 128 * rank, y1 = n * 256 + 128 * static_cast<int>(rank);
      for (int kb = 0; kb < kbs; ++kb) {
        ok = __all_sync(0xffffffffu,
                        mbar_wait(&sm.empty[stage], phase ^ 1u, &sm.abort, &g_op_status, kStWaitProducer));
        if (!ok) break;
        if (!waited) {
          pdl_wait();
          waited = true;
        }
        if (rank == 0 && lane == 0) mbar_arrive_expect_tx(&sm.full[stage], 2 * kIWStageBytes);
        __syncwarp();
        const uint32_t bar = cluster_addr(smem_u32(&sm.full[stage]), 0);
        // lane l loads box l: token rows first, then weight rows
        constexpr int kQBoxes = 128 / kIWBox, kBoxes = 2 * kQBoxes;
        if (lane < kBoxes) {
          const bool is_q = lane < kQBoxes;
          tma_load_2d_pair(stages + stage * kIWStageBytes + lane * kIWBox * 128, is_q ? &tmQ : &tmW, bar, kb * 128,
                           is_q ? y0 + lane * kIWBox : y1 + (lane - kQBoxes) * kIWBox);
        }
        last = (last & ~(1u << stage)) | (phase << stage);
        issued = max(issued, static_cast<int>(stage) + 1);
        if (++stage == kIWStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // given up: the pair's loads in flight, of which the even CTA's barriers know, land first
    if (!ok && rank == 0 && lane == 0)
      for (int i = 0; i < issued; ++i) {
        int none = 0;
        mbar_wait(&sm.full[i], (last >> i) & 1u, &none, &g_op_status, kStWaitDrain);
      }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = idesc_s8_s32(256, 256);
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++it) {
        const int buf = it & 1;
        if (!mbar_wait(&sm.tempty[buf], ((it >> 1) & 1) ^ 1, &sm.abort, &g_op_status, kStWaitMmaTmem)) break;
        tc_fence_after();
        for (int kb = 0; kb < kbs; ++kb) {
          ok = mbar_wait(&sm.full[stage], phase, &sm.abort, &g_op_status, kStWaitMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t st = stages + stage * kIWStageBytes;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_i8_pair(tmem + buf * 256u, sdesc_k128_sw128(st + 32 * k), sdesc_k128_sw128(st + 16384 + 32 * k), idesc,
                        (kb | k) > 0);
          mma_commit_pair(&sm.empty[stage]);
          if (++stage == kIWStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        mma_commit_pair(&sm.tfull[buf]);
      }
    }
  } else {
    // epilogue: lane quarter warp & 3 (32 token rows), column half (warp - 2) / 4
    const int q = warp & 3, h = (warp - 2) >> 2, et = threadIdx.x - 64;
    // rows of outputs on 32- or 16-byte boundaries are stored by their thread as whole vectors;
    // others go through shared memory, so that a warp stores neighbours (2 rows x 16 columns)
    auto on = [&](uint64_t n) { return reinterpret_cast<uintptr_t>(a.y) % n == 0 && (a.y_ld * sizeof(YT)) % n == 0; };
    const int align = on(32) ? 32 : on(16) ? 16 : 0;
    float (*turn)[17] = sm.turn[warp - 2];
    pdl_wait();
    bool dead = false;
    int it = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++it) {
      const int buf = it & 1;
      int m, n;
      iw_tile(tile, mt, nt, &m, &n);
      const int t = m * 256 + 128 * rank + 32 * q + lane;
      {
        const int c = n * 256 + et;
        sm.sw[buf][et] = c < a.N ? a.sw[c] : 0.f;
        sm.bias[buf][et] = a.bias && c < a.N ? load1_dyn(a.bias, a.bias_type, c) : 0.f;
      }
      const float sx = t < a.T ? a.sx[t] : 0.f;
      named_bar_sync(1, kIWEpiThreads);
      // after an abort the warps still meet at every tile's barrier
      if (!dead) {
        const bool ok = mbar_wait(&sm.tfull[buf], (it >> 1) & 1, &sm.abort, &g_op_status, kStWaitEpilogue);
        dead = !__all_sync(0xffffffffu, ok);
      }
      if (dead) continue;
      tc_fence_after();
      const uint32_t ta = tmem + (static_cast<uint32_t>(32 * q) << 16) + buf * 256u + 128u * h;
      // the accumulator's next 32 columns are read while these are stored
      uint32_t acc[2][32];
      tmem_ld16x2_issue(ta, ta + 16, acc[0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c0 = 32 * i;
        tmem_wait_ld32(acc[i & 1]);
        if (i < 3) {
          tmem_ld16x2_issue(ta + c0 + 32, ta + c0 + 48, acc[(i + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_u32(&sm.tempty[buf]), 0));
        }
        const float4* swp = reinterpret_cast<const float4*>(&sm.sw[buf][128 * h + c0]);
        const float4* bp = reinterpret_cast<const float4*>(&sm.bias[buf][128 * h + c0]);
        float v[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 w4 = swp[j], b4 = bp[j];
          const uint32_t* u = acc[i & 1] + 4 * j;
          v[4 * j] = fmaf(static_cast<float>(static_cast<int>(u[0])), sx * w4.x, b4.x);
          v[4 * j + 1] = fmaf(static_cast<float>(static_cast<int>(u[1])), sx * w4.y, b4.y);
          v[4 * j + 2] = fmaf(static_cast<float>(static_cast<int>(u[2])), sx * w4.z, b4.z);
          v[4 * j + 3] = fmaf(static_cast<float>(static_cast<int>(u[3])), sx * w4.w, b4.w);
        }
        const int col = n * 256 + 128 * h + c0;
        if (align) {
          if (t < a.T) store_cols32(static_cast<YT*>(a.y) + t * a.y_ld + col, a.N - col, align, v);
        } else {
          const int row0 = m * 256 + 128 * static_cast<int>(rank) + 32 * q;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) turn[lane][j] = v[16 * half + j];
            __syncwarp();
            const int cc = col + 16 * half + (lane & 15);
            if (cc < a.N)
#pragma unroll 4
              for (int r = lane >> 4; r < 32; r += 2)
                if (row0 + r < a.T) static_cast<YT*>(a.y)[(row0 + r) * a.y_ld + cc] = from_f<YT>(turn[r][lane & 15]);
          }
        }
      }
    }
  }
  // no CTA leaves while the other's products still read its shared memory: the epilogue warps
  // have seen every tile's products complete
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------- stream
constexpr int kISThreads = 320;          // producer, MMA, 8 epilogue warps
constexpr int kISEpiThreads = 256;
constexpr int kISMaxStages = 8;

struct IntStreamCtl {
  uint64_t full[kISMaxStages], empty[kISMaxStages];
  uint64_t tfull;
  uint32_t tmem_base;
  int abort;
};

// Adds up the S partial sums of token columns c0, c0 + 8, ... < c1 of the tile (a warp one column at
// a time, a lane four neighbouring outputs) and stores them; the loads of as many columns as make
// 16 vectors are in flight together.
template <class YT, int S>
__device__ __forceinline__ void is_finish(const LinearArgs& a, uint32_t part, int n0, int t0, int c0, int c1, int lane) {
  constexpr int C = S == 1 ? 8 : 16 / S;
  const int n = n0 + 4 * lane;
  float sw[4], bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sw[j] = n + j < a.N ? a.sw[n + j] : 0.f;
    bias[j] = a.bias && n + j < a.N ? load1_dyn(a.bias, a.bias_type, n + j) : 0.f;
  }
  const bool vec = n + 4 <= a.N && reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(YT)) == 0 && a.y_ld % 4 == 0;
  uint32_t from[S];
#pragma unroll
  for (int s = 0; s < S; ++s) from[s] = (S > 1 ? cluster_addr(part, s) : part) + 16 * lane;
  for (int c = c0; c < c1; c += 8 * C) {
    int4 v[C][S];
    float sx[C];
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (c + 8 * k < c1) {
#pragma unroll
        for (int s = 0; s < S; ++s) v[k][s] = ld_cluster_v4(from[s] + (c + 8 * k) * 512);
        sx[k] = a.sx[t0 + c + 8 * k];
      }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (c + 8 * k >= c1) break;
      int4 sum = v[k][0];
#pragma unroll
      for (int s = 1; s < S; ++s) {
        sum.x += v[k][s].x;
        sum.y += v[k][s].y;
        sum.z += v[k][s].z;
        sum.w += v[k][s].w;
      }
      float o[4] = {static_cast<float>(sum.x), static_cast<float>(sum.y), static_cast<float>(sum.z),
                    static_cast<float>(sum.w)};
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(o[j], sx[k] * sw[j], bias[j]);
      YT* dst = static_cast<YT*>(a.y) + (t0 + c + 8 * k) * a.y_ld + n;
      if (vec) {
        if constexpr (sizeof(YT) == 4) *reinterpret_cast<float4*>(dst) = make_float4(o[0], o[1], o[2], o[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(o[0], o[1], YT{}), pack2(o[2], o[3], YT{}));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) dst[j] = from_f<YT>(o[j]);
      }
    }
  }
}

// grid (splits * weight tiles, token tiles), clusters of `splits` CTAs along x.  Token tile: tn
// rows (a multiple of 16, at most 256); stages of 16 KB of weights and tn x 128 bytes of tokens.
// The integer partial sums [tn][128] of a split CTA reuse the stages.
template <class YT>
__global__ void __launch_bounds__(kISThreads, 2) int8_stream_kernel(const __grid_constant__ CUtensorMap tmQ,
                                                                 const __grid_constant__ CUtensorMap tmW, LinearArgs a,
                                                                 int splits, int tn, int stages, uint32_t tmem_cols) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ IntStreamCtl sm;
  uint8_t* base =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / splits * 128, t0 = blockIdx.y * tn;
  const int kbs = (a.K + 127) / 128;
  const int k0 = kbs * split / splits, k1 = kbs * (split + 1) / splits;
  const int stage_bytes = 16384 + tn * 128;
  if (threadIdx.x == 0) {
    sm.abort = 0;
    for (int i = 0; i < stages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.tfull, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  pdl_launch_dependents();

  bool ok = true;
  if (warp == 0) {
    auto load_w = [&](int stage, int kb) {
      if (lane == 0) tma_load_2d(base + stage * stage_bytes, &tmW, &sm.full[stage], kb * 128, n0);
    };
    auto load_q = [&](int stage, int kb) {
      if (lane == 1) tma_load_2d(base + stage * stage_bytes + 16384, &tmQ, &sm.full[stage], kb * 128, t0);
    };
    // weights of the first stages start before the wait for the kernel that writes q and sx
    if (!a.early_w) pdl_wait();
    const int ahead = min(stages, k1 - k0);
    for (int i = 0; i < ahead; ++i) {
      if (lane == 0) mbar_arrive_expect_tx(&sm.full[i], stage_bytes);
      __syncwarp();
      load_w(i, k0 + i);
    }
    if (a.early_w) pdl_wait();
    for (int i = 0; i < ahead; ++i) load_q(i, k0 + i);
    uint32_t stage = 0, phase = 0, last = 0;   // last: bit s = parity of stage s's latest load
    for (int kb = k0 + ahead; kb < k1; ++kb) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sm.empty[stage], phase, &sm.abort, &g_op_status, kStWaitProducer));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], stage_bytes);
      __syncwarp();
      load_w(stage, kb);
      load_q(stage, kb);
      last = (last & ~(1u << stage)) | ((phase ^ 1u) << stage);
      if (++stage == static_cast<uint32_t>(stages)) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok && lane == 0)   // given up: the loads in flight land first
      for (int i = 0; i < ahead; ++i) {
        int none = 0;
        mbar_wait(&sm.full[i], (last >> i) & 1u, &none, &g_op_status, kStWaitDrain);
      }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_s8_s32(128, tn);
      uint32_t stage = 0, phase = 0;
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(&sm.full[stage], phase, &sm.abort, &g_op_status, kStWaitMma)) break;
        tc_fence_after();
        const uint32_t st = smem_u32(base + stage * stage_bytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_i8(tmem, sdesc_k128_sw128(st + 32 * k), sdesc_k128_sw128(st + 16384 + 32 * k), idesc,
                 (kb - k0) | k);
        mma_commit(&sm.empty[stage]);
        if (++stage == static_cast<uint32_t>(stages)) {
          stage = 0;
          phase ^= 1u;
        }
      }
      mma_commit(&sm.tfull);
    }
  }
  __syncwarp();
  const int live = min(tn, a.T - t0);
  const uint32_t part = smem_u32(base);        // int [live][128] partial sums, in place of the stages
  if (warp >= 2) {
    pdl_wait();
    ok = mbar_wait(&sm.tfull, 0, &sm.abort, &g_op_status, kStWaitEpilogue);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      // every load and product of this CTA is complete: the stages are free
      const int q = warp & 3, r = 32 * q + lane;   // this thread's weight row of the tile
      for (int c0 = warp < 6 ? 0 : 32; c0 < live; c0 += 64) {
        int acc[32];
        tmem_ld32_wait(tmem + (static_cast<uint32_t>(32 * q) << 16) + c0, acc);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (c0 + i < live) st_shared_s32(part + ((c0 + i) * 128 + r) * 4, acc[i]);
      }
    }
    if (splits > 1) cluster_sync();
    else named_bar_sync(1, kISEpiThreads);
    // CTA `split` finishes its share of the token columns
    const int c0 = live * split / splits + warp - 2, c1 = live * (split + 1) / splits;
    if (splits == 8) is_finish<YT, 8>(a, part, n0, t0, c0, c1, lane);
    else if (splits == 4) is_finish<YT, 4>(a, part, n0, t0, c0, c1, lane);
    else if (splits == 2) is_finish<YT, 2>(a, part, n0, t0, c0, c1, lane);
    else is_finish<YT, 1>(a, part, n0, t0, c0, c1, lane);
    if (splits > 1) cluster_sync();   // the others have read this CTA's partial sums
  } else if (splits > 1) {
    cluster_sync();
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, tmem_cols);
}

namespace {

template <class F>
cudaError_t with_y_type(int type, F&& f) {
  return type == MOE_B200_BF16 ? f(bf16{}) : type == MOE_B200_FP16 ? f(fp16{}) : f(float{});
}

cudaError_t int8_wide_launch(const int8_t* q, int64_t q_ld, const int8_t* w, int64_t w_ld, const LinearArgs& a,
                             int sms, cudaStream_t st) {
  // (Tiles of 256 x 128 for twice the SMs at work gain nothing: an MMA of half the width takes nearly
  // as long.  512 x 4096 x 7168: 21.9 us with 256 x 256, 20.5 with 256 x 128; 18.9 in the streaming kernel,
  // which splits K.)
  const int pairs = sms / 2, tiles = ((a.T + 255) / 256) * ((a.N + 255) / 256);
  CUtensorMap mq, mw;
  if (!encode_rows_u8(&mq, q, a.K, a.T, q_ld, kIWBox) || !encode_rows_u8(&mw, w, a.K, a.N, w_ld, kIWBox))
    return cudaErrorInvalidValue;
  return with_y_type(a.y_type, [&](auto yt) {
    auto kernel = int8_wide_kernel<decltype(yt)>;
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), kIWSmemBytes);
    if (e != cudaSuccess) return e;
    return launch_cluster_pdl(kernel, dim3(2 * (tiles < pairs ? tiles : pairs)), dim3(kIWThreads), kIWSmemBytes, 2, st, mq,
                              mw, a);
  });
}

cudaError_t int8_stream_launch(const int8_t* q, int64_t q_ld, const int8_t* w, int64_t w_ld, const LinearArgs& a,
                               int sms, cudaStream_t st) {
  const int tt = (a.T + 255) / 256;
  int tn = ((a.T + tt - 1) / tt + 15) / 16 * 16;
  const int kbs = (a.K + 127) / 128, nt = (a.N + 127) / 128;
  // Split K until the CTAs fill the GPU about once (twice where two fit an SM), at least two
  // 128-byte steps each.  Clusters of eight only where two CTAs fit an SM: of one-per-SM clusters a
  // part of the GPU holds two and leaves SMs over (1000 x 512 x 4096: 18.6 us in eights).
  const int slots = tn <= 64 ? 2 * sms : sms, most = tn <= 64 ? 8 : 4;
  int splits = 1;
  while (splits < most && nt * tt * splits * 2 <= slots && kbs >= 4 * splits) splits *= 2;
  const int stage_bytes = 16384 + tn * 128;
  const int room = tn <= 64 ? 100 * 1024 : 200 * 1024;
  int stages = room / stage_bytes;
  if (stages > kISMaxStages) stages = kISMaxStages;
  uint32_t cols = 32;
  while (cols < static_cast<uint32_t>(tn)) cols *= 2;
  const size_t smem = static_cast<size_t>(stages) * stage_bytes + 1024;
  CUtensorMap mq, mw;
  if (!encode_rows_u8(&mq, q, a.K, a.T, q_ld, tn) || !encode_rows_u8(&mw, w, a.K, a.N, w_ld, 128))
    return cudaErrorInvalidValue;
  return with_y_type(a.y_type, [&](auto yt) {
    auto kernel = int8_stream_kernel<decltype(yt)>;
    static SmemOnce once;
    const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), 210 * 1024);
    if (e != cudaSuccess) return e;
    return launch_cluster_pdl(kernel, dim3(nt * splits, tt), dim3(kISThreads), smem, splits, st, mq, mw, a, splits, tn,
                              stages, cols);
  });
}

}  // namespace

// Up to 256 tokens: stream.  Beyond that, stream only where its tiles are few enough to be split over
// K and K is long enough to gain by it: 512 x 4096 x 7168 18.9 us against 21.3 wide, 512 x 2048 x 2048
// 10.3 against 9.2, 768 x 4096 x 7168 (unsplit) 27 against 22.
cudaError_t int8_gemm_launch(const int8_t* q, int64_t q_ld, const int8_t* w, int64_t w_ld, const LinearArgs& a, int sms,
                             cudaStream_t st) {
  const int64_t tiles = static_cast<int64_t>((a.T + 255) / 256) * ((a.N + 127) / 128);
  const bool stream = a.T <= 256 || (tiles * 2 <= sms && a.K >= 4096);
  return stream ? int8_stream_launch(q, q_ld, w, w_ld, a, sms, st) : int8_wide_launch(q, q_ld, w, w_ld, a, sms, st);
}

cudaError_t int8_status(cudaStream_t st, bool clear, int* v) { return take_status(st, clear, v); }

}  // namespace moe

extern "C" MOE_B200_API int moe_b200_operator_status(void* stream, int32_t clear) {
  using namespace moe;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int norm = 0, quant = 0, int8 = 0;
  cudaError_t e = norm_status(st, clear, &norm);
  if (e == cudaSuccess) e = quant_status(st, clear, &quant);
  if (e == cudaSuccess) e = int8_status(st, clear, &int8);
  if (e != cudaSuccess) return -report_cuda(e, "operator status");
  return norm ? norm : quant ? quant : int8;
}
