// What the forward and backward norm kernels (norm.cu, norm_bwd.cu) share: how a row lies in the
// registers of a group of warps, packed 32-bit arithmetic, launch shapes.
#pragma once

#include <type_traits>

#include "op_common.cuh"

namespace moe {

constexpr int kNormPerThread = 16;            // elements of a row in a thread
constexpr int kNormMaxCols = 1024 * kNormPerThread;
constexpr int kRingMaxStages = 8;
constexpr int kRingSmem = 216 * 1024;         // of an SM, shared by its CTAs

// Sixteen elements as eight pairs: two fused multiply-adds per instruction (f32x2).
struct Row16 {
  float2 v[8];
  __device__ __forceinline__ float& operator[](int q) { return (q & 1) ? v[q >> 1].y : v[q >> 1].x; }
  __device__ __forceinline__ float operator[](int q) const { return (q & 1) ? v[q >> 1].y : v[q >> 1].x; }
};

__device__ __forceinline__ uint64_t bits2(float2 a) {
  uint64_t u;
  asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(a.x), "f"(a.y));
  return u;
}
__device__ __forceinline__ float2 pair2(uint64_t u) {
  float2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(u));
  return a;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}
__device__ __forceinline__ float2 dup2(float a) { return make_float2(a, a); }

// How a row lies in its threads.  kVec, kHalf, kFull: two chunks of eight neighbours, for 16-byte
// accesses; kHalf: every first chunk exists (rows of at least 256 x their warps, so all of more than
// 256 columns); kFull: every chunk exists (the row is 16 x its threads long), so nothing is checked.
// kScattered: 128-column blocks by warp, lane + 32 m within one, so that the accesses of a warp are
// neighbours whatever the row's alignment.  kTail: the same, where only the last four elements of a
// thread may be missing (rows of at least 384 x their warps, so all of more than 1536 columns).
// kThin, kShort: the same with eight and four elements to a thread.
// In each of these a 128-column block belongs to a half warp (eight elements each) or to a warp (four
// each).  kPacked: as kVec, several rows to a warp: blockDim.x, a power of two below 32, threads each.
enum : int { kShort = -2, kThin = -1, kScattered = 0, kTail = 1, kVec = 2, kHalf = 3, kFull = 4, kPacked = 5 };
constexpr bool is_vec(int lay) { return lay >= kVec; }
constexpr int slots(int lay) { return lay == kShort ? 4 : lay == kThin ? 8 : 16; }

// (kHalf, kFull and kTail say that elements exist without a look at `cols`: they are for rows that exist,
// of the lengths named, and not for a missing row given as one of no columns.)

// The column of this thread's element q.
template <int LAY>
__device__ __forceinline__ int col_of(int q) {
  if constexpr (is_vec(LAY)) return static_cast<int>(threadIdx.x + (q >> 3) * blockDim.x) * 8 + (q & 7);
  return static_cast<int>((threadIdx.x >> 5) + (q >> 2) * (blockDim.x >> 5)) * 128 +
         static_cast<int>(threadIdx.x & 31) + 32 * (q & 3);
}
template <int LAY>
__device__ __forceinline__ bool exists(int q, int cols) {
  if (q >= slots(LAY)) return false;
  return LAY == kFull || (LAY == kHalf && q < 8) || (LAY == kTail && q < 12) || col_of<LAY>(q) < cols;
}

template <class T>
__device__ __forceinline__ void load_chunk(const T* p, float2* v) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = make_float2(a.x, a.y);
    v[1] = make_float2(a.z, a.w);
    v[2] = make_float2(b.x, b.y);
    v[3] = make_float2(b.z, b.w);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    float f[2];
    unpack2(u.x, f, T{});
    v[0] = make_float2(f[0], f[1]);
    unpack2(u.y, f, T{});
    v[1] = make_float2(f[0], f[1]);
    unpack2(u.z, f, T{});
    v[2] = make_float2(f[0], f[1]);
    unpack2(u.w, f, T{});
    v[3] = make_float2(f[0], f[1]);
  }
}

// (The row itself must exist: what lies beyond its end is not read, but where there is nothing to
// read at all, its first element may be.)
template <class T, int LAY>
__device__ __forceinline__ void load_row(const T* row, int cols, Row16& r) {
  if constexpr (is_vec(LAY)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (exists<LAY>(8 * i, cols)) {
        load_chunk(row + col_of<LAY>(8 * i), r.v + 4 * i);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r.v[4 * i + j] = dup2(0.f);
      }
    }
  } else {
    // kScattered: unconditional loads, so that all sixteen are in flight together; a branch around
    // each would wait for it (backward of 5000 x 700: 74 -> 54 us).  The last four of kTail are
    // better left out (forward of 4096 x 5001: 62 -> 57 us).
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const bool ok = exists<LAY>(q, cols);
      if (LAY == kTail || q >= slots(LAY)) {
        r[q] = ok ? to_f(row[col_of<LAY>(q)]) : 0.f;
      } else {
        const float f = to_f(row[ok ? col_of<LAY>(q) : 0]);
        r[q] = ok ? f : 0.f;
      }
    }
  }
}
template <class T, int LAY>
__device__ __forceinline__ void store_row(T* row, int cols, const Row16& r) {
  if constexpr (is_vec(LAY)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!exists<LAY>(8 * i, cols)) continue;
      T* p = row + col_of<LAY>(8 * i);
      const float2* v = r.v + 4 * i;
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
      } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0].x, v[0].y, T{}), pack2(v[1].x, v[1].y, T{}),
                                                  pack2(v[2].x, v[2].y, T{}), pack2(v[3].x, v[3].y, T{}));
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (exists<LAY>(q, cols)) row[col_of<LAY>(q)] = from_f<T>(r[q]);
  }
}
// The same with the type known at run time; `off` in elements.
template <int LAY>
__device__ __forceinline__ void load_row_dyn(const void* p, int type, int64_t off, int cols, Row16& r) {
  if (type == MOE_B200_BF16) load_row<bf16, LAY>(static_cast<const bf16*>(p) + off, cols, r);
  else if (type == MOE_B200_FP16) load_row<fp16, LAY>(static_cast<const fp16*>(p) + off, cols, r);
  else load_row<float, LAY>(static_cast<const float*>(p) + off, cols, r);
}
template <int LAY>
__device__ __forceinline__ void store_row_dyn(void* p, int type, int64_t off, int cols, const Row16& r) {
  if (type == MOE_B200_BF16) store_row<bf16, LAY>(static_cast<bf16*>(p) + off, cols, r);
  else if (type == MOE_B200_FP16) store_row<fp16, LAY>(static_cast<fp16*>(p) + off, cols, r);
  else store_row<float, LAY>(static_cast<float*>(p) + off, cols, r);
}
template <int LAY>
__device__ __forceinline__ void load_weight(const void* p, int type, float off, int cols, Row16& w) {
  load_row_dyn<LAY>(p, type, 0, cols, w);
  if (off == 0.f) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) w.v[i] = add2(w.v[i], dup2(off));
}

// Sum of squares of the elements that exist: those beyond the row are 0 in every tensor, but may
// have met an infinite factor of the row since.
template <int LAY>
__device__ __forceinline__ float squares_existing(const Row16& r, int cols) {
  if constexpr (!is_vec(LAY)) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) s = exists<LAY>(q, cols) ? fmaf(r[q], r[q], s) : s;
    return s;
  } else {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 p = mul2(r.v[4 * i], r.v[4 * i]);
#pragma unroll
      for (int j = 1; j < 4; ++j) p = fma2(r.v[4 * i + j], r.v[4 * i + j], p);
      if (exists<LAY>(8 * i, cols)) s += p.x + p.y;
    }
    return s;
  }
}
template <int LAY>
__device__ __forceinline__ float dot16(const Row16& a, const Row16& b) {
  float2 s = mul2(a.v[0], b.v[0]);
#pragma unroll
  for (int i = 1; i < slots(LAY) / 2; ++i) s = fma2(a.v[i], b.v[i], s);
  return s.x + s.y;
}

// Sums over a row of kPacked.
template <int N>
__device__ __forceinline__ void packed_sum(float (&v)[N]) {
  for (int d = blockDim.x >> 1; d >= 1; d >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], d);
}
// Threads of a row of kPacked.
inline int packed_lanes(int cols) {
  int lanes = 1;
  while (lanes * kNormPerThread < cols) lanes *= 2;
  return lanes;
}

// ---------------------------------------------------------------- rings of rows
// The row tensors that a persistent CTA streams through shared memory: rows of `bytes` bytes,
// `pitch` bytes apart, each with its place in a stage.
struct RingTensor {
  const uint8_t* base;
  int64_t pitch;
  int bytes, at;
};
constexpr int kRingTensors = 5;
struct RingPlan {
  RingTensor t[kRingTensors];
  int n, stages, stage_bytes;
};

// One thread: starts the copies of a row's tensors into a stage, completing on `bar`.
__device__ __forceinline__ void ring_fetch(const RingPlan& g, int row, uint8_t* stage, uint64_t* bar) {
  mbar_arrive_expect_tx(bar, g.stage_bytes);
#pragma unroll
  for (int i = 0; i < kRingTensors; ++i)
    if (i < g.n) bulk_load(stage + g.t[i].at, g.t[i].base + row * g.t[i].pitch, g.t[i].bytes, bar);
}

// Host: adds a tensor of 16-byte aligned rows (not if p is null).
inline void ring_add(RingPlan* g, const void* p, int64_t ld, int cols, int type) {
  if (!p) return;
  RingTensor& t = g->t[g->n++];
  t.base = static_cast<const uint8_t*>(p);
  t.pitch = ld * type_bytes(type);
  t.bytes = cols * type_bytes(type);
  t.at = g->stage_bytes;
  g->stage_bytes += t.bytes;
}

// Warps of a row and rows of a CTA: a row takes as few warps as hold it; short rows share a CTA
// of up to eight warps.
inline void norm_shape(int cols, int* warps, int* rows_per_cta) {
  *warps = (cols + 32 * kNormPerThread - 1) / (32 * kNormPerThread);
  *rows_per_cta = *warps >= 8 ? 1 : 8 / *warps;
}

// f(y type, residual type)
template <class F>
void dispatch_types(int y_type, int r_type, F&& f) {
  auto with = [&](auto yt) {
    if (r_type == MOE_B200_BF16) f(yt, bf16{});
    else if (r_type == MOE_B200_FP16) f(yt, fp16{});
    else f(yt, float{});
  };
  if (y_type == MOE_B200_BF16) with(bf16{});
  else if (y_type == MOE_B200_FP16) with(fp16{});
  else f(float{}, float{});
}
// A 32-bit y goes with a 32-bit residual.
inline bool type_pair_ok(int y, int r) {
  return is_float_type(y) && is_float_type(r) && (y != MOE_B200_FP32 || r == MOE_B200_FP32);
}

}  // namespace moe
