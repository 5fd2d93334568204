// What the forward and backward norm kernels (norm.cu, norm_bwd.cu) share: how a row lies in the
// registers of a group of warps, packed 32-bit arithmetic, launch shapes.
#pragma once

#include <type_traits>

#include "op_common.cuh"

namespace moe {

constexpr int kNormPerThread = 16;            // elements of a row in a thread
constexpr int kNormMaxCols = 1024 * kNormPerThread;
constexpr int kRingMaxStages = 8;
constexpr int kRingSmem = 200 * 1024;         // of an SM, shared by its CTAs

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

// Where a thread's element q of its row is.  VEC: two chunks of eight neighbours, for 16-byte
// accesses.  Otherwise 128-column blocks by warp, lane + 32 m within one, so that the accesses of
// a warp are neighbours whatever the row's alignment.  Either way a 128-column block belongs to a
// half warp (eight elements each) or to a warp (four each).
template <bool VEC>
__device__ __forceinline__ int col_of(int q) {
  if constexpr (VEC) return static_cast<int>(threadIdx.x + (q >> 3) * blockDim.x) * 8 + (q & 7);
  return static_cast<int>((threadIdx.x >> 5) + (q >> 2) * (blockDim.x >> 5)) * 128 +
         static_cast<int>(threadIdx.x & 31) + 32 * (q & 3);
}

template <class T, bool VEC>
__device__ __forceinline__ void load_row(const T* row, int cols, Row16& r) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v[8];
      const int e0 = col_of<true>(8 * i);
      load8<T, true>(row + e0, cols - e0, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) r[8 * i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int e = col_of<false>(q);
      r[q] = e < cols ? to_f(row[e]) : 0.f;
    }
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store_row(T* row, int cols, const Row16& r) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v[8];
      const int e0 = col_of<true>(8 * i);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r[8 * i + j];
      store8<T, true>(row + e0, cols - e0, v);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int e = col_of<false>(q);
      if (e < cols) row[e] = from_f<T>(r[q]);
    }
  }
}
// The same with the type known at run time; `off` in elements.
template <bool VEC>
__device__ __forceinline__ void load_row_dyn(const void* p, int type, int64_t off, int cols, Row16& r) {
  if (type == MOE_B200_BF16) load_row<bf16, VEC>(static_cast<const bf16*>(p) + off, cols, r);
  else if (type == MOE_B200_FP16) load_row<fp16, VEC>(static_cast<const fp16*>(p) + off, cols, r);
  else load_row<float, VEC>(static_cast<const float*>(p) + off, cols, r);
}
template <bool VEC>
__device__ __forceinline__ void store_row_dyn(void* p, int type, int64_t off, int cols, const Row16& r) {
  if (type == MOE_B200_BF16) store_row<bf16, VEC>(static_cast<bf16*>(p) + off, cols, r);
  else if (type == MOE_B200_FP16) store_row<fp16, VEC>(static_cast<fp16*>(p) + off, cols, r);
  else store_row<float, VEC>(static_cast<float*>(p) + off, cols, r);
}
template <bool VEC>
__device__ __forceinline__ void load_weight(const void* p, int type, float off, int cols, Row16& w) {
  load_row_dyn<VEC>(p, type, 0, cols, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) w.v[i] = add2(w.v[i], dup2(off));
}

// Sums over a row, of elements that exist: those beyond the row are 0 in every tensor, but a
// factor of the row may be infinite.  VEC: chunk-wise, with whole chunks in or out.
template <bool VEC>
__device__ __forceinline__ float sum_existing(const Row16& p, int cols) {
  float s = 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) s += col_of<VEC>(q) < cols ? p[q] : 0.f;
  return s;
}
__device__ __forceinline__ float dot16(const Row16& a, const Row16& b) {
  float2 s = mul2(a.v[0], b.v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) s = fma2(a.v[i], b.v[i], s);
  return s.x + s.y;
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
  if (y_type == MOE_B200_BF16) r_type == MOE_B200_FP32 ? f(bf16{}, float{}) : f(bf16{}, bf16{});
  else if (y_type == MOE_B200_FP16) r_type == MOE_B200_FP32 ? f(fp16{}, float{}) : f(fp16{}, fp16{});
  else f(float{}, float{});
}
inline bool type_pair_ok(int y, int r) {
  return is_float_type(y) && is_float_type(r) && (r == y || r == MOE_B200_FP32);
}

}  // namespace moe
