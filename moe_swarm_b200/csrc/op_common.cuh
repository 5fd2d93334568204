// What the operators around the expert layer (norm.cu, select.cu, int8.cu) share: element types,
// eight-element row chunks, warp and row reductions, host-side checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/moe_b200.h"
#include "launch_args.cuh"
#include "ptx.cuh"

namespace moe {

// Host helpers of the C entries (capi.cu).
int report_cuda(cudaError_t e, const char* what);
int op_device(int* sms);   // the current device must be sm_100; *sms = its SM count
// A byte matrix with rows `pitch` bytes apart as TMA tiles of 128 bytes x box_rows rows (SWIZZLE_128B).
bool encode_rows_u8(CUtensorMap* m, const void* base, uint64_t cols, uint64_t rows, uint64_t pitch,
                    uint32_t box_rows);

// Raises a kernel's dynamic shared memory limit once per device (a static of the launching code,
// which must use it for one kernel only).  Setting it twice in a race is harmless.
class SmemOnce {
 public:
  cudaError_t set(const void* kernel, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64 && (done_.load(std::memory_order_acquire) >> dev) & 1u) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done_.fetch_or(1ull << dev, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

// Most rows (tokens, outputs) of a call: row counters then stay clear of 32 bits.
constexpr int kOpMaxRows = 1 << 30;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int type_bytes(int t) { return t == MOE_B200_FP32 ? 4 : t == MOE_B200_E4M3 ? 1 : 2; }
inline bool is_float_type(int t) { return t == MOE_B200_BF16 || t == MOE_B200_FP16 || t == MOE_B200_FP32; }
// Whether every row of the tensor starts on a 16-byte boundary.
inline bool rows_aligned(const void* p, int64_t stride, int type) {
  return !p || (aligned16(p) && (stride * type_bytes(type)) % 16 == 0);
}

// First bounded wait of this file's kernels that ran out (0: none); one word per source file.
static __device__ int g_op_status;
// Reads (and with `clear` resets) it, synchronising the stream.
static inline cudaError_t take_status(cudaStream_t st, bool clear, int* v) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(v, g_op_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && clear && *v) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_op_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  return e;
}
cudaError_t norm_status(cudaStream_t st, bool clear, int* v);       // norm.cu and norm_bwd.cu
cudaError_t norm_bwd_status(cudaStream_t st, bool clear, int* v);
cudaError_t quant_status(cudaStream_t st, bool clear, int* v);      // int8.cu
cudaError_t int8_status(cudaStream_t st, bool clear, int* v);       // int8_gemm.cu

using bf16 = __nv_bfloat16;
using fp16 = __half;

__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(fp16 v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ fp16 from_f<fp16>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }

__device__ __forceinline__ void unpack2(uint32_t u, float* v, bf16) {
  v[0] = __uint_as_float(u << 16);
  v[1] = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t u, float* v, fp16) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  v[0] = f.x;
  v[1] = f.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bf16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, fp16) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Plain loads, not the read-only path: a tensor may be written by the kernel that this one waits
// for (pdl_wait), and a read-only load may be moved above that wait.
//
// Eight consecutive elements from p.  VEC: p is 16-byte aligned.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float* v) {
  if constexpr (!VEC) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f(p[j]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0];
    const float4 b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    unpack2(u.x, v, T{});
    unpack2(u.y, v + 2, T{});
    unpack2(u.z, v + 4, T{});
    unpack2(u.w, v + 6, T{});
  }
}

// Element `off` of p, the element type known at run time (uniform over the grid).
__device__ __forceinline__ void store1_dyn(void* p, int type, int64_t off, float v) {
  if (type == MOE_B200_BF16) static_cast<bf16*>(p)[off] = from_f<bf16>(v);
  else if (type == MOE_B200_FP16) static_cast<fp16*>(p)[off] = from_f<fp16>(v);
  else static_cast<float*>(p)[off] = v;
}
__device__ __forceinline__ float load1_dyn(const void* p, int type, int64_t off) {
  if (type == MOE_B200_BF16) return to_f(static_cast<const bf16*>(p)[off]);
  if (type == MOE_B200_FP16) return to_f(static_cast<const fp16*>(p)[off]);
  return static_cast<const float*>(p)[off];
}

// Starts a copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) from global to this
// CTA's shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sums of N values over the `warps` warps of each row of a CTA whose blockDim is (32 * warps,
// rows).  `buf` holds [rows][N][32] floats and may be reused after the next CTA barrier only.
// Every thread of the CTA calls it (one barrier, none when a row is one warp); the order of the
// additions is fixed.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int warps, float* buf) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
  if (warps == 1) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* b = buf + threadIdx.y * N * 32;
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) b[k * 32 + warp] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(lane < warps ? b[k * 32 + lane] : 0.f);
}

// The same for three values of a row of up to 16 warps, with less than half the shuffles: a warp's
// butterfly leaves each of four groups of lanes (bits 3 and 4 of the lane) with one value.
__device__ __forceinline__ void row_sum3(float (&v)[3], int warps, float* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool hi = lane & 16, odd = lane & 8;
  // lanes below 16 go on with v[0] and v[1], the others with v[2] (and nothing)
  const float send0 = hi ? v[0] : v[2], send1 = hi ? v[1] : 0.f;
  float p = (hi ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, send0, 16);
  float q = (hi ? 0.f : v[1]) + __shfl_xor_sync(0xffffffffu, send1, 16);
  float s = (odd ? q : p) + __shfl_xor_sync(0xffffffffu, odd ? p : q, 8);
#pragma unroll
  for (int d = 4; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (warps > 1) {
    float* b = buf + threadIdx.y * 3 * 32;
    const int k = lane >> 3;   // 0, 1, 2: this group's value
    if ((lane & 7) == 0 && k < 3) b[k * 32 + warp] = s;
    __syncthreads();
    const int j = lane & 7;
    s = k < 3 ? (j < warps ? b[k * 32 + j] : 0.f) + (j + 8 < warps ? b[k * 32 + j + 8] : 0.f) : 0.f;
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  }
  v[0] = __shfl_sync(0xffffffffu, s, 0);
  v[1] = __shfl_sync(0xffffffffu, s, 8);
  v[2] = __shfl_sync(0xffffffffu, s, 16);
}

// A programmatic dependent launch on `st` in clusters of `cluster` CTAs along x: the kernel may
// become resident while its predecessor drains, and calls pdl_wait() before it touches anything
// that an earlier kernel wrote or reads.
template <class... P, class... A>
cudaError_t launch_cluster_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st,
                               const A&... args) {
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = st;
  c.attrs = at;
  c.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}
template <class... P, class... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
  return launch_cluster_pdl(kernel, grid, block, smem, 1, st, args...);
}

}  // namespace moe
