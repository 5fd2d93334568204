// Linear layer in 8-bit integers with one scale per token and one per output channel.
//
//   q[t][k] = rint(v[t][k] / sx[t]) in [-127, 127],  sx[t] = max(max_k |v[t][k]| / 127, 2^-126)
//   y[t][n] = sx[t] * sw[n] * sum_k q[t][k] * w[n][k]  (+ bias[n])
//
// v is x, or silu(x2) * x1 of x = [x1 | x2] (the expert layer's order).  Sums of products are
// exact 32-bit integers (|sum| <= K * 2^14, so K <= 131056 cannot overflow).  A row holding a NaN
// or an infinity gets a NaN scale, so its outputs are NaN.
#include <type_traits>

#include "int8_gemm.cuh"

namespace moe {

constexpr int kQuantPerThread = 32;                      // four 8-element chunks
constexpr int kQuantMaxCols = 1024 * kQuantPerThread;
constexpr int kInt8MaxK = 131056;
constexpr int kInt8StreamMaxT = 256;

struct QuantArgs {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t x_ld, q_ld;
  int rows, cols, warps, type, swiglu;
};

// One row in the registers of a group of warps: maximum, then codes.
template <class XT, bool VEC>
__global__ void __launch_bounds__(1024, 1) quant_kernel(QuantArgs a) {
  __shared__ float buf[8 * 32];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int cols = row < a.rows ? a.cols : 0;
  const XT* src = static_cast<const XT*>(a.x) + row * a.x_ld;
  float v[4][8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e0 = (threadIdx.x + i * blockDim.x) * 8, n = min(8, cols - e0);
    load8<XT, VEC>(src + e0, n, v[i]);
    if (a.swiglu) {
      float g[8];
      load8<XT, VEC>(src + a.cols + e0, n, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= g[j] / (1.f + expf(-g[j]));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[i][j]));
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (a.warps > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) buf[threadIdx.y * 32 + (threadIdx.x >> 5)] = m;
    __syncthreads();
    m = lane < a.warps ? buf[threadIdx.y * 32 + lane] : 0.f;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  }
  if (row >= a.rows) return;
  const bool finite = m <= 3.4028234663852886e38f;
  const float sc = finite ? fmaxf(m / 127.f, 1.17549435082228751e-38f) : __uint_as_float(0x7fc00000u);
  const float inv = finite ? 1.f / sc : 0.f;
  if (threadIdx.x == 0) a.scale[row] = sc;
  int8_t* dst = a.q + row * a.q_ld;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e0 = (threadIdx.x + i * blockDim.x) * 8, n = min(8, cols - e0);
    if (n <= 0) continue;
    uint32_t b[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = finite ? max(-127, min(127, __float2int_rn(v[i][j] * inv))) : 0;
      b[j >> 2] |= static_cast<uint32_t>(c & 0xff) << (8 * (j & 3));
    }
    if constexpr (VEC) {
      *reinterpret_cast<uint2*>(dst + e0) = make_uint2(b[0], b[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) dst[e0 + j] = static_cast<int8_t>(b[j >> 2] >> (8 * (j & 3)));
    }
  }
}

namespace {

cudaError_t quant_launch(const QuantArgs& q0, cudaStream_t st) {
  QuantArgs q = q0;
  if (q.rows == 1) q.x_ld = q.q_ld = 0;   // a single row has no pitch
  q.warps = (q.cols + 32 * kQuantPerThread - 1) / (32 * kQuantPerThread);
  const int rpc = q.warps >= 8 ? 1 : 8 / q.warps;
  const dim3 block(q.warps * 32, rpc), grid((q.rows + rpc - 1) / rpc);
  const bool vec = q.cols % 8 == 0 && rows_aligned(q.x, q.x_ld, q.type) &&
                   (reinterpret_cast<uintptr_t>(q.q) & 7u) == 0 && q.q_ld % 8 == 0;
  auto go = [&](auto t) {
    using XT = decltype(t);
    return vec ? launch_pdl(quant_kernel<XT, true>, grid, block, 0, st, q)
               : launch_pdl(quant_kernel<XT, false>, grid, block, 0, st, q);
  };
  return q.type == MOE_B200_BF16 ? go(bf16{}) : q.type == MOE_B200_FP16 ? go(fp16{}) : go(float{});
}

int quant_check(const void* x, int type, int rows, int cols, const char** why) {
  if (rows < 0 || cols < 1 || cols > kQuantMaxCols) *why = "int8 quantisation: rows must be >= 0 and cols in [1, 32768]";
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
  const cudaError_t e = quant_launch(q, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "quantize_int8 launch");
}

MOE_B200_API size_t moe_b200_int8_linear_workspace_size(int32_t num_tokens, int32_t out_features, int32_t in_features,
                                                        int32_t x_type) {
  using namespace moe;
  if (num_tokens < 0 || out_features < 1 || in_features < 1 || in_features > kInt8MaxK) return 0;
  const size_t T = num_tokens;
  return 256 + (x_type == MOE_B200_INT8 ? 0 : align256(T * in_features) + align256(T * sizeof(float)));
}

MOE_B200_API int moe_b200_int8_linear(const moe_b200_linear_args* a, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  using namespace moe;
  if (!a) return report_error(MOE_B200_ERR_ARG, "null args");
  if (a->num_tokens < 0 || a->out_features < 1 || a->in_features < 16 || a->in_features > kInt8MaxK ||
      a->in_features % 16)
    return report_error(MOE_B200_ERR_ARG, "int8_linear: num_tokens must be >= 0, out_features >= 1 and in_features a multiple of 16 up to 131056");
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
    e = quant_launch(q, st);
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
  e = a->num_tokens <= kInt8StreamMaxT ? int8_stream_launch(q_rows, q_ld, a->weight, w_ld, l, sms, st)
                                       : int8_wide_launch(q_rows, q_ld, a->weight, w_ld, l, sms, st);
  return e == cudaSuccess ? MOE_B200_OK : report_cuda(e, "int8_linear launch");
}

}  // extern "C"
