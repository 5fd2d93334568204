// Arguments and launchers of the 8-bit integer products (int8_gemm.cu).
#pragma once

#include "op_common.cuh"

namespace moe {

struct LinearArgs {
  const float* sx;      // [T]
  const float* sw;      // [N]
  const void* bias;     // [N] or null
  void* y;
  int64_t y_ld;
  int T, N, K, y_type, bias_type;
  int early_w;          // the weights are not written by the kernel this one depends on
};

// q: int8 [T][K], rows q_ld apart; w: int8 [N][K], rows w_ld apart (both 16-byte aligned).
cudaError_t int8_gemm_launch(const int8_t* q, int64_t q_ld, const int8_t* w, int64_t w_ld, const LinearArgs& a, int sms,
                             cudaStream_t st);

}  // namespace moe
