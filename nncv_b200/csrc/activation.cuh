// Conversions between the activation types and fp32, and the activations of nncv's fixtures (ReLU, hard-sigmoid, hard-swish,
// sigmoid, SiLU: tests/Nets/MobileNetV3.mlir:345-383, tests/Nets/Yolov5s.mlir:158-169).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "ptx.cuh"

namespace nncv_b200 {
namespace {

template <typename T> __device__ __forceinline__ float ef(T v);
template <> __device__ __forceinline__ float ef<float>(float v) { return v; }
template <> __device__ __forceinline__ float ef<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float ef<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T et(float v);
template <> __device__ __forceinline__ float et<float>(float v) { return v; }
template <> __device__ __forceinline__ __half et<__half>(float v) {
  return __ushort_as_half((unsigned short)(ptx::pack_half2_sat(v, 0.f) & 0xffffu));   // saturating, NaN stays NaN
}
template <> __device__ __forceinline__ __nv_bfloat16 et<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float hard_sigmoid(float x) {
  float t = (x + 3.0f) / 6.0f;
  t = (1.0f < t) ? 1.0f : t;     // cmpf olt 1, t ; select
  t = (0.0f > t) ? 0.0f : t;     // cmpf ogt 0, t ; select
  return t;
}
__device__ __forceinline__ float sigmoid_ref(float x) { return 1.0f / (expf(-x) + 1.0f); }

// With a 16-bit result the last bits of an fp32 quotient or exponential are rounded away, so those types
// take a multiply by 1/6 and the hardware exponential / reciprocal (2 ulp of fp32) instead of IEEE division
// and expf; fp32 tensors keep the exact forms.  NaN and the clamp order are the same in both.
__device__ __forceinline__ float hard_sigmoid_fast(float x) {
  float t = (x + 3.0f) * 0.16666667f;
  t = (1.0f < t) ? 1.0f : t;
  t = (0.0f > t) ? 0.0f : t;
  return t;
}
__device__ __forceinline__ float sigmoid_fast(float x) { return __fdividef(1.0f, __expf(-x) + 1.0f); }

template <bool FAST>
__device__ __forceinline__ float activate(float x, int act) {
  switch (act) {
    case kActRelu: return !(x <= 0.0f) ? x : 0.0f;        // cmpf ugt: NaN passes
    case kActHardSigmoid: return FAST ? hard_sigmoid_fast(x) : hard_sigmoid(x);
    case kActHardSwish: return x * (FAST ? hard_sigmoid_fast(x) : hard_sigmoid(x));
    case kActSigmoid: return FAST ? sigmoid_fast(x) : sigmoid_ref(x);
    case kActSilu: return x * (FAST ? sigmoid_fast(x) : sigmoid_ref(x));
    default: return x;
  }
}

}  // namespace
}  // namespace nncv_b200
