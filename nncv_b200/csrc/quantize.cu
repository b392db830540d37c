// What makes the operands of the 8-bit matrix product: root-mean-square norm with the residual's addition, gated
// activations and plain quantisation, each with an e4m3 result that carries a scale for every block of 128 values.
//
// A block of values y:  s = max(largest finite |y|, 2^-100) / 448,  q = y / s rounded to e4m3 (448 is its largest value).
// The least scale keeps 1 / s finite for a block of zeros.  What is not finite becomes NaN -- e4m3 has no infinity -- and leaves
// the other values of its block as they are.
#include "activation.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace nncv_b200 {
namespace {

constexpr int kV = 8;             // values a thread holds of a row at a time; sixteen threads hold a block
constexpr int kGroup = 128;
constexpr float kTop = 448.0f, kLeast = 0x1p-100f;

// Eight consecutive values from column `col` of a row of K.  VEC: the row is on a 16-byte boundary and K a multiple of 8.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int col, int K, float (&v)[kV]) {
  if (VEC) {
    alignas(16) T raw[kV];
#pragma unroll
    for (int i = 0; i < (int)(kV * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(raw)[i] = col < K ? *reinterpret_cast<const uint4*>(row + col + i * (16 / sizeof(T))) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = ef<T>(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = col + e < K ? ef<T>(row[col + e]) : 0.0f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int col, int K, const float (&v)[kV]) {
  if (VEC) {
    if (col >= K) return;
    alignas(16) T raw[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) raw[e] = et<T>(v[e]);
#pragma unroll
    for (int i = 0; i < (int)(kV * sizeof(T) / 16); ++i)
      *reinterpret_cast<uint4*>(row + col + i * (16 / sizeof(T))) = reinterpret_cast<const uint4*>(raw)[i];
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      if (col + e < K) row[col + e] = et<T>(v[e]);
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;   // a NaN compares false
}
__device__ __forceinline__ float block_scale(float amax) { return fmaxf(amax, kLeast) * (1.0f / kTop); }

// Two values times 1 / s as e4m3; infinities become NaN (the conversion alone would make them 448).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi, float inv) {
  const float nan = __int_as_float(0x7fffffff);
  lo = fabsf(lo) < INFINITY ? lo * inv : nan;
  hi = fabsf(hi) < INFINITY ? hi * inv : nan;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* __restrict__ row, int col, int K, const float (&v)[kV], float inv) {
  uint32_t h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = e4m3x2(v[2 * e], v[2 * e + 1], inv);
  if (VEC) {
    if (col < K) *reinterpret_cast<uint2*>(row + col) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      if (col + e < K) row[col + e] = (uint8_t)(h[e >> 1] >> (8 * (e & 1)));
  }
}

// Writes the block that these sixteen threads hold and its scale.
template <bool VEC>
__device__ __forceinline__ void put_group(uint8_t* __restrict__ row, float* __restrict__ scales, int col, int K, const float (&v)[kV]) {
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < kV; ++e) amax = fmaxf(amax, finite_abs(v[e]));
#pragma unroll
  for (int o = 8; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float s = block_scale(amax);
  store_e4m3<VEC>(row, col, K, v, 1.0f / s);
  if (col < K && col % kGroup == 0) scales[col / kGroup] = s;
}

// ---------------------------------------------------------------- root-mean-square norm ----
// One CTA a row; the row stays in registers between the sum of squares and the result, so every tensor is read once.
template <typename T, bool VEC, bool Q, int ITER>
__global__ void __launch_bounds__(ITER <= 2 ? 1024 : 512)
rmsnorm_kernel(const T* x, long long ldx, const T* residual, const float* __restrict__ weight, float eps, T* sum, void* out,
                               float* scale, int K) {
  __shared__ float s_part[32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long row = blockIdx.x;
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float h[ITER][kV];
#pragma unroll
  for (int i = 0; i < ITER; ++i) load8<T, VEC>(x + row * ldx, (i * threads + (int)threadIdx.x) * kV, K, h[i]);
  if (residual) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      float r[kV];
      load8<T, VEC>(residual + row * K, (i * threads + (int)threadIdx.x) * kV, K, r);
#pragma unroll
      for (int e = 0; e < kV; ++e) h[i][e] += r[e];
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    if (sum) store8<T, VEC>(sum + row * K, (i * threads + (int)threadIdx.x) * kV, K, h[i]);
#pragma unroll
    for (int e = 0; e < kV; ++e) ss = fmaf(h[i][e], h[i][e], ss);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) s_part[warp] = ss;
  __syncthreads();
  float total = lane < (threads >> 5) ? s_part[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const float norm = 1.0f / sqrtf(total / (float)K + eps);
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int col = (i * threads + (int)threadIdx.x) * kV;
    float w[kV];
    if (weight) load8<float, VEC>(weight, col, K, w);
#pragma unroll
    for (int e = 0; e < kV; ++e) h[i][e] = weight ? h[i][e] * norm * w[e] : h[i][e] * norm;
    if (Q) put_group<VEC>(static_cast<uint8_t*>(out) + row * K, scale + row * ((K + kGroup - 1) / kGroup), col, K, h[i]);
    else store8<T, VEC>(static_cast<T*>(out) + row * K, col, K, h[i]);
  }
}

// ---------------------------------------------------------------- (gated) activation -------
// Sixteen threads a block of 128 columns of a row; gate * 1 where there is no `up`.
template <typename T, bool VEC, bool Q>
__global__ void __launch_bounds__(256) gated_kernel(const T* gate, const T* up, long long ld, void* out,
                                                    float* __restrict__ scale, long long groups, int kb, int K, int act) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long step = (long long)gridDim.x * (blockDim.x / 16);
  for (long long g0 = (long long)blockIdx.x * (blockDim.x / 16); g0 < groups; g0 += step) {
    const long long g = g0 + threadIdx.x / 16;
    const bool in = g < groups;
    const long long row = in ? g / kb : 0;
    const int col = in ? (int)(g - row * kb) * kGroup + (int)(threadIdx.x & 15) * kV : K;
    float v[kV];
    load8<T, VEC>(gate + row * ld, col, K, v);
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = activate<sizeof(T) == 2>(v[e], act);
    if (up) {
      float u[kV];
      load8<T, VEC>(up + row * ld, col, K, u);
#pragma unroll
      for (int e = 0; e < kV; ++e) v[e] *= u[e];
    }
    if (!VEC) {   // what an activation makes of the zeros behind the row is not part of its block
#pragma unroll
      for (int e = 0; e < kV; ++e) v[e] = col + e < K ? v[e] : 0.0f;
    } else if (col >= K) {
#pragma unroll
      for (int e = 0; e < kV; ++e) v[e] = 0.0f;
    }
    if (Q) put_group<VEC>(static_cast<uint8_t*>(out) + row * K, scale + row * kb, col, K, v);
    else store8<T, VEC>(static_cast<T*>(out) + row * K, col, K, v);
  }
}

// ---------------------------------------------------------------- blocks of 128 x 128 ------
// One CTA a block, which stays in registers between its largest value and the result: 16 threads a row of 128, 16 rows at a time.
constexpr int kBlockIter = kGroup / 16;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_block_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q,
                                                             float* __restrict__ scale, int M, int K) {
  __shared__ float s_part[8];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int kb = (K + kGroup - 1) / kGroup, bm = (int)(blockIdx.x / kb), bk = (int)(blockIdx.x % kb);
  const int col = bk * kGroup + (int)(threadIdx.x & 15) * kV;
  float v[kBlockIter][kV];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kBlockIter; ++i) {
    const int row = bm * kGroup + i * 16 + (int)(threadIdx.x >> 4);
    load8<T, VEC>(x + (long long)row * ldx, row < M ? col : K, K, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kBlockIter; ++i)
#pragma unroll
    for (int e = 0; e < kV; ++e) amax = fmaxf(amax, finite_abs(v[i][e]));
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, s_part[i]);
  const float s = block_scale(amax), inv = 1.0f / s;
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
  for (int i = 0; i < kBlockIter; ++i) {
    const int row = bm * kGroup + i * 16 + (int)(threadIdx.x >> 4);
    if (row < M) store_e4m3<VEC>(q + (long long)row * K, col, K, v[i], inv);
  }
}

inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

template <typename T, bool VEC, bool Q>
cudaError_t rmsnorm_as(const RmsNormArgs& a, cudaStream_t st) {
  const int chunks = (a.K + kV - 1) / kV;
  const int iter = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : 8;
  const int threads = ((chunks + iter - 1) / iter + 31) / 32 * 32;
#define NNCV_NORM(I_)                                                                                                                        \
  if (iter == I_)                                                                                                                            \
    return launch_pdl(rmsnorm_kernel<T, VEC, Q, I_>, dim3((unsigned)a.M), dim3(threads), 0, st, static_cast<const T*>(a.x), a.ldx,           \
                      static_cast<const T*>(a.residual), a.weight, a.eps, static_cast<T*>(a.sum), a.out, a.scale, a.K);
  NNCV_NORM(1) NNCV_NORM(2) NNCV_NORM(8)
#undef NNCV_NORM
  return cudaErrorInvalidValue;
}
template <typename T>
cudaError_t rmsnorm_of(const RmsNormArgs& a, cudaStream_t st) {
  const bool vec = a.K % kV == 0 && a.ldx * (long long)sizeof(T) % 16 == 0 && aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.weight, 16) &&
                   aligned(a.sum, 16) && aligned(a.out, a.to_e4m3 ? 8 : 16);
  if (a.to_e4m3) return vec ? rmsnorm_as<T, true, true>(a, st) : rmsnorm_as<T, false, true>(a, st);
  return vec ? rmsnorm_as<T, true, false>(a, st) : rmsnorm_as<T, false, false>(a, st);
}

template <typename T>
cudaError_t gated_of(const GatedArgs& a, cudaStream_t st) {
  const bool vec = a.K % kV == 0 && a.ld * (long long)sizeof(T) % 16 == 0 && aligned(a.gate, 16) && aligned(a.up, 16) && aligned(a.out, a.to_e4m3 ? 8 : 16);
  const int kb = (a.K + kGroup - 1) / kGroup;
  const long long groups = (long long)a.M * kb, most = (long long)(a.sm_count > 0 ? a.sm_count : 148) * 8;
  const long long need = (groups + 15) / 16;
  auto kern = a.to_e4m3 ? (vec ? gated_kernel<T, true, true> : gated_kernel<T, false, true>) : (vec ? gated_kernel<T, true, false> : gated_kernel<T, false, false>);
  return launch_pdl(kern, dim3((unsigned)(need < most ? need : most)), dim3(256), 0, st, static_cast<const T*>(a.gate), static_cast<const T*>(a.up), a.ld, a.out,
                    a.scale, groups, kb, a.K, a.act);
}

template <typename T>
cudaError_t quantize_blocks_of(const T* x, long long ldx, uint8_t* q, float* scale, int M, int K, cudaStream_t st) {
  const bool vec = K % kV == 0 && ldx * (long long)sizeof(T) % 16 == 0 && aligned(x, 16) && aligned(q, 8);
  const long long blocks = (long long)((M + kGroup - 1) / kGroup) * ((K + kGroup - 1) / kGroup);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_pdl(vec ? quantize_block_kernel<T, true> : quantize_block_kernel<T, false>, dim3((unsigned)blocks), dim3(256), 0, st, x, ldx, q, scale, M, K);
}

}  // namespace

cudaError_t launch_rmsnorm(const RmsNormArgs& a, cudaStream_t st) {
  if (a.K > kRmsNormMaxK) return cudaErrorInvalidValue;
  return a.dtype == kF32 ? rmsnorm_of<float>(a, st) : a.dtype == kF16 ? rmsnorm_of<__half>(a, st) : rmsnorm_of<__nv_bfloat16>(a, st);
}

cudaError_t launch_gated_activation(const GatedArgs& a, cudaStream_t st) {
  return a.dtype == kF32 ? gated_of<float>(a, st) : a.dtype == kF16 ? gated_of<__half>(a, st) : gated_of<__nv_bfloat16>(a, st);
}

cudaError_t launch_quantize_blocks(const void* x, long long ldx, DType dt, void* q, float* scale, int M, int K, cudaStream_t st) {
  uint8_t* o = static_cast<uint8_t*>(q);
  return dt == kF32 ? quantize_blocks_of(static_cast<const float*>(x), ldx, o, scale, M, K, st)
                    : dt == kF16 ? quantize_blocks_of(static_cast<const __half*>(x), ldx, o, scale, M, K, st)
                                 : quantize_blocks_of(static_cast<const __nv_bfloat16*>(x), ldx, o, scale, M, K, st);
}

}  // namespace nncv_b200
