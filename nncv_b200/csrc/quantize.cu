// What makes the operands of the 8-bit matrix product: root-mean-square norm with the residual's addition, gated
// activations and plain quantisation, each with an e4m3 result that carries a scale for every block of 128 values.
//
// A block of values y:  s = max(largest finite |y|, 2^-100) * (1 / 448),  q = y / s rounded to e4m3 (448 is its largest value).
// The least scale keeps 1 / s finite for a block of zeros.  What is not finite becomes NaN -- e4m3 has no infinity -- and leaves
// the other values of its block as they are.
//
// Bound by HBM where rows are whole blocks on 16-byte boundaries.  Eight threads hold the 128 columns of a block: each has 16 of them, in two
// pieces of eight that lie 64 columns apart, so that what the eight load and store at once lies in a row.  (Eight values a thread, a 64-bit division
// for each block and a test for infinities for each value took twice the time.)  Of the 6.5 TB/s of a copy: norm 4096 x 4096 bf16 with residual to
// e4m3 5.9 (20.0 us), gated SiLU 2048 x 8192 bf16 to e4m3 5.9 (14.3 us), 8192 x 2048 bf16 to e4m3 5.4 (9.4 us), 4096 x 4096 fp32 in blocks 5.8
// (14.4 us).  Further from it: norms of few columns (65536 x 128 bf16 23.6 us where the bytes take 3.9), rows off those boundaries (gated 2048 x
// 8191 40 us), fp32 norms wider than 6144 (1024 x 16384 48 us, the bytes 33.5).
#include <type_traits>

#include "activation.cuh"
#include "epilogue.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace nncv_b200 {
namespace {

constexpr int kV = 16;            // values a thread holds of a block
constexpr int kLanes = 8;         // threads that hold a block
constexpr int kGroup = 128;
constexpr float kTop = 448.0f, kLeast = 0x1p-100f;

constexpr int kPiece = 8;         // consecutive values
__device__ __forceinline__ int piece_col(int i, int t) { return (i * kLanes + t) * kPiece; }

// What a thread has of a row, as it lies in memory.  VEC: pieces are on 16-byte boundaries and K holds whole ones.
template <typename T> struct Raw {
  static constexpr int kWords = (int)sizeof(T) * kPiece / 16;
  uint4 p[kV / kPiece][kWords];
};
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(const T* row, int col0, int t, int K, Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < kV / kPiece; ++i) {
    const int col = col0 + piece_col(i, t);
    if (VEC) {
#pragma unroll
      for (int j = 0; j < Raw<T>::kWords; ++j) r.p[i][j] = col < K ? reinterpret_cast<const uint4*>(row + col)[j] : make_uint4(0, 0, 0, 0);
    } else {
      alignas(16) T e[kPiece];
#pragma unroll
      for (int j = 0; j < kPiece; ++j) e[j] = col + j < K ? row[col + j] : et<T>(0.0f);
#pragma unroll
      for (int j = 0; j < Raw<T>::kWords; ++j) r.p[i][j] = reinterpret_cast<const uint4*>(e)[j];
    }
  }
}
template <typename T>
__device__ __forceinline__ void to_float(const Raw<T>& r, float (&v)[kV]) {
  const T* e = reinterpret_cast<const T*>(r.p);
#pragma unroll
  for (int i = 0; i < kV; ++i) v[i] = ef<T>(e[i]);
}
// A piece in its type.
template <typename T>
__device__ __forceinline__ void to_type(const float* v, T* e) {
#pragma unroll
  for (int i = 0; i < kPiece; ++i) e[i] = et<T>(v[i]);
}
// fp16: finite values beyond its range become +-65504, infinite ones stay.  The plain conversion makes both infinite, so a piece that has none of
// them needs no second look (looked at one by one, wide norms took a quarter longer).
template <>
__device__ __forceinline__ void to_type<__half>(const float* v, __half* e) {
  __half2* o = reinterpret_cast<__half2*>(e);
  __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
  for (int i = 0; i < kPiece / 2; ++i) {
    o[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    most = __hmax2(most, __habs2(o[i]));   // a NaN is passed over
  }
  if (fmaxf(__low2float(most), __high2float(most)) == INFINITY) {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) e[i] = __ushort_as_half((unsigned short)epi::pack_half2_inf(v[i], 0.0f));
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_row(T* row, int col0, int t, int K, const float (&v)[kV]) {
#pragma unroll
  for (int i = 0; i < kV / kPiece; ++i) {
    const int col = col0 + piece_col(i, t);
    alignas(16) T e[kPiece];
    to_type<T>(v + i * kPiece, e);
    if (VEC) {
      if (col < K) {
#pragma unroll
        for (int j = 0; j < Raw<T>::kWords; ++j) reinterpret_cast<uint4*>(row + col)[j] = reinterpret_cast<const uint4*>(e)[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPiece; ++j)
        if (col + j < K) row[col + j] = e[j];
    }
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;   // a NaN compares false
}
template <int LANES>
__device__ __forceinline__ float max_of(float a) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}
__device__ __forceinline__ float largest(const float (&v)[kV]) {   // NaN is passed over
  float a = fabsf(v[0]);
#pragma unroll
  for (int e = 1; e < kV; ++e) a = fmaxf(a, fabsf(v[e]));
  return a;
}
__device__ __forceinline__ float largest_finite(const float (&v)[kV]) {
  float a = 0.0f;
#pragma unroll
  for (int e = 0; e < kV; ++e) a = fmaxf(a, finite_abs(v[e]));
  return a;
}
__device__ __forceinline__ void infinite_to_nan(float (&v)[kV]) {   // the conversion alone would make them 448
#pragma unroll
  for (int e = 0; e < kV; ++e) v[e] = fabsf(v[e]) < INFINITY ? v[e] : __int_as_float(0x7fffffff);
}
// Times 1 / 448 as fp32 has it: a step off the quotient for some, which the values' own quotient by it makes up for.
__device__ __forceinline__ float block_scale(float amax) { return fmaxf(amax, kLeast) * (1.0f / kTop); }
__device__ __forceinline__ float reciprocal(float s) {   // a step of fp32 off at most where 1 / s is a normal number
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Minus y / s for two values of a block.  The product with the approximate 1 / s is at most 2.5 steps of fp32 off; its remainder, by a fused
// multiply-add, times 1 / s corrects it to 2^-21 of a step before the last rounding (after P. Markstein, Computation of elementary functions
// on the IBM RISC System/6000, 1990).  So a quotient half way between two e4m3 values comes out as that and goes to the even one, where the
// product alone sent some to the other.  The sign is turned twice, so that a zero keeps its own.  8192 x 2048 bf16 in rows takes 9.4 us, with the
// product alone 9.1; 4096 x 4096 bf16 in blocks 12.3 for 11.6.
struct Divisor {
  unsigned long long s, minus_inv;
  __device__ __forceinline__ explicit Divisor(float by) : s(epi::pk(by, by)) {
    const float r = -reciprocal(by);
    minus_inv = epi::pk(r, r);
  }
  __device__ __forceinline__ void divide(float a, float b, float& qa, float& qb) const {
    const unsigned long long y = epi::pk(a, b), q = epi::mul2(y, minus_inv);
    epi::unpk(epi::fma2(epi::fma2(q, s, y), minus_inv, q), qa, qb);
  }
};
template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int col0, int t, int K, const float (&v)[kV], const Divisor& by) {
#pragma unroll
  for (int i = 0; i < kV / kPiece; ++i) {
    const int col = col0 + piece_col(i, t);
    uint32_t h[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float* y = v + i * kPiece + 4 * j;
      float q[4];
      by.divide(y[0], y[1], q[0], q[1]);
      by.divide(y[2], y[3], q[2], q[3]);
      h[j] = (e4m3x2(q[0], q[1]) | e4m3x2(q[2], q[3]) << 16) ^ 0x80808080u;
    }
    if (VEC) {
      if (col < K) *reinterpret_cast<uint2*>(row + col) = make_uint2(h[0], h[1]);
    } else {
#pragma unroll
      for (int j = 0; j < kPiece; ++j)
        if (col + j < K) row[col + j] = (uint8_t)(h[j >> 2] >> (8 * (j & 3)));
    }
  }
}

// Writes the block that these eight threads hold and its scale.  Infinities are looked for only where one is the largest
// value of some block of the warp: tested per element they took a third of the instructions.
template <bool VEC>
__device__ __forceinline__ void put_block(uint8_t* row, float* scale, int col0, int t, int K, float (&v)[kV]) {
  float amax = max_of<kLanes>(largest(v));
  if (__any_sync(0xffffffffu, !(amax < INFINITY))) {
    amax = max_of<kLanes>(largest_finite(v));
    infinite_to_nan(v);
  }
  const float s = block_scale(amax);
  store_e4m3<VEC>(row, col0, t, K, v, Divisor(s));
  if (t == 0 && col0 < K) *scale = s;
}

// x / (1 + exp(-x)) on the hardware's exponential and reciprocal: exp is off by 2 steps of fp32 and by what rounding x * log2(e) makes of
// it, far below half a step of the 16-bit values that come in.
__device__ __forceinline__ float silu16(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  return x * reciprocal(1.0f + e);
}
// SiLU and sigmoid of far gates, below kFar, are x exp(x) and exp(x): there 1 + exp(-x) is exp(-x), which passes fp32's range from -88.7 on, and the
// hardware's reciprocal of it is 0 from -87.3 on, where the result is no zero yet and a large `up` makes an ordinary value of it.
constexpr float kFar = -87.0f;
template <typename T> __device__ __forceinline__ bool any_far(const Raw<T>& r) {   // NaN is passed over
  const T* e = reinterpret_cast<const T*>(r.p);
  if constexpr (sizeof(T) == 4) {
    float a = e[0];
#pragma unroll
    for (int i = 1; i < kV; ++i) a = fminf(a, e[i]);
    return a < kFar;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* p = reinterpret_cast<const T2*>(e);
    T2 a = p[0];
#pragma unroll
    for (int i = 1; i < kV / 2; ++i) a = __hmin2(a, p[i]);
    return fminf(ef<T>(a.x), ef<T>(a.y)) < kFar;
  }
}
template <bool SILU>
__device__ __forceinline__ float far_gate(float x) {
  const float h = expf(0.5f * x);
  return (SILU ? x * h : h) * h;
}
template <typename T, int ACT>
__device__ __forceinline__ float near_gate(float x, int act) {
  return ACT == kActSilu && sizeof(T) == 2 ? silu16(x) : activate<sizeof(T) == 2>(x, ACT < 0 ? act : ACT);
}

// ---------------------------------------------------------------- root-mean-square norm ----
// The sum of a value over the CTA, in every thread; `part`: 32 floats of shared memory that nobody reads or writes meanwhile.
__device__ __forceinline__ float cta_sum(float v, float* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) part[warp] = v;
  __syncthreads();
  v = lane < (int)(blockDim.x >> 5) ? part[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ void add_raw(const Raw<T>& r, float (&h)[kV]) {
  float v[kV];
  to_float<T>(r, v);
#pragma unroll
  for (int e = 0; e < kV; ++e) h[e] += v[e];
}
template <bool VEC>
__device__ __forceinline__ void load_weight(const float* weight, int col0, int t, int K, float (&w)[kV]) {
  if (weight) {
    Raw<float> r;
    load_raw<float, VEC>(weight, col0, t, K, r);
    to_float<float>(r, w);
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e) w[e] = 1.0f;
  }
}

// Rows of up to kAheadK: a CTA takes one row after the other, which stays in registers between the sum of squares and the result, so
// that every tensor is read once; the next row is on its way while this one is worked on, and the weights stay in registers.
// (With a CTA a row, loads were under way only in the first half of its life: 4096 x 4096 bf16 with residual to e4m3 23.5 us, so 20.0.)
constexpr int kAheadK = 16384;
template <typename T, bool VEC, bool Q, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS <= 512 ? 2 : 1)
rmsnorm_kernel(const T* x, long long ldx, const T* residual, const float* weight, float eps, T* sum, void* out, float* scale, int M, int K) {
  __shared__ float s_part[2][32];
  const int t = threadIdx.x & (kLanes - 1), col0 = (int)threadIdx.x / kLanes * kGroup, kb = (K + kGroup - 1) / kGroup;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  Raw<T> a, b;
  auto load = [&](long long row) {
    load_raw<T, VEC>(x + row * ldx, col0, t, K, a);
    if (residual) load_raw<T, VEC>(residual + row * K, col0, t, K, b);
  };
  constexpr bool kKeep = THREADS < 512;   // with 64 registers a thread the weights come from L1 for every row
  float w[kV];
  if (kKeep) load_weight<VEC>(weight, col0, t, K, w);
  load(blockIdx.x);
  uint32_t turn = 0;   // the other half of s_part is written next: whoever reads this one is past the barrier of the row before
  for (long long row = blockIdx.x; row < M; row += gridDim.x, turn ^= 1u) {
    float h[kV], ss = 0.0f;
    to_float<T>(a, h);
    if (residual) add_raw<T>(b, h);
#pragma unroll
    for (int e = 0; e < kV; ++e) ss = fmaf(h[e], h[e], ss);
    if (row + gridDim.x < M) load(row + gridDim.x);
    if (sum) store_row<T, VEC>(sum + row * K, col0, t, K, h);
    const float norm = 1.0f / sqrtf(cta_sum(ss, s_part[turn]) / (float)K + eps);
    if (!kKeep) load_weight<VEC>(weight, col0, t, K, w);
#pragma unroll
    for (int e = 0; e < kV; ++e) h[e] = h[e] * norm * w[e];   // the row is of size one before the weight comes
    if (Q) put_block<VEC>(static_cast<uint8_t*>(out) + row * K, scale + row * kb + col0 / kGroup, col0, t, K, h);
    else store_row<T, VEC>(static_cast<T*>(out) + row * K, col0, t, K, h);
  }
}

// Longer rows are read twice, the second time from L2.  `sum` is written in the second pass, so that it may take the place of x
// or the residual.
constexpr int kLongThreads = 512;
template <typename T, bool VEC, bool Q>
__global__ void __launch_bounds__(kLongThreads, VEC && sizeof(T) == 2 ? 2 : 0)
rmsnorm_long_kernel(const T* x, long long ldx, const T* residual, const float* weight, float eps, T* sum, void* out, float* scale, int K) {
  __shared__ float s_part[32];
  const int t = threadIdx.x & (kLanes - 1), first = (int)threadIdx.x / kLanes * kGroup, step = kLongThreads / kLanes * kGroup, kb = (K + kGroup - 1) / kGroup;
  const long long row = blockIdx.x;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  float ss = 0.0f;
  for (int col0 = first; col0 < K; col0 += step) {
    Raw<T> a, b;
    load_raw<T, VEC>(x + row * ldx, col0, t, K, a);
    if (residual) load_raw<T, VEC>(residual + row * K, col0, t, K, b);
    float h[kV];
    to_float<T>(a, h);
    if (residual) add_raw<T>(b, h);
    float part = 0.0f;
#pragma unroll
    for (int e = 0; e < kV; ++e) part = fmaf(h[e], h[e], part);
    ss += part;
  }
  const float norm = 1.0f / sqrtf(cta_sum(ss, s_part) / (float)K + eps);
  for (int base = 0; base < K; base += step) {   // the same number of rounds for every thread: a block's threads exchange its maximum
    const int col0 = base + first;
    Raw<T> a, b;
    load_raw<T, VEC>(x + row * ldx, col0, t, K, a);
    if (residual) load_raw<T, VEC>(residual + row * K, col0, t, K, b);
    float h[kV], w[kV];
    load_weight<VEC>(weight, col0, t, K, w);
    to_float<T>(a, h);
    if (residual) add_raw<T>(b, h);
    if (sum) store_row<T, VEC>(sum + row * K, col0, t, K, h);
#pragma unroll
    for (int e = 0; e < kV; ++e) h[e] = h[e] * norm * w[e];   // the row is of size one before the weight comes
    if (Q) put_block<VEC>(static_cast<uint8_t*>(out) + row * K, scale + row * kb + col0 / kGroup, col0, t, K, h);
    else store_row<T, VEC>(static_cast<T*>(out) + row * K, col0, t, K, h);
  }
}

// ---------------------------------------------------------------- (gated) activation -------
// What a warp does whose blocks have a far gate, value by value through local memory: unrolled it took 20 registers of the kernel below, which lost a
// third of its warps.  (2048 x 8192 bf16 to e4m3 with a far gate in every block 61 us, in one of 55 21, in none 14.3.)
template <typename T, bool Q, int ACT>
__device__ __forceinline__ void gated_far(const T* gate, const T* up, void* out, float* scale, int col0, int t, int K, int act) {
  float z[kV];
#pragma unroll 1
  for (int e = 0; e < kV; ++e) {
    const int col = col0 + piece_col(e / kPiece, t) + e % kPiece;
    const float x = col < K ? ef<T>(gate[col]) : 0.0f;
    float y = x < kFar ? (act == kActSilu ? far_gate<true>(x) : far_gate<false>(x)) : near_gate<T, ACT>(x, act);
    if (up) y *= col < K ? ef<T>(up[col]) : 0.0f;
    z[e] = col < K ? y : 0.0f;
  }
  float v[kV];
#pragma unroll
  for (int e = 0; e < kV; ++e) v[e] = z[e];
  if (Q) put_block<false>(static_cast<uint8_t*>(out), scale, col0, t, K, v);
  else store_row<T, false>(static_cast<T*>(out), col0, t, K, v);
}
// The same as a call.  The kernel is faster around one but from 16 bits to e4m3 (2048 x 8192, call and body in place: sigmoid fp32 30.5 and 37.5 us,
// bf16 15.9 and 20.7, to e4m3 23.4 and 20.4).
template <typename T, bool Q, int ACT>
__device__ __noinline__ void gated_far_call(const T* gate, const T* up, void* out, float* scale, int col0, int t, int K, int act) {
  gated_far<T, Q, ACT>(gate, up, out, scale, col0, t, K, act);
}

// A thread has its part of one block, of two where there is a single tensor: then as many bytes are under way (two of two tensors: 16.5 us
// for 13.7; one of one: 9.7 for 9.0).  With two tensors of 16 bits six CTAs have room at once (40 registers a thread; left to itself with 60,
// SiLU 2048 x 8192 bf16 to e4m3 takes 16.7 us for 14.4).  ACT: the activation, or -1 for the one in `act`.
constexpr int kGatedThreads = 256, kGatedBlocks = kGatedThreads / kLanes;
template <typename T, bool VEC, bool Q, bool UP, int ACT>
__global__ void __launch_bounds__(kGatedThreads, VEC && UP && sizeof(T) == 2 ? 6 : 0)
gated_kernel(const T* gate, const T* up, long long ld, void* out, float* scale, uint32_t blocks, epi::FastDiv kb, int K, int act) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  constexpr int kUnroll = UP ? 1 : 2;
  const int t = threadIdx.x & (kLanes - 1);
  const uint32_t first = blockIdx.x * (kGatedBlocks * kUnroll) + threadIdx.x / kLanes;
  Raw<T> g[kUnroll], u[kUnroll];
  long long row[kUnroll];
  int col0[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const uint32_t b = first + i * kGatedBlocks, r = epi::div_by(b, kb);
    row[i] = b < blocks ? r : 0;
    col0[i] = b < blocks ? (int)(b - r * kb.d) * kGroup : K;
    load_raw<T, VEC>(gate + row[i] * ld, col0[i], t, K, g[i]);
    if (UP) load_raw<T, VEC>(up + row[i] * ld, col0[i], t, K, u[i]);
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if ((ACT == kActSilu || (ACT < 0 && (act == kActSilu || act == kActSigmoid))) && __any_sync(0xffffffffu, any_far<T>(g[i]))) {
      const T *gate_row = gate + row[i] * ld, *up_row = UP ? up + row[i] * ld : nullptr;
      void* out_row = static_cast<uint8_t*>(out) + row[i] * K * (Q ? 1 : (long long)sizeof(T));
      float* to_scale = Q ? scale + row[i] * kb.d + col0[i] / kGroup : nullptr;
      if (!VEC || !Q || sizeof(T) == 4) gated_far_call<T, Q, ACT>(gate_row, up_row, out_row, to_scale, col0[i], t, K, act);
      else gated_far<T, Q, ACT>(gate_row, up_row, out_row, to_scale, col0[i], t, K, act);
      continue;
    }
    float v[kV];
    to_float<T>(g[i], v);
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = near_gate<T, ACT>(v[e], act);
    if (UP) {
      float w[kV];
      to_float<T>(u[i], w);
#pragma unroll
      for (int e = 0; e < kV; ++e) v[e] *= w[e];
    }
    if (Q) {
      if (ACT != kActNone && ACT != kActSilu && !UP) {   // what the activation makes of the zeros behind the row is not part of its block
#pragma unroll
        for (int e = 0; e < kV; ++e)
          if (col0[i] + piece_col(e / kPiece, t) + e % kPiece >= K) v[e] = 0.0f;
      }
      put_block<VEC>(static_cast<uint8_t*>(out) + row[i] * K, scale + row[i] * kb.d + col0[i] / kGroup, col0[i], t, K, v);
    } else {
      store_row<T, VEC>(static_cast<T*>(out) + row[i] * K, col0[i], t, K, v);
    }
  }
}

// ---------------------------------------------------------------- blocks of 128 x 128 ------
// One CTA a block, which stays in registers between its largest value and the result: kBlockThreads / 8 rows at a time (4096 x 4096 fp32:
// 256 threads 14.3 us, 512 15.0, 1024 17.5).
constexpr int kBlockThreads = 256, kBlockRows = kBlockThreads / kLanes, kBlockIter = kGroup / kBlockRows;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBlockThreads) quantize_block_kernel(const T* x, long long ldx, uint8_t* q, float* scale, int M, int K) {
  __shared__ float s_part[kBlockThreads / 32];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int kb = (K + kGroup - 1) / kGroup, bm = (int)(blockIdx.x / kb), col0 = (int)(blockIdx.x % kb) * kGroup;
  const int t = threadIdx.x & (kLanes - 1), r0 = bm * kGroup + (int)(threadIdx.x / kLanes);
  Raw<T> raw[kBlockIter];
#pragma unroll
  for (int i = 0; i < kBlockIter; ++i) load_raw<T, VEC>(x + (long long)(r0 + i * kBlockRows) * ldx, r0 + i * kBlockRows < M ? col0 : K, t, K, raw[i]);
  float v[kBlockIter][kV], amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kBlockIter; ++i) {
    to_float<T>(raw[i], v[i]);
    amax = fmaxf(amax, largest(v[i]));
  }
  if (__syncthreads_or(!(amax < INFINITY))) {
    amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kBlockIter; ++i) {
      amax = fmaxf(amax, largest_finite(v[i]));
      infinite_to_nan(v[i]);
    }
  }
  amax = max_of<32>(amax);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBlockThreads / 32; ++i) amax = fmaxf(amax, s_part[i]);
  const float s = block_scale(amax);
  const Divisor by(s);
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
  for (int i = 0; i < kBlockIter; ++i) {
    const int row = r0 + i * kBlockRows;
    if (row < M) store_e4m3<VEC>(q + (long long)row * K, col0, t, K, v[i], by);
  }
}

inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
// Rows of x in whole pieces on 16-byte boundaries.
template <typename T>
bool pieces(const void* x, long long ld, int K) { return K % kPiece == 0 && ld * (long long)sizeof(T) % 16 == 0 && aligned(x, 16); }

template <typename T, bool VEC, bool Q>
cudaError_t rmsnorm_as(const RmsNormArgs& a, cudaStream_t st) {
  if (a.K > kAheadK)
    return launch_pdl(rmsnorm_long_kernel<T, VEC, Q>, dim3((unsigned)a.M), dim3(kLongThreads), 0, st, static_cast<const T*>(a.x), a.ldx,
                      static_cast<const T*>(a.residual), a.weight, a.eps, static_cast<T*>(a.sum), a.out, a.scale, a.K);
  const int threads = ((a.K + kGroup - 1) / kGroup * kLanes + 31) / 32 * 32;
  // as many CTAs as find room at once: 768 threads an SM with 80 registers each (4096 x 4096: 512 23.9 us, 768 19.8, 1280 21.2, measured without
  // the quotients' correction), 1024 with 64
  auto kern = threads <= 384 ? rmsnorm_kernel<T, VEC, Q, 384> : threads <= 512 ? rmsnorm_kernel<T, VEC, Q, 512> : rmsnorm_kernel<T, VEC, Q, 1024>;
  const long long grid = (long long)(a.sm_count > 0 ? a.sm_count : 148) * (threads <= 384 ? 768 / threads : 1024 / threads);
  return launch_pdl(kern, dim3((unsigned)(grid < a.M ? grid : a.M)), dim3(threads), 0, st, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.residual),
                    a.weight, a.eps, static_cast<T*>(a.sum), a.out, a.scale, a.M, a.K);
}
template <typename T>
cudaError_t rmsnorm_of(const RmsNormArgs& a, cudaStream_t st) {
  const bool vec = pieces<T>(a.x, a.ldx, a.K) && aligned(a.residual, 16) && aligned(a.weight, 16) && aligned(a.sum, 16) && aligned(a.out, a.to_e4m3 ? kPiece : 16);
  if (a.to_e4m3) return vec ? rmsnorm_as<T, true, true>(a, st) : rmsnorm_as<T, false, true>(a, st);
  return vec ? rmsnorm_as<T, true, false>(a, st) : rmsnorm_as<T, false, false>(a, st);
}

template <typename T, bool VEC, bool Q>
cudaError_t gated_as(const GatedArgs& a, cudaStream_t st) {
  const int kb = (a.K + kGroup - 1) / kGroup;
  const long long blocks = (long long)a.M * kb, each = kGatedBlocks * (a.up ? 1 : 2);
  if (blocks > 0x7fffffffLL - each) return cudaErrorInvalidValue;
  auto kern = a.up ? (a.act == kActSilu ? gated_kernel<T, VEC, Q, true, kActSilu> : gated_kernel<T, VEC, Q, true, -1>)
                   : (a.act == kActNone ? gated_kernel<T, VEC, Q, false, kActNone> : gated_kernel<T, VEC, Q, false, -1>);
  return launch_pdl(kern, dim3((unsigned)((blocks + each - 1) / each)), dim3(kGatedThreads), 0, st,
                    static_cast<const T*>(a.gate), static_cast<const T*>(a.up), a.ld, a.out, a.scale, (uint32_t)blocks, epi::fast_div((uint32_t)kb), a.K, a.act);
}
template <typename T>
cudaError_t gated_of(const GatedArgs& a, cudaStream_t st) {
  const bool vec = pieces<T>(a.gate, a.ld, a.K) && aligned(a.up, 16) && aligned(a.out, a.to_e4m3 ? kPiece : 16);
  if (a.to_e4m3) return vec ? gated_as<T, true, true>(a, st) : gated_as<T, false, true>(a, st);
  return vec ? gated_as<T, true, false>(a, st) : gated_as<T, false, false>(a, st);
}

template <typename T>
cudaError_t quantize_blocks_of(const T* x, long long ldx, uint8_t* q, float* scale, int M, int K, cudaStream_t st) {
  const bool vec = pieces<T>(x, ldx, K) && aligned(q, kPiece);
  const long long blocks = (long long)((M + kGroup - 1) / kGroup) * ((K + kGroup - 1) / kGroup);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_pdl(vec ? quantize_block_kernel<T, true> : quantize_block_kernel<T, false>, dim3((unsigned)blocks), dim3(kBlockThreads), 0, st, x, ldx, q, scale, M, K);
}

}  // namespace

cudaError_t launch_rmsnorm(const RmsNormArgs& a, cudaStream_t st) {
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
