// Matrix product in 8-bit floating point with a scale for each block of 128:
//   C[m,n] = sum over blocks b of  sa[m,b] * sb[n / 128, b] * sum over k in b of A[m,k] * B[n,k]   (+ bias[n]) (+ ReLU)
// A [M,K] and B [N,K] e4m3, row-major (B as a fully connected layer stores its weights); scales, sums and the epilogue fp32.
//
// A block of 128 values is one row of a 128-byte swizzled tile, so TMA lands it as tcgen05.mma.kind::f8f6f4 wants it: four MMAs
// of 32 a block.  The scales differ from block to block and the tensor core cannot apply them, so each block's sum is taken
// out of tensor memory and added, times its scale, to fp32 sums in the registers of eight warps; tensor memory holds the sums of
// several blocks, and the MMAs of the next ones go on meanwhile.
// Rows and columns behind M and N read as zero and are not stored.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <mutex>

#include "epilogue.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace nncv_b200 {
namespace {

constexpr int kBM = 128, kBlockK = 128;
constexpr int kEpiWarps = 8, kEpiThreads = kEpiWarps * 32, kThreads = 64 + kEpiThreads;
constexpr int kMaxStages = 8, kMaxAccs = 4;
constexpr size_t kSmemLimit = 225 * 1024;

struct GeParams {
  const float* scale_a;
  const float* scale_b;
  const float* bias;
  void* C;
  int* error_flag;
  int M, N, KB;
  int m_tiles, n_tiles;
  int c_type;    // DType
  int relu, vec;
  int stages;
};

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
gemm_e4m3_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const GeParams p) {
  constexpr uint32_t kABytes = kBM * kBlockK, kBBytes = BN * kBlockK, kStageBytes = kABytes + kBBytes;
  constexpr int kAccs = BN == 256 ? 2 : 4;
  constexpr uint32_t kTmemCols = kAccs * BN;
  constexpr int kCols = BN / 2;      // columns of a tile that one thread adds up
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_abort;
  __shared__ uint32_t s_tmem;
  __shared__ __align__(8) uint64_t s_bars[2 * kMaxStages + 2 * kMaxAccs + 1];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  const uint32_t full = ptx::smem_u32(s_bars), empty = full + 8 * kMaxStages, acc_full = empty + 8 * kMaxStages, acc_empty = acc_full + 8 * kMaxAccs;
  const uint32_t drained = acc_empty + 8 * kMaxAccs;
  {
    uint32_t dyn_bytes;
    asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_bytes));
    if (ring + (uint32_t)p.stages * kStageBytes > raw + dyn_bytes || p.stages > kMaxStages) {
      if (threadIdx.x == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrBounds);
      return;
    }
  }
  const int warp = ptx::warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(full + 8 * i, 1);
      ptx::mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kAccs; ++i) {
      ptx::mbar_init(acc_full + 8 * i, 1);
      ptx::mbar_init(acc_empty + 8 * i, kEpiWarps);
    }
    ptx::mbar_init(drained, 1);
    ptx::mbar_fence_init();
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_b);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = (uint32_t)ptx::warp_uniform((int)*reinterpret_cast<volatile uint32_t*>(&s_tmem));
  volatile int* abort_flag = &s_abort;
  const int total = p.m_tiles * p.n_tiles;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer ----
    const uint32_t issue = ptx::elect_one();
    uint32_t st = 0, ph = 0, cnt = 0;
    bool okw = true;
    for (int t = blockIdx.x; t < total && okw; t += gridDim.x) {
      const int nt = t / p.m_tiles, m0 = (t - nt * p.m_tiles) * kBM, n0 = nt * BN;
      for (int kb = 0; kb < p.KB; ++kb, ++cnt) {
        if (!ptx::warp_wait(empty + 8 * st, ph ^ 1u, abort_flag)) { okw = false; break; }
        ptx::mbar_arrive_expect_tx(full + 8 * st, kStageBytes, issue);
        ptx::tma_load_2d(ring + st * kStageBytes, &tm_a, kb * kBlockK, m0, full + 8 * st, issue);
        ptx::tma_load_2d(ring + st * kStageBytes + kABytes, &tm_b, kb * kBlockK, n0, full + 8 * st, issue);
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
      }
    }
    if (!okw) {   // copies in flight land before the CTA ends
      for (uint32_t i = cnt > (uint32_t)p.stages ? cnt - p.stages : 0; i < cnt; ++i) ptx::mbar_wait(full + 8 * (i % p.stages), (i / p.stages) & 1u);
      if (lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitProducer);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer ------
    const uint32_t issue = ptx::elect_one();
    const uint32_t idesc = ptx::umma_idesc(kBM, BN, 0);   // e4m3 times e4m3
    uint32_t st = 0, ph = 0, ac = 0, aph = 0;
    bool okw = true;
    for (int t = blockIdx.x; t < total && okw; t += gridDim.x) {
      for (int kb = 0; kb < p.KB; ++kb) {
        if (!ptx::warp_wait(acc_empty + 8 * ac, aph ^ 1u, abort_flag) || !ptx::warp_wait(full + 8 * st, ph, abort_flag)) { okw = false; break; }
        ptx::tc_fence_after();
        const uint32_t a = ptx::smem_desc_k128_lo(ring + st * kStageBytes), b = ptx::smem_desc_k128_lo(ring + st * kStageBytes + kABytes);
#pragma unroll
        for (uint32_t k4 = 0; k4 < 4; ++k4)
          ptx::umma_f8(tmem_base + ac * BN, ptx::desc_from_halves(a + k4 * 2, ptx::kSmemDescK128Hi), ptx::desc_from_halves(b + k4 * 2, ptx::kSmemDescK128Hi),
                       idesc, k4 != 0 ? 1u : 0u, issue);
        ptx::tc_commit(empty + 8 * st, issue);
        ptx::tc_commit(acc_full + 8 * ac, issue);
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        if (++ac == kAccs) { ac = 0; aph ^= 1u; }
      }
    }
    if (!okw) {   // MMAs in flight end before their memory is given back
      ptx::tc_commit(drained, issue);
      ptx::mbar_wait(drained, 0);
      if (lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitMma);
    }
  } else {
    // ------------------------------------------------------------------ scaled sums -----
    const int quad = warp & 3, half = (warp - 2) >> 2;      // tensor-memory lanes this warp may read; which columns
    const int lrow = quad * 32 + lane;
    uint32_t ac = 0, aph = 0;
    bool okw = true;
    for (int t = blockIdx.x; t < total && okw; t += gridDim.x) {
      const int nt = t / p.m_tiles, m0 = (t - nt * p.m_tiles) * kBM, n0 = nt * BN + half * kCols;
      const int row = m0 + lrow;
      const bool live = n0 < p.N && m0 + quad * 32 < p.M;   // of the warp: some of its part of the tile lies inside the matrix
      const float* sa = p.scale_a + (size_t)(row < p.M ? row : 0) * p.KB;
      const float* sb = p.scale_b + (size_t)(live ? n0 / kBlockK : 0) * p.KB;
      unsigned long long sum[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) sum[i] = 0ull;
      float next_a = __ldg(sa), next_b = __ldg(sb);
      for (int kb = 0; kb < p.KB; ++kb) {
        const float s = next_a * next_b;
        const unsigned long long s2 = epi::pk(s, s);
        if (kb + 1 < p.KB) { next_a = __ldg(sa + kb + 1); next_b = __ldg(sb + kb + 1); }
        if (!ptx::warp_wait(acc_full + 8 * ac, aph, abort_flag)) { okw = false; break; }
        ptx::tc_fence_after();
        if (live) {
          const uint32_t at = tmem_base + ((uint32_t)(quad * 32) << 16) + ac * BN + half * kCols;
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t v[32];
            ptx::tmem_ld_32x32(at + c, v);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              sum[c / 2 + i] = epi::fma2(epi::pk(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), s2, sum[c / 2 + i]);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(acc_empty + 8 * ac);
        if (++ac == kAccs) { ac = 0; aph ^= 1u; }
      }
      if (!okw || row >= p.M || !live) continue;
      const size_t o = (size_t)row * p.N;
#pragma unroll
      for (int c = 0; c < kCols; c += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) epi::unpk(sum[c / 2 + i], v[2 * i], v[2 * i + 1]);
        const int n = n0 + c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (p.bias && n + i < p.N) v[i] += __ldg(p.bias + n + i);
          if (p.relu) v[i] = !(v[i] <= 0.0f) ? v[i] : 0.0f;
        }
        if (p.c_type == kF32) {
          float* q = static_cast<float*>(p.C) + o + n;
          if (p.vec && n + 8 <= p.N) {
            reinterpret_cast<float4*>(q)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(q)[1] = make_float4(v[4], v[5], v[6], v[7]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + i < p.N) q[i] = v[i];
          }
        } else {
          unsigned short* q = static_cast<unsigned short*>(p.C) + o + n;
          uint32_t h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = epi::pack16(v[2 * i], v[2 * i + 1], p.c_type == kBF16, false);
          if (p.vec && n + 8 <= p.N) {
            *reinterpret_cast<uint4*>(q) = make_uint4(h[0], h[1], h[2], h[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + i < p.N) q[i] = (unsigned short)(h[i >> 1] >> (16 * (i & 1)));
          }
        }
      }
    }
    if (!okw && lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitEpilogue);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) ptx::tmem_dealloc(tmem_base, kTmemCols);
}

PFN_cuTensorMapEncodeTiled_v12000 ge_get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// 2-D map over a row-major [rows, K] matrix of bytes, box 128 x box_rows, 128-byte swizzle, zero fill.
bool ge_map(CUtensorMap* m, const void* ptr, long long rows, long long K, int box_rows) {
  auto enc = ge_get_encode();
  if (!enc) return false;
  cuuint64_t gdim[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t gstr[1] = {(cuuint64_t)K};
  cuuint32_t box[2] = {kBlockK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
cudaError_t launch_as(const GemmE4m3Args& a, GeParams p, cudaStream_t st) {
  const size_t stage = (size_t)(kBM + BN) * kBlockK;
  size_t n = (kSmemLimit - 1024) / stage;
  p.stages = (int)(n < kMaxStages ? n : kMaxStages);
  const size_t smem = 1024 + p.stages * stage;
  p.m_tiles = (a.M + kBM - 1) / kBM;
  p.n_tiles = (a.N + BN - 1) / BN;
  if ((long long)p.m_tiles * p.n_tiles > 0x3fffffffLL) return cudaErrorInvalidValue;
  CUtensorMap tm_a, tm_b;
  if (!ge_map(&tm_a, a.A, a.M, a.K, kBM) || !ge_map(&tm_b, a.B, a.N, a.K, BN)) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(gemm_e4m3_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int sms = a.sm_count > 0 ? a.sm_count : 148, items = p.m_tiles * p.n_tiles;
  return launch_pdl(gemm_e4m3_kernel<BN>, dim3(items < sms ? items : sms), dim3(kThreads), smem, st, tm_a, tm_b, p);
}

}  // namespace

cudaError_t launch_gemm_e4m3(const GemmE4m3Args& a, cudaStream_t st) {
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.K % 16 != 0) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(a.A) & 15) || (reinterpret_cast<uintptr_t>(a.B) & 15)) return cudaErrorMisalignedAddress;
  GeParams p{};
  p.scale_a = a.scale_a; p.scale_b = a.scale_b; p.bias = a.bias; p.C = a.C; p.error_flag = a.error_flag;
  p.M = a.M; p.N = a.N; p.KB = (a.K + kBlockK - 1) / kBlockK;
  p.c_type = a.c_dtype; p.relu = a.relu;
  p.vec = (reinterpret_cast<uintptr_t>(a.C) & 15) == 0 && (long long)a.N * (long long)dtype_size(a.c_dtype) % 16 == 0;
  const int sms = a.sm_count > 0 ? a.sm_count : 148;
  auto tiles = [&](int bn) { return (long long)((a.M + kBM - 1) / kBM) * ((a.N + bn - 1) / bn); };
  if (tiles(256) >= sms) return launch_as<256>(a, p, st);
  if (tiles(128) >= sms) return launch_as<128>(a, p, st);
  return launch_as<64>(a, p, st);
}

}  // namespace nncv_b200
