// Matrix product in 8-bit floating point with a scale for each block of 128:
//   C[m,n] = sum over blocks b of  sa[m,b] * sb[n / 128, b] * sum over k in b of A[m,k] * B[n,k]   (+ bias[n]) (+ ReLU)
// A [M,K] and B [N,K] e4m3, row-major (B as a fully connected layer stores its weights); scales, sums and the epilogue fp32.
//
// A block of 128 values is one row of a 128-byte swizzled tile, so TMA lands it as tcgen05.mma.kind::f8f6f4 wants it: four MMAs
// of 32 a block.  The scales differ from block to block and the tensor core cannot apply them, so each block's sum is taken
// out of tensor memory and added, times its scale, to fp32 sums in the registers of the epilogue warps; tensor memory holds the
// sums of several blocks, and the MMAs of the next ones go on meanwhile.
// Roles: warp 0 copies, warp 1 issues the MMAs, warps 2 and 3 bring the products of the scales, the others add up and store.
// Columns behind N read as zero, rows behind M as zero or, below 128 rows, as what lies there; neither is stored.  Every wait is bounded
// and abortable; one that runs out sets the device status word.
//
// What bounds it.  Large: the power limit.  A block of a 256 x 256 tile on a CTA pair is 512 clocks of MMAs; copies and MMAs alone take
// 540, with the sums taken out and scaled 640, with the result's stores 708 on average; the clock falls from 1.97 to 1.3 GHz.
// 8192 x 8192 x 4096 to bf16: 227 us in a burst (2420 TFLOP/s), 270 back to back; MMAs, copies and hand-overs alone 171 and 216, the
// vendor library's product with one scale a matrix 186 and 225.  The epilogue warps of an SM quarter need 256 clocks of
// multiply-adds and 180 of tensor-memory loads a block, and the two do not overlap; sixteen epilogue warps instead of eight were 7 %
// slower, one release of both parts 2 %, one wait a part 3 %, halves of tiles in the last round no faster.
// Middle sizes: what an SM takes in from L2, about 56 bytes a clock (a block of 128 x 128 is 32 KB: 600 clocks where its MMAs take 256).
// Few rows: reading B (4.4 TB/s of 6.5 at 16 x 8192 x 8192), and for one small layer what is fixed: of the 6.4 us of 1 x 4096 x 4096 (7.6 with B from memory)
// 1.9 pass until the first block is here, 2 while B comes, 1.9 while the CTAs of a cluster meet and add up.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <mutex>

#include "e4m3_tile.h"
#include "epilogue.cuh"
#include "kernels.h"
#include "pair_copies.h"
#include "ptx.cuh"

namespace nncv_b200 {
namespace {

constexpr int kBM = 128, kBlockK = 128;
constexpr int kMaxStages = 20, kMaxAccs = 4;
constexpr size_t kSmemLimit = 226 * 1024;   // beside it a few hundred bytes of static shared memory
constexpr int kGroupM = 8;                  // row tiles that are walked together with all column tiles: both operands' tiles stay in L2
constexpr int kBufs = 2;                    // staging buffers of a warp, 32 rows of 128 bytes each
constexpr int kSlots = 16;                  // blocks whose products of scales are held
constexpr int kScaleBytes = kSlots * (kBM + 4) * 8;

constexpr int threads_of(int bn) { return bn == 64 ? 256 : 384; }

struct GeParams {
  const float* scale_a;
  const float* scale_b;
  const float* bias;
  void* C;
  int* error_flag;
  int M, N, KB;
  int m_tiles, n_tiles;       // of a CTA or of a pair
  epi::FastDiv div_band, div_last;
  int a_bytes;                // of A in a stage: with fewer than 128 rows the MMAs read on into what follows, and nobody reads those rows of the sums
  int c_type;                 // DType
  int relu, vec;              // vec: rows of C start on 16-byte boundaries
  int stages;
  int splits_log;             // (as a power of two) CTAs of a cluster that share a tile's blocks; then every cluster has one tile
};

__device__ __forceinline__ void bias_relu(const GeParams& p, int n, float (&v)[8]) {
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < p.N) v[i] += __ldg(p.bias + n + i);
  }
  if (p.relu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = !(v[i] <= 0.0f) ? v[i] : 0.0f;
  }
}

// 32 rows (a lane each) of 64 columns of a warp's sums from (row, col) on: bias, ReLU, and through the warp's staging buffers out
// of the SM.  TYPE: DType of the result; PLAIN: neither bias nor ReLU.
// (900 clocks a slab: 200 until it is known that the buffer is free, 350 to convert, 250 for the fence between stores and copy.  With rows
// read back and stored in 16-byte pieces 1400 to 2000, with each lane storing its own row's pieces 3500.)
template <int TYPE, bool PLAIN>
__device__ __forceinline__ void store_slab(const GeParams& p, const CUtensorMap* tm_c, uint32_t stage, uint32_t& turn, int row, int col, int lane,
                                           const unsigned long long (&sum)[32]) {
  constexpr bool kF = TYPE == kF32;
  constexpr int kSlab = kF ? 32 : 64;   // columns of 128 bytes
  const uint32_t sw = (uint32_t)(lane & 7);
#pragma unroll
  for (int c = 0; c < 64; c += kSlab) {
    if (col + c >= p.N) break;
    const uint32_t buf = stage + turn * epi::kBufBytes, at = buf + (uint32_t)lane * 128u;
    if (lane == 0) ptx::bulk_wait_read<kBufs - 1>();   // the copy that last read this buffer is done
    __syncwarp();
    unsigned long long seek = 0;
    auto put = [&](bool inf) {
#pragma unroll
      for (int h = 0; h < kSlab / 8; ++h) {   // eight columns
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) epi::unpk(sum[c / 2 + h * 4 + i], v[2 * i], v[2 * i + 1]);
        if (!PLAIN) bias_relu(p, col + c + h * 8, v);
        if (kF) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            epi::sts128(at + ((uint32_t)(2 * h + q) ^ sw) * 16u, __float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                        __float_as_uint(v[4 * q + 3]));
        } else {
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (TYPE == kF16 && !inf) epi::seek_inf(v[2 * i], v[2 * i + 1], seek);
            o[i] = inf ? epi::pack_half2_inf(v[2 * i], v[2 * i + 1]) : epi::pack16(v[2 * i], v[2 * i + 1], TYPE == kBF16, false);
          }
          epi::sts128(at + ((uint32_t)h ^ sw) * 16u, o[0], o[1], o[2], o[3]);
        }
      }
    };
    put(false);
    if (TYPE == kF16 && epi::found_inf(seek)) put(true);   // infinite values stay infinite (asked for every eight columns: 4 % of a product, now 1)
    if (p.vec) {
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        ptx::tma_store_2d(tm_c, col + c, row, buf);   // what lies outside the matrix is not written
        ptx::bulk_commit();
      }
    } else {   // rows that are not on 16-byte boundaries: the warp writes them one after the other
      __syncwarp();
      const int rows = p.M - row < 32 ? p.M - row : 32, cols = p.N - col - c < kSlab ? p.N - col - c : kSlab;
      for (int r = 0; r < rows; ++r) {
        const size_t o = (size_t)(row + r) * p.N + col + c;
        for (int j = lane; j < cols; j += 32) {
          const uint32_t byte = (uint32_t)j * (kF ? 4u : 2u), from = buf + (uint32_t)r * 128u + ((byte >> 4) ^ (uint32_t)(r & 7)) * 16u + (byte & 15u);
          if (kF) {
            static_cast<float*>(p.C)[o + j] = epi::lds32(from);
          } else {
            uint16_t v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from));
            static_cast<uint16_t*>(p.C)[o + j] = v;
          }
        }
      }
      __syncwarp();
    }
    turn = turn + 1 == kBufs ? 0u : turn + 1;
  }
}

// v times s (a pair of the same factor) added to sum[AT / 2 ..].
template <int AT>
__device__ __forceinline__ void add_chunk(const uint32_t (&v)[32], unsigned long long s2, unsigned long long (&sum)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[AT / 2 + i] = epi::fma2(epi::pk(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), s2, sum[AT / 2 + i]);
}

// Tiles of 128 x 64 or 128 x 128 (one CTA, or a cluster that shares the tile's blocks), or of 256 x 128 or 256 x 256 on a CTA pair.  Of
// the last, an accumulator has two parts of 128 columns, which are given back one after the other, so that the MMAs of the next
// block but one start when half of this one has been read (in one part: 239 us instead of 234 at 8192 x 8192 x 4096).
template <int BN, bool PAIR>
__global__ void __launch_bounds__(threads_of(BN), 1)
gemm_e4m3_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_c,
                 const GeParams p) {
  constexpr int EW = BN == 64 ? 4 : 8;
  constexpr uint32_t kBBytes = (PAIR ? BN / 2 : BN) * kBlockK;
  constexpr int kAccs = BN == 256 ? 2 : 4;
  constexpr uint32_t kTmemCols = kAccs * BN;
  constexpr int kNS = BN == 256 ? 2 : 1, kPartN = BN / kNS;    // column parts of an accumulator; a warp has 64 columns of each
  static_assert(kPartN == 16 * EW, "");
  // products of the scales of a block, of each row for each part; the lanes of a store (4 blocks x 8 rows) meet no bank twice
  constexpr uint32_t kSlotBytes = (kBM + 4) * 4 * kNS;
  static_assert(kSlots * kSlotBytes <= (uint32_t)kScaleBytes, "");
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_abort;
  __shared__ int s_gave_up;         // of a pair, in both CTAs: a producer of theirs did
  __shared__ __align__(8) long long s_issued;   // blocks whose copies this CTA has issued
  __shared__ uint32_t s_tmem;
  __shared__ __align__(8) uint64_t s_bars[2 * kMaxStages + 3 * kMaxAccs + 1];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  const uint32_t stage_bytes = (uint32_t)p.a_bytes + kBBytes;
  const uint32_t staging = ring + (uint32_t)p.stages * stage_bytes, scales = staging + EW * kBufs * epi::kBufBytes;
  const uint32_t full = ptx::smem_u32(s_bars), empty = full + 8 * kMaxStages, acc_full = empty + 8 * kMaxStages, acc_empty = acc_full + 8 * kMaxAccs;
  const uint32_t drained = acc_empty + 16 * kMaxAccs;
  {
    uint32_t dyn_bytes;
    asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_bytes));
    if (scales + kScaleBytes > raw + dyn_bytes || p.stages > kMaxStages) {   // the same in every CTA
      if (threadIdx.x == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrBounds);
      return;
    }
  }
  const int warp = ptx::warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = PAIR || p.splits_log ? ptx::cluster_ctarank() : 0u;
  if (threadIdx.x == 0) {
    s_abort = 0;
    s_gave_up = 0;
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(full + 8 * i, 1);
      ptx::mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kAccs; ++i) ptx::mbar_init(acc_full + 8 * i, 3);   // the MMAs, and both warps that bring the scales
    for (int i = 0; i < kAccs * kNS; ++i) ptx::mbar_init(acc_empty + 8 * i, PAIR ? 2 * EW : EW);
    ptx::mbar_init(drained, 1);
    ptx::mbar_fence_init();
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_b);
  }
  if (warp == 1) {
    if (PAIR) {
      ptx::tmem_alloc_pair(ptx::smem_u32(&s_tmem), kTmemCols);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(ptx::smem_u32(&s_tmem), kTmemCols);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_sync_all();   // both CTAs' barriers exist before anyone arrives remotely
  ptx::tc_fence_after();
  const uint32_t tmem_base = (uint32_t)ptx::warp_uniform((int)*reinterpret_cast<volatile uint32_t*>(&s_tmem));
  volatile int* abort_flag = &s_abort;
  const int total = p.m_tiles * p.n_tiles;
  const int group_log = PAIR ? 1 : p.splits_log;   // CTAs that work on one tile
  const int worker = (int)blockIdx.x >> group_log, workers = (int)gridDim.x >> group_log;
  const int kb_lo = PAIR ? 0 : (p.KB * (int)rank) >> p.splits_log, kb_hi = PAIR ? p.KB : (p.KB * ((int)rank + 1)) >> p.splits_log;
  auto item = [&](int i, int& m0, int& n0) {   // tile i of this worker: first row of this CTA, first column
    const int t = worker + i * workers;
    if (t >= total) return false;
    const int band = (int)epi::div_by((uint32_t)t, p.div_band), r = t - band * kGroupM * p.n_tiles;
    const bool last = (band + 1) * kGroupM > p.m_tiles;
    const int rows = last ? p.m_tiles - band * kGroupM : kGroupM;
    const int nt = last ? (int)epi::div_by((uint32_t)r, p.div_last) : r / kGroupM, mt = band * kGroupM + r - nt * rows;
    m0 = (PAIR ? 2 * mt + (int)rank : mt) * kBM;
    n0 = nt * BN;
    return true;
  };
  // The first blocks of B start on their way to L2 while the previous kernel of the stream ends.  Nothing is read yet: should that
  // kernel write B, its stores meet the same L2 lines.
  if (warp == 0) {
    int m0, n0;
    if (item(0, m0, n0)) {
      if (PAIR) n0 += (int)rank * (kPartN / 2);
      const int most = kb_lo + p.stages < kb_hi ? kb_lo + p.stages : kb_hi;
      const uint32_t issue = ptx::elect_one();
      for (int kb = kb_lo; kb < most; ++kb)
#pragma unroll
        for (int h = 0; h < kNS; ++h) ptx::tma_prefetch_2d(&tm_b, kb * kBlockK, n0 + h * kPartN, issue);
    }
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  // 256 x 256: 384 threads start with 168 registers each (64,512); the first four warps give up what the others take:
  // 128 * 72 + 256 * 216 = 64,512
  if (warp < 4) {
    if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA producer ----
      const uint32_t issue = ptx::elect_one();
      const uint32_t full_at = PAIR ? ptx::map_to_cta(full, 0) : full;   // the bytes of a stage, of both CTAs, are counted on the leader's barrier
      uint32_t st = 0, ph = 0, used = 0;
      bool okw = true;
      int m0, n0, i = 0, kb = 0;
      for (; item(i, m0, n0); ++i) {
        if (PAIR) n0 += (int)rank * (kPartN / 2);   // each CTA brings half of the columns of every part
        for (kb = kb_lo; kb < kb_hi; ++kb) {
          if (!ptx::warp_wait(empty + 8 * st, ph ^ 1u, abort_flag)) { okw = false; break; }
          const uint32_t dst = ring + st * stage_bytes, dst_b = dst + (uint32_t)p.a_bytes;
          if (PAIR) {
            if (rank == 0) ptx::mbar_arrive_expect_tx(full + 8 * st, 2 * stage_bytes, issue);
            ptx::tma_load_2d_pair(dst, &tm_a, kb * kBlockK, m0, full_at + 8 * st, issue);
#pragma unroll
            for (int h = 0; h < kNS; ++h)
              ptx::tma_load_2d_pair(dst_b + h * (kBBytes / kNS), &tm_b, kb * kBlockK, n0 + h * kPartN, full_at + 8 * st, issue);
          } else {
            ptx::mbar_arrive_expect_tx(full + 8 * st, stage_bytes, issue);
            ptx::tma_load_2d(dst, &tm_a, kb * kBlockK, m0, full + 8 * st, issue);
            ptx::tma_load_2d(dst_b, &tm_b, kb * kBlockK, n0, full + 8 * st, issue);
          }
          used |= 1u << st;
          if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        }
        if (!okw) break;
        kb = 0;
      }
      if (PAIR && lane == 0) s_issued = (long long)i * p.KB + kb;
      if (!okw) {   // copies in flight land before the CTA ends: of a pair after both have met, else here the last round of every stage that was used
        if (PAIR) {
          if (lane == 0) {
            s_gave_up = 1;
            ptx::st_cluster(ptx::map_to_cta(ptx::smem_u32(&s_gave_up), rank ^ 1u), 1u);
          }
        } else {
          for (uint32_t j = 0; j < (uint32_t)p.stages; ++j)
            if (used >> j & 1u) ptx::mbar_wait(full + 8 * j, j < st ? ph : ph ^ 1u);
        }
        if (lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitProducer);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issuer ------
      if (!PAIR || rank == 0) {
        const uint32_t issue = ptx::elect_one();
        constexpr uint32_t idesc = ptx::umma_idesc(PAIR ? 2 * kBM : kBM, kPartN, 0);   // e4m3 times e4m3
        uint32_t st = 0, ph = 0, ac = 0, aph = 0;
        bool okw = true;
        int m0, n0;
        auto multiply = [&](int h) {
          const uint32_t a = ptx::smem_desc_k128_lo(ring + st * stage_bytes), b = ptx::smem_desc_k128_lo(ring + st * stage_bytes + (uint32_t)p.a_bytes);
          ptx::tc_fence_after();
#pragma unroll
          for (uint32_t k4 = 0; k4 < 4; ++k4) {
            const uint64_t da = ptx::desc_from_halves(a + k4 * 2, ptx::kSmemDescK128Hi);
            const uint64_t db = ptx::desc_from_halves(b + (uint32_t)h * ((kBBytes / kNS) >> 4) + k4 * 2, ptx::kSmemDescK128Hi);
            const uint32_t d = tmem_base + ac * BN + h * kPartN;
            if (PAIR) ptx::umma_f8_pair(d, da, db, idesc, k4 != 0 ? 1u : 0u, issue);
            else ptx::umma_f8(d, da, db, idesc, k4 != 0 ? 1u : 0u, issue);
          }
        };
        auto next = [&]() {
          if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
          if (++ac == kAccs) { ac = 0; aph ^= 1u; }
        };
        // One CTA: whether the next stage and accumulator are there is asked before a block's MMAs are issued; the answers take a hundred
        // clocks each, and with them in line a block took 390 clocks whatever its tile.  A pair's MMAs take longer than that, and
        // with the questions asked early it was 4 % slower.
        uint32_t seen = 0, seen_acc = 1;   // nothing has used the accumulators yet
        for (int i = 0; okw && item(i, m0, n0); ++i) {
          for (int kb = kb_lo; kb < kb_hi; ++kb) {
            if (PAIR) {
              if (!ptx::warp_spin(full + 8 * st, ph, abort_flag)) { okw = false; break; }
#pragma unroll
              for (int h = 0; h < kNS; ++h) {
                if (!ptx::warp_spin_cluster(acc_empty + 8 * (ac * kNS + h), aph ^ 1u, abort_flag)) { okw = false; break; }
                multiply(h);
              }
              if (!okw) break;
              ptx::tc_commit_pair(acc_full + 8 * ac, issue);
              ptx::tc_commit_pair(empty + 8 * st, issue);
              next();
            } else {
              if (!ptx::warp_all(seen) && !ptx::warp_spin(full + 8 * st, ph, abort_flag)) { okw = false; break; }
              if (!ptx::warp_all(seen_acc) && !ptx::warp_spin(acc_empty + 8 * ac, aph ^ 1u, abort_flag)) { okw = false; break; }
              const uint32_t st1 = st + 1 == (uint32_t)p.stages ? 0u : st + 1, ac1 = ac + 1 == kAccs ? 0u : ac + 1;
              seen = ptx::mbar_peek(full + 8 * st1, st1 == 0 ? ph ^ 1u : ph);
              seen_acc = ptx::mbar_peek(acc_empty + 8 * ac1, ac1 == 0 ? aph : aph ^ 1u);
              multiply(0);
              ptx::tc_commit(acc_full + 8 * ac, issue);
              ptx::tc_commit(empty + 8 * st, issue);
              next();
            }
          }
        }
        if (!okw) {   // MMAs in flight end before their memory is given back
          if (PAIR) ptx::tc_commit_pair(drained, issue);
          else ptx::tc_commit(drained, issue);
          ptx::mbar_wait(drained, 0);
          if (lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitMma);
        }
      }
    } else {
      // ---------------------------------------------------------------- scales ----------
      // The products of the scales of every row, for each part, go to shared memory: with loads of its own an epilogue warp lost 70 clocks a
      // block.  They come for a chunk of blocks at once, a chunk ahead of their use (a row a lane and a block at a time, 32 sectors a
      // load set the pace of the smaller tiles: 512 x 4096 x 4096 on 256 x 128 tiles 14.0 us, now 12.2).
      // A chunk is written when its first block's turn has come: the MMAs of kAccs blocks ago are complete then, so they were issued, so
      // block 2 kAccs ago, four or eight, has been read, while the slots written are those of 13 blocks ago and older.
      constexpr int kChunk = 4, kRows = 32 / kChunk, kLoads = 64 / kRows;   // blocks and rows of a load (8 x 4: 0.3 us later at the first block)
      const int k = lane & (kChunk - 1), r0 = (warp - 2) * 64 + lane / kChunk;
      uint32_t ac = 0, aph = 0, slot = 0;
      bool okw = true;
      float v[kLoads], f0 = 0.0f, f1 = 0.0f;
      auto fetch = [&](int m0, int n0, int kb) {
        const float* sa = p.scale_a + (size_t)(m0 + r0) * p.KB + kb + k;
        const float* sb = p.scale_b + (size_t)(n0 / kBlockK) * p.KB + kb + k;
        const bool in = kb + k < kb_hi;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) v[j] = in && m0 + r0 + j * kRows < p.M ? __ldg(sa + (size_t)(j * kRows) * p.KB) : 0.0f;
        f0 = in ? __ldg(sb) : 0.0f;
        if (kNS == 2) f1 = in && n0 + kPartN < p.N ? __ldg(sb + p.KB) : 0.0f;
      };
      auto tell = [&]() {   // this warp's scales of the block are there
        if (lane == 0) ptx::mbar_arrive(acc_full + 8 * ac);
        if (++ac == kAccs) { ac = 0; aph ^= 1u; }
        slot = (slot + 1) & (kSlots - 1);
      };
      int m0, n0;
      bool more = kb_lo < kb_hi && item(0, m0, n0);
      if (more) fetch(m0, n0, kb_lo);
      for (int i = 0; more && okw; ++i) {
        int next_m0, next_n0;
        more = item(i + 1, next_m0, next_n0);
        for (int kb = kb_lo; kb < kb_hi && okw; kb += kChunk) {
          if (!ptx::warp_wait(acc_full + 8 * ac, aph ^ 1u, abort_flag)) { okw = false; break; }
          const uint32_t at = scales + ((slot + (uint32_t)k) & (kSlots - 1)) * kSlotBytes + (uint32_t)r0 * (4 * kNS);
#pragma unroll
          for (uint32_t j = 0; j < kLoads; ++j) {
            if (kNS == 2) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(at + j * (8u * kRows)), "f"(v[j] * f0), "f"(v[j] * f1) : "memory");
            else asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + j * (4u * kRows)), "f"(v[j] * f0) : "memory");
          }
          if (kb + kChunk < kb_hi) fetch(m0, n0, kb + kChunk);
          else if (more) fetch(next_m0, next_n0, kb_lo);
          __syncwarp();
          tell();
          for (int j = 1; j < kChunk && kb + j < kb_hi; ++j) {
            if (!ptx::warp_wait(acc_full + 8 * ac, aph ^ 1u, abort_flag)) { okw = false; break; }
            tell();
          }
        }
        m0 = next_m0;
        n0 = next_n0;
      }
      if (!okw && lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitLoader);
    }
  } else {
    // ------------------------------------------------------------------ scaled sums -----
    // A part's 64 columns come in two loads; while one is added up the next is on its way, that of the next part or block too.
    if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quad = warp & 3, group = (warp - 4) >> 2;      // tensor-memory lanes this warp may read; which columns of each part
    const uint32_t release_at = PAIR ? ptx::map_to_cta(acc_empty, 0) : acc_empty;
    const uint32_t my_tmem = tmem_base + ((uint32_t)(quad * 32) << 16) + group * 64, my_scales = scales + (uint32_t)(quad * 32 + lane) * (4 * kNS);
    const uint32_t my_stage = staging + (uint32_t)(warp - 4) * (kBufs * epi::kBufBytes);
    uint32_t ac = 0, aph = 0, slot = 0, turn = 0;
    bool okw = true;
    auto release = [&](int h) {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) ptx::mbar_arrive_remote_cta(release_at + 8 * (ac * kNS + h));
        else ptx::mbar_arrive(release_at + 8 * (ac * kNS + h));
      }
    };
    auto advance = [&]() {
      if (++ac == kAccs) { ac = 0; aph ^= 1u; }
      slot = (slot + 1) & (kSlots - 1);
    };
    int m0, n0;
    for (int i = 0; okw && item(i, m0, n0); ++i) {
      n0 += group * 64;
      if (n0 >= p.N || m0 + quad * 32 >= p.M || kb_lo == kb_hi) {   // nothing of this warp's part of the tile lies inside the matrix
        for (int kb = kb_lo; kb < kb_hi && okw; ++kb) {
          okw = ptx::warp_wait(acc_full + 8 * ac, aph, abort_flag);
#pragma unroll
          for (int h = 0; h < kNS; ++h) release(h);
          advance();
        }
        continue;
      }
      unsigned long long sum[kNS][32], s2[kNS];
#pragma unroll
      for (int h = 0; h < kNS; ++h)
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[h][j] = 0ull;
      uint32_t v[32], w[32];
      float x = 0.0f, y = 0.0f;
      auto begin = [&](uint32_t seen) {   // the next block: wait for its sums and scales, ask for its first columns
        if (!ptx::warp_all(seen)) okw = ptx::warp_wait(acc_full + 8 * ac, aph, abort_flag);
        ptx::tc_fence_after();
        ptx::tmem_ld_32x32(my_tmem + ac * BN, v);
        const uint32_t at = my_scales + slot * kSlotBytes;
        if (kNS == 2) asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x), "=f"(y) : "r"(at));
        else x = epi::lds32(at);
      };
      begin(0);
      for (int kb = kb_lo; kb < kb_hi && okw; ++kb) {
        s2[0] = epi::pk(x, x);
        if (kNS == 2) s2[kNS - 1] = epi::pk(y, y);
        uint32_t seen = 0;   // whether the next block is there: asked for early, since the answer takes a hundred clocks
#pragma unroll
        for (int h = 0; h < kNS; ++h) {
          ptx::tmem_ld_wait();
          ptx::tmem_ld_32x32(my_tmem + ac * BN + h * kPartN + 32, w);
          if (h + 1 == kNS) {
            const uint32_t wrap = ac + 1 == kAccs ? 1u : 0u;
            seen = ptx::mbar_peek(acc_full + 8 * (wrap ? 0u : ac + 1), aph ^ wrap);
          }
          add_chunk<0>(v, s2[h], sum[h]);
          ptx::tmem_ld_wait();
          release(h);
          if (h + 1 < kNS) {
            ptx::tmem_ld_32x32(my_tmem + ac * BN + (h + 1) * kPartN, v);
          } else {
            advance();
            if (kb + 1 < kb_hi) begin(seen);
          }
          add_chunk<32>(w, s2[h], sum[h]);
        }
      }
      if (!okw) break;
      if (!PAIR && p.splits_log) {   // partial sums: rows of 256 bytes, 16-byte chunks XOR-swizzled by the row, 64 columns a group
        const uint32_t at = staging + (uint32_t)group * (kBM * 256u) + (uint32_t)(quad * 32 + lane) * 256u;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float f[4];
          epi::unpk(sum[0][2 * c], f[0], f[1]);
          epi::unpk(sum[0][2 * c + 1], f[2], f[3]);
          epi::sts128(at + (((uint32_t)c ^ (uint32_t)(lane & 7)) << 4), __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        }
        continue;
      }
      const bool plain = !p.bias && !p.relu;
#pragma unroll
      for (int h = 0; h < kNS; ++h) {
        const int row = m0 + quad * 32, col = n0 + h * kPartN;
#define NNCV_STORE(T_, P_) if (p.c_type == T_ && plain == P_) store_slab<T_, P_>(p, &tm_c, my_stage, turn, row, col, lane, sum[h]);
        NNCV_STORE(kBF16, true) NNCV_STORE(kF16, true) NNCV_STORE(kF32, true) NNCV_STORE(kBF16, false) NNCV_STORE(kF16, false) NNCV_STORE(kF32, false)
#undef NNCV_STORE
      }
    }
    if (lane == 0) ptx::bulk_wait<0>();
    if (!okw && lane == 0 && p.error_flag) atomicCAS(p.error_flag, 0, (int)kErrWaitEpilogue);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (!PAIR && p.splits_log) {
    // The CTAs of the cluster finish the tile together, four columns a thread at a time, adding the partial sums in rank order: the
    // result does not depend on timing.
    int m0, n0;
    item(0, m0, n0);
    ptx::cluster_sync_all();
    const int rows = p.M - m0 < kBM ? p.M - m0 : kBM, S = 1 << p.splits_log;
    for (int e = (int)rank * (int)blockDim.x + (int)threadIdx.x; e < rows * (BN / 4); e += S * (int)blockDim.x) {
      const int r = e / (BN / 4), c = e % (BN / 4), n = n0 + c * 4;
      if (n >= p.N) continue;
      const uint32_t at = staging + (uint32_t)(c / 16) * (kBM * 256u) + (uint32_t)r * 256u + (((uint32_t)(c % 16) ^ (uint32_t)(r & 7)) << 4);
      float4 q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < S) q[j] = ptx::ld_cluster_f4(ptx::map_to_cta(at, (uint32_t)j));
      float v[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
      for (int j = 1; j < 8; ++j)
        if (j < S) { v[0] += q[j].x; v[1] += q[j].y; v[2] += q[j].z; v[3] += q[j].w; }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (p.bias && n + j < p.N) v[j] += __ldg(p.bias + n + j);
        if (p.relu) v[j] = !(v[j] <= 0.0f) ? v[j] : 0.0f;
      }
      const size_t o = (size_t)(m0 + r) * p.N + n;
      if (p.c_type == kF32) {
        float* to = static_cast<float*>(p.C) + o;
        if (p.vec) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        else
          for (int j = 0; j < 4 && n + j < p.N; ++j) to[j] = v[j];
      } else {
        uint16_t* to = static_cast<uint16_t*>(p.C) + o;
        uint32_t h[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          h[j] = p.c_type == kBF16 ? epi::pack16(v[2 * j], v[2 * j + 1], true, false) : epi::pack_half2_inf(v[2 * j], v[2 * j + 1]);
        if (p.vec) *reinterpret_cast<uint2*>(to) = make_uint2(h[0], h[1]);
        else {
          to[0] = (uint16_t)h[0];
          if (n + 1 < p.N) to[1] = (uint16_t)(h[0] >> 16);
          if (n + 2 < p.N) to[2] = (uint16_t)h[1];
          if (n + 3 < p.N) to[3] = (uint16_t)(h[1] >> 16);
        }
      }
    }
    __syncwarp();
    ptx::cluster_sync_all();   // the peers' reads of this CTA's partial sums are over
  }
  if (PAIR) {
    ptx::cluster_sync_all();
    if (*reinterpret_cast<volatile int*>(&s_gave_up)) {   // in both CTAs; the MMAs have ended
      if (warp == 0) {
        const uint32_t issue = ptx::elect_one(), full_at = ptx::map_to_cta(full, 0);
        const long long mine = *reinterpret_cast<volatile long long*>(&s_issued);
        const long long end = pair_copies::meet_at(mine, ptx::ld_cluster_s64(ptx::map_to_cta(ptx::smem_u32(&s_issued), rank ^ 1u)));
        for (long long n = mine; n < end; ++n) {   // nobody reads what these bring
          const uint32_t st = pair_copies::spot_of(n, p.stages).stage, dst = ring + st * stage_bytes;
          if (rank == 0) ptx::mbar_arrive_expect_tx(full + 8 * st, 2 * stage_bytes, issue);
          ptx::tma_load_2d_pair(dst, &tm_a, 0, 0, full_at + 8 * st, issue);
#pragma unroll
          for (int h = 0; h < kNS; ++h) ptx::tma_load_2d_pair(dst + (uint32_t)p.a_bytes + h * (kBBytes / kNS), &tm_b, 0, 0, full_at + 8 * st, issue);
        }
        if (rank == 0)
          for (long long n = pair_copies::wait_from(end, p.stages); n < end; ++n) {
            const pair_copies::Spot at = pair_copies::spot_of(n, p.stages);
            ptx::mbar_wait(full + 8 * at.stage, at.parity);
          }
        __syncwarp();
      }
      ptx::cluster_sync_all();
    }
  }
  if (warp == 1) {
    __syncwarp();
    if (PAIR) ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    else ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
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

// 2-D map over the result, box 32 rows of 128 bytes, 128-byte swizzle.
bool ge_map_c(CUtensorMap* m, void* ptr, DType dt, long long M, long long N) {
  auto enc = ge_get_encode();
  if (!enc) return false;
  const int esz = (int)dtype_size(dt);
  cuuint64_t gdim[2] = {(cuuint64_t)N, (cuuint64_t)M};
  cuuint64_t gstr[1] = {(cuuint64_t)N * esz};
  cuuint32_t box[2] = {(cuuint32_t)(128 / esz), 32};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, dt == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, ptr, gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Shared memory of a launch with `a_rows` rows of A in a stage.
template <int BN, bool PAIR>
size_t smem_of(int a_rows, int* stages) {
  const size_t stage = (size_t)(a_rows + (PAIR ? BN / 2 : BN)) * kBlockK;
  const size_t fixed = 1024 + (size_t)(BN == 64 ? 4 : 8) * kBufs * epi::kBufBytes + kScaleBytes;
  const size_t n = (kSmemLimit - fixed) / stage;
  *stages = (int)(n < kMaxStages ? n : kMaxStages);
  return fixed + *stages * stage;
}

// Tile and CTAs that share a tile's blocks: what the caller asks for where that fits, else the model's choice.
e4m3::Choice pick(const GemmE4m3Args& a, int KB, int sms) {
  int stages;
  static const ClusterFit fit64 = cluster_fit(gemm_e4m3_kernel<64, false>, threads_of(64), smem_of<64, false>(kBM, &stages), sms);
  static const ClusterFit fit128 = cluster_fit(gemm_e4m3_kernel<128, false>, threads_of(128), smem_of<128, false>(kBM, &stages), sms);
  const e4m3::Room room{{fit64.of, fit128.of}, sms};
  return e4m3::fits(a.tile, a.splits, a.M, a.N, KB, room) ? e4m3::Choice{a.tile, a.splits} : e4m3::choose(a.M, a.N, KB, room);
}

template <int BN, bool PAIR>
cudaError_t launch_as(const GemmE4m3Args& a, GeParams p, int splits, cudaStream_t st) {
  auto kern = gemm_e4m3_kernel<BN, PAIR>;
  constexpr int kThreads = threads_of(BN), kTileM = PAIR ? 2 * kBM : kBM;
  const int a_rows = a.M < kBM ? (a.M + 7) / 8 * 8 : kBM;
  p.a_bytes = a_rows * kBlockK;
  const size_t smem = smem_of<BN, PAIR>(a_rows, &p.stages);
  p.m_tiles = (a.M + kTileM - 1) / kTileM;
  p.n_tiles = (a.N + BN - 1) / BN;
  if ((long long)p.m_tiles * p.n_tiles > 0x3fffffffLL) return cudaErrorInvalidValue;
  p.div_band = epi::fast_div((uint32_t)(kGroupM * p.n_tiles));
  p.div_last = epi::fast_div((uint32_t)(p.m_tiles % kGroupM ? p.m_tiles % kGroupM : kGroupM));
  CUtensorMap tm_a, tm_b, tm_c = {};   // a result whose rows are not on 16-byte boundaries is written without a map
  if (!ge_map(&tm_a, a.A, a.M, a.K, a_rows) || !ge_map(&tm_b, a.B, a.N, a.K, PAIR ? 64 : BN)) return cudaErrorInvalidValue;
  if (p.vec && !ge_map_c(&tm_c, a.C, a.c_dtype, a.M, a.N)) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int sms = a.sm_count > 0 ? a.sm_count : 148, items = p.m_tiles * p.n_tiles;
  while (1 << p.splits_log < splits) ++p.splits_log;
  if (!PAIR && splits == 1) return launch_pdl(kern, dim3(items < sms ? items : sms), dim3(kThreads), smem, st, tm_a, tm_b, tm_c, p);
  int size = splits, groups = items;
  if (PAIR) {
    static const int pairs = max_clusters(kern, 2, kThreads, smem, sms);
    size = 2;
    if (items > pairs) groups = pairs;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(size * groups));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, tm_a, tm_b, tm_c, p);
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
  const e4m3::Choice c = pick(a, p.KB, a.sm_count > 0 ? a.sm_count : 148);
  if (a.took) *a.took = c.tile * 16 + c.splits;
  switch (c.tile) {
    case 0: return launch_as<64, false>(a, p, c.splits, st);
    case 1: return launch_as<128, false>(a, p, c.splits, st);
    case 2: return launch_as<128, true>(a, p, 1, st);
    default: return launch_as<256, true>(a, p, 1, st);
  }
}

}  // namespace nncv_b200
