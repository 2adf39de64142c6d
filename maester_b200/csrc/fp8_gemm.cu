// C[M,N] = sum over blocks b of 2^(ea[m,b] + eb[n,b]) * sum over the 128 values of block b of A[m,:] B[n,:]
// for e4m3 codes with block exponents as fp8_blocks.cu writes them.
//
// The tensor core applies the scales itself: tcgen05.mma.kind::mxf8f6f4.block_scale multiplies every group of 32 values of the
// contraction by 2^(ea + eb) on its way into the fp32 accumulator, so the main loop is that of a plain product at the 8-bit
// rate and no partial sum passes through registers.  A scale covers 128 values here: the four instructions (K = 32) of a
// 128-deep k-block select the same exponent byte, and one 32-bit word of tensor memory serves four k-blocks.
//
// The accumulator has 32 bits, and the unit cuts off: an instruction's 32 products are lined up with the sum, what lies below its
// 25th bit or so is lost, and so are the bits of the new sum past the 24th.  Measured: sums that 24 bits hold exactly come out
// exactly, and 8192 products of one sign 65 units of 2^-24 low (256 instructions, a quarter each on average); 3 units for few rows,
// whose contraction is split in eight.
//
// CTA pairs (cta_group::2): a 256 x 256 tile per pair of SMs, each CTA stages its 128 rows of A and its half of B, 128 bytes
// deep, in a 6-stage ring (32 KiB a stage).  The exponents of four k-blocks (512 bytes for 128 rows, in the order of the
// matrix unit) come with the first of them and are copied into tensor memory by tcgen05.cp; both CTAs hold those of all
// 256 rows of B.
//
// Tensor memory: two 256-column accumulators and the exponents do not fit 512 columns, so the accumulators share 32: the
// second starts at column 224, the exponents (two sets, used in turn) are at 480.  The epilogue drains the shared columns
// first and releases them at once; the other columns are double-buffered as usual.
//
// Warp 0: TMA; warp 1: MMA issue (even CTA); warps 2-5: epilogue.  All waits are bounded; both CTAs always reach the cluster
// barriers.
//
// Measured: 16384 x 4096 x 4096 0.211 to 0.216 ms (2550 to 2600 TFLOP/s, 1.55 of the 16-bit rate of 1641), 16384 x 20480 x 2560
// 2390, 16384 x 2560 x 10240 2530.  Bound by power: the tensor pipe is active 81 % of the time at 1.56 GHz, and zeros as
// operands run at 3180.  The copies of the exponents cost 5 % there (3350 without them), the scaling itself as much again (3520
// for the plain 8-bit instruction); issuing the copies in the middle of the previous group was slower (the commit waits for them),
// and so was writing the exponents with four more warps (tcgen05.st, a commit more every four k-blocks: 242 us and more).
#include "gemm_common.cuh"
#include "host_common.cuh"
#include "sm100_pair.cuh"

namespace {
using namespace mb;

enum { OUT_BF16 = 0, OUT_F32 = 1, OUT_F32_ACC = 2 };

constexpr int BM = 128, BN = 256, BNH = 128, BK = 128;   // rows per CTA, tile columns, rows of B per CTA, bytes of K
constexpr int STAGES = 6;
constexpr int A_BYTES = BM * BK, B_BYTES = BNH * BK;
constexpr int SFA_BYTES = 512, SFB_BYTES = 1024;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int SF_BYTES = SFA_BYTES + SFB_BYTES;
constexpr int SF_STRIDE = 2048;
constexpr int THREADS = 192;
constexpr int OUT_STAGE = 4096;                         // 32 x 32 values of an epilogue warp
constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + SF_STRIDE) + 4 * OUT_STAGE + 1024 + 256;
constexpr int GROUP_M = 8;
constexpr uint32_t ACC1 = 224, SF_COL = 480, SF_SET = 16, SFB_COL = 4;

struct Params {
  void* C;
  int M, N, kblocks;
  long long ldc;
  int out;
  int vec;       // 16-byte stores are aligned
  int* status;
};

__device__ __forceinline__ void umma2_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 512 bytes of exponents (32 lanes x 16 bytes) into 4 columns of both CTAs, repeated for the four lane groups
__device__ __forceinline__ void sf_copy2(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// unswizzled operand of 8-row groups of 16 bytes
__device__ __forceinline__ uint64_t sf_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 16;
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* tmap, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar) & PEER_MASK), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// e4m3 x e4m3, power-of-two scales, fp32 accumulation; both operands K-major
constexpr uint32_t idesc_mxf8(int m, int n) {
  return (1u << 23) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// 32 x 32 accumulators of a warp (lane = row, r = columns) -> C through the warp's 4 KiB of shared memory, so that rows leave
// as whole sectors: 16 bytes a lane where C allows it, else a value a lane.  16-byte chunks of a row are swizzled so that neither
// side meets a bank twice.
__device__ __forceinline__ void store_chunk(const Params& p, const uint32_t (&r)[32], int row0, int col0, uint8_t* stage, int lane) {
  if (row0 >= p.M || col0 >= p.N) return;          // (the same for the whole warp)
  MB_CHECK_OR(p.status, row0 >= 0 && col0 >= 0 && static_cast<long long>(min(col0 + 32, p.N)) <= p.ldc, return);
  const int rows = min(32, p.M - row0), cols = min(32, p.N - col0);
  const bool whole = p.vec && cols == 32;
  __syncwarp();
  if (p.out == OUT_BF16) {
    uint4* line = reinterpret_cast<uint4*>(stage + lane * 64);
    const int x = (lane >> 1) & 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 o;
      o.x = pack_bf16(__uint_as_float(r[j * 8 + 0]), __uint_as_float(r[j * 8 + 1]));
      o.y = pack_bf16(__uint_as_float(r[j * 8 + 2]), __uint_as_float(r[j * 8 + 3]));
      o.z = pack_bf16(__uint_as_float(r[j * 8 + 4]), __uint_as_float(r[j * 8 + 5]));
      o.w = pack_bf16(__uint_as_float(r[j * 8 + 6]), __uint_as_float(r[j * 8 + 7]));
      line[j ^ x] = o;
    }
    __syncwarp();
    __nv_bfloat16* c = static_cast<__nv_bfloat16*>(p.C) + static_cast<long long>(row0) * p.ldc + col0;
    if (whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j * 8 + (lane >> 2), part = lane & 3;
        const uint4 o = reinterpret_cast<const uint4*>(stage + row * 64)[part ^ ((row >> 1) & 3)];
        if (row < rows) *reinterpret_cast<uint4*>(c + row * p.ldc + part * 8) = o;
      }
    } else if (lane < cols) {
#pragma unroll 4
      for (int row = 0; row < rows; ++row)
        c[row * p.ldc + lane] = reinterpret_cast<const __nv_bfloat16*>(stage + row * 64)[(((lane >> 3) ^ ((row >> 1) & 3)) << 3) + (lane & 7)];
    }
  } else {
    uint4* line = reinterpret_cast<uint4*>(stage + lane * 128);
#pragma unroll
    for (int j = 0; j < 8; ++j) line[j ^ (lane & 7)] = make_uint4(r[j * 4], r[j * 4 + 1], r[j * 4 + 2], r[j * 4 + 3]);
    __syncwarp();
    float* c = static_cast<float*>(p.C) + static_cast<long long>(row0) * p.ldc + col0;
    const bool acc = p.out == OUT_F32_ACC;
    if (whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = j * 4 + (lane >> 3), part = lane & 7;
        float4 o = reinterpret_cast<const float4*>(stage + row * 128)[part ^ (row & 7)];
        if (row < rows) {
          float4* to = reinterpret_cast<float4*>(c + row * p.ldc + part * 4);
          if (acc) {
            const float4 old = *to;
            o.x += old.x; o.y += old.y; o.z += old.z; o.w += old.w;
          }
          *to = o;
        }
      }
    } else if (lane < cols) {
#pragma unroll 4
      for (int row = 0; row < rows; ++row) {
        const float v = reinterpret_cast<const float*>(stage + row * 128)[(((lane >> 2) ^ (row & 7)) << 2) + (lane & 3)];
        float* to = c + row * p.ldc + lane;
        *to = (acc ? *to : 0.f) + v;
      }
    }
  }
}

__global__ void __launch_bounds__(THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf = smem + STAGES * STAGE_BYTES;
  uint8_t* out_stage = sf + STAGES * SF_STRIDE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_stage + 4 * OUT_STAGE);
  uint64_t* full = bars;                        // [STAGES] used in the even CTA
  uint64_t* empty = bars + STAGES;              // [STAGES] one per CTA
  uint64_t* acc_full = bars + 2 * STAGES;       // [2]      one per CTA
  uint64_t* acc_empty = bars + 2 * STAGES + 2;  // [2]      used in the even CTA
  uint64_t* shared_free = bars + 2 * STAGES + 4;  // shared accumulator columns drained (even CTA), one phase per tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int tm = (p.M + 2 * BM - 1) / (2 * BM), tn = (p.N + BN - 1) / BN;
  const int num_tiles = tm * tn;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    prefetch_tmap(&tmap_sa);
    prefetch_tmap(&tmap_sb);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 8);   // one arrival for each epilogue warp of both CTAs
    }
    mbar_init(shared_free, 8);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, 512);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the set-up above may run beside the kernel that writes the operands

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += npairs) {
        int mt, nt;
        mbg::tile_coords(t, tm, tn, GROUP_M, mt, nt);
        const int m0 = mt * 2 * BM + static_cast<int>(cta) * BM;
        const int n0 = nt * BN + static_cast<int>(cta) * BNH;
        for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1)) {
            atomicCAS(p.status, 0, ERR_WAIT_EMPTY);
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * STAGE_BYTES;
          const bool first = (kb & 3) == 0;
          mbar_expect_tx_leader(&full[s], STAGE_BYTES + (first ? SF_BYTES : 0));
          tma_load_2d_pair(sa, &tmap_a, &full[s], kb * BK, m0);
          tma_load_2d_pair(sa + A_BYTES, &tmap_b, &full[s], kb * BK, n0);
          if (first) {
            uint8_t* ss = sf + s * SF_STRIDE;
            tma_load_3d_pair(ss, &tmap_sa, &full[s], 0, kb >> 2, m0 / 128);
            tma_load_3d_pair(ss + SFA_BYTES, &tmap_sb, &full[s], 0, kb >> 2, nt * (BN / 128));
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && cta == 0) {
      constexpr uint32_t idesc = idesc_mxf8(2 * BM, BN);
      uint32_t it = 0, tcount = 0, group = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += npairs, ++tcount) {
        const uint32_t acc = tcount & 1;
        if (!mbar_wait(&acc_empty[acc], ((tcount >> 1) & 1) ^ 1) || (tcount && !mbar_wait(shared_free, (tcount - 1) & 1))) {
          atomicCAS(p.status, 0, ERR_WAIT_ACC_EMPTY);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (acc ? ACC1 : 0u);
        uint32_t sfc = 0;
        for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full[s], (it / STAGES) & 1)) {
            atomicCAS(p.status, 0, ERR_WAIT_FULL);
            ok = false;
            break;
          }
          tc_fence_after();
          if ((kb & 3) == 0) {
            sfc = tmem + SF_COL + (group & 1) * SF_SET;
            ++group;
            const uint32_t ss = smem_u32(sf + s * SF_STRIDE);
            sf_copy2(sfc, sf_desc(ss));
            sf_copy2(sfc + SFB_COL, sf_desc(ss + SFA_BYTES));
            sf_copy2(sfc + SFB_COL + 4, sf_desc(ss + SFA_BYTES + 512));
          }
          const uint32_t id = idesc | (static_cast<uint32_t>(kb & 3) << 29) | (static_cast<uint32_t>(kb & 3) << 4);
          const uint32_t sa = smem_u32(smem + s * STAGE_BYTES);
          const uint64_t da = make_smem_desc(sa, 16, 1024), db = make_smem_desc(sa + A_BYTES, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma2_mxf8(d, smem_desc_advance(da, k * 32), smem_desc_advance(db, k * 32), id, sfc, sfc + SFB_COL,
                       (kb | k) ? 1u : 0u);
          umma2_commit_both(&empty[s]);
        }
        if (ok) umma2_commit_both(&acc_full[acc]);
      }
    }
  } else {
    const int q = warp & 3;
    uint32_t tcount = 0;
    for (int t = pair; t < num_tiles; t += npairs, ++tcount) {
      int mt, nt;
      mbg::tile_coords(t, tm, tn, GROUP_M, mt, nt);
      const uint32_t acc = tcount & 1;
      if (!mbar_wait(&acc_full[acc], (tcount >> 1) & 1)) {
        atomicCAS(p.status, 0, ERR_WAIT_ACC_FULL);
        break;
      }
      tc_fence_after();
      const int row0 = mt * 2 * BM + static_cast<int>(cta) * BM + q * 32;
      const uint32_t taddr = tmem + (acc ? ACC1 : 0u) + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int i = 0; i < BN / 32; ++i) {
        const int c = acc ? i : (i + BN / 32 - 1) % (BN / 32);   // the shared columns first: 7 of the first, 0 of the second
        uint32_t r[32];
        tmem_ld_32x32(taddr + c * 32, r);
        tmem_ld_wait();
        if (i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(shared_free);
        }
        store_chunk(p, r, row0, nt * BN + c * 32, out_stage + q * OUT_STAGE, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(&acc_empty[acc]);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc2(tmem, 512);
  }
}

// ---- few rows of A (tokens of a decoding step): bound by reading B once
//
// The roles are swapped: 128 rows of B (output columns) are the M side of the instruction, the rows of A, rounded up to
// 16, 32 or 64, its N side, so nothing of the accumulator is wasted on rows that do not exist.  A cluster of `split` CTAs shares
// the contraction of a tile, in whole groups of four k-blocks; two CTAs an SM keep 160 KiB on the way.  The partial sums meet
// in shared memory over the cluster: CTA r receives the columns of its share of A's rows from all of them and adds them up in
// the order of the CTAs, so the bits do not depend on timing.
namespace few {

constexpr int ROWS = 128, MAX_N = 64, MAX_SPLIT = 8;
constexpr int W_BYTES = ROWS * BK, COLS = 128, SF_A = 64, SF_SETS = 16;   // columns: accumulator, then two sets of 4 + 4
constexpr int SF_STAGE = 1024;
constexpr int recv_rows(int n) { return n + MAX_SPLIT; }    // split * (n / split rounded up) is less
constexpr int stages_of(int n) { return n == 16 ? 5 : n == 32 ? 4 : 3; }   // two CTAs an SM
constexpr int smem_bytes(int n) { return stages_of(n) * (W_BYTES + n * BK + SF_STAGE) + recv_rows(n) * ROWS * 4 + 1024 + 128; }
static_assert(smem_bytes(16) <= 113 * 1024 && smem_bytes(32) <= 113 * 1024 && smem_bytes(64) <= 113 * 1024, "");

struct FewParams {
  Params p;
  int n;          // rows of A in the instruction: 16, 32 or 64
  int split;
};

__device__ __forceinline__ void umma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void sf_copy(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ uint32_t in_cta(const void* ptr, uint32_t cta) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(ptr)), "r"(cta));
  return a;
}

__device__ __forceinline__ void store_one(const Params& p, int row, int col, float v) {
  const long long at = static_cast<long long>(row) * p.ldc + col;
  if (p.out == OUT_BF16) static_cast<__nv_bfloat16*>(p.C)[at] = __float2bfloat16(v);
  else if (p.out == OUT_F32) static_cast<float*>(p.C)[at] = v;
  else static_cast<float*>(p.C)[at] += v;
}

__global__ void __launch_bounds__(THREADS, 2)
fp8_gemm_few_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb, const FewParams fp) {
  extern __shared__ uint8_t smem_raw[];
  const Params& p = fp.p;
  const int n = fp.n, split = fp.split, STAGES = stages_of(n);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = W_BYTES + n * BK;
  uint8_t* sf = smem + STAGES * stage_bytes;
  float* recv = reinterpret_cast<float*>(sf + STAGES * SF_STAGE);     // [split][n / split rounded up][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(recv + recv_rows(n) * ROWS);
  uint64_t *full = bars, *empty = bars + STAGES, *done = bars + 2 * STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = split > 1 ? cluster_ctarank() : 0u;
  const int tile = blockIdx.x / split, n0 = tile * ROWS, m0 = blockIdx.y * n;     // columns and rows of C
  const int groups = (p.kblocks + 3) / 4;
  const int kb0 = min(p.kblocks, static_cast<int>(static_cast<long long>(groups) * rank / split) * 4);
  const int kb1 = min(p.kblocks, static_cast<int>(static_cast<long long>(groups) * (rank + 1) / split) * 4);

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    prefetch_tmap(&tmap_sa);
    prefetch_tmap(&tmap_sb);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (split > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");   // waited for before the first store into another CTA
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const int it = kb - kb0, s = it % STAGES;
        if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1)) {
          atomicCAS(p.status, 0, ERR_WAIT_EMPTY);
          ok = false;
          break;
        }
        uint8_t* w = smem + s * stage_bytes;
        const bool first = (kb & 3) == 0;
        mbar_expect_tx(&full[s], stage_bytes + (first ? SF_STAGE : 0));
        tma_load_2d(w, &tmap_b, &full[s], kb * BK, n0);
        tma_load_2d(w + W_BYTES, &tmap_a, &full[s], kb * BK, m0);
        if (first) {
          tma_load_3d(sf + s * SF_STAGE, &tmap_sb, &full[s], 0, kb >> 2, tile);
          tma_load_3d(sf + s * SF_STAGE + 512, &tmap_sa, &full[s], 0, kb >> 2, m0 >> 7);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && kb0 < kb1) {
      const uint32_t idesc = idesc_mxf8(ROWS, 16) + (static_cast<uint32_t>(n - 16) >> 3 << 17);
      const uint32_t sfb = 4 + ((m0 & 127) >> 5);      // exponents of 32 rows a column
      bool ok = true;
      uint32_t set = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int it = kb - kb0, s = it % STAGES;
        if (!mbar_wait(&full[s], (it / STAGES) & 1)) {
          atomicCAS(p.status, 0, ERR_WAIT_FULL);
          ok = false;
          break;
        }
        tc_fence_after();
        if ((kb & 3) == 0) {
          ++set;
          const uint32_t ss = smem_u32(sf + s * SF_STAGE), col = tmem + SF_A + (set & 1) * SF_SETS;
          sf_copy(col, sf_desc(ss));
          sf_copy(col + 4, sf_desc(ss + 512));
        }
        const uint32_t sfc = tmem + SF_A + (set & 1) * SF_SETS;
        const uint32_t id = idesc | (static_cast<uint32_t>(kb & 3) << 29) | (static_cast<uint32_t>(kb & 3) << 4);
        const uint32_t w = smem_u32(smem + s * stage_bytes);
        const uint64_t da = make_smem_desc(w, 16, 1024), db = make_smem_desc(w + W_BYTES, 16, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mxf8(tmem, smem_desc_advance(da, k * 32), smem_desc_advance(db, k * 32), id, sfc, sfc + sfb, (it | k) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      if (ok) umma_commit(done);
    }
  } else {
    const int q = warp & 3, row = q * 32 + lane, col = n0 + row;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16);
    bool ok = kb0 < kb1;       // (a CTA without k-blocks contributes zeros)
    if (ok && !mbar_wait(done, 0)) {
      atomicCAS(p.status, 0, ERR_WAIT_ACC_FULL);
      ok = false;
    }
    tc_fence_after();
    const int share = (n + split - 1) / split, have = min(n, p.M - m0);      // rows of A that a CTA adds up, and that exist
    if (split > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    int to_cta = 0, to_row = 0;
    uint32_t to = split > 1 ? in_cta(recv + static_cast<int>(rank) * share * ROWS + row, 0) : 0u;
    for (int c0 = 0; c0 < have; c0 += 16) {
      uint32_t r[16];
      if (kb0 < kb1) {
        tmem_ld_32x16(taddr + c0, r);
        tmem_ld_wait();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = c0 + i;
        const float v = ok ? __uint_as_float(r[i]) : 0.f;
        if (split == 1) {
          if (t < have && col < p.N) store_one(p, m0 + t, col, v);
        } else if (t < have) {
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + to_row * ROWS * 4), "f"(v) : "memory");
          if (++to_row == share) {
            to_row = 0;
            to = in_cta(recv + static_cast<int>(rank) * share * ROWS + row, ++to_cta < split ? to_cta : 0);
          }
        }
      }
    }
  }
  if (split > 1) {
    if (warp < 2) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    const int share = (n + split - 1) / split, t0 = static_cast<int>(rank) * share;
    if (warp >= 2) {
      const int row = (warp & 3) * 32 + lane, col = n0 + row;
      const int t1 = min(min(n, p.M - m0), t0 + share);
      for (int t = t0; t < t1 && col < p.N; ++t) {
        float v = 0.f;
        for (int r = 0; r < split; ++r) v += recv[(r * share + t - t0) * ROWS + row];
        store_one(p, m0 + t, col, v);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, COLS);
  }
}

}  // namespace few

int make_codes_tmap(CUtensorMap* m, const void* base, uint64_t cols, uint64_t rows, uint64_t ld, uint32_t box_rows) {
  mbh::EncodeTiledFn fn = mbh::encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld};
  cuuint32_t box[2] = {128, box_rows}, es[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0 : -2;
}
// exponents: [row tiles][4-block groups][512 bytes]
int make_scales_tmap(CUtensorMap* m, const void* base, uint64_t row_tiles, uint64_t groups, uint32_t box_tiles) {
  mbh::EncodeTiledFn fn = mbh::encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[3] = {128, groups, row_tiles}, strides[2] = {512, groups * 512};
  cuuint32_t box[3] = {128, 1, box_tiles}, es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -2;
}

// Which kernel takes less time, in ns, as fitted to 336 problems of 12 to 777 rows, 256 to 20480 columns and 333 to 10240 deep
// (errors 7 and 10 %; the choice costs 0.2 % over the faster one on average).  A wave of 256 x 256 tiles costs its depth, and
// rows that are not on 16-byte boundaries their single stores; a wave of the small tiles its depth, its rows, and the meeting of
// its parts.  Examples (us, 256 x 256 tiles and small ones): 24 x 4096 x 4096 16.8 and 9.9, 64 x 20480 x 2560 21.3 and 16.9,
// 64 x 14336 x 4096 17.7 and 20.2, 256 x 4096 x 4096 17.6 and 20.2, 333 x 777 x 1100 14.5 and 11.4, 512 x 4608 x 512 7.9 and 10.7.
bool few_is_faster(long long tiles, long long units, int n, int split, int kblocks, int groups, bool vec) {
  const long long sms = mbh::sm_count(), big_waves = (tiles + sms / 2 - 1) / (sms / 2);
  const long long big = 4800 + big_waves * (1600 + 350ll * kblocks + (vec ? 0 : 4200));
  const long long ctas = units * split, waves = (ctas + 2 * sms - 1) / (2 * sms), depth = min(kblocks, (groups + split - 1) / split * 4);
  const long long of_few = 3200 + waves * (77 * n + 400 * depth + depth * n * (ctas > sms ? 2 : 1) * 57 / 100 + (split > 1 ? 138 * n / split : 0));
  return of_few < big;
}

}  // namespace

// a: [M, 128 kblocks] codes with row pitch lda and exponents sa, b: [N, 128 kblocks] likewise; out: 0 bf16, 1 fp32, 2 fp32 +=
extern "C" int mb_fp8_gemm(const void* a, const void* sa, const void* b, const void* sb, void* c, int M, int N, int kblocks,
                           long long lda, long long ldb, long long ldc, int out, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (kblocks <= 0 || kblocks > (1 << 23) || out < 0 || out > 2) return -3;
  if ((lda & 15) || (ldb & 15) || (reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(b) & 15) ||
      (reinterpret_cast<uintptr_t>(sa) & 15) || (reinterpret_cast<uintptr_t>(sb) & 15))
    return -3;
  Params p;
  p.C = c;
  p.M = M;
  p.N = N;
  p.kblocks = kblocks;
  p.ldc = ldc;
  p.out = out;
  p.vec = !(reinterpret_cast<uintptr_t>(c) & 15) && !((ldc * (out == OUT_BF16 ? 2 : 4)) & 15);
  p.status = mbh::status().dev;
  if (!p.status) return -4;
  const long long tiles = static_cast<long long>((M + 255) / 256) * ((N + BN - 1) / BN);
  if (tiles > 0x7fffffffll / 2) return -3;
  CUtensorMap ta, tb, tsa, tsb;
  const uint64_t cols = static_cast<uint64_t>(kblocks) * 128, groups = (kblocks + 3) / 4;
  const int row_tiles = (N + few::ROWS - 1) / few::ROWS;
  const int n = M <= 16 ? 16 : M <= 32 ? 32 : 64, m_tiles = (M + n - 1) / n;
  // CTAs of a tile: two an SM altogether at the most, whole groups of four k-blocks each
  const long long units = static_cast<long long>(row_tiles) * m_tiles;
  int split = static_cast<int>(min(2 * mbh::sm_count() / units, static_cast<long long>(few::MAX_SPLIT)));
  split = static_cast<int>(min(static_cast<uint64_t>(max(split, 1)), groups));
  const bool few_rows = m_tiles <= 65535 && few_is_faster(tiles, units, n, split, kblocks, static_cast<int>(groups), p.vec);
  int e = make_codes_tmap(&ta, a, cols, M, lda, few_rows ? n : BM);
  if (!e) e = make_codes_tmap(&tb, b, cols, N, ldb, BNH);
  if (!e) e = make_scales_tmap(&tsa, sa, (M + 127) / 128, groups, 1);
  if (!e) e = make_scales_tmap(&tsb, sb, (N + 127) / 128, groups, few_rows ? 1 : 2);
  if (e) return e;
  if (few_rows) {
    few::FewParams fp;
    fp.p = p;
    fp.n = n;
    fp.split = split;
    const int smem = few::smem_bytes(n);
    MB_SET_MAX_SMEM_ONCE(few::fp8_gemm_few_kernel, 113 * 1024);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(row_tiles * split, m_tiles, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, few::fp8_gemm_few_kernel, ta, tb, tsa, tsb, fp) != cudaSuccess) {
      const int e2 = mbh::check_launch("fp8_gemm_few");
      return e2 ? e2 : -100;
    }
    return mbh::check_launch("fp8_gemm_few");
  }
  MB_SET_MAX_SMEM_ONCE(fp8_gemm_kernel, SMEM_BYTES);
  const int max_pairs = mbh::sm_count() / 2;
  const int pairs = static_cast<int>(tiles < max_pairs ? tiles : max_pairs);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, fp8_gemm_kernel, ta, tb, tsa, tsb, p) != cudaSuccess) {
    const int e2 = mbh::check_launch("fp8_gemm");
    return e2 ? e2 : -100;
  }
  return mbh::check_launch("fp8_gemm");
}
