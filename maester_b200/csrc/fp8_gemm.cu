// C[M,N] = sum over blocks b of 2^(ea[m,b] + eb[n,b]) * sum over the 128 values of block b of A[m,:] B[n,:]
// for e4m3 codes with block exponents as fp8_blocks.cu writes them.
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp8.h>

namespace {

enum { OUT_BF16 = 0, OUT_F32 = 1, OUT_F32_ACC = 2 };

__device__ __forceinline__ float decode(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
__device__ __forceinline__ float scale_of(const uint8_t* s, int kt, int row, int blk) {
  const int byte = s[(static_cast<long long>(row >> 7) * kt + (blk >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (blk & 3)];
  return byte ? __uint_as_float(static_cast<uint32_t>(byte) << 23) : 0.f;
}

__global__ void __launch_bounds__(256) fp8_gemm_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ sa,
                                                       const uint8_t* __restrict__ b, const uint8_t* __restrict__ sb, void* c,
                                                       int M, int N, int kblocks, long long lda, long long ldb, long long ldc,
                                                       int out) {
  __shared__ float ta[64][33], tb[64][33];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, kt = (kblocks + 3) / 4;
  float acc[4][4] = {};
  for (int kb = 0; kb < kblocks; ++kb)
    for (int k0 = kb * 128; k0 < kb * 128 + 128; k0 += 32) {
      for (int i = tid; i < 64 * 32; i += 256) {
        const int r = i >> 5, k = i & 31;
        ta[r][k] = m0 + r < M ? decode(a[(m0 + r) * lda + k0 + k]) * scale_of(sa, kt, m0 + r, kb) : 0.f;
        tb[r][k] = n0 + r < N ? decode(b[(n0 + r) * ldb + k0 + k]) * scale_of(sb, kt, n0 + r, kb) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += ta[ty * 4 + i][k] * tb[tx * 4 + j][k];
      __syncthreads();
    }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= M || n >= N) continue;
      if (out == OUT_BF16) static_cast<__nv_bfloat16*>(c)[m * ldc + n] = __float2bfloat16(acc[i][j]);
      else if (out == OUT_F32) static_cast<float*>(c)[m * ldc + n] = acc[i][j];
      else static_cast<float*>(c)[m * ldc + n] += acc[i][j];
    }
}

}  // namespace

// a: [M, 128 kblocks] codes with row pitch lda and exponents sa, b: [N, 128 kblocks] likewise; out: 0 bf16, 1 fp32, 2 fp32 +=
extern "C" int mb_fp8_gemm(const void* a, const void* sa, const void* b, const void* sb, void* c, int M, int N, int kblocks,
                           long long lda, long long ldb, long long ldc, int out, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (kblocks <= 0 || out < 0 || out > 2) return -3;
  if ((lda & 15) || (ldb & 15) || (reinterpret_cast<uintptr_t>(a) & 15) || (reinterpret_cast<uintptr_t>(b) & 15)) return -3;
  const dim3 grid((N + 63) / 64, (M + 63) / 64);
  if (grid.y > 65535) return -3;
  fp8_gemm_kernel<<<grid, 256, 0, stream>>>(static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(sa),
                                            static_cast<const uint8_t*>(b), static_cast<const uint8_t*>(sb), c, M, N, kblocks,
                                            lda, ldb, ldc, out);
  return mbh::check_launch("fp8_gemm");
}
