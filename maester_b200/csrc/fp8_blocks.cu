// e4m3 with a power-of-two scale for every block of 128 values: quantisation.
//
// Block b of a row stands for code * 2^(byte - 127) with the smallest power that keeps |x| <= 448 * 2^k.  The division by
// a power of two is exact, so every value is rounded once.  Codes: [rows, columns rounded up to 128], the columns past the
// end are zero.  Exponent bytes come in the order in which the block-scaled tensor-core product takes them: for 128 rows and
// 4 blocks of the contraction 512 consecutive bytes, row r and block b at 16 (r mod 32) + 4 (r div 32) + b.
// A thread block owns a 128 x 128 tile of x: it reads it once and writes the codes of x (blocks along a row, or the whole
// tile as one block), of its transpose (blocks along a column), or of both.
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp8.h>

namespace {

constexpr int B = 128;
enum { ROWS = 1, COLS = 2, SQUARE = 4 };

__device__ __forceinline__ float ld_f(const float* p) { return *p; }
__device__ __forceinline__ float ld_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float pow2(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }
__device__ __forceinline__ int block_exponent(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - 127;
  const int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  return min(max(k, -117), 120);
}
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint8_t encode(float y) {
  if (!(fabsf(y) <= 3.4028234e38f)) return 0x7f;
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3));
}

template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const T* __restrict__ x, int rows, int cols, long long ld, int mode,
                                                           uint8_t* q, uint8_t* sq, uint8_t* qt, uint8_t* sqt) {
  extern __shared__ float tile[];   // [128][129]
  __shared__ uint32_t am_row[B], am_col[B];
  const int rt = blockIdx.y, ct = blockIdx.x, tid = threadIdx.x;
  const int r0 = rt * B, c0 = ct * B;
  const int ctiles = (cols + B - 1) / B, rtiles = (rows + B - 1) / B;
  if (tid < B) am_row[tid] = am_col[tid] = 0;
  __syncthreads();
  for (int i = tid; i < B * B; i += 256) {
    const int r = i >> 7, c = i & 127;
    float v = 0.f;
    if (r0 + r < rows && c0 + c < cols) v = ld_f(x + static_cast<long long>(r0 + r) * ld + c0 + c);
    tile[r * 129 + c] = v;
    const uint32_t b = finite_bits(v);
    atomicMax(&am_row[r], b);
    atomicMax(&am_col[c], b);
  }
  __syncthreads();
  if (mode & SQUARE) {
    if (tid == 0) {
      uint32_t a = 0;
      for (int i = 0; i < B; ++i) a = max(a, am_row[i]);
      am_row[0] = a;
    }
    __syncthreads();
    const uint32_t a = am_row[0];
    __syncthreads();
    if (tid < B) am_row[tid] = am_col[tid] = a;
    __syncthreads();
  }
  const bool in = rt < rtiles && ct < ctiles;
  if (mode & ROWS) {
    const long long pitch = static_cast<long long>(ctiles) * B;
    const int kt = (ctiles + 3) / 4;
    if (rt < rtiles && tid < B)
      sq[(static_cast<long long>(rt) * kt + (ct >> 2)) * 512 + (tid & 31) * 16 + (tid >> 5) * 4 + (ct & 3)] =
          (in && r0 + tid < rows) ? static_cast<uint8_t>(block_exponent(am_row[tid]) + 127) : 0;
    if (in)
      for (int i = tid; i < B * B; i += 256) {
        const int r = i >> 7, c = i & 127;
        if (r0 + r < rows) q[(r0 + r) * pitch + c0 + c] = encode(__fmul_rn(tile[r * 129 + c], pow2(-block_exponent(am_row[r]))));
      }
  }
  if (mode & COLS) {
    const long long pitch = static_cast<long long>(rtiles) * B;
    const int kt = (rtiles + 3) / 4;
    if (ct < ctiles && tid < B)
      sqt[(static_cast<long long>(ct) * kt + (rt >> 2)) * 512 + (tid & 31) * 16 + (tid >> 5) * 4 + (rt & 3)] =
          (in && c0 + tid < cols) ? static_cast<uint8_t>(block_exponent(am_col[tid]) + 127) : 0;
    if (in)
      for (int i = tid; i < B * B; i += 256) {
        const int c = i >> 7, r = i & 127;
        if (c0 + c < cols) qt[(c0 + c) * pitch + r0 + r] = encode(__fmul_rn(tile[r * 129 + c], pow2(-block_exponent(am_col[c]))));
      }
  }
}

}  // namespace

// x: [rows, cols], row pitch ld, bf16 (type 0) or fp32 (type 2).  mode: 1 codes of x into q / sq, 2 codes of x^T into
// qt / sqt, +4 one scale for each 128 x 128 tile.  sq: ceil(rows/128) x ceil(ceil(cols/128)/4) x 512 bytes, sqt likewise
// for x^T; every byte is written.
extern "C" int mb_fp8_quantize(const void* x, int type, int rows, int cols, long long ld, int mode, void* q, void* sq, void* qt,
                               void* sqt, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if ((type != 0 && type != 2) || !(mode & 3) || mode > 7) return -3;
  const int rt = (rows + B - 1) / B, ct = (cols + B - 1) / B;
  // the tiles past the end only write the padding of the exponent bytes
  const int gx = (mode & ROWS) ? (ct + 3) / 4 * 4 : ct, gy = (mode & COLS) ? (rt + 3) / 4 * 4 : rt;
  if (gy > 65535) return -3;
  const int smem = B * 129 * 4;
  uint8_t* o[4] = {static_cast<uint8_t*>(q), static_cast<uint8_t*>(sq), static_cast<uint8_t*>(qt), static_cast<uint8_t*>(sqt)};
  if (type == 0) {
    MB_SET_MAX_SMEM_ONCE(fp8_quantize_kernel<__nv_bfloat16>, smem);
    fp8_quantize_kernel<<<dim3(gx, gy), 256, smem, stream>>>(static_cast<const __nv_bfloat16*>(x), rows, cols, ld, mode, o[0],
                                                             o[1], o[2], o[3]);
  } else {
    MB_SET_MAX_SMEM_ONCE(fp8_quantize_kernel<float>, smem);
    fp8_quantize_kernel<<<dim3(gx, gy), 256, smem, stream>>>(static_cast<const float*>(x), rows, cols, ld, mode, o[0], o[1],
                                                             o[2], o[3]);
  }
  return mbh::check_launch("fp8_quantize");
}
