// y[t, n] = sum over blocks b of 2^(ex[t,b] + ew[n,b]) * sum over the 128 values of block b of xq[t,:] wq[n,:] for up to eight
// tokens: a decoding step, bound by reading the weight's codes once (14336 x 4096: 9 us at the copy rate).
//
// Everything else is kept off their way: no staging, no tensor memory, no barrier but one at the end.  A warp takes 32 rows of w
// and every 4th, 8th or 16th block of the contraction (as many warps share them), with the next block on its way.  The matrix
// instruction (16 x 8 x 32) does not care in which order the contraction comes, as long as both operands agree: the 16
// neighbouring bytes that a lane reads are its values of two instructions, of w and of x alike, so neither operand is ever
// rearranged.  The warps' sums meet in shared memory and are added in order.  The instruction cuts its sums off some 27 bits below
// the largest term; a block's sum of 128 products is then added in rounded fp32 (8192 products of one sign: at most 4 units of
// 2^-24 off, 0.01 on average).
//
// Measured with the quantiser, launches from a graph over 400 MB of weights: 4 tokens x 14336 x 4096 15.5 us (a kernel that only
// reads the codes: 10.7), 1 x 4096 x 4096 7.3 us, 1 x 2560 x 10240 10.5 us; the tcgen05 kernel for few rows of fp8_gemm.cu took
// 19.5, 11.1 and 22.6: at this size a contraction's depth is too short for its pipeline to fill.  Above eight tokens a second
// set of columns would double the instructions, and that kernel takes over (16 tokens: 23 us).  Called from the host one after
// the other a call takes 19 us, which is the host's.
//
// The tokens are quantised by the kernel of fp8_blocks.cu (doing it here instead, once for every 32 rows of w, took longer than
// the weight: 18.6 us).  This kernel starts while that one runs (programmatic launch): what it reads of w was there before
// either, and only x has to be waited for.
#include "fp8_common.cuh"
#include "host_common.cuh"

extern "C" int mb_fp8_quantize(const void* x, int type, int rows, int cols, long long ld, int mode, void* q, void* sq, void* qt,
                               void* sqt, cudaStream_t stream);
extern "C" int mb_fp8_gemm(const void* a, const void* sa, const void* b, const void* sb, void* c, int M, int N, int kblocks,
                           long long lda, long long ldb, long long ldc, int out, cudaStream_t stream);

namespace {

using namespace mbf8;

constexpr int TOKENS = 8, ROWS = 32, BLOCK = 128;

__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the codes of 32 rows and a block of the contraction, as a lane holds them, and the rows' exponents
struct Weights {
  uint4 v[2][2][2];     // rows 16 m + 8 h + g, half c of the block
  uint32_t e[2][2];
  __device__ __forceinline__ void load(const uint8_t* const (&row)[2][2], const uint8_t* const (&exps)[2][2], int kb) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 2; ++c) v[m][h][c] = load_codes(row[m][h] + kb * BLOCK + c * 64);
        e[m][h] = exps[m][h][(kb >> 2) * 512 + (kb & 3)];
      }
  }
};
struct Tokens {
  uint4 v[2];
  uint32_t e;
  __device__ __forceinline__ void load(const uint8_t* row, const uint8_t* exps, int kb) {   // (plain loads: another kernel has just written them)
    v[0] = *reinterpret_cast<const uint4*>(row + kb * BLOCK);
    v[1] = *reinterpret_cast<const uint4*>(row + kb * BLOCK + 64);
    e = exps[(kb >> 2) * 512 + (kb & 3)];
  }
};

template <typename O, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS)
fp8_few_kernel(const uint8_t* x, const uint8_t* sx, int M, int blocks, const uint8_t* __restrict__ w, const uint8_t* __restrict__ sw,
               int N, long long ldw, O* __restrict__ y, long long ldy) {
  __shared__ float sums[WARPS][TOKENS][ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, n0 = blockIdx.x * ROWS;
  const int groups = (blocks + 3) / 4;
  const uint8_t *row[2][2], *exps[2][2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = min(N - 1, n0 + m * 16 + h * 8 + g);     // (rows that do not exist: the last one, not stored)
      row[m][h] = w + r * ldw + t * 16;
      exps[m][h] = sw + static_cast<long long>(r >> 7) * groups * 512 + scale_at(r & 127, 0);
    }
  float acc[2][4] = {};
  Weights next;
  if (warp < blocks) next.load(row, exps, warp);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int token = min(g, M - 1);                            // (tokens that do not exist: the last one, not stored)
  const uint8_t *xt = x + static_cast<long long>(token) * blocks * BLOCK + t * 16, *et = sx + scale_at(token, 0);
  Tokens next_x;
  if (warp < blocks) next_x.load(xt, et, warp);
  for (int kb = warp; kb < blocks; kb += WARPS) {
    const Weights now = next;
    const Tokens b = next_x;
    if (kb + WARPS < blocks) {
      next.load(row, exps, kb + WARPS);
      next_x.load(xt, et, kb + WARPS);
    }
    const int k0 = static_cast<int>(__shfl_sync(~0u, b.e, 8 * t)) - 127, k1 = static_cast<int>(__shfl_sync(~0u, b.e, 8 * t + 4)) - 127;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float c[4] = {};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 lo = now.v[m][0][j], hi = now.v[m][1][j];
        mma(c, lo.x, hi.x, lo.y, hi.y, b.v[j].x, b.v[j].y);
        mma(c, lo.z, hi.z, lo.w, hi.w, b.v[j].z, b.v[j].w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // 2^(both exponents) in two factors: neither overflows
        const int e = static_cast<int>(now.e[m][i >> 1]) - 127 + ((i & 1) ? k1 : k0), h = e >> 1;
        acc[m][i] = fmaf(c[i] * pow2(h), pow2(e - h), acc[m][i]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[warp][2 * t + (i & 1)][m * 16 + (i >> 1) * 8 + g] = acc[m][i];
  __syncthreads();
  for (int at = threadIdx.x; at < TOKENS * ROWS; at += WARPS * 32) {
    const int to = at / ROWS, r = at % ROWS;
    if (to < M && n0 + r < N) {
      float v = sums[0][to][r];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) v += sums[k][to][r];
      if constexpr (sizeof(O) == 2) y[to * ldy + n0 + r] = __float2bfloat16(v);
      else y[to * ldy + n0 + r] = v;
    }
  }
}

template <typename O, int WARPS>
int launch(const uint8_t* x, const uint8_t* ex, int M, int blocks, const uint8_t* w, const uint8_t* ew, int N, long long ldw, void* y,
           long long ldy, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((N + ROWS - 1) / ROWS, 1, 1);
  cfg.blockDim = dim3(WARPS * 32, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, fp8_few_kernel<O, WARPS>, x, ex, M, blocks, w, ew, N, ldw, static_cast<O*>(y), ldy);
  return mbh::check_launch("fp8_few");
}
template <typename O>
int few(const uint8_t* x, const uint8_t* ex, int M, int blocks, const uint8_t* w, const uint8_t* ew, int N, long long ldw, void* y,
        long long ldy, cudaStream_t stream) {
  // twelve warps an SM hide the reads (1 x 4096 x 4096: 11.1 us with 4 warps a tile, 8.5 with 8; 4 x 14336 x 4096: 15.0 and 16.5)
  const long long tiles = (N + ROWS - 1) / ROWS, want = 12ll * mbh::sm_count();
  if (tiles * 4 >= want || blocks <= 4) return launch<O, 4>(x, ex, M, blocks, w, ew, N, ldw, y, ldy, stream);
  if (tiles * 8 >= want || blocks <= 8) return launch<O, 8>(x, ex, M, blocks, w, ew, N, ldw, y, ldy, stream);
  return launch<O, 16>(x, ex, M, blocks, w, ew, N, ldw, y, ldy, stream);
}

}  // namespace

// y = Q(x) W^T for a weight that was laid out once.  x: [M, K], row pitch ldx, bf16 (type 0) or fp32 (type 2); work (16-byte
// boundary): M x (K rounded up to 128) bytes and the exponents of as many blocks as mb_fp8_quantize writes them; w: [N, K rounded
// up to 128] codes with row pitch ldw and exponents sw; y: [M, N] of x's type, row pitch ldy
extern "C" int mb_fp8_linear(const void* x, int type, long long ldx, int M, int K, void* work, const void* w, const void* sw, int N,
                             long long ldw, void* y, long long ldy, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > (1 << 30) || (type != 0 && type != 2) || (ldw & 15) || (reinterpret_cast<uintptr_t>(w) & 15) ||
      (reinterpret_cast<uintptr_t>(work) & 15))
    return -3;
  const int blocks = (K + BLOCK - 1) / BLOCK;
  uint8_t* xc = static_cast<uint8_t*>(work);
  uint8_t* ec = xc + static_cast<long long>(M) * blocks * BLOCK;
  const int e = mb_fp8_quantize(x, type, M, K, ldx, 1, xc, ec, nullptr, nullptr, stream);
  if (e) return e;
  if (M > TOKENS)
    return mb_fp8_gemm(xc, ec, w, sw, y, M, N, blocks, static_cast<long long>(blocks) * BLOCK, ldw, ldy, type == 0 ? 0 : 1, stream);
  const uint8_t* wc = static_cast<const uint8_t*>(w);
  const uint8_t* sc = static_cast<const uint8_t*>(sw);
  return type == 0 ? few<__nv_bfloat16>(xc, ec, M, blocks, wc, sc, N, ldw, y, ldy, stream)
                   : few<float>(xc, ec, M, blocks, wc, sc, N, ldw, y, ldy, stream);
}
