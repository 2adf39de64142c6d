// e4m3 with a power-of-two scale for every block of 128 values: quantisation.
//
// Block b of a row stands for code * 2^(byte - 127) with the smallest power that keeps |x| <= 448 * 2^k.  The division by
// a power of two is exact, so every value is rounded once.  Codes: [rows, columns rounded up to 128], the columns past the
// end are zero.  Exponent bytes come in the order in which the block-scaled tensor-core product takes them: for 128 rows and
// 4 blocks of the contraction 512 consecutive bytes, row r and block b at 16 (r mod 32) + 4 (r div 32) + b.
//
// A thread block owns a 128 x 128 tile of x: it reads it once and writes the codes of x (blocks along a row, or the whole
// tile as one block), of its transpose (blocks along a column), or of both.  A thread holds 8 x 8 values: maxima along rows
// meet within 16 lanes, maxima along columns through shared memory, and the transposed codes go through a swizzled 16 KiB
// tile so that both outputs leave as whole 128-byte lines.
//
// Measured (16384 x 4096 bf16): codes of x 38 us (5290 GB/s of 6540), of x and its transpose 56 us (4760), with one scale a tile
// 49 us (5450).  The integer pipe is busy 65 to 75 % of the time (packed maxima, shifts of 16-bit values into fp32, packing of
// codes), and only 4 blocks an SM fit its registers, so neither it nor memory is full; at 6 MB (5003 x 2560, 800 blocks on 592
// places) the second wave costs as much as the first: 15 us.
#include "fp8_common.cuh"
#include "host_common.cuh"

namespace {

using namespace mbf8;

constexpr int B = 128;
enum { ROWS = 1, COLS = 2, SQUARE = 4 };

constexpr int THREADS = 256;

// 8 x 8 values of one thread.  Maxima are the ordered bits of |x| (16 bits for bf16), over what is finite: a thread that
// holds an infinity or NaN (seen from its maxima) turns infinities into NaN and takes its maxima again without them.
template <typename T>
struct Patch;

template <>
struct Patch<__nv_bfloat16> {
  uint32_t v[8][4];
  __device__ __forceinline__ void load_row(int i, const __nv_bfloat16* p, int n, bool vec) {
    if (vec && n >= 8) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) v[i][w] = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) v[i][j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[j]) << (16 * (j & 1));
    }
  }
  __device__ __forceinline__ void zero_row(int i) {
#pragma unroll
    for (int w = 0; w < 4; ++w) v[i][w] = 0u;
  }
  static __device__ __forceinline__ uint32_t mag(uint32_t w) { return w & 0x7fff7fffu; }
  static __device__ __forceinline__ bool bad(uint32_t m) { return (m & 0xffffu) >= INF16 || (m >> 16) >= INF16; }
  static __device__ __forceinline__ uint32_t finite(uint32_t m) {
    if ((m & 0xffffu) >= INF16) m &= 0xffff0000u;
    if ((m >> 16) >= INF16) m &= 0x0000ffffu;
    return m;
  }
  template <bool FILTER>
  __device__ __forceinline__ void thread_rows(uint32_t (&p)[4]) const {   // row i low, row i + 4 high
    auto f = [](uint32_t w) { return FILTER ? finite(mag(w)) : mag(w); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = __vmaxu2(__vmaxu2(f(v[i][0]), f(v[i][1])), __vmaxu2(f(v[i][2]), f(v[i][3])));
      const uint32_t b = __vmaxu2(__vmaxu2(f(v[i + 4][0]), f(v[i + 4][1])), __vmaxu2(f(v[i + 4][2]), f(v[i + 4][3])));
      p[i] = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    }
  }
  template <bool FILTER>
  __device__ __forceinline__ void thread_cols(uint32_t (&p)[4]) const {   // columns 2 w (low) and 2 w + 1 (high)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      p[w] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) p[w] = __vmaxu2(p[w], FILTER ? finite(mag(v[i][w])) : mag(v[i][w]));
    }
  }
  __device__ __forceinline__ void no_infinities() {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if ((v[i][w] & 0x7fffu) == INF16) v[i][w] |= 0x1u;
        if ((v[i][w] & 0x7fff0000u) == (INF16 << 16)) v[i][w] |= 0x10000u;
      }
  }
  // maxima of the rows over this half-warp's 128 columns: fp32 bits
  __device__ __forceinline__ void row_max(uint32_t (&am)[8]) {
    uint32_t p[4];
    thread_rows<false>(p);
    if (bad(__vmaxu2(__vmaxu2(p[0], p[1]), __vmaxu2(p[2], p[3])))) {
      no_infinities();
      thread_rows<true>(p);
    }
#pragma unroll
    for (int o = 8; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __vmaxu2(p[i], __shfl_xor_sync(~0u, p[i], o));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      am[i] = p[i] << 16;
      am[i + 4] = p[i] & 0xffff0000u;
    }
  }
  // maxima of the 8 columns over the whole tile: fp32 bits.  s: 8 warps x 128 x 16 bits
  __device__ __forceinline__ void col_max(uint32_t (&am)[8], uint32_t* s, int warp, int lane) {
    uint32_t p[4];
    thread_cols<false>(p);
    if (bad(__vmaxu2(__vmaxu2(p[0], p[1]), __vmaxu2(p[2], p[3])))) {
      no_infinities();
      thread_cols<true>(p);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) p[w] = __vmaxu2(p[w], __shfl_xor_sync(~0u, p[w], 16));
    uint4* s4 = reinterpret_cast<uint4*>(s);
    if (lane < 16) s4[warp * 16 + lane] = make_uint4(p[0], p[1], p[2], p[3]);
    __syncthreads();
    uint4 m = s4[lane & 15];
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      const uint4 o = s4[k * 16 + (lane & 15)];
      m.x = __vmaxu2(m.x, o.x); m.y = __vmaxu2(m.y, o.y); m.z = __vmaxu2(m.z, o.z); m.w = __vmaxu2(m.w, o.w);
    }
    am[0] = m.x << 16; am[1] = m.x & 0xffff0000u; am[2] = m.y << 16; am[3] = m.y & 0xffff0000u;
    am[4] = m.z << 16; am[5] = m.z & 0xffff0000u; am[6] = m.w << 16; am[7] = m.w & 0xffff0000u;
  }
  // word w of row i times the powers of two s (two bf16; exact down to 2^-126, far below the smallest code): two values
  __device__ __forceinline__ float2 scaled(int i, int w, uint32_t s) const {
    const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v[i][w]), *reinterpret_cast<__nv_bfloat162*>(&s));
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&y);
    return make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
  }
  // codes of row i, all with the scale 2^-k
  __device__ __forceinline__ uint2 row_codes(int i, int k) const {
    const uint32_t h = static_cast<uint32_t>(127 - k) << 7, s = h | (h << 16);
    uint32_t c[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) c[w] = encode2(scaled(i, w, s));
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
  // codes of columns 2 w and 2 w + 1 down the 8 rows, with the scales 2^-k0 and 2^-k1
  __device__ __forceinline__ void col_codes(int w, int k0, int k1, uint2& c0, uint2& c1) const {
    const uint32_t s = (static_cast<uint32_t>(127 - k0) << 7) | (static_cast<uint32_t>(127 - k1) << 23);
    uint32_t a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = scaled(2 * i, w, s), y = scaled(2 * i + 1, w, s);
      a[i] = encode2(make_float2(x.x, y.x));
      b[i] = encode2(make_float2(x.y, y.y));
    }
    c0 = make_uint2(a[0] | (a[1] << 16), a[2] | (a[3] << 16));
    c1 = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
  }
};

template <>
struct Patch<float> {
  float v[8][8];
  __device__ __forceinline__ void load_row(int i, const float* p, int n, bool vec) {
    if (vec && n >= 8) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
      v[i][4] = b.x; v[i][5] = b.y; v[i][6] = b.z; v[i][7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = j < n ? p[j] : 0.f;
    }
  }
  __device__ __forceinline__ void zero_row(int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
  }
  __device__ __forceinline__ uint32_t mag(int i, int j) const {   // (NaN may stand for an infinity here: neither counts)
    const uint32_t a = __float_as_uint(v[i][j]) & 0x7fffffffu;
    return a < INF32 ? a : 0u;
  }
  __device__ __forceinline__ void row_max(uint32_t (&am)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      am[i] = mag(i, 0);
#pragma unroll
      for (int j = 1; j < 8; ++j) am[i] = max(am[i], mag(i, j));
#pragma unroll
      for (int o = 8; o; o >>= 1) am[i] = max(am[i], __shfl_xor_sync(~0u, am[i], o));
    }
  }
  // s: 8 warps x 128 x 32 bits
  __device__ __forceinline__ void col_max(uint32_t (&am)[8], uint32_t* s, int warp, int lane) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      am[j] = mag(0, j);
#pragma unroll
      for (int i = 1; i < 8; ++i) am[j] = max(am[j], mag(i, j));
      am[j] = max(am[j], __shfl_xor_sync(~0u, am[j], 16));
      if (lane < 16) s[warp * 128 + lane * 8 + j] = am[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      for (int k = 0; k < 8; ++k) am[j] = max(am[j], s[k * 128 + (lane & 15) * 8 + j]);
  }
  // (the conversion would saturate an infinity; the NaN code stands for it)
  static __device__ __forceinline__ float scaled(float x, float s) {
    return fabsf(x) <= 3.4028234e38f ? __fmul_rn(x, s) : __uint_as_float(0x7fffffffu);
  }
  __device__ __forceinline__ uint2 row_codes(int i, int k) const {
    const float s = pow2(-k);
    uint32_t c[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) c[w] = encode2(make_float2(scaled(v[i][2 * w], s), scaled(v[i][2 * w + 1], s)));
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
  __device__ __forceinline__ uint2 col(int j, int k) const {
    const float s = pow2(-k);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = encode2(make_float2(scaled(v[2 * i][j], s), scaled(v[2 * i + 1][j], s)));
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
  __device__ __forceinline__ void col_codes(int w, int k0, int k1, uint2& c0, uint2& c1) const {
    c0 = col(2 * w, k0);
    c1 = col(2 * w + 1, k1);
  }
};

template <typename T, int MODE>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 4 : MODE == (ROWS | COLS) ? 1 : 2)
fp8_quantize_kernel(const T* __restrict__ src, int rows, int cols, long long ld, int vec, uint32_t across, uint8_t* q, uint8_t* sq,
                    uint8_t* qt, uint8_t* sqt) {
  __shared__ __align__(16) uint8_t tile[(MODE & COLS) ? B * B : 16];
  __shared__ __align__(16) uint32_t maxima[(MODE & COLS) ? 8 * 128 : 8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (a kernel that was launched to start beside this one may)
  const int rt = blockIdx.x / across, ct = blockIdx.x % across, tid = threadIdx.x;   // (tiles in one dimension: a second one
  // ends at 65535 of them, 8.4 million rows)
  const int ctiles = (cols + B - 1) / B, rtiles = (rows + B - 1) / B;
  if (rt >= rtiles || ct >= ctiles) {  // past the matrix: only the padding of the exponent bytes
    if (tid < B) {
      if ((MODE & ROWS) && rt < rtiles)
        sq[(static_cast<long long>(rt) * ((ctiles + 3) / 4) + (ct >> 2)) * 512 + scale_at(tid, ct & 3)] = 0;
      if ((MODE & COLS) && ct < ctiles)
        sqt[(static_cast<long long>(ct) * ((rtiles + 3) / 4) + (rt >> 2)) * 512 + scale_at(tid, rt & 3)] = 0;
    }
    return;
  }
  const int lane = tid & 31, warp = tid >> 5, c8 = tid & 15, r8 = tid >> 4;
  const int r0 = rt * B + r8 * 8, c0 = ct * B + c8 * 8;
  Patch<T> x;
  {
    const T* at = src + r0 * ld + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i, at += ld) {
      if (r0 + i < rows && c0 < cols) x.load_row(i, at, cols - c0, vec);
      else x.zero_row(i);
    }
  }
  uint32_t am[8];
  if (MODE & (ROWS | SQUARE)) x.row_max(am);
  if (MODE & SQUARE) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, am[i]);
    a = max(a, __shfl_xor_sync(~0u, a, 16));
    if (lane == 0) maxima[warp] = a;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) a = max(a, maxima[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) am[i] = a;
  }
  if (MODE & ROWS) {
    const long long pitch = static_cast<long long>(ctiles) * B;
    uint8_t* to = q + r0 * pitch + c0;
    uint8_t* st = sq + (static_cast<long long>(rt) * ((ctiles + 3) / 4) + (ct >> 2)) * 512;
#pragma unroll
    for (int i = 0; i < 8; ++i, to += pitch) {
      const int k = block_exponent(am[i]);
      if (c8 == i) st[scale_at(r8 * 8 + i, ct & 3)] = r0 + i < rows ? static_cast<uint8_t>(k + 127) : 0;
      const uint2 c = x.row_codes(i, k);
      if (r0 + i < rows) *reinterpret_cast<uint2*>(to) = c;
    }
  }
  if (MODE & COLS) {
    if (!(MODE & SQUARE)) x.col_max(am, maxima, warp, lane);
    const long long pitch = static_cast<long long>(rtiles) * B;
    uint8_t* st = sqt + (static_cast<long long>(ct) * ((rtiles + 3) / 4) + (rt >> 2)) * 512;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int k0 = block_exponent(am[2 * w]), k1 = block_exponent(am[2 * w + 1]);
      if (r8 == w) {
        st[scale_at(c8 * 8 + 2 * w, rt & 3)] = c0 + 2 * w < cols ? static_cast<uint8_t>(k0 + 127) : 0;
        st[scale_at(c8 * 8 + 2 * w + 1, rt & 3)] = c0 + 2 * w + 1 < cols ? static_cast<uint8_t>(k1 + 127) : 0;
      }
      uint2 a, b;
      x.col_codes(w, k0, k1, a, b);
      // 8 rows of a column: the 8-byte chunk r8 of that line sits at r8 ^ c8, so that the 16 lanes fill all banks
      uint8_t* line = tile + (c8 * 8 + 2 * w) * B + ((r8 ^ c8) << 3);
      *reinterpret_cast<uint2*>(line) = a;
      *reinterpret_cast<uint2*>(line + B) = b;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int c = n * 32 + (tid >> 3), part = tid & 7, x8 = c >> 3;
      uint4 o = *reinterpret_cast<const uint4*>(tile + c * B + ((part ^ (x8 >> 1)) << 4));
      if (x8 & 1) o = make_uint4(o.z, o.w, o.x, o.y);
      if (ct * B + c < cols) *reinterpret_cast<uint4*>(qt + (static_cast<long long>(ct) * B + c) * pitch + rt * B + part * 16) = o;
    }
  }
}

template <typename T>
int launch(int mode, uint32_t across, uint32_t grid, cudaStream_t stream, const void* x, int rows, int cols, long long ld, uint8_t* const* o) {
  const int vec = !(reinterpret_cast<uintptr_t>(x) & 15) && !((ld * static_cast<int>(sizeof(T))) & 15);
  const T* p = static_cast<const T*>(x);
  switch (mode) {
#define CASE(m) case m: fp8_quantize_kernel<T, m><<<grid, THREADS, 0, stream>>>(p, rows, cols, ld, vec, across, o[0], o[1], o[2], o[3]); break
    CASE(ROWS);
    CASE(COLS);
    CASE(ROWS | COLS);
    CASE(ROWS | SQUARE);
    CASE(COLS | SQUARE);
    CASE(ROWS | COLS | SQUARE);
#undef CASE
    default: return -3;
  }
  return mbh::check_launch("fp8_quantize");
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
  if (static_cast<long long>(gx) * gy > 0x7fffffffll) return -3;
  uint8_t* o[4] = {static_cast<uint8_t*>(q), static_cast<uint8_t*>(sq), static_cast<uint8_t*>(qt), static_cast<uint8_t*>(sqt)};
  return type == 0 ? launch<__nv_bfloat16>(mode, gx, gx * gy, stream, x, rows, cols, ld, o)
                   : launch<float>(mode, gx, gx * gy, stream, x, rows, cols, ld, o);
}
