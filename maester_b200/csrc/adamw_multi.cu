// One AdamW step over many tensors, with the two moments in 8 bits or in 32.
//
//   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,   p <- (1 - lr wd) p - (lr / bc1) m / (sqrt(v) / sqrt(bc2) + eps)
//
// 8-bit states: m and r = sqrt(v) are e4m3 codes with one exponent byte for every 256 values of a tensor: value =
// code * 2^(byte - 127), the smallest such power with |value| <= 448 * 2^k.  Powers of two make the division exact, so a
// value is rounded once, and encoding what was decoded gives the same values.  The root halves the range of exponents that the
// second moment needs (e4m3 then spans 2^34 of v inside a block), and a root that is not zero never becomes zero: the
// smallest code stands in, so m / r stays bounded where a block holds very different gradients.
//
// The moments are rounded to 32 bits operation by operation (no contraction), in the order written above: the codes do not
// depend on what the compiler fuses.  The root is a reciprocal root with one Newton step, whose remainder is exact (the rounded
// root but for one value in a million); the quotient m / (...) is off by two steps of its own at most, a fraction of a step of p.
//
// The step moves 18 bytes a value with 8-bit states beside 32-bit parameters and their 16-bit copy (30 with 32-bit states) and
// is bound by that.  A warp owns 256 consecutive values at a time, so a block's maximum is one warp reduction.
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp8.h>
#include <math.h>

namespace {

constexpr int BLOCK = 256;    // values that share an exponent; one warp
constexpr int WARP_BLOCKS = 8;                          // neighbouring blocks of a warp
constexpr int CHUNK = 8 * WARP_BLOCKS * BLOCK;          // values of one thread block
constexpr int THREADS = 256;
constexpr int CAP = 512;      // tensors of one launch (the table travels as a kernel argument)

struct Tensor {   // one row of the caller's table
  void* p;
  const void* g;
  __nv_bfloat16* copy;
  long long n;
  long long off;         // of its states in the flat buffers: a multiple of 256
  int first_chunk;       // filled by the launcher
  int pad;
};
struct Table {
  Tensor t[CAP];
  int count;
};
struct Hyper {
  float b1, omb1, b2, omb2, decay, step, inv_root, eps;
};

__device__ __forceinline__ float pow2(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

// smallest k in [k_min, 120] with amax <= 448 * 2^k = 1.75 * 2^(k + 8)
__device__ __forceinline__ int block_exponent(uint32_t amax_bits, int k_min) {
  const int e = static_cast<int>(amax_bits >> 23) - 127;                       // amax in [2^e, 2^(e+1)), or below 2^-126
  const int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  return min(max(k, k_min), 120);
}
__device__ __forceinline__ float floored(float y) { return y > 0.f ? fmaxf(y, 0.001953125f) : y; }   // (NaN stays)
// four codes in a word; an infinity has become NaN before
__device__ __forceinline__ uint32_t encode4(float2 a, float2 b) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ void decode4(uint32_t w, float2& a, float2& b) {
  a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3)));
  b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3)));
}

// two fp32 operations an instruction
typedef unsigned long long u64;
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<u64&>(r)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<u64&>(r)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float b) { return mul2(a, make_float2(b, b)); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<u64&>(r))
      : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)), "l"(reinterpret_cast<u64&>(c)));
  return r;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^12 sqrt(v) for v < 2^104: on 2^24 v, which is a normal number or 0
__device__ __forceinline__ float2 root2(float2 v) {
  const float2 w = mul2(v, 16777216.f);
  const float2 y = make_float2(rsqrt_approx(fmaxf(w.x, 1.1754944e-38f)), rsqrt_approx(fmaxf(w.y, 1.1754944e-38f)));
  const float2 s = mul2(w, y), left = fma2(make_float2(-s.x, -s.y), s, w);
  return fma2(left, mul2(y, 0.5f), s);
}

// four neighbouring values, read or written once
__device__ __forceinline__ float4 load4(const float* p) { return __ldcs(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 v) { __stcs(reinterpret_cast<float4*>(p), v); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  __stcs(reinterpret_cast<uint2*>(p), make_uint2(mb::pack_bf16(v.x, v.y), mb::pack_bf16(v.z, v.w)));
}

struct States {
  uint8_t *m8, *m_exp, *r8, *r_exp;   // 8 bits
  float *m32, *v32;                   // 32 bits
};

// n of four neighbouring values one by one (the end of a tensor, or off its 16-byte boundaries); 0 where there is none
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float* p, float v) { *p = v; }
__device__ __forceinline__ void narrow(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
template <typename P>
__device__ __forceinline__ void load_some(const P* p, int n, float2& a, float2& b) {
  a = make_float2(n > 0 ? widen(p[0]) : 0.f, n > 1 ? widen(p[1]) : 0.f);
  b = make_float2(n > 2 ? widen(p[2]) : 0.f, n > 3 ? widen(p[3]) : 0.f);
}
template <typename P>
__device__ __forceinline__ void store_some(P* p, int n, float2 a, float2 b) {
  if (n > 0) narrow(p, a.x);
  if (n > 1) narrow(p + 1, a.y);
  if (n > 2) narrow(p + 2, b.x);
  if (n > 3) narrow(p + 3, b.y);
}
template <typename P>
__device__ __forceinline__ void load_all(const P* p, float2& a, float2& b) {
  const float4 v = load4(p);
  a = make_float2(v.x, v.y);
  b = make_float2(v.z, v.w);
}
template <typename P>
__device__ __forceinline__ void store_all(P* p, float2 a, float2 b) { store4(p, make_float4(a.x, a.y, b.x, b.y)); }

// The next block of 256 values (n of them exist; `lines`: all, on 16-byte boundaries).  A lane owns values 4 lane .. and
// 128 + 4 lane .., so that every access of a whole block is a line.  The states behind the end of a tensor stay as they are.
// exps: biased exponents of m and r, before and after.
template <typename P, bool EIGHT>
__device__ __forceinline__ uint2 next_block(P* p, const P* g, __nv_bfloat16* copy, long long s0, int n, bool lines, const States& st,
                                            const Hyper& h, uint2 exps, int lane) {
  const int e0 = 4 * lane;
  float2 x[4], d[4], m[4], v[4];
  uint32_t mw[2], rw[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = e0 + 128 * j;
    if (lines) {
      load_all(g + e, d[2 * j], d[2 * j + 1]);
      load_all(p + e, x[2 * j], x[2 * j + 1]);
    } else {
      load_some(g + e, n - e, d[2 * j], d[2 * j + 1]);
      load_some(p + e, n - e, x[2 * j], x[2 * j + 1]);
    }
    if (EIGHT) {     // (the state buffers go on to the end of the block, zeros there)
      mw[j] = __ldcs(reinterpret_cast<const uint32_t*>(st.m8 + s0 + e));
      rw[j] = __ldcs(reinterpret_cast<const uint32_t*>(st.r8 + s0 + e));
    } else {
      load_all(st.m32 + s0 + e, m[2 * j], m[2 * j + 1]);
      load_all(st.v32 + s0 + e, v[2 * j], v[2 * j + 1]);
    }
  }
  if (EIGHT) {
    const float sm = pow2(static_cast<int>(exps.x) - 127), sr = pow2(static_cast<int>(exps.y) - 127);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      decode4(mw[j], m[2 * j], m[2 * j + 1]);
      decode4(rw[j], v[2 * j], v[2 * j + 1]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = mul2(m[j], sm);
      const float2 r = mul2(v[j], sr);
      v[j] = mul2(r, r);
    }
  }
  float am = 0.f, av = 0.f;     // largest finite or infinite value (fmaxf passes NaN over)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // (one by one: a packed product and sum are contracted, and ties between two codes then go the other way)
    m[j].x = __fadd_rn(__fmul_rn(m[j].x, h.b1), __fmul_rn(d[j].x, h.omb1));
    m[j].y = __fadd_rn(__fmul_rn(m[j].y, h.b1), __fmul_rn(d[j].y, h.omb1));
    v[j].x = __fadd_rn(__fmul_rn(v[j].x, h.b2), __fmul_rn(__fmul_rn(d[j].x, d[j].x), h.omb2));
    v[j].y = __fadd_rn(__fmul_rn(v[j].y, h.b2), __fmul_rn(__fmul_rn(d[j].y, d[j].y), h.omb2));
    if (EIGHT) am = fmaxf(fmaxf(am, fabsf(m[j].x)), fabsf(m[j].y));
    av = fmaxf(fmaxf(av, v[j].x), v[j].y);
  }
  if (!EIGHT) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = e0 + 128 * j;
      if (lines) {
        store_all(st.m32 + s0 + e, m[2 * j], m[2 * j + 1]);
        store_all(st.v32 + s0 + e, v[2 * j], v[2 * j + 1]);
      } else {
        store_some(st.m32 + s0 + e, n - e, m[2 * j], m[2 * j + 1]);
        store_some(st.v32 + s0 + e, n - e, v[2 * j], v[2 * j + 1]);
      }
    }
  }
  const bool vast = !(av < 2.028241e31f);      // 2^104 and more
#pragma unroll
  for (int j = 0; j < 4; ++j) {    // v becomes 2^12 times its root
    if (vast) v[j] = make_float2(__fmul_rn(__fsqrt_rn(v[j].x), 4096.f), __fmul_rn(__fsqrt_rn(v[j].y), 4096.f));
    else v[j] = root2(v[j]);
    const float2 den = add2(mul2(v[j], h.inv_root * 0.000244140625f), make_float2(h.eps, h.eps));
    const float2 u = mul2(make_float2(__fdividef(m[j].x, den.x), __fdividef(m[j].y, den.y)), -h.step);
    x[j] = add2(mul2(x[j], h.decay), u);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = e0 + 128 * j;
    if (lines) {
      store_all(p + e, x[2 * j], x[2 * j + 1]);
      if (copy) store_all(copy + e, x[2 * j], x[2 * j + 1]);
    } else {
      store_some(p + e, n - e, x[2 * j], x[2 * j + 1]);
      if (copy) store_some(copy + e, n - e, x[2 * j], x[2 * j + 1]);
    }
  }
  if (EIGHT) {
    uint32_t bm = __float_as_uint(am), br = __float_as_uint(av);
    bm = __reduce_max_sync(~0u, bm);
    br = __reduce_max_sync(~0u, br);
    if (bm >= 0x7f800000u || br >= 0x7f800000u) {   // an infinity: it becomes the NaN code and sets no scale
      bm = br = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float* a[4] = {&m[j].x, &m[j].y, &v[j].x, &v[j].y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t b = __float_as_uint(*a[i]) & 0x7fffffffu;
          if (b >= 0x7f800000u) *a[i] = __uint_as_float(0x7fffffffu);
          else if (i < 2) bm = max(bm, b);
          else br = max(br, b);
        }
      }
      bm = __reduce_max_sync(~0u, bm);
      br = __reduce_max_sync(~0u, br);
      br = __float_as_uint(__fmul_rn(__uint_as_float(br), 0.000244140625f));
    } else {        // the largest root is the root of the largest v
      const float2 r = root2(make_float2(__uint_as_float(br), 0.f));
      br = __float_as_uint(br >= 0x73800000u /* 2^104 */ ? __fsqrt_rn(__uint_as_float(br)) : __fmul_rn(r.x, 0.000244140625f));
    }
    const int km = block_exponent(bm, -117), kr = block_exponent(br, -54);
    const float im = pow2(-km), ir = pow2(-kr) * 0.000244140625f;
    exps = make_uint2(km + 127, kr + 127);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = mul2(m[j], im);
      v[j] = mul2(v[j], ir);
      v[j] = make_float2(floored(v[j].x), floored(v[j].y));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = e0 + 128 * j;
      // behind the end everything was 0 and stays 0: whole words
      __stcs(reinterpret_cast<uint32_t*>(st.m8 + s0 + e), encode4(m[2 * j], m[2 * j + 1]));
      __stcs(reinterpret_cast<uint32_t*>(st.r8 + s0 + e), encode4(v[2 * j], v[2 * j + 1]));
    }
  }
  return exps;
}

template <typename P, bool EIGHT>
__global__ void __launch_bounds__(THREADS, 3) adamw_multi_kernel(const __grid_constant__ Table tab, const Hyper h, const States st) {
  int lo = 0, hi = tab.count - 1;
  const int chunk = blockIdx.x;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first_chunk <= chunk) lo = mid; else hi = mid - 1;
  }
  const Tensor& t = tab.t[lo];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c0 = static_cast<long long>(chunk - t.first_chunk) * CHUNK, n = t.n;
  P* p = static_cast<P*>(t.p);
  const P* g = static_cast<const P*>(t.g);
  __nv_bfloat16* copy = t.copy;
  const long long off = t.off;
  const bool lines = !((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & (4 * sizeof(P) - 1)) &&
                     !(reinterpret_cast<uintptr_t>(copy) & 7);
  // A warp's blocks are neighbours: their exponents are read together before the first and written together after the last.
  // (Read and written block by block, bytes of one 32-byte sector were on their way in both directions all the time: 1247
  // instead of 565 us for 200M values.)
  const long long w0 = c0 + static_cast<long long>(warp) * WARP_BLOCKS * BLOCK;
  if (w0 >= n) return;
  const int blocks = static_cast<int>(min(static_cast<long long>(WARP_BLOCKS), (n - w0 + BLOCK - 1) / BLOCK));
  uint8_t* exp_at = nullptr;
  uint32_t exps = 0;               // lane b: m's exponent of block b, lane 16 + b: r's
  if (EIGHT && (lane & 15) < blocks) {
    exp_at = (lane < 16 ? st.m_exp : st.r_exp) + (off + w0) / BLOCK + (lane & 15);
    exps = *exp_at;
  }
  for (int b = 0; b < blocks; ++b) {
    const long long i0 = w0 + static_cast<long long>(b) * BLOCK;
    uint2 e = make_uint2(__shfl_sync(~0u, exps, b), __shfl_sync(~0u, exps, 16 + b));
    const int have = static_cast<int>(min(n - i0, static_cast<long long>(BLOCK)));
    e = next_block<P, EIGHT>(p + i0, g + i0, copy ? copy + i0 : nullptr, off + i0, have, lines && have == BLOCK, st, h, e, lane);
    if ((lane & 15) == b) exps = lane < 16 ? e.x : e.y;
  }
  if (EIGHT && exp_at) *exp_at = static_cast<uint8_t>(exps);
}

}  // namespace

// tensors: host array of `count` rows (struct Tensor above), all of one type: 32-bit (p_bf16 = 0) or bf16 values with
// gradients of the same type.  bits 8: m, m_exp, r, r_exp; bits 32: m, r hold fp32 moments and the exponents are null.
// hyper: 8 host floats in the order of struct Hyper.
extern "C" int mb_adamw_multi(const void* tensors, int count, int p_bf16, int bits, void* m, void* m_exp, void* r,
                              void* r_exp, const float* hyper, cudaStream_t stream) {
  if (count < 0 || (bits != 8 && bits != 32)) return -3;
  const Tensor* rows = static_cast<const Tensor*>(tensors);
  Hyper h;
  h.b1 = hyper[0]; h.omb1 = hyper[1]; h.b2 = hyper[2]; h.omb2 = hyper[3];
  h.decay = hyper[4]; h.step = hyper[5]; h.inv_root = hyper[6]; h.eps = hyper[7];
  int at = 0;
  while (at < count) {
    Table tab;
    tab.count = 0;
    long long chunks = 0;
    while (at < count && tab.count < CAP) {
      Tensor t = rows[at];
      if (t.n < 0 || (t.off & (BLOCK - 1))) return -3;
      const long long c = (t.n + CHUNK - 1) / CHUNK;
      if (chunks + c > 0x7fffffffll) {
        if (!tab.count) return -3;
        break;
      }
      ++at;
      if (!c) continue;
      t.first_chunk = static_cast<int>(chunks);
      tab.t[tab.count++] = t;
      chunks += c;
    }
    if (!tab.count) continue;
    const unsigned grid = static_cast<unsigned>(chunks);
    const States st{static_cast<uint8_t*>(m), static_cast<uint8_t*>(m_exp), static_cast<uint8_t*>(r), static_cast<uint8_t*>(r_exp),
                    static_cast<float*>(m), static_cast<float*>(r)};
    if (bits == 8) {
      if (p_bf16) adamw_multi_kernel<__nv_bfloat16, true><<<grid, THREADS, 0, stream>>>(tab, h, st);
      else adamw_multi_kernel<float, true><<<grid, THREADS, 0, stream>>>(tab, h, st);
    } else {
      if (p_bf16) adamw_multi_kernel<__nv_bfloat16, false><<<grid, THREADS, 0, stream>>>(tab, h, st);
      else adamw_multi_kernel<float, false><<<grid, THREADS, 0, stream>>>(tab, h, st);
    }
    const int e = mbh::check_launch("adamw_multi");
    if (e) return e;
  }
  return 0;
}
