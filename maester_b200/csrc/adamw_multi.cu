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
// Every operation is rounded to 32 bits on its own (no contraction), in the order written above: the codes do not depend
// on what the compiler fuses, and equal inputs give equal bits on every path.
//
// The step moves 18 bytes a value with 8-bit states beside 32-bit parameters and their 16-bit copy (30 with 32-bit
// states) and is bound by that.  A warp owns 256 consecutive values, so a block's maximum is one warp reduction.
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp8.h>
#include <math.h>

namespace {

constexpr int BLOCK = 256;    // values that share an exponent; one warp
constexpr int CHUNK = 8192;   // values of one thread block
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

__device__ __forceinline__ float ld_f(const float* p) { return *p; }
__device__ __forceinline__ float ld_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ float pow2(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

// smallest k in [k_min, 120] with amax <= 448 * 2^k = 1.75 * 2^(k + 8)
__device__ __forceinline__ int block_exponent(uint32_t amax_bits, int k_min) {
  const int e = static_cast<int>(amax_bits >> 23) - 127;                       // amax in [2^e, 2^(e+1)), or below 2^-126
  const int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  return min(max(k, k_min), 120);
}
__device__ __forceinline__ uint32_t finite_bits(float x) {                      // |x| as an ordered whole number; 0 if not finite
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint8_t encode(float y) {
  if (!(fabsf(y) <= 3.4028234e38f)) return 0x7f;                                // NaN and infinities
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ float decode(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
__device__ __forceinline__ float floored(float y) { return y > 0.f ? fmaxf(y, 0.001953125f) : y; }   // (NaN stays)
// four codes in a word; finite values
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float4 decode4(uint32_t w) {
  const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3)));
  const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3)));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}

struct Moments {
  float m, v, root;
};
__device__ __forceinline__ Moments moments(float m, float v, float g, const Hyper& h) {
  Moments o;
  o.m = __fadd_rn(__fmul_rn(m, h.b1), __fmul_rn(g, h.omb1));
  o.v = __fadd_rn(__fmul_rn(v, h.b2), __fmul_rn(__fmul_rn(g, g), h.omb2));
  o.root = __fsqrt_rn(o.v);
  return o;
}
__device__ __forceinline__ float update(float p, const Moments& o, const Hyper& h) {
  const float den = __fadd_rn(__fmul_rn(o.root, h.inv_root), h.eps);
  return __fsub_rn(__fmul_rn(p, h.decay), __fmul_rn(__fdiv_rn(o.m, den), h.step));
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

// A block of 256 values, its tensor's last one, or one that does not start on a 16-byte boundary: value by value.
template <typename P, bool EIGHT>
__device__ __noinline__ void block_by_value(P* p, const P* g, __nv_bfloat16* copy, int n, long long s0, const States& st,
                                            const Hyper& h, int lane) {
  Moments o[BLOCK / 32];
  float scale_m = 0.f, scale_r = 0.f;
  if (EIGHT) {
    scale_m = pow2(static_cast<int>(st.m_exp[s0 / BLOCK]) - 127);
    scale_r = pow2(static_cast<int>(st.r_exp[s0 / BLOCK]) - 127);
  }
  uint32_t am = 0, ar = 0;
#pragma unroll
  for (int j = 0; j < BLOCK / 32; ++j) {
    const int e = j * 32 + lane;
    o[j] = Moments{0.f, 0.f, 0.f};
    if (e < n) {
      float m, v;
      if (EIGHT) {
        m = decode(st.m8[s0 + e]) * scale_m;
        const float r = decode(st.r8[s0 + e]) * scale_r;
        v = __fmul_rn(r, r);
      } else {
        m = st.m32[s0 + e];
        v = st.v32[s0 + e];
      }
      o[j] = moments(m, v, ld_f(g + e), h);
      const float np = update(ld_f(p + e), o[j], h);
      st_f(p + e, np);
      if (copy) copy[e] = __float2bfloat16(np);
      if (!EIGHT) {
        st.m32[s0 + e] = o[j].m;
        st.v32[s0 + e] = o[j].v;
      }
      am = max(am, finite_bits(o[j].m));
      ar = max(ar, finite_bits(o[j].root));
    }
  }
  if (EIGHT) {
    const int km = block_exponent(__reduce_max_sync(~0u, am), -117), kr = block_exponent(__reduce_max_sync(~0u, ar), -54);
    if (lane == 0) {
      st.m_exp[s0 / BLOCK] = static_cast<uint8_t>(km + 127);
      st.r_exp[s0 / BLOCK] = static_cast<uint8_t>(kr + 127);
    }
    const float im = pow2(-km), ir = pow2(-kr);
#pragma unroll
    for (int j = 0; j < BLOCK / 32; ++j) {
      const int e = j * 32 + lane;
      if (e < n) {
        st.m8[s0 + e] = encode(__fmul_rn(o[j].m, im));
        st.r8[s0 + e] = encode(floored(__fmul_rn(o[j].root, ir)));
      }
    }
  }
}

// A whole block on 16-byte boundaries: a lane owns values 4 lane .. and 128 + 4 lane .., so that every access is a line.
template <typename P, bool EIGHT>
__device__ __forceinline__ void block_by_line(P* p, const P* g, __nv_bfloat16* copy, long long s0, const States& st, const Hyper& h,
                                              int lane) {
  const int e0 = 4 * lane;
  float4 pv[2], gv[2], mv[2], vv[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    gv[j] = load4(g + e0 + 128 * j);
    pv[j] = load4(p + e0 + 128 * j);
  }
  if (EIGHT) {
    uint32_t mw[2], rw[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mw[j] = __ldcs(reinterpret_cast<const uint32_t*>(st.m8 + s0 + e0 + 128 * j));
      rw[j] = __ldcs(reinterpret_cast<const uint32_t*>(st.r8 + s0 + e0 + 128 * j));
    }
    const float sm = pow2(static_cast<int>(st.m_exp[s0 / BLOCK]) - 127), sr = pow2(static_cast<int>(st.r_exp[s0 / BLOCK]) - 127);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mv[j] = decode4(mw[j]);
      vv[j] = decode4(rw[j]);
      float* m = &mv[j].x;
      float* v = &vv[j].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = __fmul_rn(m[i], sm);
        const float r = __fmul_rn(v[i], sr);
        v[i] = __fmul_rn(r, r);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mv[j] = load4(st.m32 + s0 + e0 + 128 * j);
      vv[j] = load4(st.v32 + s0 + e0 + 128 * j);
    }
  }
  uint32_t am = 0, ar = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float* m = &mv[j].x;
    float* v = &vv[j].x;
    float* x = &pv[j].x;
    const float* d = &gv[j].x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Moments o = moments(m[i], v[i], d[i], h);
      x[i] = update(x[i], o, h);
      m[i] = o.m;
      v[i] = EIGHT ? o.root : o.v;
      if (EIGHT) {
        am = max(am, __float_as_uint(o.m) & 0x7fffffffu);
        ar = max(ar, __float_as_uint(o.root) & 0x7fffffffu);
      }
    }
    store4(p + e0 + 128 * j, pv[j]);
    if (copy) store4(copy + e0 + 128 * j, pv[j]);
    if (!EIGHT) {
      store4(st.m32 + s0 + e0 + 128 * j, mv[j]);
      store4(st.v32 + s0 + e0 + 128 * j, vv[j]);
    }
  }
  if (EIGHT) {
    am = __reduce_max_sync(~0u, am);
    ar = __reduce_max_sync(~0u, ar);
    if (am >= 0x7f800000u || ar >= 0x7f800000u) {   // something is not finite: it becomes the NaN code and sets no scale
      am = ar = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* m = &mv[j].x;
        float* r = &vv[j].x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          am = max(am, finite_bits(m[i]));
          ar = max(ar, finite_bits(r[i]));
          if (!finite_bits(m[i]) && m[i] != 0.f) m[i] = __uint_as_float(0x7fffffffu);
          if (!finite_bits(r[i]) && r[i] != 0.f) r[i] = __uint_as_float(0x7fffffffu);
        }
      }
      am = __reduce_max_sync(~0u, am);
      ar = __reduce_max_sync(~0u, ar);
    }
    const int km = block_exponent(am, -117), kr = block_exponent(ar, -54);
    const float im = pow2(-km), ir = pow2(-kr);
    if (lane == 0) {
      st.m_exp[s0 / BLOCK] = static_cast<uint8_t>(km + 127);
      st.r_exp[s0 / BLOCK] = static_cast<uint8_t>(kr + 127);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float* m = &mv[j].x;
      const float* r = &vv[j].x;
      __stcs(reinterpret_cast<uint32_t*>(st.m8 + s0 + e0 + 128 * j),
             encode4(__fmul_rn(m[0], im), __fmul_rn(m[1], im), __fmul_rn(m[2], im), __fmul_rn(m[3], im)));
      __stcs(reinterpret_cast<uint32_t*>(st.r8 + s0 + e0 + 128 * j),
             encode4(floored(__fmul_rn(r[0], ir)), floored(__fmul_rn(r[1], ir)), floored(__fmul_rn(r[2], ir)), floored(__fmul_rn(r[3], ir))));
    }
  }
}

template <typename P, bool EIGHT>
__global__ void __launch_bounds__(THREADS, 4) adamw_multi_kernel(const __grid_constant__ Table tab, const Hyper h, const States st) {
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
  for (int b = warp; b < CHUNK / BLOCK; b += THREADS / 32) {
    const long long i0 = c0 + static_cast<long long>(b) * BLOCK;
    if (i0 >= n) break;
    if (lines && i0 + BLOCK <= n)
      block_by_line<P, EIGHT>(p + i0, g + i0, copy ? copy + i0 : nullptr, off + i0, st, h, lane);
    else
      block_by_value<P, EIGHT>(p + i0, g + i0, copy ? copy + i0 : nullptr, static_cast<int>(min(n - i0, static_cast<long long>(BLOCK))),
                               off + i0, st, h, lane);
  }
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
