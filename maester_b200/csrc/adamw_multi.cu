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
// A moving average changes by a few percent a step, or by a thousandth, and neighbouring codes are 6 to 12 percent apart: rounded
// to nearest it would stand still (the second moment never decays at b2 >= 0.95, and hardly grows at 0.999).  So a value becomes
// one of its two neighbouring codes lo < hi, at random, and its expectation stays what it was: m the upper one with probability
// (m - lo) / (hi - lo), the root r with (r^2 - lo^2) / (hi^2 - lo^2), which keeps the expectation of v (keeping that of r would
// add the variance of every rounding to v).  (r^2 is v to 2^-23: holding v itself to the end costs 8 registers a thread, 3 % of the
// time with fp32 and 8 % with bf16 parameters.)  A parameter's first step rounds to nearest: nothing has gone before it that a
// rounding could hold fast, and the error is half as large where the bias correction weighs it most.  The random numbers are a
// hash of the step number and the value's place, so that runs repeat.
//
// The moments are rounded to 32 bits operation by operation (no contraction), in the order written above: the codes do not
// depend on what the compiler fuses.  The root is a reciprocal root with one Newton step, whose remainder is exact (the rounded
// root but for one value in a million); the quotient m / (...) is off by two steps of its own at most, a fraction of a step of p.
//
// The step moves 18 bytes a value with 8-bit states beside 32-bit parameters and their 16-bit copy (30 with 32-bit states) and
// is bound by that.  A warp owns 256 consecutive values at a time, so a block's maximum is one warp reduction.
//
// Measured (24 tensors of 4096 x 4096; copy rate 6540 GB/s): fp32 parameters with a copy 1130 us with 8-bit states (6420 GB/s),
// 1801 us with 32-bit ones (6710); bf16 parameters 856 us with 8-bit states (4710: the codes cost more instructions than the 10
// bytes of a value cost time), 1341 us with 32-bit ones (6610).  Of the 8-bit times the noise costs some 40 and 90 us (hash,
// neighbouring codes, comparison: 15 instructions a value).  Small tensors are the host's: 45 to 55 us for 20 of them.
#include "fp8_common.cuh"
#include "host_common.cuh"
#include <math.h>

namespace {

using namespace mbf8;

constexpr int BLOCK = 256;    // values that share an exponent; one warp
constexpr int THREADS = 128;                            // (256: bf16 parameters 3 % slower)
// neighbouring blocks of a warp (with 32-bit states 8 are 2 % slower; with 8-bit ones 4 are as much slower)
constexpr int warp_blocks(bool eight) { return eight ? 8 : 4; }
constexpr int chunk_of(bool eight) { return THREADS / 32 * warp_blocks(eight) * BLOCK; }   // values of one thread block
constexpr int CAP_SMALL = 32, CAP_LARGE = 512;   // tensors of one launch: the table travels as a kernel argument of
// 1.5 or 24 KiB (20 tensors: 10 us of the host's time with the small one, 14 with the large one)

struct Tensor {   // one row of the caller's table
  void* p;
  const void* g;
  __nv_bfloat16* copy;
  long long n;
  long long off;         // of its states in the flat buffers: a multiple of 256
  int first_chunk;       // filled by the launcher
  int pad;
};
template <int CAP>
struct Table {
  Tensor t[CAP];
  int count;
};
struct Hyper {
  float b1, omb1, b2, omb2, decay, step, inv_root, eps;
  uint32_t key;    // stands for the step number in the noise of the codes' rounding
  int noisy;       // 0: codes are rounded to nearest
  float one;   // 1, unknown to the compiler: a packed product and sum would be contracted, and ties between two codes go the
};             // other way then; a fused operation with it is a plain sum

__device__ __forceinline__ float floored(float y) { return y > 0.f ? fmaxf(y, 0.001953125f) : y; }   // (NaN stays)
// four codes in a word; an infinity has become NaN before
__device__ __forceinline__ uint32_t encode4(float2 a, float2 b) { return encode2(a) | (encode2(b) << 16); }
__device__ __forceinline__ void decode4(uint32_t w, float2& a, float2& b) {
  a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3)));
  b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3)));
}

// two fp32 operations an instruction
typedef unsigned long long u64;
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
__device__ __forceinline__ float rcp_approx(float x) {   // 0 above 2^126
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// sqrt(v) for v in [2^-102, 2^104): the remainder v - s^2 is exact
constexpr float ROOT_FROM = 1.9721523e-31f, ROOT_TO = 2.028241e31f;
__device__ __forceinline__ float2 root2(float2 v) {
  const float2 y = make_float2(rsqrt_approx(v.x), rsqrt_approx(v.y));
  const float2 s = mul2(v, y), left = fma2(make_float2(-s.x, -s.y), s, v);
  return fma2(left, mul2(y, 0.5f), s);
}
// any v: 0, tiny and vast ones, infinities and NaN too
__device__ __forceinline__ float any_root(float v) {
  if (v >= ROOT_FROM && v < ROOT_TO) return root2(make_float2(v, 1.f)).x;
  return __fsqrt_rn(v);
}

// Eight neighbouring values, read or written once: 32 bytes of fp32 or 16 of bf16 in one access
__device__ __forceinline__ void load_all(const float* p, float2 (&a)[4]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(a[0].x), "=f"(a[0].y), "=f"(a[1].x), "=f"(a[1].y), "=f"(a[2].x), "=f"(a[2].y), "=f"(a[3].x), "=f"(a[3].y)
               : "l"(p));
}
__device__ __forceinline__ void widen_all(uint4 w, float2 (&a)[4]) {
  a[0] = make_float2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u));
  a[1] = make_float2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  a[2] = make_float2(__uint_as_float(w.z << 16), __uint_as_float(w.z & 0xffff0000u));
  a[3] = make_float2(__uint_as_float(w.w << 16), __uint_as_float(w.w & 0xffff0000u));
}
__device__ __forceinline__ void load_all(const __nv_bfloat16* p, float2 (&a)[4]) {
  widen_all(__ldcs(reinterpret_cast<const uint4*>(p)), a);
}
__device__ __forceinline__ void store_all(float* p, const float2 (&a)[4]) {
  asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
               ::"f"(a[0].x), "f"(a[0].y), "f"(a[1].x), "f"(a[1].y), "f"(a[2].x), "f"(a[2].y), "f"(a[3].x), "f"(a[3].y), "l"(p)
               : "memory");
}
__device__ __forceinline__ void store_all(__nv_bfloat16* p, const float2 (&a)[4]) {
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(mb::pack_bf16(a[0].x, a[0].y), mb::pack_bf16(a[1].x, a[1].y),
                                                 mb::pack_bf16(a[2].x, a[2].y), mb::pack_bf16(a[3].x, a[3].y)));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// ---- noise: 32 random bits for each of the 8 values of a lane, a hash of their group's place and a linear congruence after it.
// The lower 23 bits round the root, the upper 20 the first moment (what they share weighs 2^-10 and less in the latter's).
__device__ __forceinline__ uint32_t first_noise(uint32_t group, uint32_t key) {
  uint32_t x = group * 0x9E3779B9u + key;
  x = (x ^ (x >> 16)) * 0xB7E15163u;
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t next_noise(uint32_t x) { return x * 0x6A09E667u + 0xBB67AE85u; }
__device__ __forceinline__ float one_plus(uint32_t bits) { return __uint_as_float(0x3f800000u | (bits & 0x7fffffu)); }

constexpr float NORMAL = 0.015625f;   // 2^-6: below it codes keep the distance 2^-9
// the largest code that is at most a in [0, 448], after `add` units of 2^-20 of a code's last place; its distance to the next
__device__ __forceinline__ float code_below(float a, uint32_t add, float& gap) {
  const float low = a < NORMAL ? NORMAL : 0.f;
  const uint32_t z = (__float_as_uint(__fadd_rn(a, low)) + add) & 0xfff00000u;
  gap = __uint_as_float(z & 0x7f800000u) * 0.125f;
  return __uint_as_float(z) - low;
}
// m / 2^k and a root / 2^k as one of the two neighbouring codes; NaN stays
__device__ __forceinline__ float round_noisy(float y, uint32_t bits) {
  float gap;
  const float r = copysignf(code_below(fabsf(y), bits >> 12, gap), y);
  return y == y ? r : y;
}
__device__ __forceinline__ float round_root_noisy(float y, uint32_t bits) {
  float gap;
  const float lo = code_below(y, 0u, gap), q = gap * (2.f * lo + gap);      // hi^2 - lo^2: exact, as lo^2 - q is
  float r = __fmul_rn(y, y) > fmaf(one_plus(bits), q, fmaf(lo, lo, -q)) ? lo + gap : lo;    // lo^2 + u q
  if (y > 0.f) r = fmaxf(r, 0.001953125f);
  return y == y ? r : y;
}
// the same for eight values that are no smaller than NORMAL
__device__ __forceinline__ void round_all(float2 (&m)[4], float2 (&r)[4], uint32_t x) {
  const float2 two = make_float2(2.f, 2.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a = x, b = next_noise(x);
    x = next_noise(b);
    m[j].x = __uint_as_float((__float_as_uint(m[j].x) + (a >> 12)) & 0xfff00000u);
    m[j].y = __uint_as_float((__float_as_uint(m[j].y) + (b >> 12)) & 0xfff00000u);
    const uint32_t lx = __float_as_uint(r[j].x) & 0xfff00000u, ly = __float_as_uint(r[j].y) & 0xfff00000u;
    const float2 lo = make_float2(__uint_as_float(lx), __uint_as_float(ly));
    const float2 gap = mul2(make_float2(__uint_as_float(lx & 0x7f800000u), __uint_as_float(ly & 0x7f800000u)), 0.125f);
    const float2 q = mul2(gap, fma2(lo, two, gap)), w = mul2(r[j], r[j]);
    const float2 t = fma2(make_float2(one_plus(a), one_plus(b)), q, fma2(lo, lo, make_float2(-q.x, -q.y)));
    r[j] = make_float2(__uint_as_float(w.x > t.x ? lx + 0x100000u : lx), __uint_as_float(w.y > t.y ? ly + 0x100000u : ly));
  }
}

struct States {
  uint8_t *m8, *m_exp, *r8, *r_exp;   // 8 bits
  float *m32, *v32;                   // 32 bits
};

// n of eight neighbouring values one by one (the end of a tensor, or off its 32-byte boundaries); 0 where there is none
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float* p, float v) { *p = v; }
__device__ __forceinline__ void narrow(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
template <typename P>
__device__ __forceinline__ void load_some(const P* p, int n, float2 (&a)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = make_float2(n > 2 * i ? widen(p[2 * i]) : 0.f, n > 2 * i + 1 ? widen(p[2 * i + 1]) : 0.f);
}
template <typename P>
__device__ __forceinline__ void store_some(P* p, int n, const float2 (&a)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n > 2 * i) narrow(p + 2 * i, a[i].x);
    if (n > 2 * i + 1) narrow(p + 2 * i + 1, a[i].y);
  }
}

// What a lane reads of a block of 16-bit values with 8-bit states.  Such a block is few bytes and much arithmetic: the next one
// is read while one is worked on (446 -> 397 us for 200M values; with 32-bit values the registers are worth more).
struct Ahead {
  uint4 x, d;
  uint2 m, r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, const __nv_bfloat16* g, const States& st, long long s0, int e) {
    d = __ldcs(reinterpret_cast<const uint4*>(g + e));
    x = __ldcs(reinterpret_cast<const uint4*>(p + e));
    m = __ldcs(reinterpret_cast<const uint2*>(st.m8 + s0 + e));
    r = __ldcs(reinterpret_cast<const uint2*>(st.r8 + s0 + e));
  }
  __device__ __forceinline__ void load(const float*, const float*, const States&, long long, int) {}
};

// A block of 256 values (n of them exist; `lines`: all, on 32-byte boundaries), 8 of them a lane's.  The states behind the end
// of a tensor stay as they are.  exps: biased exponents of m and r, before and after.  read: this block if AHEAD and lines;
// the following one afterwards, if it is whole (`more`).
template <typename P, bool EIGHT>
__device__ __forceinline__ uint2 next_block(P* p, const P* g, __nv_bfloat16* copy, long long s0, int n, bool lines, const States& st,
                                            const Hyper& h, uint2 exps, int lane, Ahead& read, bool more) {
  constexpr bool AHEAD = EIGHT && sizeof(P) == 2;
  const int e = 8 * lane;
  float2 x[4], d[4], m[4], v[4];
  uint2 mw, rw;
  if (AHEAD && lines) {
    widen_all(read.d, d);
    widen_all(read.x, x);
  } else if (lines) {
    load_all(g + e, d);
    load_all(p + e, x);
  } else {
    load_some(g + e, n - e, d);
    load_some(p + e, n - e, x);
  }
  if (EIGHT) {     // (the state buffers go on to the end of the block, zeros there)
    mw = AHEAD && lines ? read.m : __ldcs(reinterpret_cast<const uint2*>(st.m8 + s0 + e));
    rw = AHEAD && lines ? read.r : __ldcs(reinterpret_cast<const uint2*>(st.r8 + s0 + e));
    if (AHEAD && more) read.load(p + BLOCK, g + BLOCK, st, s0 + BLOCK, e);
  } else {
    load_all(st.m32 + s0 + e, m);
    load_all(st.v32 + s0 + e, v);
  }
  if (EIGHT) {
    const float sm = pow2(static_cast<int>(exps.x) - 127), sr = pow2(static_cast<int>(exps.y) - 127);
    decode4(mw.x, m[0], m[1]);
    decode4(mw.y, m[2], m[3]);
    decode4(rw.x, v[0], v[1]);
    decode4(rw.y, v[2], v[3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = mul2(m[j], sm);
      const float2 r = mul2(v[j], sr);
      v[j] = mul2(r, r);
    }
  }
  float am = 0.f, av = 0.f;                       // NaN if there is one
  float least = INFINITY;                         // over what is not NaN
  const float2 one = make_float2(h.one, h.one);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = fma2(mul2(m[j], h.b1), one, mul2(d[j], h.omb1));
    v[j] = fma2(mul2(v[j], h.b2), one, mul2(mul2(d[j], d[j]), h.omb2));
    if (EIGHT) am = max_nan(max_nan(am, fabsf(m[j].x)), fabsf(m[j].y));
    av = max_nan(max_nan(av, v[j].x), v[j].y);
    least = fminf(fminf(least, v[j].x), v[j].y);
  }
  if (!EIGHT) {
    if (lines) {
      store_all(st.m32 + s0 + e, m);
      store_all(st.v32 + s0 + e, v);
    } else {
      store_some(st.m32 + s0 + e, n - e, m);
      store_some(st.v32 + s0 + e, n - e, v);
    }
  }
  if (least >= ROOT_FROM && av < ROOT_TO) {      // v becomes its root (NaN stays)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = root2(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_float2(any_root(v[j].x), any_root(v[j].y));
  }
  const float2 c = make_float2(h.inv_root, h.inv_root), eps = make_float2(h.eps, h.eps), step = make_float2(-h.step, -h.step);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 den = fma2(v[j], c, eps);
    const float2 u = mul2(m[j], make_float2(rcp_approx(den.x), rcp_approx(den.y)));
    x[j] = fma2(u, step, mul2(x[j], h.decay));
  }
  if (lines) {
    store_all(p + e, x);
    if (copy) store_all(copy + e, x);
  } else {
    store_some(p + e, n - e, x);
    if (copy) store_some(copy + e, n - e, x);
  }
  if (EIGHT) {
    uint32_t bm = __float_as_uint(am), br = __float_as_uint(av);
    bm = __reduce_max_sync(~0u, bm);
    br = __reduce_max_sync(~0u, br);
    const bool odd = bm >= 0x7f800000u || br >= 0x7f800000u;
    if (odd) {               // an infinity becomes the NaN code; neither it nor NaN sets a scale
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
    } else {
      br = __float_as_uint(any_root(__uint_as_float(br)));       // the largest root is the root of the largest v
    }
    const int km = block_exponent(bm, -117), kr = block_exponent(br, -54);
    const float im = pow2(-km), ir = pow2(-kr);
    exps = make_uint2(km + 127, kr + 127);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = mul2(m[j], im);
      v[j] = mul2(v[j], ir);
    }
    if (h.noisy) {
      const uint32_t x = first_noise(static_cast<uint32_t>((s0 >> 3) + lane), h.key);
      float small = INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) small = fminf(fminf(small, fabsf(m[j].x)), fabsf(m[j].y));
      // (a whole warp goes one way; the margin over 2^-12 covers the roots' roundings)
      if (!__any_sync(~0u, odd || !(least * (ir * ir) >= 2.45e-4f && small >= NORMAL))) {
        round_all(m, v, x);
      } else {
        uint32_t y = x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a = y, b = next_noise(y);
          y = next_noise(b);
          m[j] = make_float2(round_noisy(m[j].x, a), round_noisy(m[j].y, b));
          v[j] = make_float2(round_root_noisy(v[j].x, a), round_root_noisy(v[j].y, b));
        }
      }
    } else if (!(least * (ir * ir) >= 3.9e-6f)) {
      // (a lane whose smallest root is at least the smallest code has nothing to lift; the margin covers the roots' roundings)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = make_float2(floored(v[j].x), floored(v[j].y));
    }
    // (behind the end everything was 0 and stays 0: whole words)
    __stcs(reinterpret_cast<uint2*>(st.m8 + s0 + e), make_uint2(encode4(m[0], m[1]), encode4(m[2], m[3])));
    __stcs(reinterpret_cast<uint2*>(st.r8 + s0 + e), make_uint2(encode4(v[0], v[1]), encode4(v[2], v[3])));
  }
  return exps;
}

template <typename P, bool EIGHT, int CAP>
__global__ void __launch_bounds__(THREADS, 8)
adamw_multi_kernel(const __grid_constant__ Table<CAP> tab, const Hyper h, const States st) {
  constexpr int WARP_BLOCKS = warp_blocks(EIGHT), CHUNK = chunk_of(EIGHT);
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
  const bool lines = !((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & (8 * sizeof(P) - 1)) &&
                     !(reinterpret_cast<uintptr_t>(copy) & 15);
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
  Ahead read;
  if (EIGHT && lines && w0 + BLOCK <= n) read.load(p + w0, g + w0, st, off + w0, 8 * lane);
  for (int b = 0; b < blocks; ++b) {
    const long long i0 = w0 + static_cast<long long>(b) * BLOCK;
    uint2 e = make_uint2(__shfl_sync(~0u, exps, b), __shfl_sync(~0u, exps, 16 + b));
    const int have = static_cast<int>(min(n - i0, static_cast<long long>(BLOCK)));
    e = next_block<P, EIGHT>(p + i0, g + i0, copy ? copy + i0 : nullptr, off + i0, have, lines && have == BLOCK, st, h, e, lane, read,
                             lines && b + 1 < blocks && i0 + 2 * BLOCK <= n);
    if ((lane & 15) == b) exps = lane < 16 ? e.x : e.y;
  }
  if (EIGHT && exp_at) *exp_at = static_cast<uint8_t>(exps);
}

// Launches for rows [at, count) of the caller's table, as many as one takes; returns 0 and moves `at` on.
template <int CAP>
int launch(const Tensor* rows, int& at, int count, bool bf16, bool eight, const Hyper& h, const States& st, cudaStream_t stream) {
  Table<CAP> tab;
  tab.count = 0;
  long long chunks = 0;
  while (at < count && tab.count < CAP) {
    Tensor t = rows[at];
    if (t.n < 0 || (t.off & (BLOCK - 1))) return -3;
    const long long c = (t.n + chunk_of(eight) - 1) / chunk_of(eight);
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
  if (!tab.count) return 0;
  const unsigned grid = static_cast<unsigned>(chunks);
  if (eight) {
    if (bf16) adamw_multi_kernel<__nv_bfloat16, true, CAP><<<grid, THREADS, 0, stream>>>(tab, h, st);
    else adamw_multi_kernel<float, true, CAP><<<grid, THREADS, 0, stream>>>(tab, h, st);
  } else {
    if (bf16) adamw_multi_kernel<__nv_bfloat16, false, CAP><<<grid, THREADS, 0, stream>>>(tab, h, st);
    else adamw_multi_kernel<float, false, CAP><<<grid, THREADS, 0, stream>>>(tab, h, st);
  }
  return mbh::check_launch("adamw_multi");
}

}  // namespace

// tensors: host array of `count` rows (struct Tensor above), all of one type: 32-bit (p_bf16 = 0) or bf16 values with
// gradients of the same type.  bits 8: m, m_exp, r, r_exp; bits 32: m, r hold fp32 moments and the exponents are null.
// hyper: 8 host floats in the order of struct Hyper.  key: 32 bits that stand for the step number in the noise of the codes'
// rounding; negative: they are rounded to nearest.
extern "C" int mb_adamw_multi(const void* tensors, int count, int p_bf16, int bits, void* m, void* m_exp, void* r,
                              void* r_exp, const float* hyper, long long key, cudaStream_t stream) {
  if (count < 0 || (bits != 8 && bits != 32)) return -3;
  const Tensor* rows = static_cast<const Tensor*>(tensors);
  Hyper h;
  h.b1 = hyper[0]; h.omb1 = hyper[1]; h.b2 = hyper[2]; h.omb2 = hyper[3];
  h.decay = hyper[4]; h.step = hyper[5]; h.inv_root = hyper[6]; h.eps = hyper[7];
  h.key = static_cast<uint32_t>(key);
  h.noisy = key >= 0;
  h.one = 1.f;
  const States st{static_cast<uint8_t*>(m), static_cast<uint8_t*>(m_exp), static_cast<uint8_t*>(r), static_cast<uint8_t*>(r_exp),
                  static_cast<float*>(m), static_cast<float*>(r)};
  for (int at = 0; at < count;) {
    const int e = count - at <= CAP_SMALL ? launch<CAP_SMALL>(rows, at, count, p_bf16, bits == 8, h, st, stream)
                                          : launch<CAP_LARGE>(rows, at, count, p_bf16, bits == 8, h, st, stream);
    if (e) return e;
  }
  return 0;
}
