// Log-probabilities of given tokens, row entropies and the best alternatives from a matrix of logits, and the gradient.
//
// With z = scale * x, m = max z, s = sum exp(z - m) and t = sum (z - m) exp(z - m):
//   log p_j = (z_j - m) - log s,    H = log s - t / s   (every term of t has one sign: no cancellation)
//   dx_j = scale * [ g (1[j = token] - p_j) - gH p_j (log p_j + H) + sum_a ga (1[j = alternative a] - p_j) ]
// Statistics are 32-bit whatever the type of the logits.  -inf logits have probability 0 and gradient 0; a row without a
// finite logit, or with NaN or +inf, has no distribution and comes out as NaN.
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace {

constexpr long long IGNORE = -100;
constexpr int MAX_TOP = 64;
constexpr float LOG2E = 1.4426950408889634f;

enum { T_BF16 = 0, T_F16 = 1, T_F32 = 2 };

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void from_f(__half* p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void from_f(float* p, float v) { *p = v; }

// Whole number that orders as the value does: -0 with +0, NaN above +inf.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// (max, sum, weighted sum) of two parts of a row
__device__ __forceinline__ void merge(float& m, float& s, float& t, float m2, float s2, float t2, float k) {
  const float n = fmaxf(m, m2);
  if (n == -INFINITY) {  // neither part has a finite value: only NaN sums have to survive
    s += s2;
    t += t2;
    return;
  }
  const float d1 = fmaxf((m - n) * k, -1e4f), d2 = fmaxf((m2 - n) * k, -1e4f);
  const float c1 = exp2f(d1), c2 = exp2f(d2);
  t = (t + s * d1) * c1 + (t2 + s2 * d2) * c2;
  s = s * c1 + s2 * c2;
  m = n;
}

template <typename T>
__global__ void __launch_bounds__(512) logprobs_fwd_kernel(const T* __restrict__ x, const long long* __restrict__ tokens,
                                                           int rows, int V, long long ld, float scale,
                                                           float* __restrict__ logprob, float* __restrict__ entropy,
                                                           int top, float* __restrict__ top_lp, long long* __restrict__ top_id,
                                                           float4* __restrict__ stats, int* status) {
  __shared__ float sm[16], ss[16], st[16];
  __shared__ unsigned long long sk[16];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long tok = tokens ? tokens[row] : 0;
  const bool bad = tok < 0 || tok >= V;
  if (bad && tokens) {
    const float v = tok == IGNORE ? 0.f : NAN;
    if (tok != IGNORE && tid == 0) atomicCAS(status, 0, mb::ERR_BAD_ARG);
    if (tid == 0) {
      logprob[row] = v;
      if (entropy) entropy[row] = v;
      if (stats) stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int j = tid; j < top; j += blockDim.x) {
      top_lp[static_cast<long long>(row) * top + j] = -INFINITY;
      top_id[static_cast<long long>(row) * top + j] = -1;
    }
    return;
  }
  const T* xr = x + static_cast<long long>(row) * ld;
  const float k = scale * LOG2E;
  float m = -INFINITY, s = 0.f, t = 0.f;
  for (int j = tid; j < V; j += blockDim.x) {
    const float v = to_f(xr[j]);
    const float n = fmaxf(m, v);
    const float base = n == -INFINITY ? 0.f : n;
    const float d = (v - base) * k, c = n == m || m == -INFINITY ? 0.f : fmaxf((m - n) * k, -1e4f);
    const float e = exp2f(d), f = exp2f(c);
    t = (t + s * c) * f + e * fmaxf(d, -1e4f);
    s = s * f + e;
    m = n;
  }
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(~0u, m, o), s2 = __shfl_xor_sync(~0u, s, o), t2 = __shfl_xor_sync(~0u, t, o);
    merge(m, s, t, m2, s2, t2, k);
  }
  if (lane == 0) { sm[warp] = m; ss[warp] = s; st[warp] = t; }
  __syncthreads();
  m = sm[0]; s = ss[0]; t = st[0];
  for (int w = 1; w < 16; ++w) merge(m, s, t, sm[w], ss[w], st[w], k);
  const float log_s = logf(s);
  if (tid == 0) {
    const float h = log_s - t / s * 0.6931471805599453f;
    if (tokens) logprob[row] = (to_f(xr[tok]) - m) * scale - log_s;
    if (entropy) entropy[row] = h;
    if (stats) stats[row] = make_float4(m, log_s, h, 0.f);
  }
  unsigned long long last = ~0ull;
  for (int a = 0; a < top; ++a) {
    unsigned long long best = 0;
    for (int j = tid; j < V; j += blockDim.x) {
      const unsigned long long key = (static_cast<unsigned long long>(order_of(to_f(xr[j]))) << 32) | (0xffffffffu - j);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o; o >>= 1) {
      const unsigned long long b2 = __shfl_xor_sync(~0u, best, o);
      best = best > b2 ? best : b2;
    }
    __syncthreads();
    if (lane == 0) sk[warp] = best;
    __syncthreads();
    best = sk[0];
    for (int w = 1; w < 16; ++w) best = best > sk[w] ? best : sk[w];
    last = best;
    if (tid == 0) {
      const long long id = 0xffffffffu - static_cast<uint32_t>(best);
      top_id[static_cast<long long>(row) * top + a] = id;
      top_lp[static_cast<long long>(row) * top + a] = (to_f(xr[id]) - m) * scale - log_s;
    }
  }
}

template <typename T, typename G>
__global__ void __launch_bounds__(512) logprobs_bwd_kernel(const T* __restrict__ x, const long long* __restrict__ tokens,
                                                           int rows, int V, long long ld, float scale,
                                                           const float4* __restrict__ stats, const float* __restrict__ g_lp,
                                                           const float* __restrict__ g_ent, int top,
                                                           const long long* __restrict__ top_id,
                                                           const float* __restrict__ g_top, G* __restrict__ dx,
                                                           long long ld_dx) {
  const int row = blockIdx.x, tid = threadIdx.x;
  const long long tok = tokens ? tokens[row] : -1;
  G* dr = dx + static_cast<long long>(row) * ld_dx;
  if (tokens && (tok < 0 || tok >= V)) {
    for (int j = tid; j < V; j += blockDim.x) from_f(dr + j, tok == IGNORE ? 0.f : NAN);
    return;
  }
  const T* xr = x + static_cast<long long>(row) * ld;
  const float4 r = stats[row];
  const float gl = g_lp && tokens ? g_lp[row] : 0.f, ge = g_ent ? g_ent[row] : 0.f;
  float all = gl;
  for (int a = 0; a < top; ++a) all += g_top[static_cast<long long>(row) * top + a];
  auto grad = [&](int j) {
    const float lp = (to_f(xr[j]) - r.x) * scale - r.y;
    const float p = exp2f(lp * LOG2E);
    return -p * (all + ge * (fmaxf(lp, -1e4f) + r.z)) + (j == tok ? gl : 0.f);
  };
  for (int j = tid; j < V; j += blockDim.x) from_f(dr + j, grad(j) * scale);
  __syncthreads();
  for (int a = tid; a < top; a += blockDim.x) {
    const int j = static_cast<int>(top_id[static_cast<long long>(row) * top + a]);
    from_f(dr + j, (grad(j) + g_top[static_cast<long long>(row) * top + a]) * scale);
  }
}

}  // namespace

extern "C" int mb_logprobs_fwd(const void* x, const long long* tokens, int type, int rows, int V, long long ld, float scale,
                               float* logprob, float* entropy, int top, float* top_lp, long long* top_id, void* stats,
                               cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || top < 0 || top > MAX_TOP || top > V || type < 0 || type > 2) return -3;
  int* st = mbh::status().dev;
  if (!st) return -4;
  float4* f4 = static_cast<float4*>(stats);
  if (type == T_BF16)
    logprobs_fwd_kernel<<<rows, 512, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), tokens, rows, V, ld, scale, logprob,
                                                  entropy, top, top_lp, top_id, f4, st);
  else if (type == T_F16)
    logprobs_fwd_kernel<<<rows, 512, 0, stream>>>(static_cast<const __half*>(x), tokens, rows, V, ld, scale, logprob,
                                                  entropy, top, top_lp, top_id, f4, st);
  else
    logprobs_fwd_kernel<<<rows, 512, 0, stream>>>(static_cast<const float*>(x), tokens, rows, V, ld, scale, logprob,
                                                  entropy, top, top_lp, top_id, f4, st);
  return mbh::check_launch("logprobs_fwd");
}

// out_type: type of dx; equal to `type`, or bf16 beside 32-bit logits (the gradient that a matrix product reads next)
extern "C" int mb_logprobs_bwd(const void* x, const long long* tokens, int type, int rows, int V, long long ld, float scale,
                               const void* stats, const float* g_lp, const float* g_ent, int top, const long long* top_id,
                               const float* g_top, void* dx, int out_type, long long ld_dx, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || top < 0 || top > MAX_TOP || type < 0 || type > 2) return -3;
  const float4* f4 = static_cast<const float4*>(stats);
#define LAUNCH(T, G)                                                                                                     \
  logprobs_bwd_kernel<<<rows, 512, 0, stream>>>(static_cast<const T*>(x), tokens, rows, V, ld, scale, f4, g_lp, g_ent, top, \
                                                top_id, g_top, static_cast<G*>(dx), ld_dx)
  if (type == T_BF16 && out_type == T_BF16) LAUNCH(__nv_bfloat16, __nv_bfloat16);
  else if (type == T_F16 && out_type == T_F16) LAUNCH(__half, __half);
  else if (type == T_F32 && out_type == T_F32) LAUNCH(float, float);
  else if (type == T_F32 && out_type == T_BF16) LAUNCH(float, __nv_bfloat16);
  else return -3;
#undef LAUNCH
  return mbh::check_launch("logprobs_bwd");
}
