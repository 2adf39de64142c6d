// Log-probabilities of given tokens, row entropies and the best alternatives from a matrix of logits, and the gradient.
//
// With z = scale * x, m = max z, s = sum exp(z - m) and t = sum (z - m) exp(z - m):
//   log p_j = (z_j - m) - log s,    H = log s - t / s   (every term of t has one sign: no cancellation)
//   dx_j = scale * [ g (1[j = token] - p_j) - gH p_j (log p_j + H) + sum_a ga (1[j = alternative a] - p_j) ]
// Statistics are 32-bit whatever the type of the logits.  -inf logits have probability 0 and gradient 0; a row without a
// finite logit, or with NaN or +inf, has no distribution and comes out as NaN.
//
// Forward: one pass over the logits.  A row belongs to one block of 256 threads, or to a cluster of 2, 4 or 8 of them when
// rows are few (their partial results meet in the first block's shared memory).  Every thread keeps its own running (max, sum,
// weighted sum); it takes the maximum of 32 values first, so the sums are rescaled once for 32.
// The alternatives come out of the same pass: a threshold below which no value can be among the best `top` starts as the
// top-th largest of the 256 threads' first maxima, and what reaches it (some `top` values of every 8192 at first) goes into a
// short list of its warp.  A full list is cut down to its best `top`, which raises the threshold for the whole block.  Keys are
// (ordered value, inverted index), all different: equal values come out by the lowest index, whatever the order of the work.
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace {

constexpr long long IGNORE = -100;
constexpr int MAX_TOP = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float FAR = 1000.f;      // exp(-1000) is 0 in fp32: distances are cut there so that a weight of 0 never meets infinity
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int CAP = 128;           // entries of a warp's list
constexpr int MAX_CLUSTER = 8;
typedef unsigned long long u64;

enum { T_BF16 = 0, T_F16 = 1, T_F32 = 2 };

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void from_f(__half* p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void from_f(float* p, float v) { *p = v; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of logits
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  uint32_t w[4];
  __device__ __forceinline__ float at(int i) const { return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16)); }
  // largest value; NaN if there is one
  __device__ __forceinline__ float top() const {
    auto v = [&](int i) { return *reinterpret_cast<const __nv_bfloat162*>(&w[i]); };
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(v(0), v(1)), __hmax2_nan(v(2), v(3)));
    return to_f(__hmax_nan(m.x, m.y));
  }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  uint32_t w[4];
  __device__ __forceinline__ float at(int i) const {
    const __half2 v = *reinterpret_cast<const __half2*>(&w[i >> 1]);
    return to_f((i & 1) ? v.y : v.x);
  }
  __device__ __forceinline__ float top() const {
    auto v = [&](int i) { return *reinterpret_cast<const __half2*>(&w[i]); };
    const __half2 m = __hmax2_nan(__hmax2_nan(v(0), v(1)), __hmax2_nan(v(2), v(3)));
    return to_f(__hmax_nan(m.x, m.y));
  }
};
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
template <>
struct Vec<float> {
  static constexpr int N = 4;
  uint32_t w[4];
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
  __device__ __forceinline__ float top() const { return max_nan(max_nan(at(0), at(1)), max_nan(at(2), at(3))); }
};
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {   // read once: not kept in L1
  Vec<T> v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
      : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]) : "l"(p));
  return v;
}

// Whole number that orders as the value does: -0 with +0, NaN above +inf; never 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ u64 entry_of(float v, uint32_t idx) { return (static_cast<u64>(order_of(v)) << 32) | (0xffffffffu - idx); }
__device__ __forceinline__ long long index_of(u64 e) { return 0xffffffffu - static_cast<uint32_t>(e); }

// Running (maximum m of x, sum s of exp(scale (x - m)), sum t of (x - m) exp(scale (x - m))).
struct Sums {
  float m, s, t;
};
// two parts of a row.  t + s d: with d <= 0 the old terms move by d each.  (A part without a finite value has m = -inf and
// s = t = 0, or NaN, which has to survive.)
__device__ __forceinline__ Sums merge(const Sums& a, const Sums& b, float k, float far) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  if (r.m == -INFINITY) {
    r.s = a.s + b.s;
    r.t = a.t + b.t;
    return r;
  }
  const float da = fmaxf(a.m - r.m, -far), db = fmaxf(b.m - r.m, -far);
  const float ca = ex2(da * k), cb = ex2(db * k);
  r.t = (a.t + a.s * da) * ca + (b.t + b.s * db) * cb;
  r.s = a.s * ca + b.s * cb;
  return r;
}

// Add the values of `v` (largest: cm) to the sums.
template <typename T, int U, bool ENT>
__device__ __forceinline__ void add_values(Sums& a, const Vec<T> (&v)[U], float cm, float k, float far) {
  if (cm > a.m || a.m == -INFINITY) {
    if (cm == -INFINITY) return;               // nothing but -inf so far (NaN goes on: it has to reach the sums)
    if (a.m != -INFINITY && cm == cm) {
      const float d = fmaxf(a.m - cm, -far), c = ex2(d * k);
      a.t = (a.t + a.s * d) * c;
      a.s *= c;
    }
    a.m = cm == cm ? cm : fmaxf(a.m, 0.f);
  }
  const float m = a.m;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) {
      float d = v[u].at(i) - m;
      const float e = ex2(d * k);
      s += e;
      if (ENT) t = fmaf(e, fmaxf(d, -far), t);   // (-inf has weight 0 and must not meet it as 0 * inf)
    }
  }
  a.s += s;
  if (ENT) a.t += t;
}

// ---- lists of candidates
struct Lists {
  u64 entry[WARPS][CAP];
  u64 merged[WARPS * CAP];       // survivors of this block; in the first block of a cluster, the blocks' best
  alignas(16) uint32_t first[THREADS];   // maxima of the threads' first values
  u64 threshold;                 // an entry below it is not among the best
  uint32_t first_min;
  int count[WARPS];
  int survivors;
};

// Cut a warp's full list down to its best `top`, best first; their last entry becomes the threshold.
__device__ __noinline__ void cut_list(Lists& l, int warp, int lane, int top) {
  u64 mine[CAP / 32];
  int rank[CAP / 32];
#pragma unroll
  for (int i = 0; i < CAP / 32; ++i) {
    mine[i] = l.entry[warp][i * 32 + lane];
    rank[i] = 0;
  }
#pragma unroll 4
  for (int j = 0; j < CAP; ++j) {
    const u64 e = l.entry[warp][j];
#pragma unroll
    for (int i = 0; i < CAP / 32; ++i) rank[i] += e > mine[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < CAP / 32; ++i) {
    if (rank[i] < top) l.entry[warp][rank[i]] = mine[i];
    if (rank[i] == top - 1) atomicMax(&l.threshold, mine[i]);
  }
  if (lane == 0) l.count[warp] = top;
  __syncwarp();
}

// Values above the threshold go into the warp's list; value i of vector u has index idx0[u] + i, `valid` says which exist.
// All lanes of the warp call this together.  When the list is full it is cut down and the values that found no room are
// offered again, against the raised threshold.
template <typename T, int U>
__device__ __noinline__ void offer(Lists& l, const Vec<T> (&v)[U], const uint32_t (&idx0)[U], uint32_t valid, int warp, int lane,
                                   int top) {
  constexpr int N = Vec<T>::N;
  uint32_t stored = 0;
  for (;;) {
    const u64 thr = *const_cast<volatile u64*>(&l.threshold);
    uint32_t left = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t bit = 1u << (u * N + i);
        if (!(valid & bit) || (stored & bit)) continue;
        const u64 e = entry_of(v[u].at(i), idx0[u] + i);
        if (e <= thr) continue;
        const int at = atomicAdd(&l.count[warp], 1);
        if (at < CAP) {
          l.entry[warp][at] = e;
          stored |= bit;
        } else {
          left |= bit;
        }
      }
    __syncwarp();
    if (*const_cast<volatile int*>(&l.count[warp]) < CAP) return;   // (a list that is just full is cut as well)
    cut_list(l, warp, lane, top);
    if (!__any_sync(~0u, left)) return;
  }
}

// Best `top` entries of the block, best first, into out (missing ones 0).  All threads call this; a barrier is inside.
__device__ __forceinline__ void block_best(Lists& l, u64* out, int top, int tid) {
  __syncthreads();
  const u64 thr = l.threshold;
  for (int i = tid; i < WARPS * CAP; i += THREADS) {
    const int w = i / CAP, j = i % CAP;
    if (j < l.count[w]) {
      const u64 e = l.entry[w][j];
      if (e >= thr) l.merged[atomicAdd(&l.survivors, 1)] = e;   // (the entry that set the threshold is among the best)
    }
  }
  if (tid < top) out[tid] = 0;
  __syncthreads();
  const int n = l.survivors;
  for (int i = tid; i < n; i += THREADS) {
    const u64 e = l.merged[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += l.merged[j] > e;
    if (rank < top) out[rank] = e;
  }
  __syncthreads();
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_block(const void* p, uint32_t block) {   // the same variable in another block
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(mb::smem_u32(p)), "r"(block));
  return a;
}

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(THREADS, 4)
logprobs_fwd_kernel(const T* __restrict__ x, const long long* __restrict__ tokens, int V, long long ld, float scale, int blocks,
                    float* __restrict__ logprob, float* __restrict__ entropy, int top, float* __restrict__ top_lp,
                    long long* __restrict__ top_id, float4* __restrict__ stats, int* status) {
  constexpr int N = Vec<T>::N, U = 4;
  __shared__ Sums parts[WARPS];
  __shared__ Sums block_parts[MAX_CLUSTER];       // first block: one of each block of the cluster
  __shared__ __align__(16) uint8_t lists_raw[TOP ? sizeof(Lists) : 16];
  __shared__ u64 best[TOP ? MAX_TOP : 1];
  __shared__ u64 block_best_of[TOP ? MAX_CLUSTER * MAX_TOP : 1];
  Lists& l = *reinterpret_cast<Lists*>(lists_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t block = blocks > 1 ? cluster_rank() : 0u;
  const long long row = blockIdx.x / blocks;
  const long long tok = tokens ? tokens[row] : 0;
  if (tok < 0 || tok >= V) {     // (the same for every block of the row)
    if (block == 0) {
      const float v = tok == IGNORE ? 0.f : NAN;
      if (tok != IGNORE && tid == 0) atomicCAS(status, 0, mb::ERR_BAD_ARG);
      if (tid == 0) {
        logprob[row] = v;
        if (entropy) entropy[row] = v;
        if (stats) stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      for (int j = tid; j < top; j += THREADS) {
        top_lp[row * top + j] = -INFINITY;
        top_id[row * top + j] = -1;
      }
    }
    return;
  }
  if (blocks > 1) cluster_arrive();   // (waited for before the first store into another block: it has started by then)
  const T* xr = x + row * ld;
  const float k = scale * LOG2E, far = fminf(FAR / scale, 3e38f);
  // vectors start at the first 16-byte boundary of the row; what lies before it and behind the last one goes one by one
  const int head = min(V, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / sizeof(T)));
  const int vectors = (V - head) / N, per = (vectors + blocks - 1) / blocks;
  const int v0 = min(vectors, static_cast<int>(block) * per), v1 = min(vectors, v0 + per);
  const T* xv = xr + head;
  Sums a{-INFINITY, 0.f, 0.f};
  if (TOP) {
    if (tid < WARPS) l.count[tid] = 0;
    if (tid == 0) {
      l.survivors = 0;
      l.threshold = 0;
      l.first_min = 0xffffffffu;
    }
  }
  // one value of a ragged end for some threads of the first block
  Vec<T> edge[1];
  uint32_t edge_at[1] = {0u};
  bool has_edge = false;
  {
    const int tail0 = head + vectors * N, ends = head + V - tail0;
    if (block == 0 && tid < ends) {
      const int j = tid < head ? tid : tail0 + tid - head;
      const float v = to_f(xr[j]);
      has_edge = true;
      edge_at[0] = j;
      edge[0].w[0] = sizeof(T) == 4 ? __float_as_uint(v) : static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(xr)[j]);
      edge[0].w[1] = edge[0].w[2] = edge[0].w[3] = 0u;
      if (v != -INFINITY) {
        a.m = v == v ? v : 0.f;
        const float e = ex2((v - a.m) * k);
        a.s = e;
        a.t = e * (v - a.m);
      }
    }
  }
  bool first = true;
  for (int i0 = v0; i0 < v1 || (TOP && first); i0 += THREADS * U) {
    Vec<T> v[U];
    uint32_t idx0[U], valid = 0;
    float cm = -INFINITY;
    if (i0 + THREADS * U <= v1) {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load_vec(xv + static_cast<long long>(i0 + u * THREADS + tid) * N);
      valid = (U * N == 32) ? ~0u : (1u << (U * N)) - 1u;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = i0 + u * THREADS + tid;
        if (at < v1) {
          v[u] = load_vec(xv + static_cast<long long>(at) * N);
          valid |= ((1u << N) - 1u) << (u * N);
        } else {   // -inf: no weight
          const uint32_t none = sizeof(T) == 4 ? 0xff800000u : sizeof(T) == 2 && __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
          v[u].w[0] = v[u].w[1] = v[u].w[2] = v[u].w[3] = none;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      idx0[u] = static_cast<uint32_t>(head + (i0 + u * THREADS + tid) * N);
      cm = max_nan(cm, v[u].top());
    }
    if (TOP && first) {
      // the top-th largest of the threads' maxima: at least `top` values reach it
      const float edge_v = has_edge ? edge[0].at(0) : -INFINITY;
      l.first[tid] = valid || has_edge ? order_of(max_nan(cm, edge_v)) : 0u;
      __syncthreads();
      const uint32_t mine = l.first[tid];
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < THREADS; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(&l.first[j]);
        above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      }
      if (above < top) atomicMin(&l.first_min, mine);
      __syncthreads();
      if (tid == 0 && l.first_min) l.threshold = (static_cast<u64>(l.first_min) << 32) - 1;
      __syncthreads();
      first = false;
      if (__any_sync(~0u, has_edge)) offer<T, 1>(l, edge, edge_at, has_edge ? 1u : 0u, warp, lane, top);
    }
    if (TOP) {
      const u64 thr = *const_cast<volatile u64*>(&l.threshold);
      if (__any_sync(~0u, valid && !(cm < value_of(static_cast<uint32_t>(thr >> 32))))) offer<T, U>(l, v, idx0, valid, warp, lane, top);
    }
    add_values<T, U, ENT>(a, v, cm, k, far);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(~0u, a.m, o);
    b.s = __shfl_xor_sync(~0u, a.s, o);
    b.t = __shfl_xor_sync(~0u, a.t, o);
    a = merge(a, b, k, far);
  }
  if (lane == 0) parts[warp] = a;
  if (TOP) block_best(l, best, top, tid);
  else __syncthreads();
  a = parts[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) a = merge(a, parts[w], k, far);
  if (blocks > 1) {
    cluster_wait();
    if (tid == 0) {
      const uint32_t to = in_block(&block_parts[block], 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(a.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(a.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(a.t) : "memory");
    }
    if (TOP && tid < top)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_block(&block_best_of[block * top + tid], 0)), "l"(best[tid]) : "memory");
    cluster_arrive();
    cluster_wait();
    if (block) return;
    a = block_parts[0];
    for (int b = 1; b < blocks; ++b) a = merge(a, block_parts[b], k, far);
    if (TOP) {
      const int n = blocks * top;
      for (int i = tid; i < n; i += THREADS) {
        const u64 e = block_best_of[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += block_best_of[j] > e;
        if (e && rank < top) best[rank] = e;
      }
      __syncthreads();
    }
  }
  const float log_s = logf(a.s);
  if (tid == 0) {
    const float h = log_s - a.t / a.s * scale;
    if (tokens) logprob[row] = (to_f(xr[tok]) - a.m) * scale - log_s;
    if (ENT && entropy) entropy[row] = h;
    if (stats) stats[row] = make_float4(a.m, log_s, h, 0.f);
  }
  if (TOP && tid < top) {
    const long long id = index_of(best[tid]);
    top_id[row * top + tid] = id;
    top_lp[row * top + tid] = (to_f(xr[id]) - a.m) * scale - log_s;
  }
}

// Gradient: reads the logits once more and writes as much.  A block owns `per` vectors of a row (16 bytes of output); where
// rows of x and dx do not share their 16-byte boundaries it goes value by value, neighbours in neighbouring lanes.
struct RowGrad {
  float m, k, log2_s, c0, c1, hot;
  // p * (c0 + c1 log2 p): c1 carries the entropy's part
  template <bool ENT>
  __device__ __forceinline__ float at(float x) const {
    const float l = fmaf(x - m, k, -log2_s), p = ex2(l);
    return ENT ? p * fmaf(fmaxf(l, -1e4f), c1, c0) : p * c0;
  }
};
template <typename G>
struct OutVec {   // 16 bytes of gradients
  static constexpr int N = 16 / sizeof(G);
  G v[N];
};

template <typename T, typename G, bool ENT>
__global__ void __launch_bounds__(THREADS, 4)
logprobs_bwd_kernel(const T* __restrict__ x, const long long* __restrict__ tokens, int V, long long ld, float scale, int blocks,
                    int per, const float4* __restrict__ stats, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                    int top, const long long* __restrict__ top_id, const float* __restrict__ g_top, G* __restrict__ dx,
                    long long ld_dx) {
  constexpr int N = OutVec<G>::N, L = N / Vec<T>::N, U = sizeof(T) == sizeof(G) ? 4 : 2;
  const int tid = threadIdx.x, block = blockIdx.x % blocks;
  const long long row = blockIdx.x / blocks, tok = tokens ? tokens[row] : -1;
  const T* xr = x + row * ld;
  G* dr = dx + row * ld_dx;
  const int head0 = min(V, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(dr) & 15)) & 15) / sizeof(G)));
  const bool vec = !(reinterpret_cast<uintptr_t>(xr + head0) & 15);
  // this block's vectors [v0, v1) from element `head` on, and single elements [e0, e1) and, first block, the ragged ends
  const int head = vec ? head0 : 0, vectors = vec ? (V - head) / N : 0;
  const int v0 = min(vectors, block * per), v1 = min(vectors, v0 + per);
  const int e0 = vec ? 0 : min(static_cast<long long>(V), static_cast<long long>(block) * per * N);
  const int e1 = vec ? 0 : min(static_cast<long long>(V), e0 + static_cast<long long>(per) * N);
  const int tail0 = head + vectors * N, ends = vec && block == 0 ? head + V - tail0 : 0;
  if (tokens && (tok < 0 || tok >= V)) {
    const float v = tok == IGNORE ? 0.f : NAN;
    OutVec<G> o;
#pragma unroll
    for (int i = 0; i < N; ++i) from_f(&o.v[i], v);
    for (int i = v0 + tid; i < v1; i += THREADS)
      *reinterpret_cast<uint4*>(dr + head + static_cast<long long>(i) * N) = *reinterpret_cast<const uint4*>(&o);
    for (int j = e0 + tid; j < e1; j += THREADS) from_f(dr + j, v);
    if (tid < ends) from_f(dr + (tid < head ? tid : tail0 + tid - head), v);
    return;
  }
  const float4 r = stats[row];
  const float gl = g_lp ? g_lp[row] : 0.f, ge = ENT ? g_ent[row] : 0.f;
  float all = gl;
  for (int a = 0; a < top; ++a) all += g_top[row * top + a];
  const RowGrad f{r.x, scale * LOG2E, r.y * LOG2E, -scale * (all + ge * r.z), -scale * ge * LN2, gl * scale};
  auto one = [&](int j) { return f.at<ENT>(to_f(xr[j])) + (j == tok ? f.hot : 0.f); };
  for (int i0 = v0; i0 < v1; i0 += THREADS * U) {
    Vec<T> in[U][L];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i0 + u * THREADS + tid;
      if (at < v1) {
#pragma unroll
        for (int i = 0; i < L; ++i) in[u][i] = load_vec(xr + head + static_cast<long long>(at) * N + i * Vec<T>::N);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i0 + u * THREADS + tid;
      if (at >= v1) break;
      const int j0 = head + at * N;
      float g[N];
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] = f.at<ENT>(in[u][i / Vec<T>::N].at(i % Vec<T>::N));
      if (static_cast<unsigned long long>(tok - j0) < N) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] += tok - j0 == i ? f.hot : 0.f;
      }
      __align__(16) OutVec<G> o;
#pragma unroll
      for (int i = 0; i < N; ++i) from_f(&o.v[i], g[i]);
      *reinterpret_cast<uint4*>(dr + j0) = *reinterpret_cast<const uint4*>(&o);
    }
  }
#pragma unroll 8
  for (int j = e0 + tid; j < e1; j += THREADS) from_f(dr + j, one(j));
  if (tid < ends) {
    const int j = tid < head ? tid : tail0 + tid - head;
    from_f(dr + j, one(j));
  }
  if (top) {   // the alternatives' own terms, over what was just written
    __syncthreads();
    for (int a = tid; a < top; a += THREADS) {
      const int j = static_cast<int>(top_id[row * top + a]);
      const int at = (j - head) / N;
      const bool mine = vec ? (j < head || j >= tail0 ? block == 0 : at >= v0 && at < v1) : j >= e0 && j < e1;
      if (mine) from_f(dr + j, one(j) + g_top[row * top + a] * scale);
    }
  }
}

// Blocks of a row: enough of them for about six waves, so that the last, partial wave costs little; every block keeps at least
// one full turn of its loop (1024 vectors).
int blocks_per_row(int rows, int V, int elem) {
  const long long slots = 4ll * mbh::sm_count(), vectors = static_cast<long long>(V) * elem / 16;
  int b = 1;
  while (b < MAX_CLUSTER && rows * static_cast<long long>(b) < 6 * slots && vectors >= 2048ll * b) b *= 2;
  return b;
}

template <typename T, bool ENT, bool TOP>
int launch_fwd(const void* x, const long long* tokens, int rows, int V, long long ld, float scale, float* logprob,
               float* entropy, int top, float* top_lp, long long* top_id, float4* stats, cudaStream_t stream) {
  int* status = mbh::status().dev;
  if (!status) return -4;
  const int blocks = blocks_per_row(rows, V, sizeof(T));
  if (static_cast<long long>(rows) * blocks > 0x7fffffffll) return -3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * blocks, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, ENT, TOP>, static_cast<const T*>(x), tokens, V, ld, scale, blocks, logprob,
                     entropy, top, top_lp, top_id, stats, status);
  return mbh::check_launch("logprobs_fwd");
}
template <typename T>
int fwd(const void* x, const long long* tokens, int rows, int V, long long ld, float scale, float* logprob, float* entropy,
        int top, float* top_lp, long long* top_id, float4* stats, cudaStream_t stream) {
  const bool ent = entropy || stats;   // (the entropy's gradient needs the entropy)
  if (top)
    return ent ? launch_fwd<T, true, true>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, stats, stream)
               : launch_fwd<T, false, true>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, stats, stream);
  return ent ? launch_fwd<T, true, false>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, stats, stream)
             : launch_fwd<T, false, false>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, stats, stream);
}

}  // namespace

// x: [rows, V] with row pitch ld, type 0 bf16, 1 fp16, 2 fp32; tokens int64 [rows] or null; entropy, stats (float4 [rows] for
// the backward pass) and the alternatives (top > 0: fp32 and int64 [rows, top]) may be null
extern "C" int mb_logprobs_fwd(const void* x, const long long* tokens, int type, int rows, int V, long long ld, float scale,
                               float* logprob, float* entropy, int top, float* top_lp, long long* top_id, void* stats,
                               cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > 0x7fffffff - 65536 || top < 0 || top > MAX_TOP || top > V) return -3;
  float4* f4 = static_cast<float4*>(stats);
  if (type == T_BF16) return fwd<__nv_bfloat16>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, f4, stream);
  if (type == T_F16) return fwd<__half>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, f4, stream);
  if (type == T_F32) return fwd<float>(x, tokens, rows, V, ld, scale, logprob, entropy, top, top_lp, top_id, f4, stream);
  return -3;
}

namespace {

template <typename T, typename G>
int bwd(const void* x, const long long* tokens, int rows, int V, long long ld, float scale, const float4* stats,
        const float* g_lp, const float* g_ent, int top, const long long* top_id, const float* g_top, void* dx, long long ld_dx,
        cudaStream_t stream) {
  constexpr int N = 16 / sizeof(G);
  const int vectors = (V + N - 1) / N;
  // a block takes 4096 vectors (its row's numbers are read once for 64 KiB), fewer where that would leave SMs idle
  int per = 4096;
  while (per > 512 && static_cast<long long>(rows) * ((vectors + per - 1) / per) < 8ll * mbh::sm_count()) per /= 2;
  const int blocks = (vectors + per - 1) / per;
  if (static_cast<long long>(rows) * blocks > 0x7fffffffll) return -3;
  const T* xt = static_cast<const T*>(x);
  G* dt = static_cast<G*>(dx);
  if (g_ent)
    logprobs_bwd_kernel<T, G, true><<<rows * blocks, THREADS, 0, stream>>>(xt, tokens, V, ld, scale, blocks, per, stats, g_lp, g_ent,
                                                                          top, top_id, g_top, dt, ld_dx);
  else
    logprobs_bwd_kernel<T, G, false><<<rows * blocks, THREADS, 0, stream>>>(xt, tokens, V, ld, scale, blocks, per, stats, g_lp,
                                                                           g_ent, top, top_id, g_top, dt, ld_dx);
  return mbh::check_launch("logprobs_bwd");
}

}  // namespace

// out_type: type of dx; equal to `type`, or bf16 beside 32-bit logits (the gradient that a matrix product reads next).
// g_lp, g_ent (fp32 [rows]) and g_top (fp32 [rows, top], with top_id) may be null; g_lp is null where tokens are
extern "C" int mb_logprobs_bwd(const void* x, const long long* tokens, int type, int rows, int V, long long ld, float scale,
                               const void* stats, const float* g_lp, const float* g_ent, int top, const long long* top_id,
                               const float* g_top, void* dx, int out_type, long long ld_dx, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > 0x7fffffff - 65536 || top < 0 || top > MAX_TOP || (g_lp && !tokens)) return -3;
  const float4* f4 = static_cast<const float4*>(stats);
#define ARGS x, tokens, rows, V, ld, scale, f4, g_lp, g_ent, top, top_id, g_top, dx, ld_dx, stream
  if (type == T_BF16 && out_type == T_BF16) return bwd<__nv_bfloat16, __nv_bfloat16>(ARGS);
  if (type == T_F16 && out_type == T_F16) return bwd<__half, __half>(ARGS);
  if (type == T_F32 && out_type == T_F32) return bwd<float, float>(ARGS);
  if (type == T_F32 && out_type == T_BF16) return bwd<float, __nv_bfloat16>(ARGS);
#undef ARGS
  return -3;
}
