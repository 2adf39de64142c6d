// Log-probabilities of given tokens, row entropies and the best alternatives from a matrix of logits, and the gradient.
//
// With z = scale * x, m = max z, s = sum exp(z - m) and t = sum (z - m) exp(z - m):
//   log p_j = (z_j - m) - log s,    H = log s - t / s   (every term of t has one sign: no cancellation)
//   dx_j = scale * [ g (1[j = token] - p_j) - gH p_j (log p_j + H) + sum_a ga (1[j = alternative a] - p_j) ]
// Statistics are 32-bit whatever the type of the logits.  -inf logits have probability 0 and the gradient 0, but for the own term
// (g, ga) of the token and of alternatives; a row without a finite logit, or with NaN or +inf, has no distribution and comes out
// as NaN.
//
// Forward: one pass over the logits, bound by reading them.  A row belongs to one block of 256 threads, or to a cluster of 2, 4
// or 8 of them when rows are few (their results meet in the first block's shared memory), or to a block of 128 threads when
// rows are many and short: what a block does after its last vector does not overlap with its own copies, and smaller blocks
// leave more neighbours that go on.  Every thread copies its own next vectors into its own slots of shared memory (cp.async),
// STAGES turns ahead: no thread waits for another's copy, and 128 KiB an SM are on the way while a block puts a row's results
// together (three turns ahead: no faster; five blocks an SM: slower by a twentieth, the registers spill).  Resident blocks that
// take row after row, with copies across the ends of rows, were slower: SMs differ in their distance to memory, and a fixed
// share of the rows leaves the fast ones idle at the end; 176 against 163 us for 4099 x 128256 bf16.
// A thread keeps its own running (max, sum, weighted sum) and takes the maximum of 32 values first, so the sums are rescaled
// once for 32; two fp32 operations an instruction.
//
// Alternatives: 1024 cells (a quarter or an eighth of a thread's turns) keep their maxima.  At least `top` values reach the
// top-th largest of 64 or 128 groups of threads, and hardly more do, so the second look goes to some `top` cells (a thousandth
// of the row each, mostly still in L2).  What reaches that threshold goes into short lists, one a warp; a full list is cut down
// to its best `top`, which raises the threshold for the whole block.  Entries are (ordered value, inverted index), all
// different: equal values come out by the lowest index, whatever the order of the work.  With one maximum a thread the second
// look was four times as long: 240 against 202 us for 4099 x 128256 bf16, 20 alternatives; a threshold found bit by bit and
// lists filled by one vector a warp at a time cost 370 - 243 us of it at 64.
//
// Measured (bf16, copy rate of the same GPU: 6540 GB/s): 4096 x 128256 162 us without entropy (6470 GB/s), 179 with, 194 with 5
// alternatives, 204 with 20, 245 with 64; 8192 x 32000 92, 100, 126, 135, 200; 16 x 262144, where a launch and a row's chain of
// steps count, 10 to 17.  The entropy costs its instructions (two more of some nine for two values), the alternatives the
// steps after the last vector, some 9000 cycles of a row.  Gradient: 330 us for 4096 x 128256 (6370 GB/s).
#include "host_common.cuh"
#include "sm100.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace {

constexpr long long IGNORE = -100;
constexpr int MAX_TOP = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float FAR = 1000.f;      // exp(-1000) is 0 in fp32: distances are cut there so that a weight of 0 never meets infinity
constexpr int THREADS = 256;       // of a block of the backward pass
constexpr int CAP = 96;            // entries of a warp's list: MAX_TOP and one of each lane
constexpr int TURN = 4;            // vectors of a thread's turn
constexpr int STAGES = 2;          // turns in flight
constexpr int ON_SM = 1024;        // threads of an SM (64 registers each)
constexpr int CELLS = 1024;        // of a row part, each with a maximum of its own
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
  static constexpr bool PACKED = true;
  static constexpr float LOWEST = -3.3895314e38f;
  uint32_t w[4];
  static __device__ __forceinline__ uint32_t both(float v) { return mb::pack_bf16(v, v); }
  // neighbours 2 i and 2 i + 1, nothing below `low` (NaN stays)
  __device__ __forceinline__ float2 pair(int i, uint32_t low) const {
    const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), *reinterpret_cast<const __nv_bfloat162*>(&low));
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&v);
    return make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
  }
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
  static constexpr bool PACKED = true;
  static constexpr float LOWEST = -65504.f;
  uint32_t w[4];
  static __device__ __forceinline__ uint32_t both(float v) {
    const __half2 h = __float2half2_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ float2 pair(int i, uint32_t low) const {
    return __half22float2(__hmax2_nan(*reinterpret_cast<const __half2*>(&w[i]), *reinterpret_cast<const __half2*>(&low)));
  }
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
  static constexpr bool PACKED = false;
  static constexpr float LOWEST = 0.f;
  uint32_t w[4];
  static __device__ __forceinline__ uint32_t both(float) { return 0u; }
  __device__ __forceinline__ float2 pair(int i, uint32_t) const { return make_float2(at(2 * i), at(2 * i + 1)); }
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

// two fp32 operations an instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<u64&>(r)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<u64&>(r))
      : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)), "l"(reinterpret_cast<u64&>(c)));
  return r;
}

// Running maximum m of x, sum s of 2^z and sum t of z 2^z with z = k x - base(m), k = scale log2(e).  base(m) is k m as rounded:
// one fused operation gives z, and the difference to k m (at most 2) is taken out of log s at the end.  Where |k m| is 2^26 or
// more, or overflows (rows of the lowest finite value as a mask), z = k (x - m): the base is k m itself.
struct Sums {
  float m, s, t;
};
constexpr float ZFAR = -1500.f;      // 2^-1500 is 0
__device__ __forceinline__ float base(float m, float k) { return __fmul_rn(m, k); }   // (never contracted: it is one number)
__device__ __forceinline__ bool plain(float m, float k) { return fabsf(base(m, k)) < 67108864.f; }
__device__ __forceinline__ float lost(float m, float k) { return plain(m, k) ? fmaf(m, k, -base(m, k)) : 0.f; }
// base(from) - base(to), at least ZFAR; `from` <= `to`, `to` finite or +inf, `from` may be -inf
__device__ __forceinline__ float base_step(float from, float to, float k) {
  const float d = plain(from, k) && plain(to, k) ? __fsub_rn(base(from, k), base(to, k))
                                                 : (from - to) * k + (lost(to, k) - lost(from, k));
  return fmaxf(d, ZFAR);
}
// the sums of `a` on the base of m >= a.m.  (t + s d: every old z moves by d.)
__device__ __forceinline__ void rebase(Sums& a, float m, float k) {
  const float d = base_step(a.m, m, k), c = ex2(d);
  a.t = (a.t + a.s * d) * c;
  a.s *= c;
  a.m = m;
}
// over n = 32 or 8 lanes; a part without a finite value has m = -inf and s = t = 0, or NaN, which has to survive
template <int LANES>
__device__ __forceinline__ Sums merge_lanes(Sums a, float k) {
  float m = a.m;
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (m != -INFINITY) rebase(a, m, k);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, o);
    a.t += __shfl_xor_sync(~0u, a.t, o);
  }
  return a;
}

// Add the values of `v` (largest: cm, NaN if there is one) to the sums.
template <typename T, int U, bool ENT>
__device__ __forceinline__ void add_values(Sums& a, const Vec<T> (&v)[U], float cm, float k, float far) {
  if (!(cm <= a.m) || a.m == -INFINITY) {
    if (cm == -INFINITY) return;               // nothing but -inf so far (NaN goes on: it has to reach the sums)
    const float m = cm == cm ? cm : fmaxf(a.m, 0.f);
    if (a.m == -INFINITY) a.m = m;
    else rebase(a, fmaxf(m, a.m), k);
  }
  // Two values an instruction.  What is so far below the maximum that its weight is 0 is lifted to a finite value first, so
  // that -inf does not meet the weight 0 in the entropy's sum: 16-bit logits in packed form where there is room below m
  const float m = a.m, low = m - fmaxf(far, 0.02f * fabsf(m));
  float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
  const float2 k2 = make_float2(k, k);
  if (plain(m, k) && (!ENT || (Vec<T>::PACKED && low >= Vec<T>::LOWEST))) {
    const uint32_t low2 = Vec<T>::both(low);
    const float2 nb = make_float2(-base(m, k), -base(m, k));
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < Vec<T>::N / 2; ++i) {
        const float2 x = ENT ? v[u].pair(i, low2) : make_float2(v[u].at(2 * i), v[u].at(2 * i + 1));
        const float2 z = fma2(x, k2, nb), e = make_float2(ex2(z.x), ex2(z.y));
        s = add2(s, e);
        if (ENT) t = fma2(e, z, t);
      }
  } else {
    const bool p = plain(m, k);
    const float2 nm = p ? make_float2(0.f, 0.f) : make_float2(-m, -m), nb = p ? make_float2(-base(m, k), -base(m, k)) : make_float2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < Vec<T>::N / 2; ++i) {
        float2 z = fma2(add2(make_float2(v[u].at(2 * i), v[u].at(2 * i + 1)), nm), k2, nb);
        const float2 e = make_float2(ex2(z.x), ex2(z.y));
        s = add2(s, e);
        if (ENT) {
          z.x = fmaxf(z.x, ZFAR);
          z.y = fmaxf(z.y, ZFAR);
          t = fma2(e, z, t);
        }
      }
  }
  a.s += s.x + s.y;
  if (ENT) a.t += t.x + t.y;
}

// ---- lists of candidates (they lie where the copies lay)
template <int TH>
struct Lists {
  static constexpr int WARPS = TH / 32;
  u64 entry[WARPS][CAP];
  u64 merged[WARPS * CAP];   // survivors of this block
  u64 threshold;                 // an entry below it is not among the best
  alignas(16) uint32_t maxima[128];          // of 64 or 128 groups of threads (as ordered whole numbers)
  uint16_t queue[CELLS];   // cells that reach the threshold
  int queued;
  int count[WARPS];
  int survivors;
};

// Cut a warp's list of n entries (n >= top) down to its best `top`, best first; their last one becomes the threshold.
template <int TH>
__device__ __noinline__ void cut_list(Lists<TH>& l, int warp, int lane, int n, int top) {
  static_assert(CAP % 32 == 0 && CAP >= MAX_TOP + 32, "");
  u64 mine[CAP / 32];
  int rank[CAP / 32];
#pragma unroll
  for (int i = 0; i < CAP / 32; ++i) {
    mine[i] = i * 32 + lane < n ? l.entry[warp][i * 32 + lane] : 0;
    rank[i] = 0;
  }
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const u64 e = l.entry[warp][j];
#pragma unroll
    for (int i = 0; i < CAP / 32; ++i) rank[i] += e > mine[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < CAP / 32; ++i) {
    if (mine[i] && rank[i] < top) l.entry[warp][rank[i]] = mine[i];
    if (mine[i] && rank[i] == top - 1) atomicMax(&l.threshold, mine[i]);
  }
  __syncwarp();
}

// The top-th largest of G keys, of which this thread (and GROUP - 1 neighbours that share the work) holds `mine`, becomes the
// threshold: its upper half, as the lowest entry with it.  Every key is compared with every other, G / GROUP comparisons a
// thread; the lower half of a key is its place, so that all differ.
template <int G, int TH>
__device__ __forceinline__ void set_threshold(Lists<TH>& l, uint32_t mine, int tid, int top) {
  constexpr int GROUP = TH / G, PER = G / GROUP;
  const int from = tid % GROUP * PER;
  int rank = 0;
#pragma unroll 4
  for (int i = 0; i < PER; i += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(&l.maxima[from + i]);
    rank += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
  }
#pragma unroll
  for (int o = GROUP / 2; o; o >>= 1) rank += __shfl_xor_sync(~0u, rank, o);
  if (rank == top - 1 && tid % GROUP == 0) l.threshold = static_cast<u64>(mine & 0xffff0000u) << 32;
}

// Entries of at least the threshold go into the warp's list (n entries, returned).  Every lane brings a vector whose first value
// has index j0 (valid: there is one).  The whole warp calls this together.
template <typename T, int TH>
__device__ __forceinline__ int offer(Lists<TH>& l, const Vec<T>& v, bool valid, uint32_t j0, int n, int warp, int lane, int top) {
  u64 thr = *const_cast<volatile u64*>(&l.threshold);
  float least = value_of(static_cast<uint32_t>(thr >> 32));      // (may be NaN: then all are looked at)
  if (!__any_sync(~0u, valid && !(v.top() < least))) return n;
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) {
    if (!__any_sync(~0u, valid && !(v.at(i) < least))) continue;
    const u64 e = valid ? entry_of(v.at(i), j0 + i) : 0;
    uint32_t kept = __ballot_sync(~0u, e >= thr);
    if (n + __popc(kept) > CAP) {
      __syncwarp();
      cut_list(l, warp, lane, n, top);
      n = top;
      thr = *const_cast<volatile u64*>(&l.threshold);
      least = value_of(static_cast<uint32_t>(thr >> 32));
      kept = __ballot_sync(~0u, e >= thr);
    }
    if (kept >> lane & 1) l.entry[warp][n + __popc(kept & ((1u << lane) - 1u))] = e;
    n += __popc(kept);
  }
  return n;
}

// Best `top` of the entries get(0 .. n - 1), of which 0 is none, best first, into out (missing ones 0).  All threads call this
// with l.survivors = 0; barriers are inside, and one at the end.
template <int TH, typename Get>
__device__ __forceinline__ void best_of(Lists<TH>& l, int n, Get get, u64* out, int top, int tid) {
  const int lane = tid & 31;
  for (int i0 = 0; i0 < n; i0 += TH) {
    const u64 e = i0 + tid < n ? get(i0 + tid) : 0;
    const uint32_t kept = __ballot_sync(~0u, e != 0);
    if (!kept) continue;
    int at = 0;
    if (lane == 0) at = atomicAdd(&l.survivors, __popc(kept));
    at = __shfl_sync(~0u, at, 0);
    if (e) l.merged[at + __popc(kept & ((1u << lane) - 1u))] = e;
  }
  if (tid < top) out[tid] = 0;
  __syncthreads();
  const int m = l.survivors;
  // four lanes an entry, each against a quarter of the others
  for (int i0 = tid / 32 * 8; i0 < m; i0 += TH / 4) {
    const int i = i0 + lane / 4;
    const u64 e = i < m ? l.merged[i] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = lane & 3; j < m; j += 4) rank += l.merged[j] > e;
    rank += __shfl_xor_sync(~0u, rank, 1);
    rank += __shfl_xor_sync(~0u, rank, 2);
    if (e && !(lane & 3) && rank < top) out[rank] = e;
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

// The part of a row that a block reads: vectors [v0, v1) counted from the first 16-byte boundary, `head` values into the row.
template <typename T>
struct Part {
  const T* row;
  int head, vectors, v0, v1;
  __device__ __forceinline__ Part(const T* x, int V, int blocks, int block) : row(x) {
    head = min(V, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    vectors = (V - head) / Vec<T>::N;
    const int per = (vectors + blocks - 1) / blocks;
    v0 = min(vectors, block * per);
    v1 = min(vectors, v0 + per);
  }
};

__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mb::smem_u32(to)), "l"(from) : "memory");
}

struct FwdArgs {
  const long long* tokens;
  int rows, V;
  long long ld;
  float scale;
  int blocks;                // of a row
  float *logprob, *entropy;
  int top;
  float* top_lp;
  long long* top_id;
  float4* stats;
  int* status;
};

template <typename T, bool ENT, bool TOP, int TH>
__global__ void __launch_bounds__(TH, ON_SM / TH) logprobs_fwd_kernel(const T* __restrict__ x, const FwdArgs p) {
  constexpr int N = Vec<T>::N, U = TURN, WARPS = TH / 32, PARTS = CELLS / TH;
  __shared__ Sums parts[WARPS];
  __shared__ Sums block_parts[MAX_CLUSTER];          // first block: one of each block of the cluster
  __shared__ u64 block_best_of[TOP ? MAX_CLUSTER * MAX_TOP : 1];
  __shared__ u64 best[TOP ? MAX_TOP : 1];
  extern __shared__ __align__(16) uint8_t dynamic[];
  uint4* slots = reinterpret_cast<uint4*>(dynamic);  // [STAGES][U][TH]
  Lists<TH>& l = *reinterpret_cast<Lists<TH>*>(dynamic);     // ... after the last of them has been read
  static_assert(sizeof(Lists<TH>) <= STAGES * U * TH * 16, "");
  __shared__ uint16_t cells[TOP ? CELLS : 1];   // upper half of (the largest value as an ordered whole number)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.V, blocks = p.blocks, top = p.top;
  const int block = blocks > 1 ? static_cast<int>(cluster_rank()) : 0;
  const long long row = blockIdx.x / blocks;
  const float scale = p.scale, k = scale * LOG2E, far = fminf(FAR / scale, 3e38f);
  const long long tok = p.tokens ? __ldg(p.tokens + row) : 0;
  if (tok < 0 || tok >= V) {     // (the same for every block of the row)
    if (block == 0) {
      const float v = tok == IGNORE ? 0.f : NAN;
      if (tok != IGNORE && tid == 0) atomicCAS(p.status, 0, mb::ERR_BAD_ARG);
      if (tid == 0) {
        p.logprob[row] = v;
        if (p.entropy) p.entropy[row] = v;
        if (p.stats) p.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (TOP && tid < top) {
        p.top_lp[row * top + tid] = -INFINITY;
        p.top_id[row * top + tid] = -1;
      }
    }
    return;
  }
  if (blocks > 1) cluster_arrive();   // (waited for before the first store into another block: it has started by then)
  const Part<T> q(x + row * p.ld, V, blocks, block);
  const T* from = q.row + q.head;
  int copied = q.v0, into = 0;
  auto copy_turn = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = copied + u * TH + tid;
      if (at < q.v1) copy16(&slots[(into * U + u) * TH + tid], from + static_cast<long long>(at) * N);
    }
    copied += TH * U;
    into = into + 1 == STAGES ? 0 : into + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i) copy_turn();

  const float at_token = tid == 0 ? to_f(q.row[tok]) : 0.f;
  Sums a{-INFINITY, 0.f, 0.f};
  // one value of a ragged end for some lanes of the first warp of the first block
  float edge_v = -INFINITY;
  int edge_at = 0;
  bool has_edge = false;
  {
    const int tail0 = q.head + q.vectors * N, ends = q.head + V - tail0;   // (at most 14)
    if (block == 0 && tid < ends) {
      edge_at = tid < q.head ? tid : tail0 + tid - q.head;
      has_edge = true;
      const float v = edge_v = to_f(q.row[edge_at]);
      if (v != -INFINITY) {
        a.m = v == v ? v : 0.f;
        const float z = plain(a.m, k) ? fmaf(v, k, -base(a.m, k)) : (v - a.m) * k, e = ex2(z);
        a.s = e;
        a.t = e * z;
      }
    }
  }
  const int turns = (q.v1 - q.v0 + TH * U - 1) / (TH * U), part = max(1, (turns + PARTS - 1) / PARTS);   // turns of a cell
  float most = edge_v;    // largest value of the cell; NaN if there is one
  uint32_t highest = 0;   // of the thread's cells
  int cell = tid, left = part;
  auto end_cell = [&]() {
    const uint32_t key = order_of(most);
    cells[cell] = static_cast<uint16_t>(key >> 16);
    highest = max(highest, key);
    cell += TH;
    most = -INFINITY;
    left = part;
  };
  int stage = 0;
  for (int i0 = q.v0; i0 < q.v1; i0 += TH * U) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    Vec<T> v[U];
    float cm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 w = slots[(stage * U + u) * TH + tid];
      v[u].w[0] = w.x; v[u].w[1] = w.y; v[u].w[2] = w.z; v[u].w[3] = w.w;
      if (i0 + u * TH + tid >= q.v1) {   // nothing there: -inf, no weight
        const uint32_t none = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
        v[u].w[0] = v[u].w[1] = v[u].w[2] = v[u].w[3] = none;
      }
      cm = max_nan(cm, v[u].top());
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    copy_turn();          // into the slots that were just read
    if (TOP) {
      most = max_nan(most, cm);
      if (--left == 0) end_cell();
    }
    add_values<T, U, ENT>(a, v, cm, k, far);
  }
  a = merge_lanes<32>(a, k);
  if (lane == 0) parts[warp] = a;
  if (TOP) {
    if (left != part || cell == tid) end_cell();
    // 64 groups of threads where `top` is at most half their number, else 128: the fewer, the shorter the search, and only
    // cells that reach the threshold themselves are looked at again
    const int in_group = TH / (top <= 32 ? 64 : 128);
    uint32_t group = highest;
    if (in_group >= 2) group = max(group, __shfl_xor_sync(~0u, group, 1));
    if (in_group >= 4) group = max(group, __shfl_xor_sync(~0u, group, 2));
    __syncthreads();       // (the copies have been read: the lists take their place)
    group = (group & 0xffff0000u) | (TH - tid / in_group);
    if (tid % in_group == 0) l.maxima[tid / in_group] = group;
    if (tid == 0) l.survivors = l.queued = 0;
    __syncthreads();
    if (top <= 32) set_threshold<64>(l, group, tid, top);
    else set_threshold<128>(l, group, tid, top);
    __syncthreads();
    const u64 thr = l.threshold;
    const uint32_t reached = static_cast<uint32_t>(thr >> 32);
    if (__any_sync(~0u, highest >= reached))
      for (int c = tid; c < cell; c += TH) {      // (every thread has as many cells)
        const bool take = cells[c] >= reached >> 16;
        const uint32_t kept = __ballot_sync(~0u, take);
        int at = 0;
        if (lane == 0 && kept) at = atomicAdd(&l.queued, __popc(kept));
        at = __shfl_sync(~0u, at, 0) + __popc(kept & ((1u << lane) - 1u));
        if (take) l.queue[at] = static_cast<uint16_t>(c);
      }
    __syncthreads();
    int listed = 0;
    if (warp == 0) {   // the ragged ends: at most 14 values
      const u64 e = has_edge ? entry_of(edge_v, edge_at) : 0;
      const uint32_t kept = __ballot_sync(~0u, has_edge && e >= thr);
      if (kept >> lane & 1) l.entry[0][__popc(kept & ((1u << lane) - 1u))] = e;
      listed = __popc(kept);
    }
    const int of_cell = part * U, items = l.queued * of_cell;   // vectors (at most the block's and the ends of its cells)
    for (int i0 = lane * WARPS + warp; i0 - lane * WARPS < items; i0 += TH * 2) {   // (neighbours to different warps)
      Vec<T> v[2];
      uint32_t j0[2];
      bool valid[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int item = i0 + u * TH, w = item / of_cell, c = item < items ? l.queue[w] : 0;
        const int at = item < items ? q.v0 + (c / TH * of_cell + item - w * of_cell) * TH + c % TH : q.v1;
        valid[u] = at < q.v1;
        j0[u] = static_cast<uint32_t>(q.head + at * N);
        if (valid[u]) v[u] = load_vec(q.row + j0[u]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) listed = offer<T, TH>(l, v[u], valid[u], j0[u], listed, warp, lane, top);
    }
    if (lane == 0) l.count[warp] = listed;
    __syncthreads();
    const u64 least = l.threshold;       // (the entry that set it is among the best)
    best_of(l, WARPS * CAP, [&](int i) {
      const u64 e = i % CAP < l.count[i / CAP] ? l.entry[i / CAP][i % CAP] : 0;
      return e >= least ? e : 0;
    }, best, top, tid);
  } else {
    __syncthreads();
  }
  if (blocks > 1) {
    cluster_wait();
    if (warp == 0) {
      a = merge_lanes<WARPS>(parts[lane & (WARPS - 1)], k);
      if (lane == 0) {
        const uint32_t to = in_block(&block_parts[block], 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(a.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(a.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(a.t) : "memory");
      }
    }
    if (TOP && tid == 0) l.survivors = 0;
    if (TOP && tid < top)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_block(&block_best_of[block * top + tid], 0)), "l"(best[tid])
                   : "memory");
    cluster_arrive();
    cluster_wait();
    if (block) return;
    if (TOP) {
      // every list holds `share` entries of at least the lowest of their share-th ones: together at least `top`
      const int share = (top + blocks - 1) / blocks;
      u64 least = ~0ull;
      for (int b = 0; b < blocks; ++b) least = min(least, block_best_of[b * top + share - 1]);
      best_of(l, blocks * top, [&](int i) {
        const u64 e = block_best_of[i];
        return e >= least ? e : 0;
      }, best, top, tid);
    }
  }
  if (warp < (TOP ? (top + 31) / 32 : 1)) {
    const int at = lane & (WARPS - 1);
    Sums part{-INFINITY, 0.f, 0.f};
    if (blocks == 1) part = parts[at];
    else if (at < blocks) part = block_parts[at];
    a = merge_lanes<WARPS>(part, k);
    // (log s on the base of m: what k m lost in its rounding is taken out)
    const float log_s = logf(a.s) - lost(a.m, k) * LN2;
    if (tid == 0) {
      const float mean = a.t / a.s, h = logf(a.s) - mean * LN2;     // mean: of z under p
      if (p.tokens) p.logprob[row] = (at_token - a.m) * scale - log_s;
      if (ENT && p.entropy) p.entropy[row] = h;
      if (p.stats) p.stats[row] = make_float4(a.m, 1.f / a.s, mean, 0.f);
    }
    if (TOP && tid < top) {
      const u64 e = best[tid];
      p.top_id[row * top + tid] = index_of(e);
      p.top_lp[row * top + tid] = (value_of(static_cast<uint32_t>(e >> 32)) - a.m) * scale - log_s;
    }
  }
}

// Gradient: reads the logits once more and writes as much.  A block owns `per` vectors of a row (16 bytes of output); where
// rows of x and dx do not share their 16-byte boundaries it goes value by value, neighbours in neighbouring lanes.
// With z and s as above p = 2^z / s and log p + H = (z - mean z) ln 2: neither needs a logarithm.
struct RowGrad {
  float m, k, nb, mean, c0, c1, hot;      // z = k (x - m) + nb, with m = 0 and nb = -base where the base is small enough
  // 2^z (c0 + c1 (z - mean)): both carry -scale / s, c1 the entropy's part
  template <bool ENT>
  __device__ __forceinline__ float at(float x) const {
    const float z = fmaf(x - m, k, nb), e = ex2(z);
    return ENT ? e * fmaf(fmaxf(z, ZFAR) - mean, c1, c0) : e * c0;
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
  const float k = scale * LOG2E, per_s = -scale * r.y;
  const bool p = plain(r.x, k);
  const RowGrad f{p ? 0.f : r.x, k, p ? -base(r.x, k) : 0.f, r.z, per_s * all, per_s * ge * LN2, gl * scale};
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

// Blocks of a row, and whether they are the small ones: the split with the fewest waves times the length of one.  A block costs
// its vectors and about 1500 more (its start, the reductions, the alternatives), a cluster's barrier some 500; small blocks run
// at half the speed, twice as many at a time.  (8192 x 32000 bf16, 5 alternatives: 126 us with small blocks, 160 with large ones;
// 4099 x 128256: 211 and 200; 2048 x 50257: 54 and 62.)
int blocks_per_row(int rows, int V, int elem, bool& small) {
  const long long sms = mbh::sm_count(), slots = ON_SM / 256 * sms, vectors = static_cast<long long>(V) * elem / 16;
  int best = 1;
  long long least = 0;
  for (int b = 1; b <= MAX_CLUSTER; b *= 2) {
    const long long clusters = slots / b, turns = (rows + clusters - 1) / clusters;
    const long long cost = turns * ((vectors + b - 1) / b + 1500 + (b > 1 ? 500 : 0));
    if (b == 1 || cost < least) {
      least = cost;
      best = b;
    }
  }
  const long long of_small = ON_SM / 128 * sms, cost = (rows + of_small - 1) / of_small * (2 * vectors + 1500);
  small = cost < least;
  return small ? 1 : best;
}

template <typename T, bool ENT, bool TOP, int TH>
int launch_fwd(const void* x, const FwdArgs& p, cudaStream_t stream) {
  constexpr int smem = STAGES * TURN * TH * 16;
  MB_SET_MAX_SMEM_ONCE((logprobs_fwd_kernel<T, ENT, TOP, TH>), smem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * p.blocks, 1, 1);
  cfg.blockDim = dim3(TH, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.blocks > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, ENT, TOP, TH>, static_cast<const T*>(x), p);
  return mbh::check_launch("logprobs_fwd");
}
template <typename T, int TH>
int fwd(const void* x, const FwdArgs& p, cudaStream_t stream) {
  const bool ent = p.entropy || p.stats;   // (the entropy's gradient needs the entropy)
  if (p.top) return ent ? launch_fwd<T, true, true, TH>(x, p, stream) : launch_fwd<T, false, true, TH>(x, p, stream);
  return ent ? launch_fwd<T, true, false, TH>(x, p, stream) : launch_fwd<T, false, false, TH>(x, p, stream);
}
template <typename T>
int fwd(const void* x, FwdArgs& p, cudaStream_t stream) {
  bool small;
  p.blocks = blocks_per_row(p.rows, p.V, sizeof(T), small);
  if (static_cast<long long>(p.rows) * p.blocks > 0x7fffffffll) p.blocks = 1;
  return small ? fwd<T, 128>(x, p, stream) : fwd<T, 256>(x, p, stream);
}

}  // namespace

// x: [rows, V] with row pitch ld, type 0 bf16, 1 fp16, 2 fp32; tokens int64 [rows] or null; entropy, stats (float4 [rows] for
// the backward pass) and the alternatives (top > 0: fp32 and int64 [rows, top]) may be null
extern "C" int mb_logprobs_fwd(const void* x, const long long* tokens, int type, int rows, int V, long long ld, float scale,
                               float* logprob, float* entropy, int top, float* top_lp, long long* top_id, void* stats,
                               cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > 0x7fffffff - 65536 || top < 0 || top > MAX_TOP || top > V) return -3;
  if (type < T_BF16 || type > T_F32) return -3;
  int* status = mbh::status().dev;
  if (!status) return -4;
  FwdArgs p{tokens, rows, V, ld, scale, 1, logprob, entropy, top, top_lp, top_id,
                  static_cast<float4*>(stats), status};
  return type == T_BF16 ? fwd<__nv_bfloat16>(x, p, stream) : type == T_F16 ? fwd<__half>(x, p, stream) : fwd<float>(x, p, stream);
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
