// A linear layer in 8 bits, forward and backward: the quantisation passes and products of one direction behind one call.
//
// A layer of a few hundred tokens spends its time in calls, not in kernels: one call for three launches takes some 15 us of
// the host's time in the forward pass, three calls took 27.
//
// A packed matrix is its codes [rows, 128 blocks] with its exponent bytes behind them.
#include "fp8_common.cuh"
#include "host_common.cuh"

extern "C" int mb_fp8_quantize(const void* x, int type, int rows, int cols, long long ld, int mode, void* q, void* sq, void* qt,
                               void* sqt, cudaStream_t stream);
extern "C" int mb_fp8_gemm(const void* a, const void* sa, const void* b, const void* sb, void* c, int M, int N, int kblocks,
                           long long lda, long long ldb, long long ldc, int out, cudaStream_t stream);

namespace {

constexpr int ROWS = 1, COLS = 2, SQUARE = 4;   // modes of mb_fp8_quantize

struct Packed {
  uint8_t* codes = nullptr;
  int rows = 0, blocks = 0;
  Packed(void* at, int rows_, int values) : codes(static_cast<uint8_t*>(at)), rows(rows_), blocks((values + 127) / 128) {}
  long long pitch() const { return blocks * 128ll; }
  uint8_t* scales() const { return codes ? codes + rows * pitch() : nullptr; }
  uint8_t* end() const { return scales() + (rows + 127) / 128 * ((blocks + 3) / 4) * 512ll; }
};

int quantize(const void* x, int type, int rows, int cols, long long ld, int square, const Packed& q, const Packed& qt,
             cudaStream_t stream) {
  const int mode = (q.codes ? ROWS : 0) | (qt.codes ? COLS : 0) | square;
  return mode & (ROWS | COLS) ? mb_fp8_quantize(x, type, rows, cols, ld, mode, q.codes, q.scales(), qt.codes, qt.scales(), stream) : 0;
}
int product(const Packed& a, const Packed& b, void* c, long long ldc, int out, cudaStream_t stream) {
  return mb_fp8_gemm(a.codes, a.scales(), b.codes, b.scales(), c, a.rows, b.rows, a.blocks, a.pitch(), b.pitch(), ldc, out, stream);
}

}  // namespace

// y [M, N] = Q(x) Q(w)^T for x [M, K] and w [N, K] (type 0 bf16, 2 fp32; y has x's).  x_t, w_t (either may be null): packed
// codes of the transposes, for the backward pass.  work: a packed [M, K] and a packed [N, K].
extern "C" int mb_fp8_linear_fwd(const void* x, int x_type, long long ldx, const void* w, int w_type, long long ldw, int M, int K,
                                 int N, void* work, void* x_t, void* w_t, void* y, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0) return -3;
  const Packed xq(work, M, K), wq(xq.end(), N, K);
  int e = quantize(x, x_type, M, K, ldx, 0, xq, Packed(x_t, K, M), stream);
  if (!e) e = quantize(w, w_type, N, K, ldw, SQUARE, wq, Packed(w_t, K, N), stream);
  return e ? e : product(xq, wq, y, N, x_type == 0 ? 0 : 1, stream);
}

// From dy [M, N]: dx [M, K] of its type (w_t given) and dw [N, K] with row pitch ld_dw (x_t given; out 0 bf16, 1 fp32,
// 2 fp32 +=).  work: a packed [M, N] where there is a dx, then a packed [N, M] where there is a dw.
extern "C" int mb_fp8_linear_bwd(const void* dy, int type, long long ld, int M, int K, int N, void* work, void* w_t, void* x_t,
                                 void* dx, void* dw, long long ld_dw, int out, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0) return -3;
  const Packed dyq(w_t ? work : nullptr, M, N), dyt(!x_t ? nullptr : w_t ? dyq.end() : work, N, M);
  int e = quantize(dy, type, M, N, ld, 0, dyq, dyt, stream);
  if (!e && w_t) e = product(dyq, Packed(w_t, K, N), dx, K, type == 0 ? 0 : 1, stream);
  if (!e && x_t) e = product(dyt, Packed(x_t, K, M), dw, ld_dw, out, stream);
  return e;
}
