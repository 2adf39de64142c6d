"""8-bit linear layers: codes bit for bit against the plain definition, products against 64 bits.

Tolerance of a product of K values with fp32 sums: every addition is off by at most one step (2^-23) of a partial sum that
sum |a||b| bounds, K of them one after the other at the worst; the result is rounded once more (half a step).
"""
import pytest
import torch

from maester_b200 import ops
from maester_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


def _blocks(rows, cols, dtype=torch.bfloat16, spread=1.0):
    """Rows and columns of very different size, some zeros."""
    x = torch.randn(rows, cols, device="cuda") * torch.exp(torch.randn(rows, 1, device="cuda") * spread)
    x = x * torch.exp(torch.randn(1, cols, device="cuda") * spread)
    return torch.where(torch.rand_like(x) < 0.05, torch.zeros_like(x), x).to(dtype)


def _close(got, a, b, base=0.0, dtype=None):
    """got = a @ b.T (+ base) for fp64 a, b"""
    want = a @ b.T + base
    tol = a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().T + abs(base)) + want.abs() * HALF[dtype or got.dtype] * 1.01 + 1e-38
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3g} of the tolerance"


SIZES = [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (128, 128), (129, 257), (64, 1000), (333, 1100), (700, 520), (1, 5000)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("square", [False, True])
def test_codes(rows, cols, dtype, square):
    wide = _blocks(rows, cols + 3, dtype)
    for x in (wide[:, :cols].contiguous(), wide[:, 3:], wide[:, :cols].T.contiguous().T):
        for transpose in (False, True):
            got = ops.quantize_fp8(x, square=square, transpose=transpose)
            codes, exps = ref.fp8_quantize(x.T if transpose else x, square)
            assert got.shape == ((cols, rows) if transpose else (rows, cols))
            assert torch.equal(got.data.view(torch.uint8), codes.view(torch.uint8))
            assert torch.equal(got.exponents(), exps)
            assert torch.equal(got.scales, ref.fp8_pack_exponents(exps))
            # half a step of a code, or of the smallest step of the block
            v, want = got.dequantize().double(), (x.T if transpose else x).double()
            unit = ref.pow2(exps.int() - 127).double().repeat_interleave(128, 1)[:, :want.shape[1]]
            assert ((v - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, unit * 2.0 ** -10)).all()


def test_codes_of_special_values():
    x = torch.zeros(6, 300, device="cuda")
    x[1, 5] = float("nan")
    x[1, 6], x[1, 130] = 3.0, float("inf")
    x[2] = 1e-44                                        # below every scale
    x[3, :128], x[3, 200] = 3.3e38, -3.3e38
    x[4] = torch.exp2(torch.arange(300, device="cuda") / 4 - 30)
    x[5] = 448.0 * 2.0 ** -20                           # exactly at the border of a scale
    x[5, 128] = 448.0 * 2.0 ** -20 * (1 + 2.0 ** -23)   # and just above it
    got = ops.quantize_fp8(x)
    codes, exps = ref.fp8_quantize(x)
    assert torch.equal(got.exponents(), exps) and torch.equal(got.data.view(torch.uint8), codes.view(torch.uint8))
    v = got.dequantize()
    assert v[1, 5].isnan() and v[1, 130].isnan() and v[1, 6] == 3.0 and not v[0].any() and not v[2].any()
    assert (exps[5].int() - 127).tolist() == [-20, -19, -20]


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (4, 256, 512), (7, 1000, 640), (16, 136, 4096), (100, 72, 77),
                                   (128, 256, 128), (129, 257, 129), (256, 512, 1024), (333, 777, 1100), (1000, 520, 2100),
                                   (70, 3000, 384), (2500, 130, 700), (600, 9, 5000), (1, 4097, 8192), (64, 2050, 2560)])
def test_product(M, N, K):
    a, b = ops.quantize_fp8(_blocks(M, K)), ops.quantize_fp8(_blocks(N, K))
    da, db = a.dequantize().double(), b.dequantize().double()
    _close(ops.matmul_fp8(a, b), da, db)
    _close(ops.matmul_fp8(a, b, out_dtype=torch.float32), da, db)
    wide = torch.full((M + 1, N + 5), 7.0, device="cuda")
    assert ops.matmul_fp8(a, b, out=wide[:M, 2:2 + N], accumulate=True) is not None
    _close(wide[:M, 2:2 + N], da, db, 7.0)
    assert (wide[M] == 7).all() and (wide[:, :2] == 7).all() and (wide[:, 2 + N:] == 7).all()
    wide = torch.full((M + 1, N + 3), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.matmul_fp8(a, b, out=wide[:M, 1:1 + N])
    _close(wide[:M, 1:1 + N], da, db)
    assert (wide[M] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 1 + N:] == 7).all()


def test_product_scales_far_apart():
    """Every block of the contraction at another power of two: a scale that is taken for a neighbour's would show."""
    M, N, K = 300, 400, 128 * 13
    unit = torch.exp2(torch.randint(-20, 20, (13,), device="cuda").float()).repeat_interleave(128)
    a = ops.quantize_fp8(torch.randn(M, K, device="cuda") * unit)
    b = ops.quantize_fp8(torch.randn(N, K, device="cuda") / unit * torch.exp2(torch.randint(-9, 9, (N, 1), device="cuda").float()))
    _close(ops.matmul_fp8(a, b, out_dtype=torch.float32), a.dequantize().double(), b.dequantize().double())


def test_nan_stays_in_its_rows():
    x, w = torch.randn(200, 300, device="cuda"), torch.randn(150, 300, device="cuda")
    x[3, 7], w[9, 299] = float("nan"), float("inf")
    y = ops.matmul_fp8(ops.quantize_fp8(x), ops.quantize_fp8(w), out_dtype=torch.float32)
    bad = torch.zeros(200, 150, dtype=torch.bool, device="cuda")
    bad[3], bad[:, 9] = True, True
    assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("lead,K,N", [((1,), 64, 40), ((3,), 300, 128), ((2, 65), 256, 333), ((5, 7, 11), 130, 600), ((1500,), 512, 257)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(lead, K, N, dtype):
    x = _blocks(torch.Size(lead).numel(), K, dtype).view(*lead, K).requires_grad_(True)
    w = _blocks(N, K, dtype).requires_grad_(True)
    y = ops.linear_fp8(x, w)
    dy = _blocks(torch.Size(lead).numel(), N, dtype).view(*lead, N)
    dx, dw = torch.autograd.grad(y, [x, w], dy, retain_graph=True)
    q = lambda t, square=False: ref.fp8_dequantize(*ref.fp8_quantize(t, square))[:, :t.shape[1]].double()
    x2, dy2, wq = x.detach().reshape(-1, K), dy.reshape(-1, N), q(w.detach(), True)
    _close(y.detach().reshape(-1, N), q(x2), wq)
    _close(dx.reshape(-1, K), q(dy2), wq.T)
    _close(dw, q(dy2.T), q(x2.T))
    assert y.dtype == dx.dtype == dtype and dw.dtype == dtype
    # a frozen weight, a frozen input, an accumulation buffer
    w1 = w.detach()
    assert torch.equal(torch.autograd.grad(ops.linear_fp8(x, w1), x, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(ops.linear_fp8(x.detach(), w), w, dy)[0], dw)
    w2 = w.detach().clone().requires_grad_(True)
    w2.main_grad = torch.full((N, K), 2.0, device="cuda")
    ops.linear_fp8(x, w2).backward(dy)
    _close(w2.main_grad, q(dy2.T), q(x2.T), 2.0)
    assert w2.grad is None
    # the weight laid out once
    with torch.no_grad():
        held = ops.linear_fp8(x, ops.quantize_fp8(w, square=True))
        _close(held.reshape(-1, N), q(x2), wq)      # (a few tokens take another path: the same sum in another order)
        assert torch.equal(held, y) or x2.shape[0] <= 8
        assert torch.equal(ops.linear_fp8(x, w), y)
    # gradients of a broadcast output
    s, = torch.autograd.grad(ops.linear_fp8(x, w1).sum(), x)
    _close(s.reshape(-1, K), torch.ones(x2.shape[0], N, device="cuda", dtype=torch.float64), wq.T)


@pytest.mark.parametrize("M", [1, 2, 3, 5, 7, 8])
@pytest.mark.parametrize("K,N", [(1, 1), (16, 33), (127, 64), (128, 31), (130, 257), (640, 1000), (4096, 96), (5000, 40), (1100, 777)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_few_tokens(M, K, N, dtype):
    """Tokens that are quantised on the way, rows off their 16-byte boundaries, scales far apart, columns that are not there."""
    wide = _blocks(M, K + 5, dtype, 2.0)
    w = ops.quantize_fp8(_blocks(N, K, spread=2.0), square=K % 2 == 0)
    for x in (wide[:, :K].contiguous(), wide[:, 5:]):
        y = ops.linear_fp8(x, w)
        a = ref.fp8_dequantize(*ref.fp8_quantize(x))[:, :K].double()
        assert y.dtype == dtype
        _close(y, a, w.dequantize().double())
    x = torch.ones(M, K, device="cuda", dtype=dtype)
    x[M - 1, K - 1] = float("inf")
    y = ops.linear_fp8(x, w)
    assert y[M - 1].isnan().all() and y[:M - 1].isfinite().all()


def test_capture_streams_and_repeats():
    w = ops.quantize_fp8(torch.randn(520, 640, device="cuda", dtype=torch.bfloat16), square=True)
    x = torch.randn(77, 640, device="cuda", dtype=torch.bfloat16)
    want = ops.linear_fp8(x, w)
    for _ in range(3):
        assert torch.equal(ops.linear_fp8(x, w), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.linear_fp8(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    buf = x.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear_fp8(buf, w)
        graphs.append((g, y))
    buf.copy_(x * 3)
    fresh = ops.linear_fp8(buf, w)
    for g, y in graphs + graphs:
        g.replay()
        assert torch.equal(y, fresh)


def test_fp32_sums_keep_their_bits():
    """A long contraction whose sum is small beside its parts: the product keeps fp32 sums (half a step of the largest
    partial sum an addition), not fewer bits."""
    K = 8192
    a = torch.ones(128, K, device="cuda")
    a[:, 1::2] = -1
    b = torch.ones(256, K, device="cuda")
    b[:, 0] = 1 + 1 / 8
    y = ops.matmul_fp8(ops.quantize_fp8(a), ops.quantize_fp8(b), out_dtype=torch.float32)
    assert torch.equal(y, torch.full_like(y, 0.125))
