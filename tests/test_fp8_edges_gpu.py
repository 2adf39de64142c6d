"""8-bit products on the GPU: results of one column or row, very many rows, the precision of the sums."""
import pytest
import torch

from maester_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", [(8, 1), (700, 1), (1, 333), (1, 1), (1, 20480)])
def test_results_of_one_column_or_row(M, N, dtype):
    """The stride of a dimension of one says nothing."""
    a, b = ops.quantize_fp8(torch.randn(M, 300, device="cuda")), ops.quantize_fp8(torch.randn(N, 300, device="cuda"))
    want = ops.matmul_fp8(a, b, out_dtype=dtype)
    if N == 1:
        buf = torch.full((M, 3), 7.0, device="cuda", dtype=dtype)
        out = buf.as_strided((M, 1), (3, 5))
    else:
        buf = torch.full((N,), 7.0, device="cuda", dtype=dtype)
        out = buf.as_strided((1, N), (1, 1))
    assert torch.equal(ops.matmul_fp8(a, b, out=out), want)
    if N == 1:
        assert (buf[:, 1:] == 7).all()
    if dtype == torch.float32:
        assert torch.equal(ops.matmul_fp8(a, b, out=out, accumulate=True), want + want)


def test_more_rows_than_a_grid_dimension_counts():
    n, at = 65535 * 128 + 257, 65534 * 128
    x = torch.randn(n, 4, device="cuda")
    q, part = ops.quantize_fp8(x), ops.quantize_fp8(x[at:])
    assert torch.equal(q.data[at:].view(torch.uint8), part.data.view(torch.uint8))
    assert torch.equal(q.scales[at // 128:], part.scales)
    t, square = ops.quantize_fp8(x, transpose=True), ops.quantize_fp8(x, square=True)
    assert torch.equal(t.data[:, at:].view(torch.uint8), ops.quantize_fp8(x[at:], transpose=True).data.view(torch.uint8))
    assert torch.equal(square.scales[at // 128:], ops.quantize_fp8(x[at:], square=True).scales)
    w = ops.quantize_fp8(torch.randn(8, 4, device="cuda"), square=True)
    assert torch.equal(ops.linear_fp8(x, w)[at:], ops.linear_fp8(x[at:], w))


def _product(kind, x, w):
    """Through the kernel for CTA pairs (many rows), for few rows, or for up to eight tokens."""
    qx, qw = ops.quantize_fp8(x), ops.quantize_fp8(w, square=True)
    y = ops.linear_fp8(x, qw) if kind == "tokens" else ops.matmul_fp8(qx, qw, out_dtype=torch.float32)
    return qx.dequantize(), qw.dequantize(), y


KERNELS = [("pairs", 512, 4608), ("few rows", 24, 4096), ("tokens", 4, 4096)]


@pytest.mark.parametrize("kind,M,N", KERNELS, ids=lambda v: v if isinstance(v, str) else "")
@pytest.mark.parametrize("K,inside,unit", [(128, True, 2.0 ** -4), (9216, True, 2.0 ** -4), (9216, False, 2.0 ** -1)])
def test_sums_keep_24_bits_beside_a_large_one(kind, M, N, K, inside, unit):
    """Large products of one sign, then small ones, then as many large ones of the other sign, inside every block of 128 or block
    by block.  In any order the partial sums are multiples of ``unit`` below 2^24 of them: 32-bit sums are exact, and sums of
    fewer bits lose the small products."""
    at = torch.arange(K)
    if inside:      # (16 neighbouring values of which the first 8 are one instruction's, in either half of a block)
        first, half = at % 16 < 8, at % 128 // 64
        plus, minus, large = first & (half == 0), ~first & (half == 1), 128.0
    else:
        block, n = at // 128, K // 128
        plus, minus, large = block < n // 3, block >= n - n // 3, 16.0
    x, w = torch.full((K,), 1.0), torch.full((K,), unit)
    x[plus | minus] = 128.0
    w[plus], w[minus] = large, -large
    want = (x.double() * w.double()).sum().item()
    assert want == unit * (~(plus | minus)).sum().item() and 128 * large * plus.sum().item() / unit * (128 / K if inside else 1) < 2 ** 24
    a, b, y = _product(kind, x.repeat(M, 1).cuda(), w.repeat(N, 1).cuda())
    assert torch.equal(a[0].cpu(), x) and torch.equal(b[0].cpu(), w)       # (all of them are codes)
    assert (y == want).all()


@pytest.mark.parametrize("kind,M,N", KERNELS, ids=lambda v: v if isinstance(v, str) else "")
def test_sums_of_one_sign(kind, M, N):
    """The matrix unit adds 32 products to a 32-bit sum at a time and cuts off: the sum after each of the K / 32 instructions by
    up to 2^-23 of it, every product by up to 2^-25 of the sum beside it, which is on average half of the last one:
    K / 32 (2^-23 + 32 2^-25) / 2 of the result.  (A sum of 16 bits would be cut by 2^-15 each time, 32 times as much.)"""
    K = 8192
    torch.manual_seed(0)
    a, b, y = _product(kind, torch.rand(M, K, device="cuda") + 0.5, torch.rand(N, K, device="cuda") + 0.5)
    want = a.double() @ b.double().T
    assert ((y - want).abs() <= K / 32 * (2.0 ** -23 + 32 * 2.0 ** -25) / 2 * want).all()


def test_codes_that_start_off_a_boundary_are_refused():
    q = ops.quantize_fp8(torch.randn(40, 200, device="cuda"), square=True)
    for at, ok in ((16, True), (8, False), (1, False)):
        codes = torch.zeros(40 * 256 + at, device="cuda", dtype=torch.uint8)[at:].view(torch.float8_e4m3fn).view(40, 256)
        scales = torch.zeros(q.scales.numel() + at, device="cuda", dtype=torch.uint8)[at:].view(q.scales.shape)
        codes.copy_(q.data)
        scales.copy_(q.scales)
        for args in ((codes, q.scales), (q.data, scales)):
            if ok:
                w = ops.Fp8Blocks(*args, 200)
                x = torch.randn(3, 200, device="cuda")
                assert torch.equal(ops.linear_fp8(x, w), ops.linear_fp8(x, q))
            else:
                with pytest.raises(ValueError, match="16-byte"):
                    ops.Fp8Blocks(*args, 200)
