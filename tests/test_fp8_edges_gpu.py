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
