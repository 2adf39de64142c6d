"""``linear_logprobs`` on the GPU off the native products' path: types other than bf16, widths that 8 does not divide."""
import pytest
import torch

from test_logprobs_plain import check_linear

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


@pytest.mark.parametrize("rows,width,vocab,types", [
    (11, 20, 50, (torch.bfloat16, torch.bfloat16)), (300, 20, 1001, (torch.bfloat16, torch.bfloat16)),
    (300, 64, 1001, (torch.float16, torch.float16)), (300, 64, 515, (torch.float32, torch.float32)),
    (40, 24, 129, (torch.bfloat16, torch.float32)), (40, 24, 129, (torch.float32, torch.bfloat16))], ids=str)
@pytest.mark.parametrize("main_grad", [False, True])
@pytest.mark.parametrize("chunked", [False, True])
def test_against_64_bits(rows, width, vocab, types, main_grad, chunked, monkeypatch):
    from maester_b200.ops import logprobs as L
    if chunked:
        monkeypatch.setattr(L, "_chunks", lambda n, V: [(r, min(n, r + 37)) for r in range(0, n, 37)])
    torch.manual_seed(0)
    check_linear(torch.randn(rows, width, device="cuda").to(types[0]), torch.randn(vocab, width, device="cuda").to(types[1]),
                 main_grad)
