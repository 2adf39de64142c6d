"""Token log-probabilities on the GPU: very many rows, gradients of logits that start anywhere."""
import pytest
import torch

from maester_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


def test_more_rows_than_an_eighth_of_a_grid():
    n, at = (1 << 28) + 133, (1 << 28) - 1000
    x = torch.randn(n, 4, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    tokens = torch.randint(0, 4, (n,), device="cuda", dtype=torch.int32)
    out = ops.token_logprobs(x, tokens)
    part = x.detach()[at:].clone().requires_grad_(True)
    want = ops.token_logprobs(part, tokens[at:])
    assert torch.equal(out.logprobs[at:], want.logprobs)
    out.logprobs.backward(torch.ones_like(out.logprobs))
    want.logprobs.backward(torch.ones_like(want.logprobs))
    assert torch.equal(x.grad[at:], part.grad)
