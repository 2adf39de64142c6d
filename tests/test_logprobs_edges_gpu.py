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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V,start,pitch", [(5, 4099, 3, 4111), (3, 40_003, 1, 40_008), (130, 2048, 5, 2056), (2, 9, 7, 16),
                                                (1, 20_000, 2, 20_002), (64, 5001, 4, 5008)])
def test_gradients_of_logits_that_start_anywhere(rows, V, start, pitch, dtype):
    """Rows that share no 16-byte boundary with their gradient go value by value, several blocks to a row: every value against
    64 bits.  A probability's exponent is off by a rounding of z (|z| 2^-24, here |z| < 40) and by the sums' 2^-20, the
    gradient by the same relative to each term, plus its own rounding."""
    g = torch.Generator(device="cuda").manual_seed(rows + V)
    wide = (torch.randn(rows, pitch, device="cuda", generator=g) * 3).to(dtype)
    x = wide[:, start:start + V].requires_grad_(True)
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=g)
    tokens[rows // 2] = V - 1
    top = min(5, V)
    go, ge, gt = (torch.randn(s, device="cuda", generator=g) for s in ((rows,), (rows,), (rows, top)))
    out = ops.token_logprobs(x, tokens, scale=1.2, entropy=True, top=top)
    got, = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], [x], [go, ge, gt])
    z = x.detach().double() * 1.2
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    ent = -(p * logp).sum(1, keepdim=True)
    terms = torch.zeros_like(p).scatter_add_(1, tokens[:, None], go.double()[:, None]).scatter_add_(1, out.top_tokens, gt.double())
    size = terms.abs() + p * (go.double()[:, None].abs() + gt.double().abs().sum(1, keepdim=True)) \
        + ge.double().abs()[:, None] * p * (logp.abs() + ent)
    want = 1.2 * (terms - p * (go.double()[:, None] + gt.double().sum(1, keepdim=True)) - ge.double()[:, None] * p * (logp + ent))
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-38
    assert ((got - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -17 * 1.2 * size + tiny).all()
    assert out.top_tokens[0, 0] == x[0].argmax()
