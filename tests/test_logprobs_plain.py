"""Token log-probabilities off the kernels' path: rows without a distribution, masks of the lowest value, logits in 32 bits."""
import math

import pytest
import torch

from maester_b200 import ops

LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("fill", [-math.inf, math.nan, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_skipped_rows_have_no_gradient(fill, dtype):
    x = torch.randn(4, 20).to(dtype)
    x[1] = fill
    x[2, 3] = fill
    x.requires_grad_(True)
    tokens = torch.tensor([5, -100, -100, 7])
    out = ops.token_logprobs(x, tokens, entropy=True, top=3)
    assert out.logprobs[1] == 0 and out.entropy[1] == 0 and (out.top_tokens[1:3] == -1).all()
    (out.logprobs.sum() + out.entropy.sum() + out.top_logprobs[[0, 3]].sum()).backward()
    assert not x.grad[1:3].any() and x.grad[[0, 3]].isfinite().all() and x.grad[[0, 3]].any()


@pytest.mark.parametrize("scale", [0.5, 1.0, 2.0, 1e6])
def test_rows_of_the_lowest_value(scale):
    """Equal logits are equally likely, however low they are; a value that stands out of them takes all."""
    x = torch.full((2, 16), LOWEST)
    x[1, 4] = 3.0
    x.requires_grad_(True)
    out = ops.token_logprobs(x, torch.tensor([2, 4]), scale=scale, entropy=True, top=2)
    want = torch.tensor([-math.log(16), 0.0])
    assert torch.allclose(out.logprobs, want, atol=1e-6) and torch.allclose(out.entropy, -want, atol=1e-6)
    assert out.top_tokens.tolist() == [[0, 1], [4, 0]]
    (out.logprobs.sum() + out.entropy.sum()).backward()
    p = torch.zeros(2, 16)
    p[0], p[1, 4] = 1 / 16, 1.0
    want = scale * (torch.nn.functional.one_hot(torch.tensor([2, 4]), 16) - p)
    assert torch.allclose(x.grad, want, atol=2e-6 * scale)


def test_rows_without_a_distribution_are_nan():
    x = torch.zeros(3, 8)
    x[0], x[1, 2], x[2, 5] = -math.inf, math.nan, math.inf
    x.requires_grad_(True)
    out = ops.token_logprobs(x, torch.tensor([0, 2, 5]), entropy=True, top=2)
    assert out.logprobs.isnan().all() and out.entropy.isnan().all() and out.top_logprobs.isnan().all()
    assert out.top_tokens[1, 0] == 2 and out.top_tokens[2, 0] == 5
