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


def _exact(h, w, tokens, scale, g):
    z = h.double() @ w.double().T * scale
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    lp, ent = logp.gather(1, tokens[:, None])[:, 0], -(p * logp).sum(1)
    one = torch.nn.functional.one_hot(tokens, w.shape[0])
    dz = scale * (g[0][:, None] * (one - p) - g[1][:, None] * p * (logp + ent[:, None]))
    return lp, ent, logp, dz @ w.double(), dz.T @ h.double()


def check_linear(h, w, main_grad):
    """``linear_logprobs`` of h [R, D] and w [V, D] against 64 bits.  Logits are sums of D products of values of which each is
    exact in 32 bits: off by (D + 2) 2^-24 sum |h||w| and the scale's rounding; a log-probability and an entropy by some of
    those (twice, and the entropy times the spread of the logits), and by 2^-20 for the sums over V."""
    R, D, V, scale = h.shape[0], h.shape[1], w.shape[0], 1.3
    g = torch.randn(2, R, generator=torch.Generator().manual_seed(4)).to(h.device)
    tokens = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(5)).to(h.device)
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    if main_grad:
        w.main_grad = torch.ones(V, D, device=w.device)
    out = ops.linear_logprobs(h, w, tokens, logit_scale=scale, entropy=True, top=3)
    lp, ent, logp, dh, dw = _exact(h.detach(), w.detach(), tokens, scale, g.double())
    off = scale * (D + 4) * 2.0 ** -24 * (h.detach().double().abs() @ w.detach().double().abs().T).max().item()
    spread = (logp.max() - logp.min()).item()
    assert out.logprobs.dtype == torch.float32
    assert (out.logprobs - lp).abs().max() <= 2 * off + 2.0 ** -20 * (1 + spread)
    assert (out.entropy - ent).abs().max() <= 2 * (1 + spread) * off + 2.0 ** -20 * (1 + spread)
    assert (out.top_logprobs - logp.sort(1, descending=True).values[:, :3]).abs().max() <= 2 * off + 2.0 ** -20 * (1 + spread)
    torch.autograd.backward([out.logprobs, out.entropy], [g[0], g[1]])
    got = w.main_grad - 1 if main_grad else w.grad
    assert (w.grad is None) == main_grad and h.grad.dtype == h.dtype
    for a, b, t in ((h.grad, dh, h.dtype), (got, dw, torch.float32 if main_grad else w.dtype)):
        # the gradient's own rounding, and the logits' roundings carried through the softmax (twice `off` relative, with the
        # entropy's term times the spread), over a sum of R or V terms
        bound = torch.finfo(t).eps / 2 * b.abs() + (4 * (1 + spread) * off + 2.0 ** -18) * b.abs().max()
        assert ((a - b).abs() <= bound).all()


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
                                   (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("main_grad", [False, True])
def test_linear_logprobs_hold_32_bit_logits_a_chunk_at_a_time(types, main_grad, monkeypatch):
    from maester_b200.ops import logprobs as L
    from maester_b200.ops import reference as ref
    seen = []
    whole = ref.token_logprobs
    monkeypatch.setattr(ref, "token_logprobs", lambda x, *a: (seen.append((x.dtype, x.shape[0])), whole(x, *a))[1])
    monkeypatch.setattr(L, "_chunks", lambda rows, V: [(r, min(rows, r + 4)) for r in range(0, rows, 4)] or [(0, 0)])
    torch.manual_seed(0)
    check_linear(torch.randn(11, 20).to(types[0]), torch.randn(50, 20).to(types[1]), main_grad)
    assert set(seen) == {(torch.float32, 4), (torch.float32, 3)}


def test_linear_logprobs_of_no_rows_and_64_bits():
    out = ops.linear_logprobs(torch.randn(2, 0, 6), torch.randn(9, 6), entropy=True, top=2)
    assert out.entropy.shape == (2, 0) and out.top_tokens.shape == (2, 0, 2)
    h, w = torch.randn(5, 6, dtype=torch.float64), torch.randn(9, 6, dtype=torch.float64)
    t = torch.tensor([1, 2, -100, 8, 0])
    f = lambda h, w: (lambda o: o.logprobs.sum() + 0.3 * o.entropy.sum() + o.top_logprobs[[0, 1, 3, 4]].sum())(
        ops.linear_logprobs(h, w, t, logit_scale=0.7, entropy=True, top=2))
    assert torch.autograd.gradcheck(f, (h.requires_grad_(True), w.requires_grad_(True)))
    with pytest.raises(TypeError):
        ops.linear_logprobs(torch.ones(2, 6, dtype=torch.int64), torch.ones(9, 6, dtype=torch.int64), entropy=True)
