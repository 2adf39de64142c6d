"""The 8-bit linear layer, the log-probabilities and AdamW over many tensors as one training step and as one sampling step,
on the GPU: eager, captured and replayed, and on two streams at a time."""
import pytest
import torch

from maester_b200 import ops
from maester_b200.optimizers import AdamWMulti

pytestmark = pytest.mark.gpu
D, H, V = 200, 136, 1003


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


def _weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, device="cuda", generator=g) * 0.1).bfloat16()) for s in ((H, D), (V, H))]


def _batch(tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, D, device="cuda", generator=g).bfloat16()
    t = torch.randint(0, V, (tokens,), device="cuda", generator=g)
    t[tokens // 2] = -100       # padding
    return x, t


def _loss(x, t, w1, head):
    h = ops.linear_fp8(x, w1)
    out = ops.token_logprobs(ops.linear_fp8(h, head), t, entropy=True, top=3)
    return -(out.logprobs.sum() + 0.01 * out.entropy.sum()) / t.numel(), out


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_a_training_step(tokens):
    """Gradients are those of the formulas on the values that the codes stand for.  Every operand of a product is off by at
    most 2^-4 of its largest neighbour's share (half a step of e4m3), which the comparison avoids by taking the same codes:
    what is left is fp32 sums of up to 1003 products (2^-14 of their absolute sum is 32 times the worst case of a tree) and
    one bf16 rounding of an output (2^-8)."""
    w1, head = _weights()
    opt = AdamWMulti([w1, head], lr=1e-2)
    deq = lambda m, **kw: ops.quantize_fp8(m, **kw).dequantize().double()
    for step in range(3):
        x, t = _batch(tokens, step)
        h = ops.linear_fp8(x, w1)
        h.retain_grad()
        logits = ops.linear_fp8(h, head)
        logits.retain_grad()
        out = ops.token_logprobs(logits, t, entropy=True, top=3)
        opt.zero_grad()
        (-(out.logprobs.sum() + 0.01 * out.entropy.sum()) / tokens).backward()
        z = logits.detach().double()
        logp = torch.log_softmax(z, 1)
        p, live = logp.exp(), (t != -100).double()[:, None]
        one = torch.nn.functional.one_hot(t.clamp_min(0), V).double()
        ent = -(p * logp).sum(1, keepdim=True)
        dz = -live * (one - p - 0.01 * p * (logp + ent)) / tokens
        assert ((logits.grad.double() - dz).abs() <= 2.0 ** -8 * dz.abs() + 2.0 ** -16 / tokens).all()
        for a, b, got in ((deq(logits.grad), deq(head, square=True, transpose=True), h.grad),
                          (deq(logits.grad, transpose=True), deq(h.detach(), transpose=True), head.grad),
                          (deq(h.grad, transpose=True), deq(x, transpose=True), w1.grad)):
            bound = 2.0 ** -8 * (a @ b.T).abs() + 2.0 ** -14 * (a.abs() @ b.abs().T) + 1e-30
            assert ((got.double() - a @ b.T).abs() <= bound).all()
        before = head.detach().clone()
        opt.step()
        # (without a live token the gradient is 0, and weight decay, 1e-4 of a value, is below half a step of bf16, 2^-9)
        assert torch.equal(before, head) == (not live.any()) and head.isfinite().all() and w1.isfinite().all()


def test_captured_with_its_backward_pass():
    """Two graphs (two sizes) out of one memory pool, replayed in turn with new inputs, give what eager calls give, bit for bit."""
    w = [p.detach().requires_grad_() for p in _weights()]
    sides = []
    pool = torch.cuda.graph_pool_handle()
    for tokens in (300, 24):
        x, t = _batch(tokens, 0)

        def run(x=x, t=t):
            loss, out = _loss(x, t, *w)
            return [loss.detach(), out.logprobs.detach(), out.top_tokens, *torch.autograd.grad(loss, w)]

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            result = run()
        sides.append((g, x, t, result, run))
    for seed in (1, 2):
        for g, x, t, result, run in sides:
            nx, nt = _batch(x.shape[0], seed)
            x.copy_(nx)
            t.copy_(nt)
            g.replay()
            got = [r.clone() for r in result]       # (the other graph's memory is this one's)
            assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_two_streams_at_a_time():
    w = [p.detach() for p in _weights()]
    held = [ops.quantize_fp8(p, square=True) for p in w]
    batches = [_batch(n, n) for n in (1, 8, 9, 700)]

    def run(x, t):
        out = ops.token_logprobs(ops.linear_fp8(ops.linear_fp8(x, held[0]), held[1]), t, entropy=True, top=20)
        return out

    want = [run(*b) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, b in zip(streams, batches):
            with torch.cuda.stream(s):
                got.append(run(*b))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % len(batches)]))


def test_sampling_step_by_step_is_the_whole_prompt():
    """A token alone gets the logits, numbers and alternatives that it gets among others: rows do not depend on the batch in
    values (sums are taken in another order: fp32 sums of up to 200 products, then one bf16 step of the logits)."""
    w = ops.quantize_fp8(torch.randn(V, D, device="cuda").bfloat16() * 0.3, square=True)
    x, t = _batch(500, 3)
    whole = ops.linear_fp8(x, w).double()
    scale = ops.quantize_fp8(x).dequantize().double().abs() @ w.dequantize().double().abs().T
    for i in (0, 250, 499):
        row = ops.linear_fp8(x[i:i + 1], w).double()
        assert ((row - whole[i]).abs() <= 2.0 ** -7 * whole[i].abs() + 2.0 ** -14 * scale[i]).all()
    all_at_once = ops.token_logprobs(whole.bfloat16(), t, top=5)
    one = ops.token_logprobs(whole[7:8].bfloat16(), t[7:8], top=5)
    assert torch.equal(one.top_tokens[0], all_at_once.top_tokens[7])
    assert abs(one.logprobs.item() - all_at_once.logprobs[7].item()) <= 1e-5
