"""Token log-probabilities, 8-bit linear layers and AdamW over many tensors on the CPU: definitions, refusals, checkpoints."""
import copy
import math

import pytest
import torch

from maester_b200 import ops
from maester_b200.ops import reference as ref
from maester_b200.optimizers import AdamWMulti, FusedAdamW


# ---------------------------------------------------------------- log-probabilities
def test_logprobs_definition():
    x = torch.randn(6, 50, dtype=torch.float64) * 3
    x[2, :20] = -math.inf
    tokens = torch.tensor([0, 3, 30, -100, 49, 7])
    got = ops.token_logprobs(x, tokens, scale=0.8, entropy=True, top=4)
    logp = torch.log_softmax(x * 0.8, 1)
    for r, t in enumerate(tokens.tolist()):
        if t == -100:
            assert got.logprobs[r] == 0 and got.entropy[r] == 0 and (got.top_tokens[r] == -1).all()
            continue
        p = logp[r].exp()
        assert abs(got.logprobs[r] - logp[r, t]) < 1e-12
        assert abs(got.entropy[r] + sum(a * math.log(a) for a in p.tolist() if a > 0)) < 1e-12
        assert got.top_tokens[r].tolist() == sorted(range(50), key=lambda j: (-x[r, j].item(), j))[:4]
        assert torch.allclose(got.top_logprobs[r], logp[r, got.top_tokens[r]])
    x.requires_grad_(True)
    f = lambda v: (lambda o: o.logprobs.sum() + 0.3 * o.entropy.sum())(ops.token_logprobs(v[3:], tokens[3:], entropy=True))
    assert torch.autograd.gradcheck(f, (x,))


def test_logprobs_ties_take_the_lowest_id():
    x = torch.tensor([[1.0, 2.0, 2.0, -0.0, 0.0, 2.0]])
    assert ops.token_logprobs(x, top=5).top_tokens.tolist() == [[1, 2, 5, 0, 3]]


def test_linear_logprobs_is_the_composition():
    h, w = torch.randn(4, 3, 16), torch.randn(21, 16)
    tokens = torch.randint(0, 21, (4, 3))
    a = ops.linear_logprobs(h, w, tokens, logit_scale=1.3, entropy=True, top=2)
    b = ops.token_logprobs(h @ w.T, tokens, scale=1.3, entropy=True, top=2)
    assert a.top_tokens.shape == (4, 3, 2) and all(torch.allclose(i, j, atol=1e-6) for i, j in zip(a[:3], b[:3]))
    loss = ref.linear_cross_entropy(h.view(-1, 16), w, tokens.view(-1), 1.3)
    assert abs(loss + a.logprobs.mean()) < 1e-5


@pytest.mark.parametrize("kw,error", [
    (dict(tokens=torch.zeros(3, dtype=torch.int64)), ValueError), (dict(tokens=torch.zeros(4)), TypeError),
    (dict(), ValueError), (dict(entropy=True, scale=0.0), ValueError), (dict(entropy=True, scale=-1.0), ValueError),
    (dict(entropy=True, scale=math.nan), ValueError), (dict(top=9), ValueError), (dict(top=-1), ValueError),
    (dict(top=1.5), ValueError), (dict(tokens=torch.tensor([0, 1, 8, 2])), ValueError),
    (dict(tokens=torch.tensor([0, 1, -1, 2])), ValueError)])
def test_logprobs_refusals(kw, error):
    with pytest.raises(error):
        ops.token_logprobs(torch.randn(4, 8), **kw)
    with pytest.raises(error):
        kw = {("logit_scale" if k == "scale" else k): v for k, v in kw.items()}
        ops.linear_logprobs(torch.randn(4, 6), torch.randn(8, 6), **kw)


def test_sizes_that_no_kernel_counts():
    from maester_b200.ops import cuda as C
    C._fit(5, 2 ** 31 - 2 ** 16 - 1)
    with pytest.raises(ValueError, match="below"):
        C._fit(5, 2 ** 31)


@pytest.mark.parametrize("scale", [1e-9, 1e9, math.inf, 10 ** 400, "1", None])
def test_logprobs_refuse_a_scale_that_fp32_cannot_carry(scale):
    with pytest.raises(ValueError, match="scale"):
        ops.token_logprobs(torch.randn(2, 8), entropy=True, scale=scale)


def test_logprobs_refuse_more_alternatives_than_the_limit():
    with pytest.raises(ValueError, match="64"):
        ops.token_logprobs(torch.randn(2, 100), top=65)
    with pytest.raises(TypeError):
        ops.token_logprobs(torch.zeros(2, 100, dtype=torch.int64), entropy=True)
    with pytest.raises(ValueError, match="empty"):
        ops.token_logprobs(torch.randn(2, 0), entropy=True)
    with pytest.raises(ValueError, match="fit"):
        ops.linear_logprobs(torch.randn(4, 6), torch.randn(8, 5), entropy=True)


# ---------------------------------------------------------------- 8-bit blocks
def test_every_code_is_a_fixed_point():
    """Quantising what was dequantised gives the same values.  (A maximum in (224, 232) * 2^k rounds to 224 * 2^k, which is
    448 * 2^(k - 1): the second time the block's scale is half as large, and every code's value is one of its codes too.)"""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[codes.isfinite()]
    x = torch.cat([codes, codes]).view(2, 254) * torch.tensor([[2.0 ** -30], [2.0 ** 9]])
    q = ops.quantize_fp8(x)
    assert torch.equal(q.dequantize(), x)
    y = torch.randn(300, 513) * torch.exp(torch.randn(300, 1) * 3)
    for square in (False, True):
        a = ops.quantize_fp8(y, square=square)
        b = ops.quantize_fp8(a.dequantize(), square=square)
        assert torch.equal(a.dequantize(), b.dequantize())


def test_rounding_is_to_the_nearest_code():
    x = torch.randn(40, 1000)
    q = ops.quantize_fp8(x)
    unit = torch.exp2(q.exponents().double() - 127).repeat_interleave(128, 1)[:, :1000]
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[codes.isfinite()].unique()
    y = (x.double() / unit).reshape(-1)
    at = torch.searchsorted(codes, y).clamp(1, len(codes) - 1)
    best = torch.minimum((codes[at] - y).abs(), (codes[at - 1] - y).abs())
    assert torch.equal((q.dequantize().double() / unit).reshape(-1).sub(y).abs(), best)
    assert q.dequantize().abs().amax() <= 448 * unit.max()


def test_a_square_scale_is_shared_with_the_transpose():
    w = torch.randn(200, 300) * torch.exp(torch.randn(200, 1))
    a, b = ops.quantize_fp8(w, square=True), ops.quantize_fp8(w, square=True, transpose=True)
    assert torch.equal(a.dequantize(), b.dequantize().T)


def test_linear_fp8_cpu_gradients():
    x, w = torch.randn(9, 150, requires_grad=True), torch.randn(33, 150, requires_grad=True)
    dy = torch.randn(9, 33)
    y = ops.linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    q = lambda t, s=False: ops.quantize_fp8(t, square=s).dequantize()
    assert torch.allclose(y, q(x) @ q(w, True).T, rtol=1e-5, atol=1e-4)
    assert torch.allclose(dx, q(dy) @ q(w, True), rtol=1e-5, atol=1e-4)
    assert torch.allclose(dw, q(dy.T) @ q(x.T).T, rtol=1e-5, atol=1e-4)
    # within the roundings of both operands (2^-4 each at the most) of the unrounded product's gradient
    assert (dx - dy @ w).norm() < 0.125 * (dy.abs() @ w.abs()).norm()
    w.main_grad = torch.ones(33, 150)
    ops.linear_fp8(x, w).backward(dy)
    assert w.grad is None and torch.allclose(w.main_grad, 1 + dw, rtol=1e-5, atol=1e-4)
    assert ops.linear_fp8(x[:0], w).shape == (0, 33)
    with torch.no_grad():
        assert torch.equal(ops.linear_fp8(x, ops.quantize_fp8(w, square=True)), y)


def test_fp8_refusals():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    h = ops.quantize_fp8(w, square=True)
    for bad, error in ((lambda: ops.linear_fp8(x[:, :63], w), ValueError), (lambda: ops.linear_fp8(x.half(), w), TypeError),
                       (lambda: ops.linear_fp8(x, w.double()), TypeError), (lambda: ops.linear_fp8(x, w[0]), TypeError),
                       (lambda: ops.linear_fp8(x.requires_grad_(True), h), RuntimeError),
                       (lambda: ops.quantize_fp8(w[0]), ValueError), (lambda: ops.quantize_fp8(w[:0]), ValueError),
                       (lambda: ops.quantize_fp8(w.long()), TypeError),
                       (lambda: ops.matmul_fp8(h, ops.quantize_fp8(torch.randn(3, 65))), ValueError),
                       (lambda: ops.matmul_fp8(h, h, accumulate=True), ValueError),
                       (lambda: ops.matmul_fp8(h, h, out_dtype=torch.float16), TypeError),
                       (lambda: ops.matmul_fp8(h, h, out=torch.zeros(8, 8, dtype=torch.bfloat16), accumulate=True), TypeError),
                       (lambda: ops.matmul_fp8(h, h, out=torch.zeros(8, 9)), ValueError),
                       (lambda: ops.matmul_fp8(h, h, out=torch.zeros(8, 16)[:, ::2]), ValueError),
                       (lambda: ops.matmul_fp8(h, h, out=torch.zeros(1, 8).expand(8, 8)), ValueError),
                       (lambda: ops.Fp8Blocks(h.data, h.scales, 129), ValueError),
                       (lambda: ops.Fp8Blocks(h.data[:, :64], h.scales, 64), TypeError),
                       (lambda: ops.Fp8Blocks(h.data, h.scales[:, :, :16], 64), ValueError),
                       (lambda: ops.Fp8Blocks(h.data.float(), h.scales, 64), TypeError)):
        with pytest.raises(error):
            bad()


# ---------------------------------------------------------------- AdamW over many tensors
def _model(dtype=torch.float32):
    torch.manual_seed(1)
    return [torch.nn.Parameter((torch.randn(s) * 0.1).to(dtype)) for s in ((30, 20), (7,), (300,), (2, 3, 50), (1,))]


def _grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=g) * 0.1).to(p.dtype)


def test_32_bit_states_follow_torch_adamw():
    a, b = _model(), _model()
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    oa, ob = AdamWMulti(a, state_bits=32, **kw), torch.optim.AdamW(b, **kw)
    for s in range(5):
        _grads(a, s)
        _grads(b, s)
        oa.step()
        ob.step()
        for p, q in zip(a, b):   # some ten fp32 roundings of a step of size lr, five steps
            assert torch.allclose(p, q, rtol=0, atol=5 * (16 * 2.0 ** -24 * (1e-2 + p.abs().max().item())))


def test_step_numbers_that_differ():
    """Parameters that missed steps count their own: each is updated once by a step, whatever number it is at."""
    a, b = _model(), _model()
    oa, ob = AdamWMulti(a, state_bits=32, lr=1e-2), torch.optim.AdamW(b, lr=1e-2)
    for s in range(5):
        _grads(a, s)
        _grads(b, s)
        for i in range(s, len(a)):   # after step s parameters 0 .. s - 1 have been updated
            a[i].grad = b[i].grad = None
        oa.step()
        ob.step()
        assert [x.step for x in oa._slots.values()] == [max(0, s - i) for i in range(len(a))]
        for p, q in zip(a, b):
            assert torch.allclose(p, q, rtol=0, atol=5 * (16 * 2.0 ** -24 * (1e-2 + p.abs().max().item())))


def test_8_bit_states_stay_near_32_bit_ones():
    """A code is off by at most 2^-4 of its value (or half the smallest step of its block) before each update; an element's
    update therefore stays within a fraction of the learning rate of the exact one."""
    a, b = _model(), _model()
    oa, ob = AdamWMulti(a, lr=1e-3, betas=(0.9, 0.95), weight_decay=0.0), AdamWMulti(b, lr=1e-3, betas=(0.9, 0.95),
                                                                                     weight_decay=0.0, state_bits=32)
    for s in range(20):
        _grads(a, s)
        _grads(b, s)
        oa.step()
        ob.step()
    for p, q in zip(a, b):
        assert (p - q).abs().max() < 20 * 1e-3 * 0.5 and (p - q).norm() < 0.2 * 20 * 1e-3 * math.sqrt(p.numel())


def test_a_root_never_becomes_zero():
    x = torch.zeros(512)
    x[0], x[1], x[300] = 1.0, 1e-12, 1e-30
    codes, exps = ref.state_encode(x, root=True)
    v = ref.state_decode(codes, exps)
    assert (v > 0).tolist() == (x > 0).tolist() and v[0] == 1.0
    p = torch.nn.Parameter(torch.zeros(256))
    opt = AdamWMulti([p], lr=1.0, weight_decay=0.0)
    p.grad = torch.full((256,), 1e-12)
    p.grad[0] = 1e6                       # far above what the block can hold beside the others
    for _ in range(4):
        opt.step()
        p.grad[1:] = 0.0
    assert p.detach()[1:].abs().max() <= 4.0   # each update is at most about lr


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict_holds_plain_moments_and_changes_nothing(bits):
    a = _model()
    opt = AdamWMulti(a, lr=1e-2, state_bits=bits)
    for s in range(3):
        _grads(a, s)
        opt.step()
    sd = opt.state_dict()
    assert set(sd["state"][0]) == {"step", "exp_avg", "exp_avg_sq"} and sd["state"][3]["exp_avg"].shape == (2, 3, 50)
    assert sd["state"][0]["step"].item() == 3 and sd["state"][0]["exp_avg"].dtype == torch.float32
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    two = AdamWMulti(b, lr=5.0, state_bits=bits)
    two.load_state_dict(sd)
    assert two.param_groups[0]["lr"] == 1e-2
    for p, q in zip(a, b):   # the same values (a block's scale may be half as large, see above)
        assert all(torch.equal(x, y) for x, y in zip(opt._moments(p), two._moments(q)))
    _grads(a, 7)
    _grads(b, 7)
    opt.step()
    two.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # a plain AdamW takes the same file
    three = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in a], lr=1e-2)
    groups = three.state_dict()["param_groups"]
    three.load_state_dict({"state": sd["state"], "param_groups": groups})
    assert torch.equal(three.state[three.param_groups[0]["params"][0]]["exp_avg"], sd["state"][0]["exp_avg"])


def test_checkpoint_through_the_container(tmp_path):
    import torch.distributed.checkpoint as dcp
    from maester_b200.checkpoint import OptimizerWrapper
    from maester_b200.config import Config
    from maester_b200.optimizers import build_optimizers

    def make(cls, **extra):
        torch.manual_seed(0)
        m = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 5))
        cfg = Config(optimizer_groups=[{"opt_class": f"maester_b200.optimizers.{cls}", "min_dim": 0,
                                        "opt_cfg": {"lr": 1e-2, "betas": [0.9, 0.95], **extra}}])
        return m, build_optimizers(m, cfg)

    m, opt = make("AdamWMulti", state_bits=8)
    for _ in range(2):
        opt.zero_grad()
        m(torch.randn(4, 20)).square().sum().backward()
        opt.step()
    dcp.save({"optimizer": OptimizerWrapper(m, opt)}, checkpoint_id=str(tmp_path / "c"), no_dist=True)
    m2, opt2 = make("AdamWMulti", state_bits=8)
    dcp.load({"optimizer": OptimizerWrapper(m2, opt2)}, checkpoint_id=str(tmp_path / "c"), no_dist=True)
    a, b = opt.optimizers[0], opt2.optimizers[0]
    for p, q in zip(m.parameters(), m2.parameters()):
        assert all(torch.equal(x, y) for x, y in zip(a._moments(p), b._moments(q))) and a._moments(p)[1].any()
    assert [s.step for s in b._slots.values()] == [2] * 4
    # the files of a 32-bit run have the same keys
    m3, opt3 = make("FusedAdamW")
    m3(torch.randn(4, 20)).square().sum().backward()
    opt3.step()
    assert {k for k in opt3.state_dict() if k.startswith("state.")} == {k for k in opt.state_dict() if k.startswith("state.")}
    assert isinstance(opt3.optimizers[0], FusedAdamW)


def test_adamw_multi_refusals():
    p = torch.nn.Parameter(torch.randn(4, 4))
    for bad, error in ((lambda: AdamWMulti([p], state_bits=4), ValueError), (lambda: AdamWMulti([p], lr=-1.0), ValueError),
                       (lambda: AdamWMulti([p], betas=(0.9, 1.0)), ValueError),
                       (lambda: AdamWMulti([p], weight_decay=-0.1), ValueError),
                       (lambda: AdamWMulti([torch.nn.Parameter(torch.zeros(3, dtype=torch.float16))]), TypeError),
                       (lambda: AdamWMulti([torch.nn.Parameter(torch.zeros(4, 3).T)]), ValueError),
                       (lambda: AdamWMulti([p]).add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))]}), RuntimeError),
                       (lambda: AdamWMulti([p]).attach_copies({p: torch.zeros(16)}), ValueError),
                       (lambda: AdamWMulti([p]).attach_copies({p: torch.zeros(15, dtype=torch.bfloat16)}), ValueError),
                       (lambda: AdamWMulti([p]).load_param_state(p, {"exp_avg": torch.zeros(3)}), ValueError)):
        with pytest.raises(error):
            bad()
    flat = torch.zeros(20)
    twice = (flat[:12], flat[11:]), (flat, flat), (flat.view(4, 5), flat)
    for pair in twice:
        with pytest.raises(ValueError, match="share memory"):
            AdamWMulti([torch.nn.Parameter(x) for x in pair])
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="twice"):
        AdamWMulti([p, p])
    AdamWMulti([torch.nn.Parameter(x) for x in (flat[:10], flat[10:], flat[:0])])
    with pytest.raises(TypeError, match="state_dict"):
        copy.deepcopy(AdamWMulti([p]))
    opt = AdamWMulti([p])
    for sparse in (torch.zeros(4, 4).to_sparse(), torch.eye(4).to_sparse()):
        p.grad = sparse
        with pytest.raises(RuntimeError, match="dense"):
            opt.step()


# ---------------------------------------------------------------- together
def test_a_training_step_of_the_three():
    """Product in 8 bits, log-probabilities with their gradient, update with 8-bit states: it runs and its gradients are the
    formulas' (how far the loss falls says nothing)."""
    torch.manual_seed(0)
    x, tokens = torch.randn(12, 64), torch.randint(0, 50, (12,))
    w1, head = torch.nn.Parameter(torch.randn(32, 64) * 0.1), torch.nn.Parameter(torch.randn(50, 32) * 0.1)
    opt = AdamWMulti([w1, head], lr=1e-2)
    for _ in range(3):
        h = ops.linear_fp8(x, w1)
        out = ops.linear_logprobs(h, head, tokens, entropy=True, top=2)
        loss = -(out.logprobs.mean() + 0.01 * out.entropy.mean())
        opt.zero_grad()
        loss.backward()
        z = (h.detach() @ head.detach().T).double()
        logp = torch.log_softmax(z, 1)
        p = logp.exp()
        ent = -(p * logp).sum(1, keepdim=True)
        dz = -(torch.nn.functional.one_hot(tokens, 50) - p - 0.01 * p * (logp + ent)) / 12
        assert torch.allclose(head.grad.double(), dz.T @ h.detach().double(), atol=1e-6)
        dh = (dz @ head.detach().double()).float()
        q = lambda t: ops.quantize_fp8(t).dequantize()
        assert torch.allclose(w1.grad, q(dh.T) @ q(x.T).T, atol=1e-2 * w1.grad.abs().max().item())
        before = head.detach().clone()
        opt.step()
        assert not torch.equal(before, head)
