"""``AdamWMulti`` on the GPU against the plain definition, whose operations are rounded one by one.

The moments (codes, exponents, 32-bit states) agree bit for bit.  A parameter's update u is m / (root * c + eps) * step: the
kernel's quotient is off by two steps of fp32 (2^-22 relative) at most, its root by one in rare cases, and adding it rounds p
once: per step |p| 2^-23 + 3 |u| 2^-23 with |u| <= |p before| + |p after|; a 16-bit parameter may round to its neighbour.
The plain form runs on GPU tensors too: its square root and division are correctly rounded there.
"""
import pytest
import torch

from maester_b200.ops import reference as ref
from maester_b200.optimizers import AdamWMulti

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


def _params(sizes, dtype, shift=0):
    """Separate tensors; ``shift`` puts them off a 16-byte boundary."""
    out = []
    for n in sizes:
        buf = torch.randn(n + shift, device="cuda").mul_(0.1).to(dtype)
        out.append(torch.nn.Parameter(buf[shift:]))
    return out


def _grads(params, step, special=False, shift=0):
    g = torch.Generator(device="cuda").manual_seed(step)
    for i, p in enumerate(params):
        v = torch.randn(p.numel() + shift, device="cuda", generator=g) * 10.0 ** (i % 7 - 5)
        v = v * torch.exp(torch.randn(v.shape, device="cuda", generator=g) * 2)
        v = torch.where(torch.rand(v.shape, device="cuda", generator=g) < 0.1, torch.zeros_like(v), v)
        if special and v.numel() > 40:
            v[shift + 7], v[shift + 11], v[shift + 13] = float("nan"), float("inf"), 1e30
        p.grad = v.to(p.dtype)[shift:].view(p.shape)


def _twin(params):
    return [torch.nn.Parameter(p.detach().clone()) for p in params]


def _plain(opt):
    opt._launch = opt._plain
    return opt


def _same(a, b):
    a, b = a.detach().cpu(), b.detach().cpu()
    if a.dtype == torch.float8_e4m3fn:
        return torch.equal(a.view(torch.uint8) & 0x7f, b.view(torch.uint8) & 0x7f) and torch.equal(
            a.float().nan_to_num(9.0), b.float().nan_to_num(9.0))     # (the sign of a NaN code says nothing)
    return torch.equal(a.nan_to_num(9.0, 8.0, 7.0), b.nan_to_num(9.0, 8.0, 7.0)) if a.is_floating_point() else torch.equal(a, b)


class _Near:
    """The bound above, summed over the steps."""

    def __init__(self, params):
        self.before = [p.detach().double().abs() for p in params]
        self.tol = [torch.zeros_like(b) for b in self.before]

    def check(self, a, b):
        for i, (p, q) in enumerate(zip(a, b)):
            x, y = p.detach().double(), q.detach().double()
            step = 2.0 ** (-23 if p.dtype == torch.float32 else -7)
            self.tol[i] += step * y.abs().nan_to_num(0.0) + 3 * 2.0 ** -23 * (y.abs() + self.before[i]).nan_to_num(0.0)
            self.before[i] = y.abs()
            assert torch.equal(x.isnan(), y.isnan()) and ((x - y).abs() <= self.tol[i])[~x.isnan()].all()


SIZES = [(1,), (255, 256, 257), (3, 8191, 8192, 8193, 1), (100_003, 17, 65536, 5), tuple(range(1, 700, 7)), (1 << 20,)]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[-1]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("shift", [0, 1])
def test_steps(sizes, dtype, bits, shift):
    a = _params(sizes, dtype, shift)
    b = _twin(a)
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1, state_bits=bits)
    oa, ob = AdamWMulti(a, **kw), _plain(AdamWMulti(b, **kw))
    near, copies = _Near(b), {}
    if dtype == torch.float32:
        copies = {p: torch.zeros(p.numel() + shift, device="cuda", dtype=torch.bfloat16)[shift:] for p in a[::2]}
        oa.attach_copies(copies)
    for step in range(4):
        _grads(a, step, special=step == 2, shift=shift)
        for p, q in zip(a, b):
            q.grad = p.grad
        if step == 1 and len(a) > 1:
            a[0].grad = b[0].grad = None                     # left alone, its step number too
        oa.step()
        ob.step()
        near.check(a, b)
        for k, v in oa.state_buffers().items():
            assert _same(v, ob.state_buffers()[k]), k
    for p, c in copies.items():
        assert _same(c, p.detach().to(torch.bfloat16))


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_and_many_tensors(bits):
    """More tensors than one launch takes, two groups with settings of their own, both types."""
    a = _params([(i * 37) % 900 + 1 for i in range(1100)], torch.float32) + _params([300, 4000], torch.bfloat16)
    b = _twin(a)

    def make(ps):
        return AdamWMulti([{"params": ps[:700], "lr": 1e-2, "weight_decay": 0.3}, {"params": ps[700:], "betas": (0.8, 0.99)}],
                          lr=3e-3, state_bits=bits)
    oa, ob = make(a), _plain(make(b))
    near = _Near(b)
    for step in range(3):
        _grads(a, step)
        for p, q in zip(a, b):
            q.grad = p.grad
        oa.step()
        ob.step()
        near.check(a, b)
    assert all(_same(v, ob.state_buffers()[k]) for k, v in oa.state_buffers().items())


def test_update_against_64_bits():
    """From a state of zeros the codes play no part: fp32 roundings only (8 of them on the update, each u = 2^-24)."""
    p, = _params([5000], torch.float32)
    p0, u = p.detach().double().clone(), 2.0 ** -24
    _grads([p], 3)
    g = p.grad.double()
    opt = AdamWMulti([p], lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    opt.step()
    upd = 1e-2 * (0.1 * g / 0.1) / ((0.05 * g * g / 0.05).sqrt() + 1e-8)
    want = p0 * (1 - 1e-3) - upd
    assert ((p.detach().double() - want).abs() <= 3 * u * (p0.abs() + upd.abs()) + 16 * u * upd.abs()).all()


def test_what_surrounds_a_tensor_stays():
    buf = torch.full((3000,), 5.0, device="cuda")
    low = torch.full((3000,), 5.0, device="cuda", dtype=torch.bfloat16)
    p = torch.nn.Parameter(buf[1001:2002])
    opt = AdamWMulti([p], lr=0.1)
    opt.attach_copies({p: low[1001:2002]})
    p.grad = torch.ones_like(p)
    opt.step()
    assert (buf[:1001] == 5).all() and (buf[2002:] == 5).all() and (buf[1001:2002] != 5).all()
    assert (low[:1001] == 5).all() and (low[2002:] == 5).all() and (low[1001:2002] != 5).all()


def test_strided_gradients_streams_and_capture():
    p = torch.nn.Parameter(torch.randn(64, 48, device="cuda"))
    q = torch.nn.Parameter(p.detach().clone())
    g = torch.randn(48, 64, device="cuda")
    p.grad, q.grad = g.T, g.T.contiguous()
    AdamWMulti([p], lr=0.1).step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        AdamWMulti([q], lr=0.1).step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(p, q)
    opt = AdamWMulti([p], lr=0.1)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()


def test_parameters_that_move():
    """A parameter whose memory is replaced is updated where it is then; one that is no longer what it was is refused."""
    a, b = _params([700, 33, 5000], torch.float32), _params([700, 33, 5000], torch.float32)
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    oa, ob = AdamWMulti(a, lr=0.1), AdamWMulti(b, lr=0.1)
    for step in range(3):
        _grads(a, step)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        old = a[1].data
        if step == 1:
            a[1].data = old.clone()
            before = old.clone()
        oa.step()
        ob.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        if step == 1:
            assert torch.equal(old, before)
    good = a[2].data
    for bad in (good.bfloat16(), good[:100].clone(), good.cpu(), torch.zeros(10000, device="cuda")[::2]):
        a[2].grad = None
        a[2].data = bad
        with pytest.raises(RuntimeError, match="replaced"):
            oa.step()
    a[2].data = good
    a[2].grad = torch.zeros(5000, device="cuda")
    oa.step()


def test_saved_and_loaded_on_the_gpu():
    a = _params([1000, 77], torch.float32)
    opt = AdamWMulti(a, lr=1e-2)
    for step in range(3):
        _grads(a, step)
        opt.step()
    twin = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = AdamWMulti(twin, lr=1e-2)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(a, twin):
        assert all(torch.equal(x, y) for x, y in zip(opt._moments(p), other._moments(q)))
    _grads(a, 9)
    for p, q in zip(a, twin):
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, twin))


@pytest.mark.parametrize("bits", [8, 32])
def test_trainer_writes_the_compute_copy(bits):
    """Through the optimizer builder and the sharding runtime: the bf16 parameters of the next forward are the rounded
    masters."""
    from maester_b200.config import Config
    from maester_b200.datasets.synthetic import SyntheticLoader
    from maester_b200.trainer import Trainer
    losses = {}
    for name, extra in (("torch.optim.AdamW", {}), ("maester_b200.optimizers.AdamWMulti", {"state_bits": bits})):
        torch.manual_seed(0)
        cfg = Config(model_name="gemma3", flavor="debug", seq_len=256, train_batch_size=2, data_parallel_shard_degree=1,
                     enable_checkpoint=False,
                     optimizer_groups=[{"opt_class": name, "min_dim": 0,
                                        "opt_cfg": {"lr": 1e-3, "betas": (0.9, 0.95), "weight_decay": 0.0, **extra}}])
        tr = Trainer(cfg)
        loader = SyntheticLoader(2, 256, tr.model_args.vocab_size, "uniform:16:256")
        losses[name] = [tr.train_step(next(loader)).item() for _ in range(3)]
        if extra:
            assert tr.optimizers.optimizers[0].writes_lowp
            assert torch.equal(tr.sharded.full, tr.sharded.master.to(torch.bfloat16))
    a, b = losses.values()
    assert all(x == x for x in a + b)
    # the same model before the first update; the row losses are added by atomics, 512 fp32 additions in any order
    assert abs(a[0] - b[0]) <= 512 * 2.0 ** -24 * a[0]
