"""State dicts and checkpoints of ``AdamWMulti``: what they leave out, other optimizers, memory."""
import copy

import pytest
import torch

from maester_b200.optimizers import AdamWMulti


def _params():
    torch.manual_seed(3)
    return [torch.nn.Parameter(torch.randn(n)) for n in (300, 7, 40)]


def _run(opt, params, steps, skip=()):
    for s in range(steps):
        g = torch.Generator().manual_seed(s)
        for i, p in enumerate(params):
            p.grad = None if i in skip else torch.randn(p.shape, generator=g)
        opt.step()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("what", ["empty", "partial", "fields"])
def test_a_loaded_state_replaces_the_present_one(bits, what):
    """As torch.optim's: a parameter that the state does not have starts afresh."""
    params = _params()
    opt = AdamWMulti(params, lr=1e-2, state_bits=bits)
    fresh = {k: v.clone() for k, v in opt.state_buffers().items()}
    if what == "partial":
        _run(opt, params, 2, skip=(1,))
    snapshot = copy.deepcopy(opt.state_dict())
    if what == "empty":
        snapshot["state"] = torch.optim.AdamW(params).state_dict()["state"]
    elif what == "partial":
        del snapshot["state"][1]
    else:
        snapshot["state"] = {i: {"exp_avg": torch.ones(p.shape)} for i, p in enumerate(params)}
    _run(opt, params, 3)
    opt.load_state_dict(snapshot)
    for i, p in enumerate(params):
        m, v = opt._moments(p)
        gone = what == "empty" or (what == "partial" and i == 1)
        assert opt._slots[p].step == (0 if gone or what == "fields" else 2)
        assert bool(m.any()) != gone and bool(v.any()) == (what == "partial" and i != 1)
    if what == "empty":
        assert all(torch.equal(a.float(), fresh[k].float()) for k, a in opt.state_buffers().items())


def _container(cls, **extra):
    from maester_b200.config import Config
    from maester_b200.optimizers import build_optimizers
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 5))
    cfg = Config(optimizer_groups=[{"opt_class": cls, "min_dim": 0,
                                    "opt_cfg": {"lr": 1e-2, "betas": [0.9, 0.95], "weight_decay": 0.1, **extra}}])
    return m, build_optimizers(m, cfg)


def _train(m, opt, seeds):
    for s in seeds:
        x = torch.randn(4, 20, generator=torch.Generator().manual_seed(s))
        opt.zero_grad()
        m(x).square().sum().backward()
        opt.step()


def _held(opt, p):
    o = opt.optimizers[0]
    st = o.param_state(p) if hasattr(o, "param_state") else o.state[p]
    return st["exp_avg"], st["exp_avg_sq"], float(st["step"])


@pytest.mark.parametrize("other", ["maester_b200.optimizers.FusedAdamW", "torch.optim.AdamW"])
@pytest.mark.parametrize("direction", ["from", "to"])
@pytest.mark.parametrize("bits", [8, 32])
def test_job_checkpoints_pass_between_optimizers(tmp_path, other, direction, bits):
    """A job's checkpoint goes on under another AdamW: moments, step numbers, settings, and the step that follows.  (Into 8
    bits: a code is off by half a step at the most, 2^-4 of a first moment and, for the squares, 2^-3 + 2^-8.)"""
    import torch.distributed.checkpoint as dcp
    from maester_b200.checkpoint import OptimizerWrapper
    mine = ("maester_b200.optimizers.AdamWMulti", dict(state_bits=bits))
    a, b = (mine, (other, {})) if direction == "to" else ((other, {}), mine)
    m, opt = _container(a[0], **a[1])
    _train(m, opt, range(3))
    opt.param_groups[0]["lr"] = 3e-3
    dcp.save({"optimizer": OptimizerWrapper(m, opt)}, checkpoint_id=str(tmp_path / "c"), no_dist=True)
    m2, opt2 = _container(b[0], **b[1])
    _train(m2, opt2, [9])                   # (torch's has no states to load into before its first step)
    m2.load_state_dict(m.state_dict())
    dcp.load({"optimizer": OptimizerWrapper(m2, opt2)}, checkpoint_id=str(tmp_path / "c"), no_dist=True)
    assert opt2.param_groups[0]["lr"] == 3e-3 and tuple(opt2.param_groups[0]["betas"]) == (0.9, 0.95)
    coarse = bits == 8 and direction == "from"
    for p, q in zip(m.parameters(), m2.parameters()):
        (ma, va, sa), (mb, vb, sb) = _held(opt, p), _held(opt2, q)
        assert sa == sb == 3
        if coarse:      # (below 2^-6 of a block's largest value 448: half a code's distance there)
            assert ((ma - mb).abs() <= ma.abs() * 2 ** -4 + ma.abs().max() * 2 ** -17).all()
            assert ((va.sqrt() - vb.sqrt()).abs() <= va.sqrt() * 2 ** -4 + va.max().sqrt() * 2 ** -17).all()
        else:
            assert torch.equal(ma, mb) and torch.equal(va, vb)
    before = [p.detach().clone() for p in m.parameters()]
    _train(m, opt, [5])
    _train(m2, opt2, [5])
    for p, q, old in zip(m.parameters(), m2.parameters(), before):
        step = (p.detach() - old).abs().max()
        # 32 bits into 32 bits: fp32 roundings; else the states' roundings, at most an eighth of an update or so
        assert (p - q).abs().max() <= (0.3 * step if coarse else 16 * 2.0 ** -24 * (old.abs().max() + step))


def test_state_dicts_pass_between_optimizers():
    params = _params()
    opt = AdamWMulti(params, lr=1e-2, state_bits=32)
    _run(opt, params, 2)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    plain = torch.optim.AdamW(twin)
    plain.load_state_dict(copy.deepcopy(opt.state_dict()))
    _run(opt, params, 1)
    _run(plain, twin, 1)
    for p, q in zip(params, twin):
        assert torch.allclose(p, q, rtol=0, atol=16 * 2.0 ** -24 * (1e-2 + p.abs().max().item()))


@pytest.mark.parametrize("key", ["maximize", "amsgrad"])
def test_settings_that_it_does_not_follow_are_refused(key):
    params = _params()
    plain = torch.optim.AdamW(params, **{key: True})
    opt = AdamWMulti(params)
    opt.load_state_dict(plain.state_dict())
    for p in params:
        p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match=key):
        opt.step()


def test_a_state_is_found_by_the_names_that_its_groups_give():
    """As torch.optim's: the entries of ``state`` are named by the groups' ``params``, whatever they are."""
    params = _params()
    opt = AdamWMulti(params, lr=1e-2)
    _run(opt, params, 2)
    sd = copy.deepcopy(opt.state_dict())
    names = ["c", "a", "b"]
    sd["state"] = {names[i]: s for i, s in sd["state"].items()}
    sd["param_groups"][0]["params"] = names
    want = [opt._moments(p)[0].clone() for p in params]
    _run(opt, params, 1)
    opt.load_state_dict(sd)
    assert all(torch.equal(opt._moments(p)[0], m) and opt._slots[p].step == 2 for p, m in zip(params, want))
    del sd["param_groups"][0]["params"][0]
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert all(opt._slots[p].step == 2 for p in params)


def test_torch_checkpoint_helpers_leave_the_states_alone():
    """They take an optimizer whose ``state`` is empty for one that has never stepped, and let it step with zeros."""
    from torch.distributed.checkpoint.state_dict import get_optimizer_state_dict, set_optimizer_state_dict
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 5))
    params = list(m.parameters())
    opt = AdamWMulti(params, lr=1e-2)
    _run(opt, params, 2)
    opt.zero_grad()
    want = [[x.clone() for x in opt._moments(p)] for p in params]
    for again in range(2):
        sd = get_optimizer_state_dict(m, opt)
        assert [s.step for s in opt._slots.values()] == [2] * 4
        for p, w in zip(params, want):
            assert all(torch.equal(x, y) for x, y in zip(opt._moments(p), w))
        assert torch.equal(sd["state"]["1.weight"]["exp_avg"], want[2][0].view(5, 30))
        _run(opt, params, 1)
        opt.zero_grad()
        set_optimizer_state_dict(m, opt, sd)
    assert [s.step for s in opt._slots.values()] == [2] * 4
    for p, w in zip(params, want):
        assert all(torch.equal(x, y) for x, y in zip(opt._moments(p), w))
