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
