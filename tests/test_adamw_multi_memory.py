"""``AdamWMulti`` and memory that goes away, moves or changes size under it (host side)."""
import pytest
import torch

from maester_b200.optimizers import AdamWMulti


def _addresses(opt):
    return [int(a) for b in opt._batches for a in b.table[:, 2]]


def _stepped(opt, params):
    for p in params:
        p.grad = torch.ones_like(p)
    opt.step()


def test_copies_are_written_where_they_are():
    """A copy's memory may be freed between steps (its storage resized to nothing) and come back elsewhere: it is never
    written through an address of before."""
    params = [torch.nn.Parameter(torch.randn(n)) for n in (300, 40)]
    opt = AdamWMulti(params, lr=0.1)
    buffer = torch.zeros(400, dtype=torch.bfloat16)
    opt.attach_copies({params[0]: buffer[:300], params[1]: buffer[300:340]})   # (the second does not start the storage)
    _stepped(opt, params)
    assert _addresses(opt) == [buffer.data_ptr(), buffer.data_ptr() + 600]
    assert all(torch.equal(c, p.detach().bfloat16()) for c, p in zip((buffer[:300], buffer[300:340]), params))
    size = buffer.untyped_storage().nbytes()
    buffer.untyped_storage().resize_(0)
    _stepped(opt, params)                      # (parameters are updated; a copy without memory is left out)
    assert _addresses(opt) == [0, 0]
    buffer.untyped_storage().resize_(size)
    buffer.zero_()
    _stepped(opt, params)
    assert _addresses(opt) == [buffer.data_ptr(), buffer.data_ptr() + 600]
    assert all(torch.equal(c, p.detach().bfloat16()) for c, p in zip((buffer[:300], buffer[300:340]), params))
    big = torch.zeros(100, dtype=torch.bfloat16)
    opt = AdamWMulti(params[1:], lr=0.1)
    opt.attach_copies({params[1]: big[:40]})
    big.resize_(100_000)                       # moves the storage
    _stepped(opt, params[1:])
    assert _addresses(opt) == [big.data_ptr()] and torch.equal(big[:40], params[1].detach().bfloat16())


def test_a_copy_whose_storage_shrank_is_refused():
    p = torch.nn.Parameter(torch.randn(300))
    opt = AdamWMulti([p], lr=0.1)
    low = torch.zeros(300, dtype=torch.bfloat16)
    opt.attach_copies({p: low})
    low.untyped_storage().resize_(100)
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="copy"):
        _stepped(opt, [p])
    assert torch.equal(p, before) and opt._slots[p].step == 0


@pytest.mark.parametrize("change", ["shorter", "type", "freed", "freed view"])
def test_a_parameter_that_is_no_longer_what_it_was_is_refused(change):
    """The address and the layout may be those of before: a step would go on over memory that is no longer the parameter's."""
    flat = torch.randn(1500)
    p = torch.nn.Parameter(flat[500:] if change == "freed view" else torch.randn(1000))
    other = torch.nn.Parameter(torch.randn(7))
    opt = AdamWMulti([other, p], lr=0.1)
    _stepped(opt, [other, p])
    before = other.detach().clone()
    if change == "shorter":
        p.data = p.data[:100]
    elif change == "type":
        p.grad = None
        p.data = p.data.view(torch.bfloat16)[:1000]
    elif change == "freed":
        p.data.untyped_storage().resize_(0)
    else:
        flat.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="replaced"):
        opt.step()
    assert torch.equal(other, before) and opt._slots[other].step == 1       # (nothing of a refused step has run)


def test_parameters_that_come_to_share_memory_are_refused():
    a, b = torch.nn.Parameter(torch.randn(50)), torch.nn.Parameter(torch.randn(70))
    opt = AdamWMulti([{"params": [a]}, {"params": [b], "lr": 0.2}], lr=0.1)
    _stepped(opt, [a, b])
    kept, before = b.data, a.detach().clone()
    b.data = torch.cat([a.data, torch.zeros(40)])[:70]
    a.data = b.data[:50]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="share memory"):
            _stepped(opt, [a, b])
    assert torch.equal(a, before)
    b.data = kept
    _stepped(opt, [a, b])
    assert not torch.equal(a, before)


def test_copies_that_share_memory_are_refused():
    p, q = torch.nn.Parameter(torch.randn(50)), torch.nn.Parameter(torch.randn(70))
    opt = AdamWMulti([p, q], lr=0.1)
    low = torch.zeros(100, dtype=torch.bfloat16)
    for copies in ({p: low[:50], q: low[30:100]}, {p: p.data.view(torch.bfloat16)[:50]}, {q: p.data.view(torch.bfloat16)[30:]}):
        with pytest.raises(ValueError):
            opt.attach_copies(copies)
    assert all(s.copy is None for s in opt._slots.values())
    opt.attach_copies({p: low[:50]})
    with pytest.raises(ValueError, match="share memory"):
        opt.attach_copies({q: low[30:]})
    opt.attach_copies({q: torch.zeros(70, dtype=torch.bfloat16)})
    _stepped(opt, [p, q])
    assert torch.equal(low[:50], p.detach().bfloat16())


def test_parameters_may_move_while_copies_have_no_memory():
    params = [torch.nn.Parameter(torch.randn(300)) for _ in range(2)]
    opt = AdamWMulti(params, lr=0.1)
    low = [torch.zeros(500, dtype=torch.bfloat16) for _ in range(2)]
    opt.attach_copies({params[0]: low[0][10:310], params[1]: low[1][100:400]})
    for x in low:
        x.untyped_storage().resize_(0)
    params[0].data = params[0].data.clone()
    before = params[0].detach().clone()
    _stepped(opt, params)
    assert not torch.equal(params[0], before)
