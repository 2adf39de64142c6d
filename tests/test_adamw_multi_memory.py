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
