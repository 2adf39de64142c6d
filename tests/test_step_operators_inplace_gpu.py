"""Operators that write into a caller's tensor tell autograd, on the GPU as on the CPU."""
import pytest
import torch

from maester_b200 import ops
from maester_b200.optimizers import AdamWMulti

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
def test_a_graph_of_before_the_step_is_refused(bits):
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    w, other = (torch.nn.Parameter(torch.randn(8, 8, device="cuda")) for _ in range(2))
    low = torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    opt = AdamWMulti([w, other], lr=0.1, state_bits=bits)
    opt.attach_copies({w: low})
    for _ in range(2):
        y, z = (x @ w).sum(), (x @ other).sum()
        w.grad = torch.ones_like(w)
        seen = w._version, low._version
        opt.step()
        assert w._version > seen[0] and low._version > seen[1]
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
        z.backward()                        # (a parameter without a gradient was left alone)
        other.grad = None


def test_a_product_into_a_tensor_that_is_needed():
    a = ops.quantize_fp8(torch.randn(8, 128, device="cuda"))
    out = torch.zeros(8, 8, device="cuda")
    y = (out * torch.ones(8, 8, device="cuda", requires_grad=True)).sum()
    ops.matmul_fp8(a, a, out=out)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        inside = torch.zeros(8, 8, device="cuda")
        ops.matmul_fp8(a, a, out=inside)
    ops.matmul_fp8(a, a, out=inside)
    assert torch.equal(inside, out)
