"""Saving and loading ``AdamWMulti`` takes no device memory beyond that of one parameter's moments."""
import pytest
import torch

from maester_b200.optimizers import AdamWMulti

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
def test_peak_memory_of_a_checkpoint(tmp_path, bits):
    import torch.distributed.checkpoint as dcp
    from maester_b200.checkpoint import OptimizerWrapper
    from maester_b200.config import Config
    from maester_b200.optimizers import build_optimizers
    one = 1 << 20                                     # values of a parameter
    m = torch.nn.ParameterDict({f"w{i}": torch.nn.Parameter(torch.randn(one // 1024, 1024, device="cuda")) for i in range(16)})
    cfg = Config(optimizer_groups=[{"opt_class": "maester_b200.optimizers.AdamWMulti", "min_dim": 0,
                                    "opt_cfg": {"lr": 1e-2, "state_bits": bits}}])
    opt = build_optimizers(m, cfg)
    for p in m.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    inner = opt.optimizers[0]
    before = {k: v.clone() for k, v in inner.state_buffers().items()}

    def peak(what):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        what()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - held

    # fp32 moments of all parameters are 16 x 8 MiB; encoding or decoding one takes a dozen temporaries of its size at most
    limit = 16 * 4 * one
    path = str(tmp_path / "c")
    assert peak(lambda: dcp.save({"optimizer": OptimizerWrapper(m, opt)}, checkpoint_id=path, no_dist=True)) < limit
    opt.step()
    assert peak(lambda: dcp.load({"optimizer": OptimizerWrapper(m, opt)}, checkpoint_id=path, no_dist=True)) < limit
    assert peak(lambda: inner.load_state_dict(inner.state_dict())) < limit
    for k, v in inner.state_buffers().items():
        if bits == 32:
            assert torch.equal(v, before[k])
    assert all(s.step == 1 for s in inner._slots.values())
