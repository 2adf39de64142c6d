"""State that is held on the host under a device mesh is written and read as pieces of the whole tensors, where a DTensor over
the mesh would have put them.  (Here the mesh is the host's too: the ranks take the pieces all the same.)"""
import torch

from test_checkpoint_cpu import _ep_save_resume, _run_save_resume, _tp_save
from test_parallel_cpu import _batches, _cfg, _full_weights, run_ranks

MULTI = [{"opt_class": "maester_b200.optimizers.AdamWMulti", "min_dim": 0,
          "opt_cfg": {"lr": 1e-3, "betas": (0.9, 0.95), "weight_decay": 0.1, "state_bits": 8}}]


def _as_pieces(rank, world, inner, *args):
    from maester_b200 import checkpoint
    seen = []
    whole = checkpoint._as_host_piece

    def piece(local, mesh, placements, shape):
        from torch.distributed.tensor import DTensor
        t = whole(local, mesh, placements, shape)
        stride = torch.empty(shape, device="meta").stride()
        d = DTensor.from_local(local, mesh, placements, run_check=False, shape=shape, stride=stride)
        want = [(tuple(c.offsets), tuple(c.sizes)) for c in d.__create_chunk_list__() if 0 not in c.sizes]
        assert [(tuple(c.offsets), tuple(c.sizes)) for c in t.__create_chunk_list__()] == want
        assert t.data_ptr() == local.data_ptr() and t.size() == shape
        seen.append(len(want))
        return t
    checkpoint._on_mesh_device = lambda local, mesh: False
    checkpoint._as_host_piece = piece
    out = inner(rank, world, *args)
    assert seen
    return out


def test_two_rank_save_and_resume(tmp_path):
    full = _full_weights(_cfg())
    kw = dict(data_parallel_shard_degree=2, optimizer_groups=MULTI)
    assert run_ranks(2, _as_pieces, _run_save_resume, kw, str(tmp_path), full, _batches(4, 4, 64, 512)) == [True, True]


def test_expert_parallel_round_trip(tmp_path):
    from test_expert_parallel_cpu import _cfg as ep_cfg
    full = _full_weights(ep_cfg(train_batch_size=8))
    assert all(r > 0 for r in run_ranks(4, _as_pieces, _ep_save_resume, str(tmp_path), full, _batches(2, 8, 32, 2000)))


def test_tensor_parallel_pieces(tmp_path):
    full = _full_weights(_cfg())
    assert run_ranks(4, _as_pieces, _tp_save, str(tmp_path), full, [], 2) == [True] * 4
    from maester_b200.convert.io import read_dcp_model
    flat = read_dcp_model(tmp_path / "job" / "checkpoints" / "step-2")
    assert set(flat) == set(full) and all(torch.equal(flat[k], full[k]) for k in full)
