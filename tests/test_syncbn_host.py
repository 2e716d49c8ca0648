"""Cross-rank batch-norm statistics without a GPU: what is refused."""
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _trainer(world):
    from dpig_amd.trainer import DPIG_Encoder_GAN_BodyROI_FgBg, GradAllReduce
    tr = object.__new__(DPIG_Encoder_GAN_BodyROI_FgBg)
    tr.device = torch.device("cpu")
    tr.allreduce = GradAllReduce()
    tr.allreduce.world, tr.allreduce.enabled = world, world > 1
    return tr


@pytest.mark.parametrize("world", [2, 8])
def test_captured_steps_with_statistics_over_several_ranks_are_refused(monkeypatch, world):
    from dpig_amd import autograd as A
    monkeypatch.setattr(A, "_SYNC_BN_GROUP", [True, None])
    tr = _trainer(world)
    with pytest.raises(RuntimeError, match="batch-norm statistics over %d ranks" % world):
        tr.enable_graphs({}, {})
    assert not hasattr(tr, "_static_g")                      # nothing was begun


@pytest.mark.parametrize("world,sync", [(1, True), (2, False)])
def test_the_other_configurations_are_not_refused(monkeypatch, world, sync):
    """One rank, or statistics per rank: enable_graphs goes on (to its first use of the device, which a stand-in ends)."""
    from dpig_amd import autograd as A, trainer
    monkeypatch.setattr(A, "_SYNC_BN_GROUP", [sync, None])

    class Went(Exception):
        pass

    def stream(*a, **k):
        raise Went()
    monkeypatch.setattr(trainer.torch.cuda, "Stream", stream)
    with pytest.raises(Went):
        _trainer(world).enable_graphs({}, {})


def test_the_one_gpu_rehearsal_leaves_the_statistics_over_ranks_out():
    text = open(os.path.join(ROOT, "scripts", "run_scale.sh")).read()
    lines = [k for k in text.splitlines() if "DPIG_SYNC_BN=1" in k]
    assert lines and all(k.endswith("-- --no-graph") for k in lines)
    head = text[:text.index(lines[0])].splitlines()[-2:]
    assert any("$DRY -eq 0" in k for k in head)
