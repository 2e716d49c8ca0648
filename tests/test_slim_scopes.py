"""Variable names of slim.gated_res_block (no kernel runs: the block itself is stood in for)."""
import numpy as np
import pytest
import torch


@pytest.fixture
def block(monkeypatch):
    """gated_res_block on the CPU -> the variables it hands to the operator, in order."""
    import dpig_amd.tflib as lib
    from dpig_amd import autograd as A, slim
    lib.delete_all_params(); slim.reset_scopes(); lib.set_device(torch.device("cpu"))
    np.random.seed(0)
    monkeypatch.setattr(A, "gated_resblock", lambda x, s1, o1, w1, b1, w2, b2, s2, o2, gate, res, *a: (s1, o1, w1, b1, w2, b2, s2, o2, res))
    yield slim.gated_res_block
    lib.delete_all_params(); slim.reset_scopes()


def _names():
    import dpig_amd.tflib as lib
    return sorted(lib._params)


LEAVES = ["entry_offset", "entry_scale", "exit_offset", "exit_scale", "fully_connected/biases", "fully_connected/weights",
          "fully_connected_1/biases", "fully_connected_1/weights", "res_scale"]


def test_a_scope_given_twice_shares_every_variable(block):
    x = torch.zeros(2, 40)
    a, b = block(x, 24, scope="Net/blk"), block(x, 24, scope="Net/blk")
    assert len(a) == 9 and all(p is q for p, q in zip(a, b))
    assert _names() == ["Net/blk/" + n for n in LEAVES]
    c = block(x, 24, scope="Net/other")
    assert not any(p is q for p in a for q in c) and len(_names()) == 18


def test_blocks_without_a_scope_count_on(block):
    from dpig_amd import slim
    x = torch.zeros(2, 40)
    with slim.variable_scope("Emb"):
        a = block(x, 24)
        block(x, 24, scope="Emb/own")                       # (leaves the counters alone)
        b = block(x)
    with slim.variable_scope("Emb", reuse=True):
        again = block(x, 24)
    assert all(p is q for p, q in zip(a, again)) and not any(p is q for p in a for q in b)
    fc = [n for n in _names() if "fully_connected" in n and "own" not in n]
    assert fc == sorted("Emb/fully_connected%s/%s" % (k, t) for k in ("", "_1", "_2", "_3") for t in ("weights", "biases"))
