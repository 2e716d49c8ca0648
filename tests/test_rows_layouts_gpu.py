"""The row operators where rows abound and the channels lie just above a power of two: a quarter of the lanes with three vectors each (bf16), and what takes
two vectors there.  Checks and bounds are those of test_rows_gpu.py."""
import pytest
import torch

import rows_reference as R
import test_rows_gpu as T

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16

# just above and below the row counts from which the layouts change, at both ends of each range of channels; whole rows and ragged ones
WHOLE = [(32800, 136), (32768, 192), (16400, 264), (16384, 384), (8200, 520), (8192, 640), (8192, 768), (4100, 1032), (4096, 1536)]
RAGGED = [(32800, 131), (32770, 189), (16400, 301), (8200, 601), (4100, 1030), (4098, 1275)]
BELOW = [(32760, 160), (16376, 320), (8184, 600), (4092, 1280)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", WHOLE + RAGGED + BELOW)
def test_norm_and_its_gradient(dev, rows, C, dtype):
    T.test_rownorm(dev, rows, C, dtype, "layer" if C % 16 else "rms")


@pytest.mark.parametrize("dtype,fmt", [(F32, "int8"), (BF16, "e4m3"), (BF16, "int8")])
@pytest.mark.parametrize("rows,C", WHOLE + RAGGED)
def test_norm_with_its_checkpoint(dev, rows, C, dtype, fmt):
    T.test_rownorm_checkpoint(dev, rows, C, dtype, fmt)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,groups", [(32800, 136, 8), (32770, 189, None), (16400, 264, 400), (16400, 301, 16400), (8200, 520, None), (8192, 640, 8),
                                           (8200, 601, 4), (8192, 768, 1), (4100, 1032, 4100), (4096, 1536, 64), (4098, 1275, 6)])
def test_gated_exit_and_its_gradient(dev, rows, C, groups, dtype):
    T.test_gated_residual(dev, rows, C, groups, dtype, "layer" if C % 16 else "rms")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(32800, 136), (16400, 301), (8192, 640), (4100, 1030)])
def test_gated_exit_with_the_next_norm_and_checkpoints(dev, rows, C, dtype):
    T.test_gated_residual_with_the_next_norm_and_checkpoints(dev, rows, C, dtype, "e4m3")


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,groups", [(32800, 136, 8), (32770, 189, 2), (16400, 301, 1), (8192, 640, 8), (8200, 601, 4), (4100, 1032, 20), (4098, 1275, 6)])
def test_exit_gradient_from_checkpoints_of_groups(dev, rows, C, groups, dtype, fmt):
    """(The shared test of checkpoints has a gate per row, which takes another form of the gradient.)"""
    H = T._H()
    f, dy = T._rand(rows, C, 2, dtype), T._rand(rows, C, 3, dtype)
    scale, offset, res, gate = T._vec(C, 4), T._vec(C, 5, 0.0), T._vec(C, 6, 0.4), T._rand(groups, C, 7)
    _, mean, rstd, a = H.rownorm_fwd(f.to(dev), None, None, T.EPS, "layer", save8=fmt)
    df, ds, do, dg, dr = H.gated_residual_bwd(dy.to(dev), a, scale.to(dev), offset.to(dev), gate.to(dev), res.to(dev), mean, rstd, "layer")
    v, d, rs = H.act8_load(a).double().cpu(), dy.double(), rstd.double().cpu()
    per = rows // groups
    G = gate.double().repeat_interleave(per, 0)
    m = G * res.double()
    n, nmag = v * scale.double() + offset.double(), (v * scale.double()).abs() + offset.double().abs()
    T._close(df, R.norm_backward(d * m * scale.double(), v, rs, "layer"), 2 * R.backward_error(d * m * scale.double(), v, rs), dtype)
    T._close(ds, (d * m * v).sum(0), R.sums_error(d * m * v, rows))
    T._close(do, (d * m).sum(0), R.sums_error(d * m, rows))
    T._close(dr, (d * G * n).sum(0), R.sums_error(d * G * nmag, rows))
    t, tm = ((d * res.double() * k).reshape(groups, per, C) for k in (n, nmag))
    T._close(dg, t.sum(1), torch.stack([R.sums_error(q, per) for q in tm]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", WHOLE + RAGGED)
def test_a_rows_result_does_not_depend_on_the_layout(dev, rows, C, dtype):
    """The last rows of a large call are, bit for bit, what a small call on them gives: entry with and without a checkpoint, exits with and without the next
    norm, gates per row and per group."""
    H = T._H()
    x, f = T._rand(rows, C, 1, dtype).to(dev), T._rand(rows, C, 2, dtype).to(dev)
    s, o, r = (T._vec(C, i).to(dev) for i in (1, 2, 3))
    gate = T._rand(rows, C, 4, dtype).to(dev)
    n = 50
    xt, ft, gt = (t[-n:].contiguous() for t in (x, f, gate))
    for save in (None, "e4m3"):
        y, mean, rstd, a = H.rownorm_fwd(x, s, o, T.EPS, "layer", save8=save)
        yt, mt, rt, at = H.rownorm_fwd(xt, s, o, T.EPS, "layer", save8=save)
        assert torch.equal(y[-n:], yt) and torch.equal(mean[-n:], mt) and torch.equal(rstd[-n:], rt)
        assert save is None or (torch.equal(a.codes[-n:], at.codes) and torch.equal(a.scales[-n:], at.scales))
    for nxt in (None, (s, o, T.EPS, "rms")):
        for g, t in ((gate, gt), (None, None), (gate[0], gate[0])):
            p, q = H.gated_residual_fwd(x, f, s, o, g, r, T.EPS, "layer", next_norm=nxt), H.gated_residual_fwd(xt, ft, s, o, t, r, T.EPS, "layer", next_norm=nxt)
            assert torch.equal(p[0][-n:], q[0]) and torch.equal(p[1][-n:], q[1]) and torch.equal(p[2][-n:], q[2])
            assert nxt is None or (torch.equal(p[4][0][-n:], q[4][0]) and torch.equal(p[4][2][-n:], q[4][2]))
