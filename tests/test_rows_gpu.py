"""Entry norm and gated residual exit of a block on rows of channels, forward and backward, against float64 forms of their formulas."""
import pytest
import torch

import rows_reference as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5


def _H():
    import dpig_amd.hip_ops as H
    return H


def _rand(rows, C, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g)) + 0.3).to(dtype)


def _vec(C, seed, about=1.0):
    g = torch.Generator().manual_seed(seed)
    return about + 0.2 * torch.randn(C, generator=g)


def _close(got, ref, bound, dtype=F32):
    err = (got.double().cpu() - ref).abs()
    bound = bound + R.STORE[dtype] * (ref.abs() + bound) + 1e-37
    assert got.dtype == dtype and bool((err <= bound).all()), "worst %.3g of its bound" % float((err / bound).max())


# every lane layout (C <= 64, 128, 256, 512, 1024, 2048, 8192), whole and ragged rows, one row to many
SHAPES = [(1, 1), (5, 7), (3, 64), (33, 40), (130, 128), (64, 512), (77, 250), (300, 256), (29, 513), (1024, 640), (9, 1025), (21, 2048), (6, 2500),
          (3, 8192), (20000, 96)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", SHAPES)
def test_rownorm(dev, rows, C, dtype, kind):
    H = _H()
    x, dy, acc = _rand(rows, C, 1, dtype), _rand(rows, C, 2, dtype), _rand(rows, C, 3, dtype)
    scale, offset = _vec(C, 4), _vec(C, 5, 0.0)
    y, mean, rstd, saved = H.rownorm_fwd(x.to(dev), scale.to(dev), offset.to(dev), EPS, kind)
    xh, m, r = R.normed(x, kind, EPS)
    e = R.normed_error(x, xh, r, C)
    assert saved is None and (mean is None) == (kind == "rms")
    _close(y, xh * scale.double() + offset.double(), e * scale.double().abs() + 2 * R.U * ((xh * scale.double()).abs() + offset.double().abs()), dtype)
    _close(rstd, r, r * R.U * (34 + 41 * x.double().abs().amax(1) * r))
    if mean is not None:
        _close(mean, m, 41 * R.U * x.double().abs().amax(1))
    # backward from x, with the statistics as they were left
    mu = mean.double().cpu() if mean is not None else torch.zeros(rows, dtype=torch.float64)
    rs = rstd.double().cpu()
    xh = (x.double() - mu[:, None]) * rs[:, None]
    d = dy.double()
    g = d * scale.double()
    for accum in (None, acc):
        dx, ds, do = H.rownorm_bwd(dy.to(dev), x.to(dev), scale.to(dev), mean, rstd, kind, accum=None if accum is None else accum.to(dev))
        ref = R.norm_backward(g, xh, rs, kind) + (0 if accum is None else accum.double())
        _close(dx, ref, R.backward_error(g, xh, rs) + 2 * R.U * ref.abs() + (0 if accum is None else 2 * R.U * accum.double().abs()), dtype)
        _close(ds, (d * xh).sum(0), R.sums_error(d * xh, rows))
        _close(do, d.sum(0), R.sums_error(d, rows))
    dx2, none, none2 = H.rownorm_bwd(dy.to(dev), x.to(dev), scale.to(dev), mean, rstd, kind, accum=acc.to(dev), want_params=False)
    assert none is None and none2 is None and torch.equal(dx, dx2)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", SHAPES)
def test_rownorm_checkpoint(dev, rows, C, dtype, fmt):
    """The checkpoint of xh that the forward pass leaves, and the backward pass from it."""
    H = _H()
    kind = "layer" if rows % 2 else "rms"
    x, dy = _rand(rows, C, 1, dtype), _rand(rows, C, 2, dtype)
    scale = _vec(C, 4)
    y, mean, rstd, a = H.rownorm_fwd(x.to(dev), scale.to(dev), None, EPS, kind, save8=fmt)
    y2, _, rstd2, _ = H.rownorm_fwd(x.to(dev), scale.to(dev), None, EPS, kind)
    assert torch.equal(y, y2) and torch.equal(rstd, rstd2)                # saving changes nothing else
    xh, _, r = R.normed(x, kind, EPS)
    v = H.act8_load(a).double().cpu()
    s = torch.exp2(a.scales.cpu().double() - 127).repeat_interleave(32, 1)[:, :C]
    # a rounding of the format (half a step: 2^-4 relative, or half of the smallest step; a whole one below it) of xh as fp32 has it
    half = torch.maximum(2.0 ** -4 * xh.abs(), s * 2.0 ** -9) if fmt == "e4m3" else torch.where(xh.abs() < s, s, s / 2)
    assert bool(((v - xh).abs() <= half * (1 + 1e-3) + R.normed_error(x, xh, r, C)).all())
    if C % 32:
        pad = a.codes.cpu()[:, C:]
        assert bool((pad == (0 if fmt == "e4m3" else 128)).all())
    rs = rstd.double().cpu()
    d = dy.double()
    g = d * scale.double()
    dx, ds, do = H.rownorm_bwd(dy.to(dev), a, scale.to(dev), mean, rstd, kind)
    _close(dx, R.norm_backward(g, v, rs, kind), R.backward_error(g, v, rs), dtype)
    _close(ds, (d * v).sum(0), R.sums_error(d * v, rows))
    _close(do, d.sum(0), R.sums_error(d, rows))


GATES = [(1, 1, 1), (5, 7, 5), (33, 40, 3), (64, 512, 64), (64, 512, None), (300, 256, 1), (300, 256, 15), (77, 250, 77), (320, 640, 2), (768, 129, 48),
         (21, 2048, 7), (6, 2500, 6), (40, 2500, 2), (8192, 96, 512), (20000, 96, 4), (6000, 64, 2000), (4100, 36, 4100)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,groups", GATES)
def test_gated_residual(dev, rows, C, groups, dtype, kind):
    H = _H()
    x, f, dy = _rand(rows, C, 1, dtype), _rand(rows, C, 2, dtype), _rand(rows, C, 3, dtype)
    scale, offset, res = _vec(C, 4), _vec(C, 5, 0.0), _vec(C, 6, 0.4)
    gate = None if groups is None else _rand(groups, C, 7)
    per = rows // (groups or 1)
    gd = None if gate is None else gate.to(dev)
    args = (scale.to(dev), offset.to(dev), gd, res.to(dev))
    out, mean, rstd, _, after = H.gated_residual_fwd(x.to(dev), f.to(dev), *args, EPS, kind)
    assert after is None
    fh, _, r = R.normed(f, kind, EPS)
    G = torch.ones(rows, C, dtype=torch.float64) if gate is None else gate.double().repeat_interleave(per, 0)
    m = G * res.double()
    n = fh * scale.double() + offset.double()
    mag = m.abs() * ((fh * scale.double()).abs() + offset.double().abs())
    _close(out, x.double() + m * n, R.normed_error(f, fh, r, C) * (m * scale.double()).abs() + R.U * (6 * mag + x.double().abs()), dtype)
    # backward
    mu = mean.double().cpu() if mean is not None else torch.zeros(rows, dtype=torch.float64)
    rs = rstd.double().cpu()
    fh = (f.double() - mu[:, None]) * rs[:, None]
    n = fh * scale.double() + offset.double()
    nmag = (fh * scale.double()).abs() + offset.double().abs()
    d = dy.double()
    w = m * scale.double()
    df, ds, do, dg, dr = H.gated_residual_bwd(dy.to(dev), f.to(dev), *args, mean, rstd, kind)
    _close(df, R.norm_backward(d * w, fh, rs, kind), 2 * R.backward_error(d * w, fh, rs), dtype)
    # (A and B are summed apart and combined: the magnitudes that round are |scale A| + |offset B|)
    _close(ds, (d * m * fh).sum(0), R.sums_error(d * m * fh, rows))
    _close(do, (d * m).sum(0), R.sums_error(d * m, rows))
    _close(dr, (d * G * n).sum(0), R.sums_error(d * G * nmag, rows))
    if gate is None:
        assert dg is None
    else:
        assert dg.shape == gate.shape
        t = (d * res.double() * n).reshape(groups, per, C)
        tm = (d * res.double() * nmag).reshape(groups, per, C)
        _close(dg, t.sum(1), torch.stack([R.sums_error(q, per) for q in tm]) if groups <= 64 else R.U * (per / 64 + 68) * tm.abs().sum(1))
    again = H.gated_residual_bwd(dy.to(dev), f.to(dev), *args, mean, rstd, kind)
    for a, b in zip((df, ds, do, dg, dr), again):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(1, 9), (64, 512), (77, 250), (300, 128), (40, 2500), (5, 1000)])
def test_gated_residual_with_the_next_norm_and_checkpoints(dev, rows, C, dtype, fmt):
    """Everything from one pass equals the separate calls bit for bit."""
    H = _H()
    x, f = _rand(rows, C, 1, dtype).to(dev), _rand(rows, C, 2, dtype).to(dev)
    scale, offset, res, s2, o2 = (_vec(C, 10 + i).to(dev) for i in range(5))
    gate = _rand(rows, C, 7, dtype).to(dev)
    plain = H.gated_residual_fwd(x, f, scale, offset, gate, res, EPS, "layer")
    out, mean, rstd, a, after = H.gated_residual_fwd(x, f, scale, offset, gate, res, EPS, "layer", save8=fmt, next_norm=(s2, o2, 1e-3, "rms"),
                                                     next_save8=fmt)
    assert torch.equal(out, plain[0]) and torch.equal(mean, plain[1]) and torch.equal(rstd, plain[2])
    h, m2, r2, a2 = after
    y, my, ry, ay = H.rownorm_fwd(out, s2, o2, 1e-3, "rms", save8=fmt)
    assert m2 is None and my is None and torch.equal(h, y) and torch.equal(r2, ry)
    assert torch.equal(a2.codes, ay.codes) and torch.equal(a2.scales, ay.scales)
    _, _, _, af = H.rownorm_fwd(f, None, None, EPS, "layer", save8=fmt)
    assert torch.equal(a.codes, af.codes) and torch.equal(a.scales, af.scales)
    dy = _rand(rows, C, 3, dtype).to(dev)
    df, ds, do, dg, dr = H.gated_residual_bwd(dy, a, scale, offset, gate, res, mean, rstd, "layer")
    v = H.act8_load(a).double().cpu()
    d, G, rs = dy.double().cpu(), gate.double().cpu(), rstd.double().cpu()
    w = G * (res * 1.0).double().cpu() * scale.double().cpu()
    _close(df, R.norm_backward(d * w, v, rs, "layer"), 2 * R.backward_error(d * w, v, rs), dtype)
    t = d * res.double().cpu() * (v * scale.double().cpu() + offset.double().cpu())
    tm = (d * res.double().cpu()).abs() * ((v * scale.double().cpu()).abs() + offset.double().cpu().abs())
    _close(dg, t, 8 * R.U * tm, dtype)


def test_gradients_are_those_of_differences(dev):
    """df, dgate, dscale, doffset, dres_scale against central differences of the float64 form (step 1e-4: truncation below 1e-6, fp32 below 1e-4)."""
    H = _H()
    rows, C, groups = 6, 20, 3
    t = {"f": _rand(rows, C, 1).double(), "scale": _vec(C, 2).double(), "offset": _vec(C, 3, 0.0).double(), "gate": _rand(groups, C, 4).double(),
         "res": _vec(C, 5, 0.5).double()}
    dy = _rand(rows, C, 6)

    def loss(q):
        fh, _, _ = R.normed(q["f"], "layer", EPS)
        return float((dy.double() * q["res"] * q["gate"].repeat_interleave(rows // groups, 0) * (fh * q["scale"] + q["offset"])).sum())

    f = t["f"].float().to(dev)
    args = [t[k].float().to(dev) for k in ("scale", "offset", "gate", "res")]
    _, mean, rstd, _, _ = H.gated_residual_fwd(f, f, *args, EPS, "layer")
    got = dict(zip(("f", "scale", "offset", "gate", "res"), H.gated_residual_bwd(dy.to(dev), f, *args, mean, rstd, "layer")))
    for k, v in t.items():
        num = torch.empty_like(v).reshape(-1)
        for i in range(v.numel()):
            hi, lo = {n: q.clone() for n, q in t.items()}, {n: q.clone() for n, q in t.items()}
            hi[k].reshape(-1)[i] += 1e-4
            lo[k].reshape(-1)[i] -= 1e-4
            num[i] = (loss(hi) - loss(lo)) / 2e-4
        assert float((got[k].double().cpu().reshape(-1) - num).abs().max()) < 2e-4 * max(1.0, float(num.abs().max())), k


def test_strides_gate_shapes_and_rows_without_any(dev):
    H = _H()
    wide = torch.randn(2, 4, 3, 300, generator=torch.Generator().manual_seed(1)).to(dev)
    x, f = wide[..., 5:105], wide[..., 150:250]
    xc, fc = x.contiguous(), f.contiguous()
    s, o, r = (_vec(100, i).to(dev) for i in (1, 2, 3))
    gate = torch.randn(2, 1, 1, 100, generator=torch.Generator().manual_seed(2)).to(dev)
    a = H.gated_residual_fwd(x, f, s, o, gate, r)
    b = H.gated_residual_fwd(xc.reshape(24, 100), fc.reshape(24, 100), s, o, gate.reshape(2, 100), r)
    assert a[0].shape == x.shape and torch.equal(a[0].reshape(24, 100), b[0])
    full = gate.expand(2, 4, 3, 100)
    assert torch.equal(H.gated_residual_fwd(x, f, s, o, full, r)[0], a[0])
    one = H.gated_residual_fwd(x, f, s, o, gate[0, 0, 0], r)[0]
    assert torch.equal(one[0], a[0][0])
    dx, ds, do, dg, dr = H.gated_residual_bwd(x, f, s, o, gate, r, a[1], a[2])
    assert dg.shape == gate.shape
    e = H.gated_residual_bwd(xc, fc, s, o, gate, r, a[1], a[2])
    for p, q in zip((dx, ds, do, dg, dr), e):
        assert torch.equal(p, q)
    y, mean, rstd, _ = H.rownorm_fwd(x, s, o)
    assert torch.equal(y, H.rownorm_fwd(xc, s, o)[0])
    p, q = H.rownorm_bwd(f, x, s, mean, rstd, accum=x), H.rownorm_bwd(fc, xc, s, mean, rstd, accum=xc)
    assert all(torch.equal(u, v) for u, v in zip(p, q))
    # expanded rows (stride 0) and a transposed view are copied
    row = xc[0, 0, :1]
    assert torch.equal(H.rownorm_fwd(row.expand(5, 100), s, o)[0], H.rownorm_fwd(row.repeat(5, 1), s, o)[0])
    # no rows at all
    z = torch.empty(0, 100, device=dev)
    y, mean, rstd, sv = H.rownorm_fwd(z, s, o, save8="int8")
    assert y.shape == (0, 100) and sv.codes.shape == (0, 128)
    dx, ds, do = H.rownorm_bwd(z, z, s, mean, rstd)
    assert dx.shape == (0, 100) and float(ds.abs().sum() + do.abs().sum()) == 0.0
    assert H.gated_residual_fwd(z, z, s, o, None, r)[0].shape == (0, 100)


def test_values_that_are_not_finite_stay_in_their_rows(dev):
    H = _H()
    x = _rand(40, 96, 1)
    x[3, 5], x[9, 95], x[20, 0] = float("nan"), float("inf"), float("-inf")
    y, mean, rstd, a = H.rownorm_fwd(x.to(dev), None, None, EPS, "layer", save8="e4m3")
    bad = torch.isnan(y).all(1).cpu().nonzero().flatten().tolist()
    assert bad == [3, 9, 20] and bool(torch.isfinite(y.cpu()[[i for i in range(40) if i not in bad]]).all())
    assert (a.scales.cpu() == 255).all(1).nonzero().flatten().tolist() == bad
    big = torch.full((3, 96), 1e25)                                       # squares beyond fp32: rstd = 0, and with it xh
    big[:, ::2] *= -1
    big[1] = torch.randn(96, generator=torch.Generator().manual_seed(3))
    for kind in ("layer", "rms"):
        y, _, rstd, _ = H.rownorm_fwd(big.to(dev), None, None, EPS, kind, save8="int8")
        assert rstd.cpu()[[0, 2]].tolist() == [0.0, 0.0] and float(y[[0, 2]].abs().sum()) == 0.0 and float(y[1].abs().max()) > 1
    z = torch.zeros(4, 96, device=dev)                                    # a row of zeros: xh = 0, not NaN
    y, _, rstd, _ = H.rownorm_fwd(z, None, None, EPS, "rms")
    assert float(y.abs().sum()) == 0.0 and bool(torch.isfinite(rstd).all())


def test_refusals(dev):
    H = _H()
    x = torch.randn(6, 40, device=dev)
    s = torch.ones(40, device=dev)
    y, mean, rstd, a = H.rownorm_fwd(x, s, s, save8="e4m3")
    for call in (lambda: H.rownorm_fwd(x, s, s, kind="batch"), lambda: H.rownorm_fwd(x, s[:39]), lambda: H.rownorm_fwd(x, s.bfloat16()),
                 lambda: H.rownorm_fwd(x.double()), lambda: H.rownorm_fwd(x.cpu()), lambda: H.rownorm_fwd(x[:, :0]),
                 lambda: H.rownorm_fwd(torch.zeros(2, 8193, device=dev)), lambda: H.rownorm_fwd(x, save8="int4"),
                 lambda: H.rownorm_bwd(x, x[:5], s, mean, rstd), lambda: H.rownorm_bwd(x, x.bfloat16(), s, mean, rstd),
                 lambda: H.rownorm_bwd(x, x, s, None, rstd), lambda: H.rownorm_bwd(x, a, s, mean, None),
                 lambda: H.rownorm_bwd(x[:, :39], a, s[:39].contiguous(), mean, rstd), lambda: H.rownorm_bwd(x, x, s, mean[:5], rstd),
                 lambda: H.gated_residual_fwd(x, x[:5]), lambda: H.gated_residual_fwd(x, x, gate=torch.ones(4, 40, device=dev)),
                 lambda: H.gated_residual_fwd(x, x, gate=torch.ones(6, 39, device=dev)), lambda: H.gated_residual_fwd(x, x, gate=torch.ones(6, 40)),
                 lambda: H.gated_residual_fwd(x, x, next_save8="int8"), lambda: H.gated_residual_fwd(x, x, next_norm=(s, s, 1e-5, "none")),
                 lambda: H.gated_residual_fwd(x.reshape(2, 3, 40), x.reshape(2, 3, 40), gate=torch.ones(3, 40, device=dev))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_two_streams_and_graph_replays(dev, dtype):
    """The same calls on two streams at once and captured into two graphs give the eager bits; eager work runs between the replays."""
    H = _H()
    rows, C = 4000, 384
    s, o, r = (_vec(C, i).to(dev) for i in (1, 2, 3))
    data = [[_rand(rows, C, 10 * k + i, dtype).to(dev) for i in range(3)] + [_rand(8, C, 10 * k + 4).to(dev)] for k in range(2)]

    def work(x, f, dy, gate):
        out, mean, rstd, a, after = H.gated_residual_fwd(x, f, s, o, gate, r, save8="e4m3", next_norm=(s, o, EPS, "rms"), next_save8="int8")
        back = H.gated_residual_bwd(dy, a, s, o, gate, r, mean, rstd)
        dx = H.rownorm_bwd(dy, after[3], s, after[1], after[2], "rms", accum=back[0])
        dw = H.linear_wgrad8(after[3], dy, scale=s, offset=o, want_bias=True)
        return [out, after[0]] + list(back) + list(dx) + list(dw)

    want = [[t.clone() for t in work(*d)] for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for k in range(2):
            streams[k].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[k]):
                got[k] = work(*data[k])
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(*data[k]))
        graphs.append(g)
    for rep in range(4):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k])), rep
        for t in work(*data[rep % 2]):
            float(t.float().sum())


def test_rows_beyond_32_bit_offsets(dev):
    """2^31 elements and more: the last rows are what a small call on them gives, bit for bit."""
    H = _H()
    rows, C = 270000, 8192
    x = torch.empty(rows, C, dtype=BF16, device=dev)
    x[:16] = 0
    x[16:] = 1
    g = torch.Generator(device=dev).manual_seed(1)
    x[-40:] = torch.randn(40, C, generator=g, device=dev).to(BF16)
    s, o, r = (_vec(C, i).to(dev) for i in (1, 2, 3))
    tail = x[-40:].clone()
    y, mean, rstd, a = H.rownorm_fwd(x, s, o, save8="int8")
    y2, mean2, rstd2, a2 = H.rownorm_fwd(tail, s, o, save8="int8")
    assert torch.equal(y[-40:], y2) and torch.equal(rstd[-40:], rstd2) and torch.equal(a.codes[-40:], a2.codes) and torch.equal(a.scales[-40:], a2.scales)
    assert float(y[:16].float().sub(o).abs().max()) < 0.02 * float(o.abs().max())
    dx = H.rownorm_bwd(x, a, s, mean, rstd, accum=y, want_params=False)[0]
    assert torch.equal(dx[-40:], H.rownorm_bwd(tail, a2, s, mean2, rstd2, accum=y2, want_params=False)[0])
    del dx
    gate = x[-rows:]
    out = H.gated_residual_fwd(x, y, s, o, gate, r)[0]
    assert torch.equal(out[-40:], H.gated_residual_fwd(tail, y2, s, o, tail, r)[0])
    del out, y
    q = H.act8_store(x, "e4m3")
    assert torch.equal(q.codes[-40:], H.act8_store(tail, "e4m3").codes)
    z = H.act8_load(q, BF16)
    assert torch.equal(z[-40:], H.act8_load(H.act8_store(tail, "e4m3"), BF16))
    assert torch.equal(H.act8_act_bwd(x, q, 1)[-40:], torch.where(tail > 0, tail, torch.zeros_like(tail)))
    # a filter gradient whose dy is a slice of rows 8192 apart; integers, so that every order of the sum is exact
    del z, q
    x.copy_(torch.randint(-2, 3, (rows, 1), generator=g, device=dev).to(BF16).expand(rows, C))
    act = torch.randint(-8, 9, (rows, 40), generator=g, device=dev).float()
    dw, db = H.linear_wgrad8(H.act8_store(act, "int8"), x[:, 8:24], want_bias=True)
    assert torch.equal(dw.double(), act.double().t().contiguous() @ x[:, 8:24].double()) and torch.equal(db.double(), x[:, 8:24].double().sum(0))


def test_a_tensor_of_another_device_is_refused(dev):
    H = _H()
    with pytest.raises(RuntimeError, match="current device"):
        H._on_current(torch.device("cuda", torch.cuda.current_device() + 1), "x")


@pytest.mark.parametrize("rows,C,groups", [(96, 200, 4), (640, 64, 20), (40, 130, 20), (33 * 64, 96, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bf16_gates(dev, rows, C, groups, dtype):
    """A bf16 gate per group, in every form: what the same gate in fp32 gives; its gradient is that one rounded."""
    H = _H()
    x, f, dy = (_rand(rows, C, i, dtype).to(dev) for i in (1, 2, 3))
    s, o, r = (_vec(C, i).to(dev) for i in (1, 2, 3))
    gate = _rand(groups, C, 4, BF16).to(dev)
    a, b = H.gated_residual_fwd(x, f, s, o, gate, r), H.gated_residual_fwd(x, f, s, o, gate.float(), r)
    assert torch.equal(a[0], b[0])
    p, q = (H.gated_residual_bwd(dy, f, s, o, g, r, a[1], a[2]) for g in (gate, gate.float()))
    assert p[3].dtype == BF16 and torch.equal(p[3], q[3].to(BF16))
    for k in (0, 1, 2, 4):
        assert torch.equal(p[k], q[k])


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("C,ld", [(64, 80), (37, 45), (250, 256)])
def test_strided_results_leave_what_lies_between_their_rows(dev, bf16, C, ld):
    """The C entries with row strides of their own: nothing is written between the rows, before the first or behind the last."""
    from dpig_amd import _lib
    h, rows, dt = _lib.lib(), 70, BF16 if bf16 else F32
    st = _lib.stream_ptr()

    def field():
        return torch.full((rows + 2, ld), 7.0, dtype=dt, device=dev)

    def inside(t):
        return t.view(-1)[ld + 3:].as_strided((rows, C), (ld, 1))

    def check(t, want):
        assert torch.equal(inside(t), want)
        inside(t).fill_(7.0)
        assert bool((t == 7.0).all())
    H = _H()
    x, f, dy = (_rand(rows, C, i, dt).to(dev) for i in (1, 2, 3))
    s, o = _vec(C, 1).to(dev), _vec(C, 2).to(dev)
    m, r, m2, r2 = torch.empty(4, rows, device=dev).unbind(0)
    P = lambda t: t.data_ptr()      # noqa: E731
    y, hh = field(), field()
    assert h.dpig_rownorm_fwd(P(x), bf16, C, rows, C, 0, P(s), P(o), EPS, P(inside(y)), ld, P(m), P(r), 0, None, None, st) == 0
    check(y, H.rownorm_fwd(x, s, o)[0])
    assert h.dpig_gated_residual_fwd(P(x), C, P(f), C, bf16, rows, C, 0, P(s), P(o), EPS, None, 0, 0, None, P(inside(y)), ld, P(m), P(r), 0, None, None,
                                     0, P(s), P(o), EPS, P(inside(hh)), ld, P(m2), P(r2), 0, None, None, st) == 0
    out, mean, rstd, _, after = H.gated_residual_fwd(x, f, s, o, next_norm=(s, o, EPS, "layer"))
    check(y, out)
    check(hh, after[0])
    assert h.dpig_gated_residual_bwd(P(dy), bf16, C, P(f), C, 0, None, None, rows, C, 0, P(s), P(o), None, 0, 0, None, P(mean), P(rstd), P(inside(y)), ld,
                                     None, None, None, None, None, 0, st) == 0
    check(y, H.gated_residual_bwd(dy, f, s, o, None, None, mean, rstd, want_params=False)[0])
    a = H.act8_store(x, "int8")
    assert h.dpig_act8_load(P(a.codes), P(a.scales), rows, C, 1, P(inside(y)), bf16, ld, st) == 0
    check(y, H.act8_load(a, dt))
    assert h.dpig_act8_act_bwd(P(dy), bf16, C, P(a.codes), rows, C, 1, 2, 0.2, P(inside(y)), ld, st) == 0
    check(y, H.act8_act_bwd(dy, a, 2))


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows,C,groups", [(3000, 37, 3000), (3000, 250, 6), (600, 1100, 20), (64, 512, 64)])
def test_results_in_place_of_an_operand(dev, bf16, rows, C, groups):
    """The C entries with y = x, out = x, out = f, df = dout, dx = dy and dx = accum give the bits of separate results."""
    from dpig_amd import _lib
    h, dt, H = _lib.lib(), BF16 if bf16 else F32, _H()
    st = _lib.stream_ptr()
    P = lambda t: t.data_ptr()      # noqa: E731
    x, f, dy, acc = (_rand(rows, C, i, dt).to(dev) for i in (1, 2, 3, 4))
    s, o, r = (_vec(C, i).to(dev) for i in (1, 2, 3))
    gate = _rand(groups, C, 5).to(dev)
    m, q = torch.empty(2, rows, device=dev).unbind(0)
    y = H.rownorm_fwd(x, s, o)[0]
    t = x.clone()
    assert h.dpig_rownorm_fwd(P(t), bf16, C, rows, C, 0, P(s), P(o), EPS, P(t), C, P(m), P(q), 0, None, None, st) == 0
    assert torch.equal(t, y)
    out, mean, rstd, _, _ = H.gated_residual_fwd(x, f, s, o, gate, r)
    for k in range(2):
        a = [x.clone(), f.clone()]
        assert h.dpig_gated_residual_fwd(P(a[0]), C, P(a[1]), C, bf16, rows, C, 0, P(s), P(o), EPS, P(gate), 0, groups, P(r), P(a[k]), C, P(m), P(q), 0, None,
                                         None, 0, None, None, 0.0, None, 0, None, None, 0, None, None, st) == 0
        assert torch.equal(a[k], out)
    df = H.gated_residual_bwd(dy, f, s, o, gate, r, mean, rstd, want_params=False)[0]
    t = dy.clone()
    assert h.dpig_gated_residual_bwd(P(t), bf16, C, P(f), C, 0, None, None, rows, C, 0, P(s), P(o), P(gate), 0, groups, P(r), P(mean), P(rstd), P(t), C,
                                     None, None, None, None, None, 0, st) == 0
    assert torch.equal(t, df)
    dx = H.rownorm_bwd(dy, f, s, mean, rstd, accum=acc, want_params=False)[0]
    for k in range(2):
        a = [dy.clone(), acc.clone()]
        assert h.dpig_rownorm_bwd(P(a[0]), bf16, C, P(f), C, 0, None, None, rows, C, 0, P(s), P(mean), P(rstd), P(a[1]), C, P(a[k]), C, None, None, None, 0,
                                  st) == 0
        assert torch.equal(a[k], dx)


def test_layers_without_rows(dev):
    """No rows: empty results, zero gradients, through the autograd functions and the registry layers."""
    from dpig_amd import autograd as A
    for fmt in (None, "int8"):
        x = torch.zeros(0, 64, device=dev, requires_grad=True)
        f = torch.zeros(0, 64, device=dev, requires_grad=True)
        s, o, r = (_vec(64, i).to(dev).requires_grad_(True) for i in (1, 2, 3))
        h = A.rownorm(x, s, o, save8=fmt)
        y = A.gated_residual(h, f, s, o, None, r, save8=fmt)
        assert y.shape == (0, 64)
        y.sum().backward()
        assert x.grad.shape == (0, 64) and f.grad.shape == (0, 64)
        assert all(float(t.grad.abs().sum()) == 0.0 for t in (s, o, r))
