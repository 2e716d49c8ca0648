"""8-bit activation checkpoints: codes, scales and values against a float64 restatement, bit for bit, and the filter gradient that reads them."""
import pytest
import torch

import rows_reference as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _H():
    import dpig_amd.hip_ops as H
    return H


def _same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    assert a.shape == b.shape
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), (torch.nan_to_num(a) - torch.nan_to_num(b)).abs().max()


def _check_store(x, fmt):
    H = _H()
    a = H.act8_store(x, fmt)
    C = x.shape[-1]
    codes, scales, values = R.checkpoint(x.reshape(-1, C), fmt)
    assert a.shape == tuple(x.shape) and a.nbytes == codes.numel() + scales.numel()
    assert torch.equal(a.scales.cpu(), scales)
    zero = 0 if fmt == "e4m3" else 128
    dead = (scales == 255).repeat_interleave(32, 1)
    assert bool((a.codes.cpu()[dead] == zero).all())
    got, want = a.codes.cpu()[~dead], codes[~dead]
    if fmt == "e4m3":                                                     # (the two zeros are one value)
        got, want = torch.where(got == 128, torch.zeros_like(got), got), torch.where(want == 128, torch.zeros_like(want), want)
    assert torch.equal(got, want)
    for dt in (F32, BF16):
        y = H.act8_load(a, dt)
        assert y.dtype == dt and y.shape == x.shape
        _same(y.reshape(-1, C), values)                                  # exact in both types
    return a


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 31), (3, 32), (7, 33), (64, 512), (129, 250), (1000, 96), (5, 2100), (70001, 8)])
def test_store_and_load_are_exact(dev, rows, C, dtype, fmt):
    g = torch.Generator().manual_seed(rows * 31 + C)
    x = torch.randn(rows, C, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    x = torch.relu(x) if C % 2 else x
    _check_store(x.to(dtype).to(dev), fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_every_bf16_value_and_the_edges_of_the_scales(dev, fmt):
    """Every bf16 bit pattern beside a large, a middle and no neighbour; infinities and NaNs; amax on and beside the format's edge."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    x = torch.zeros(65536, 96, dtype=BF16)
    x[:, 0] = bits
    x[:, 40] = bits
    x[:, 63] = 1.0
    x[:, 65] = bits
    x[:, 95] = bits.flip(0)
    _check_store(x.to(dev), fmt)
    m = R.MOST[fmt]
    rows = []
    for e in (-120, -116, -100, -20, 0, 15, 100, 118, 119):
        for f in (m, m * (1 + 2.0 ** -23), m * (1 - 2.0 ** -24), m / 2, m * 1.5):
            v = torch.zeros(32, dtype=torch.float64)
            v[0], v[1], v[2], v[3], v[4] = f, m * 0.0009, -m * 0.3, 2.0 ** -10, 0.5
            rows.append((v * 2.0 ** e).float())
    rows += [torch.full((32,), t) for t in (3.4028234663852886e38, -1e-45, 0.0, -0.0)]
    _check_store(torch.stack(rows).to(dev), fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_relu_outputs_mask_survives(dev, fmt):
    H = _H()
    g = torch.Generator().manual_seed(3)
    y = torch.relu(torch.randn(257, 250, generator=g)) * torch.exp(8 * torch.randn(257, 250, generator=g))
    dy = torch.randn(257, 250, generator=g)
    a = H.act8_store(y.to(dev), fmt)
    for act, off in ((1, 0.0), (2, 0.2)):
        for dt in (F32, BF16):
            d = dy.to(dt).to(dev)
            z = H.act8_act_bwd(d, a, act, 0.2)
            assert z.dtype == dt
            want = d.float().cpu() * torch.where(y > 0, torch.tensor(1.0), torch.tensor(off))
            assert torch.equal(z.cpu(), want.to(dt))
    y[5, 7] = float("nan")                                              # the whole group reads as a NaN: not positive
    a = H.act8_store(y.to(dev), fmt)
    z = H.act8_act_bwd(torch.ones(257, 250, device=dev), a, 1)
    assert float(z[5, :32].abs().sum()) == 0.0


def test_strided_rows_and_other_ranks(dev):
    H = _H()
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(4, 6, 5, 200, generator=g).to(dev)
    x = wide[..., 17:81]                                                # a channel slice: rows 200 apart, 4-byte aligned
    a = H.act8_store(x, "int8")
    b = H.act8_store(x.contiguous(), "int8")
    assert a.shape == (4, 6, 5, 64) and torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    t = torch.randn(70, 48, generator=g).to(dev).t()                    # columns as rows: copied
    a, b = H.act8_store(t, "e4m3"), H.act8_store(t.contiguous(), "e4m3")
    assert torch.equal(a.codes, b.codes)
    assert H.act8_load(H.act8_store(torch.randn(3, 0, 5, 8, device=dev)[..., :8].reshape(0, 8), "e4m3")).shape == (0, 8)
    v = torch.randn(33, generator=g).to(dev)                            # one row
    _same(H.act8_load(H.act8_store(v, "e4m3"))[None], R.checkpoint(v[None], "e4m3")[2])


# ---- the filter gradient ---------------------------------------------------------------------------------------------------------------
def _operands(rows, C, K, dtype, fmt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.relu(torch.randn(rows, C, generator=g)) * torch.exp(torch.randn(C, generator=g))
    return x, torch.randn(rows, K, generator=g).to(dtype), 1 + 0.2 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)


def _check_wgrad(dw, db, values, dy, scale, offset, rows):
    """A sum of `rows` products, in three terms each for fp32 dy: at most 3 rows + 80 roundings of partial sums no larger than the sum of
    magnitudes, elementwise; and as roundings of a random walk, whose errors add up to U sqrt(3 rows) / 2 of its length, eight times that in the norm."""
    v, d = values, dy.double().cpu()
    sc = torch.ones(v.shape[1], dtype=torch.float64) if scale is None else scale.double()
    of = torch.zeros(v.shape[1], dtype=torch.float64) if offset is None else offset.double()
    ref = (v * sc + of).t() @ d
    mag = (v * sc).abs().t() @ d.abs() + of.abs()[:, None] * d.abs().sum(0)
    err = (dw.double().cpu() - ref).abs()
    assert bool((err <= R.U * (3 * rows + 80) * mag).all()), (err / mag).max()
    assert float(err.norm()) <= R.U * (4 * (3 * rows) ** 0.5 + 16) * max(float(ref.norm()), float((mag / rows ** 0.5).norm()))
    if db is not None:
        e = (db.double().cpu() - d.sum(0)).abs()
        assert bool((e <= R.U * (rows / 16 + 64) * d.abs().sum(0)).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,K", [(1, 1, 1), (2, 33, 7), (64, 512, 512), (65, 128, 130), (100, 250, 390), (1000, 64, 8), (4097, 96, 264),
                                      (20011, 130, 100)])
def test_linear_wgrad8(dev, rows, C, K, dtype, fmt):
    H = _H()
    x, dy, scale, offset = _operands(rows, C, K, dtype, fmt, rows + C + K)
    a = H.act8_store(x.to(dev), fmt)
    values = R.checkpoint(x, fmt)[2]
    d = dy.to(dev)
    dw = H.linear_wgrad8(a, d)
    _check_wgrad(dw, None, values, dy, None, None, rows)
    dw, db = H.linear_wgrad8(a, d, scale=scale.to(dev), offset=offset.to(dev), want_bias=True)
    _check_wgrad(dw, db, values, dy, scale, offset, rows)
    dw2, db2 = H.linear_wgrad8(a, d, scale=scale.to(dev), offset=offset.to(dev), want_bias=True)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)                   # fixed order
    # accumulate into given buffers
    out, b = torch.ones(C, K, device=dev), torch.ones(K, device=dev)
    H.linear_wgrad8(a, d, offset=offset.to(dev), out=out, beta=0.5, db=b, db_beta=2.0)
    ref = (values + offset.double()).t() @ dy.double() + 0.5
    mag = (values.abs() + offset.double().abs()).t() @ dy.double().abs() + 1
    assert bool(((out.double().cpu() - ref).abs() <= R.U * (3 * rows + 90) * mag).all())
    assert bool(((b.double().cpu() - dy.double().sum(0) - 2).abs() <= R.U * (rows / 16 + 64) * (dy.double().abs().sum(0) + 2)).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,K", [(3000, 300, 200), (17, 140, 260), (129, 512, 128), (2049, 40, 640), (9000, 257, 129)])
def test_linear_wgrad8_of_integers_is_exact(dev, rows, C, K, dtype):
    """Integers whose sums stay below 2^24: every product and sum is exact, so a misplaced element shows whole."""
    H = _H()
    g = torch.Generator().manual_seed(rows)
    q = torch.randint(-100, 101, (rows, C), generator=g)
    q[:, ::32] = 100                                                    # (the group's scale is 2^0)
    dy = torch.randint(-3, 4, (rows, K), generator=g)
    a = H.act8_store(q.float().to(dev), "int8")
    assert bool((a.scales == 127).all())
    dw, db = H.linear_wgrad8(a, dy.to(dtype).to(dev), want_bias=True)
    assert torch.equal(dw.cpu().double(), q.double().t() @ dy.double())
    assert torch.equal(db.cpu().double(), dy.double().sum(0))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(128, 300), (131, 64), (640, 130)])
def test_linear_wgrad8_reads_every_value_exactly(dev, rows, C, dtype, fmt):
    """dy the identity: dw is the checkpoint's values transposed, whatever their sizes."""
    H = _H()
    g = torch.Generator().manual_seed(C)
    x = torch.randn(rows, C, generator=g) * torch.exp(12 * torch.randn(rows, C, generator=g))
    x[0, :8] = torch.tensor([3.4e38, -3.4e38, 1e-30, -1e-38, 1e-44, 0.0, 2.0 ** 127, -1.9 * 2.0 ** 126])
    a = H.act8_store(x.to(dev), fmt)
    dw, db = H.linear_wgrad8(a, torch.eye(rows, dtype=dtype, device=dev), want_bias=True)
    assert torch.equal(dw.double().cpu(), R.checkpoint(x, fmt)[2].t().contiguous())
    assert torch.equal(db.cpu(), torch.ones(rows))


# the 256 x 128 tile is taken above 10^10 products (fp32 dy: a third of that)
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,C,K,dtype", [(90001, 250, 520, BF16), (90001, 250, 519, BF16), (140001, 500, 520, BF16), (140001, 512, 513, BF16),
                                              (80001, 200, 260, F32)])
def test_linear_wgrad8_large_tiles_are_exact_on_integers(dev, rows, C, K, dtype, fmt):
    H = _H()
    g = torch.Generator(device=dev).manual_seed(rows)
    q = torch.randint(-8, 9, (rows, C), generator=g, device=dev).float()        # (both formats hold these as they are)
    dy = torch.randint(-3, 4, (rows, K), generator=g, device=dev)
    dw, db = H.linear_wgrad8(H.act8_store(q, fmt), dy.to(dtype), want_bias=True)
    want = q.double().t().contiguous() @ dy.double()
    assert torch.equal(dw.double(), want) and torch.equal(db.double(), dy.double().sum(0))


@pytest.mark.parametrize("rows", [40, 3000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_wgrad8_adds_into_given_buffers(dev, rows, dtype):
    """beta and db_beta without an affine part, written in place (few rows) and joined (many)."""
    H = _H()
    g = torch.Generator().manual_seed(rows)
    q, dy = torch.randint(-9, 10, (rows, 70), generator=g), torch.randint(-3, 4, (rows, 50), generator=g)
    out, db = torch.full((70, 50), 2.0, device=dev), torch.full((50,), 3.0, device=dev)
    H.linear_wgrad8(H.act8_store(q.float().to(dev), "int8"), dy.to(dtype).to(dev), out=out, beta=0.5, db=db, db_beta=2.0)
    assert torch.equal(out.double().cpu(), q.double().t() @ dy.double() + 1) and torch.equal(db.double().cpu(), dy.double().sum(0) + 6)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_linear_wgrad8_strides_and_not_finite_values(dev, fmt):
    H = _H()
    x, dy, _, _ = _operands(300, 70, 90, F32, fmt, 9)
    big = H.linear_wgrad8(H.act8_store(x.to(dev), fmt), torch.full((300, 4), 3.4e38, device=dev) * torch.tensor([1.0, -1.0, 0.0, 1e-30], device=dev))
    assert bool(torch.isfinite(big[:, 2:]).all()) and not bool(torch.isnan(big).any())       # (finite, however large: no NaN)
    x[11, 40] = float("inf")
    wide = torch.randn(300, 128)
    wide[:, 3:93] = dy
    a = H.act8_store(x.to(dev), fmt)
    dw = H.linear_wgrad8(a, wide.to(dev)[:, 3:93])
    bad = torch.isnan(dw).all(1).cpu()
    assert bad.nonzero().flatten().tolist() == list(range(32, 64))        # the group that held the infinity, and nothing else
    x[11, 40] = 0
    ref = H.linear_wgrad8(H.act8_store(x.to(dev), fmt), dy.to(dev))
    keep = ~bad
    assert torch.equal(dw.cpu()[keep], ref.cpu()[keep])
    d4 = torch.randn(4, 5, 15, 90)                                       # channel-last maps: rows are the pixels
    assert torch.equal(H.linear_wgrad8(a, d4.to(dev))[:32], H.linear_wgrad8(a, d4.reshape(300, 90).to(dev))[:32])
    z = H.Act8(torch.empty(0, 96, dtype=torch.uint8, device=dev), torch.empty(0, 3, dtype=torch.uint8, device=dev), (0, 70), "int8")
    dw, db = H.linear_wgrad8(z, torch.empty(0, 90, device=dev), want_bias=True)
    assert dw.shape == (70, 90) and float(dw.abs().sum()) == 0.0 and float(db.abs().sum()) == 0.0


def test_refusals(dev):
    H = _H()
    x = torch.randn(6, 40, device=dev)
    a = H.act8_store(x, "e4m3")
    for call in (lambda: H.act8_store(x, "e5m2"), lambda: H.act8_store(x.half()), lambda: H.act8_store(x.cpu()), lambda: H.act8_store(x[:, :0]),
                 lambda: H.act8_load(a, torch.float16), lambda: H.act8_act_bwd(x[:5], a, 1), lambda: H.act8_act_bwd(x, a, 0),
                 lambda: H.linear_wgrad8(a, x[:5]), lambda: H.linear_wgrad8(a, x, scale=x[0, :39].contiguous()),
                 lambda: H.linear_wgrad8(a, x, out=torch.empty(40, 39, device=dev)), lambda: H.linear_wgrad8(a, x, db=torch.empty(40)),
                 lambda: H.Act8(a.codes[:, :32], a.scales, (6, 40), "e4m3"), lambda: H.Act8(a.codes, a.scales, (5, 40), "e4m3")):
        with pytest.raises(RuntimeError):
            call()


# the 256 x 256 generator's fully connected layer has 163840 inputs at its full width: more than a checkpoint's product takes (32768)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C,K", [(5, 40000, 3), (33, 40, 40000), (64, 32769, 33), (1, 163840, 64)])
def test_linear_wgrad8_of_wide_matrices_is_exact_on_integers(dev, rows, C, K, dtype):
    H = _H()
    g = torch.Generator(device=dev).manual_seed(rows)
    q = torch.randint(-8, 9, (rows, C), generator=g, device=dev).float()
    dy = torch.randint(-3, 4, (rows, K), generator=g, device=dev)
    scale, offset = (torch.randint(1, 4, (C,), generator=g, device=dev).float() for _ in range(2))
    a, d = H.act8_store(q, "int8"), dy.to(dtype)
    want, sums = q.double().t().contiguous() @ dy.double(), dy.double().sum(0)
    assert torch.equal(H.linear_wgrad8(a, d).double(), want)
    dw, db = H.linear_wgrad8(a, d, scale=scale, offset=offset, want_bias=True)
    affine = want * scale.double()[:, None] + offset.double()[:, None] * sums
    assert torch.equal(dw.double(), affine) and torch.equal(db.double(), sums)
    out, b = torch.full((C, K), 2.0, device=dev), torch.full((K,), 3.0, device=dev)
    r = H.linear_wgrad8(a, d, offset=offset, out=out, beta=0.5, db=b, db_beta=2.0)
    assert r[0] is out and r[1] is b
    assert torch.equal(out.double(), want + offset.double()[:, None] * sums + 1) and torch.equal(b.double(), sums + 6)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_wgrad8_of_rows_far_apart(dev, dtype):
    """Rows of dy more than 2^22 elements apart: copied together first."""
    H = _H()
    g = torch.Generator(device=dev).manual_seed(1)
    ld, rows = (1 << 22) + 64, 4
    q, dy = torch.randint(-8, 9, (rows, 40), generator=g, device=dev).float(), torch.randint(-3, 4, (rows, 24), generator=g, device=dev).to(dtype)
    wide = torch.empty(rows * ld, dtype=dtype, device=dev).as_strided((rows, 24), (ld, 1))
    wide.copy_(dy)
    dw, db = H.linear_wgrad8(H.act8_store(q, "int8"), wide, want_bias=True)
    assert torch.equal(dw.double(), q.double().t().contiguous() @ dy.double()) and torch.equal(db.double(), dy.double().sum(0))


# the 256 x 256 tile is taken from 2^36 products on where it pads no more than 9 / 8 of what 256 x 128 does (the shapes above do)
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,C,K", [(270000, 510, 512), (270001, 512, 511), (270017, 250, 1021), (120031, 760, 766)])
def test_linear_wgrad8_largest_tiles_are_exact_on_integers(dev, rows, C, K, fmt):
    test_linear_wgrad8_large_tiles_are_exact_on_integers(dev, rows, C, K, BF16, fmt)
