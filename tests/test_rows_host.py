"""Residual-block operators on rows of channels: argument checks and workspace plans of the C entries (host code: no device is touched), and the Python
layer's refusals on the CPU."""
import pytest
import torch

EINVAL, EALIGN, ENOMEM = -22, -14, -12


@pytest.fixture(scope="module")
def h():
    import __graft_entry__
    __graft_entry__.build()
    from dpig_amd import _lib
    return _lib.lib()


P = 4096          # a pointer that is never followed


def _err(h, rc, code, text):
    assert rc == code, (rc, h.dpig_last_error())
    assert text in h.dpig_last_error().decode(), h.dpig_last_error()


def test_act8_entries_refuse(h):
    _err(h, h.dpig_act8_store(P, 0, 64, 4, 64, 2, P, P, None), EINVAL, "format")
    _err(h, h.dpig_act8_store(P, 0, 63, 4, 64, 0, P, P, None), EINVAL, "stride")
    _err(h, h.dpig_act8_store(None, 0, 64, 4, 64, 0, P, P, None), EINVAL, "null")
    _err(h, h.dpig_act8_store(P, 0, 64, 0, 64, 0, P, P, None), EINVAL, "shape")
    _err(h, h.dpig_act8_store(P, 0, 64, 4, 64, 0, P + 8, P, None), EALIGN, "aligned")
    _err(h, h.dpig_act8_load(P, None, 4, 64, 0, P, 0, 64, None), EINVAL, "null")
    _err(h, h.dpig_act8_load(P, P, 4, 64, 0, P, 0, 60, None), EINVAL, "stride")
    _err(h, h.dpig_act8_act_bwd(P, 0, 64, P, 4, 64, 0, 0, 0.2, P, 64, None), EINVAL, "ReLU")
    _err(h, h.dpig_act8_act_bwd(P, 0, 64, P, 4, 64, 7, 1, 0.2, P, 64, None), EINVAL, "format")


def test_norm_entries_refuse(h):
    def fwd(ldx=64, rows=4, C=64, kind=0, ldy=64, m=P, fmt=0, c=None, q=None):
        return h.dpig_rownorm_fwd(P, 0, ldx, rows, C, kind, P, P, 1e-5, P, ldy, m, P, fmt, c, q, None)
    _err(h, fwd(C=8193, ldx=9000, ldy=9000), EINVAL, "channels")
    _err(h, fwd(C=0), EINVAL, "channels")
    _err(h, fwd(rows=0), EINVAL, "row count")
    _err(h, fwd(kind=2), EINVAL, "kind")
    _err(h, fwd(m=None), EINVAL, "null")
    _err(h, fwd(ldy=63), EINVAL, "stride")
    _err(h, fwd(c=P), EINVAL, "codes and scales")
    _err(h, fwd(c=P, q=P, fmt=5), EINVAL, "format")
    _err(h, fwd(c=P + 4, q=P), EALIGN, "aligned")
    n = h.dpig_rownorm_bwd_workspace_bytes(1000, 64)

    def bwd(x=P, c=None, q=None, r=P, ws=P, nb=n, m=P):
        return h.dpig_rownorm_bwd(P, 0, 64, x, 64, 0, c, q, 1000, 64, 0, P, m, r, None, 0, P, 64, P, P, ws, nb, None)
    _err(h, bwd(c=P, q=P), EINVAL, "exactly one")
    _err(h, bwd(x=None), EINVAL, "exactly one")
    _err(h, bwd(x=None, c=P), EINVAL, "codes and scales")
    _err(h, bwd(m=None), EINVAL, "null")
    _err(h, bwd(r=None), EINVAL, "null")
    _err(h, bwd(nb=n - 1), ENOMEM, "workspace")
    _err(h, bwd(ws=None), ENOMEM, "workspace")


def test_gated_residual_entries_refuse(h):
    def fwd(rows=12, gate=P, groups=4, hh=None, k2=0, m2=P, ldo=64):
        return h.dpig_gated_residual_fwd(P, 64, P, 64, 0, rows, 64, 0, P, P, 1e-5, gate, 0, groups, P, P, ldo, P, P, 0, None, None, k2, P, P, 1e-5, hh, 64,
                                         m2, P, 0, None, None, None)
    _err(h, fwd(groups=5), EINVAL, "groups")
    _err(h, fwd(groups=0), EINVAL, "groups")
    _err(h, fwd(ldo=1), EINVAL, "stride")
    _err(h, fwd(hh=P, k2=9), EINVAL, "kind")
    _err(h, fwd(hh=P, m2=None), EINVAL, "next norm")

    def bwd(gate=P, groups=4, dgate=P, nb=1 << 20):
        return h.dpig_gated_residual_bwd(P, 0, 64, P, 64, 0, None, None, 12, 64, 0, P, P, gate, 0, groups, P, P, P, P, 64, P, P, dgate, P, P, nb, None)
    _err(h, bwd(groups=7), EINVAL, "groups")
    _err(h, bwd(gate=None), EINVAL, "without a gate")
    _err(h, bwd(nb=0), ENOMEM, "workspace")


def test_linear_wgrad8_refuses(h):
    def call(rows=100, C=64, K=48, ldy=48, fmt=0, codes=P, dw=P, scale=None, ws=None, nb=0):
        return h.dpig_linear_wgrad8(codes, P, fmt, rows, C, P, 0, ldy, K, scale, None, dw, 0.0, P, 0.0, ws, nb, None)
    _err(h, call(fmt=2), EINVAL, "format")
    _err(h, call(ldy=47), EINVAL, "stride")
    _err(h, call(ldy=(1 << 22) + 1), EINVAL, "stride")
    _err(h, call(rows=0), EINVAL, "shape")
    _err(h, call(C=40000), EINVAL, "shape")
    _err(h, call(rows=(1 << 30) + 1), EINVAL, "shape")
    _err(h, call(dw=None), EINVAL, "null")
    _err(h, call(codes=P + 8), EALIGN, "aligned")
    _err(h, call(scale=P), ENOMEM, "workspace")                 # an affine part is folded in where the sums are joined
    assert h.dpig_linear_wgrad8_workspace_bytes(64, 512, 512, 512, 0, 0) == 0      # few rows: written in place
    assert h.dpig_linear_wgrad8_workspace_bytes(64, 512, 512, 512, 0, 1) > 0
    assert h.dpig_linear_wgrad8_workspace_bytes(64, 512, 500, 512, 0, 1) == 0      # (a bad descriptor: no size)


@pytest.mark.parametrize("C", [1, 8, 64, 65, 130, 384, 640, 1000, 2048, 5000, 8192])
@pytest.mark.parametrize("rows", [1, 7, 64, 4096, 131072, 1 << 22])
def test_workspace_plans_are_bounded(h, rows, C):
    """At most two workgroups a CU leave partial sums (a piece per group at least), so the scratch stays far below the operands."""
    n = h.dpig_rownorm_bwd_workspace_bytes(rows, C)
    assert 8 * C <= n <= 8 * C * min(rows, 512)
    for groups in (1, 2, 16, 64, rows):
        if rows % groups == 0:
            g = h.dpig_gated_residual_bwd_workspace_bytes(rows, C, groups)
            assert 8 * C <= g <= 8 * C * (max(1024, min(groups, rows // 16) + 256) + 1024)
    assert h.dpig_gated_residual_bwd_workspace_bytes(rows, C, 0) == n
    if rows > 1:
        assert h.dpig_gated_residual_bwd_workspace_bytes(rows, C, rows - 1) in (0, h.dpig_gated_residual_bwd_workspace_bytes(rows, C, 1) if rows == 2 else 0)
    w = h.dpig_linear_wgrad8_workspace_bytes(rows, C, 256, 256, 1, 1)
    assert 0 < w <= 4 * 260 * (C + 256) * 384


def test_python_layer_refuses_on_the_cpu():
    import dpig_amd.autograd as A
    import dpig_amd.hip_ops as H
    x = torch.zeros(4, 40)
    a = H.Act8(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), (2, 2, 40), "int8")
    assert a.nbytes == 4 * 66 and a.shape == (2, 2, 40)
    for call in (lambda: H.act8_store(x), lambda: H.act8_load(a), lambda: H.rownorm_fwd(x), lambda: H.gated_residual_fwd(x, x),
                 lambda: H.linear_wgrad8(a, x), lambda: H.act8_act_bwd(x, a, 1)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    for bad in (lambda: H.Act8(a.codes, a.scales, (4, 65), "int8"), lambda: H.Act8(a.codes, a.scales, (4, 40), "fp8"),
                lambda: H.Act8(a.codes.float(), a.scales, (4, 40), "int8"), lambda: H.Act8(a.codes, a.scales, (4, 0), "int8"),
                lambda: H.Act8(a.codes.t().contiguous().t(), a.scales, (4, 40), "int8"), lambda: H.Act8(a.codes, a.scales, (), "int8"),
                lambda: A.set_activation_checkpoint("fp16"), lambda: H.rownorm_fwd(x, kind="group"), lambda: H.rownorm_fwd(x, save8="e5m2")):
        with pytest.raises(RuntimeError):
            bad()
    assert A.SAVE8[0] is None


def test_narrow_tensors_stay_as_they_are():
    """A checkpoint pads the channels to 32: three channels would grow."""
    import dpig_amd.autograd as A

    class T(object):
        is_cuda = True

        def __init__(self, C, size):
            self.shape, self.size = (2, 4, 4, C), size

        def element_size(self):
            return self.size
    assert not A._worth8(T(3, 4), "int8") and not A._worth8(T(16, 2), "int8") and not A._worth8(T(64, 4), None)
    assert A._worth8(T(16, 4), "int8") and A._worth8(T(32, 2), "int8") and A._worth8(T(640, 2), "e4m3")
