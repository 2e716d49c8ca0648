"""Plain float64 forms (CPU) of the residual-block operators on rows of channels, written from their formulas."""
import torch

U = 2.0 ** -24                      # half a step of fp32, relative
STORE = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
MOST = {"e4m3": 448.0, "int8": 127.0}
LEAST = {"e4m3": 2.0 ** -9, "int8": 1.0}
EXP = {"e4m3": (-116, 119), "int8": (-116, 121)}


def checkpoint(x, fmt):
    """(codes uint8 [rows, ld], scales uint8 [rows, ld / 32], values float64 [rows, C]) of x [rows, C]."""
    x = x.double().cpu()
    rows, C = x.shape
    ld = -(-C // 32) * 32
    p = torch.zeros(rows, ld, dtype=torch.float64)
    p[:, :C] = x
    p = p.reshape(rows, ld // 32, 32)
    bad = ~torch.isfinite(p).all(-1, keepdim=True)
    z = torch.where(bad, torch.zeros_like(p), p)
    amax = z.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, EXP[fmt][0])
    for k in range(EXP[fmt][0], EXP[fmt][1]):                 # the smallest exponent that holds the largest value
        e = torch.where(amax > MOST[fmt] * 2.0 ** k, torch.full_like(e, k + 1), e)
    v = z / torch.exp2(e)
    if fmt == "e4m3":
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    else:
        step = torch.ones_like(v)
    q = (torch.round(v / step) * step).clamp(-MOST[fmt], MOST[fmt])
    q = torch.where((q == 0) & (z != 0), torch.sign(z) * LEAST[fmt], q)
    if fmt == "e4m3":
        codes = q.float().to(torch.float8_e4m3fn).view(torch.uint8)
        assert torch.equal(codes.view(torch.float8_e4m3fn).double(), q)
    else:
        codes = (q + 128).to(torch.uint8)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    values = torch.where(bad, torch.full_like(p, float("nan")), q * torch.exp2(e))
    return codes.reshape(rows, ld), scales.reshape(rows, ld // 32), values.reshape(rows, ld)[:, :C]


def normed(x, kind, eps):
    """(xh, mean, rstd) in float64."""
    x = x.double().cpu()
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    return (x - mean) * rstd, mean[:, 0], rstd[:, 0]


def normed_error(x, xh, rstd, C):
    """Bound on the error of xh in fp32.  A row's sum runs over at most 32 values in a lane and 8 more steps: the mean is off by at most 40 U max|x|,
    so is x - mean (41 U), and the variance by 45 U relative and twice the mean's error; half of that is the reciprocal root's, + 4 U of its own."""
    big = x.double().cpu().abs().amax(1, keepdim=True) * rstd[:, None]
    return U * (41 * big + xh.abs() * (30 + 41 * big))


def norm_backward(g, xh, rstd, kind):
    m1 = g.mean(1, keepdim=True) if kind == "layer" else 0.0
    return rstd[:, None] * (g - m1 - xh * (g * xh).mean(1, keepdim=True))


def backward_error(g, xh, rstd):
    """Bound on norm_backward's error in fp32: each of its means carries at most 40 roundings of its terms, g and xh three each."""
    return U * rstd[:, None] * (6 * g.abs() + 50 * g.abs().mean(1, keepdim=True) + xh.abs() * 56 * (g * xh).abs().mean(1, keepdim=True))


def sums_error(terms, rows):
    """Column sums over `rows`: at most rows / 64 + 64 roundings in a row (a lane's rows, the lanes of a workgroup, the workgroups), each of
    at most U of the sum of magnitudes; 4 more for the terms themselves."""
    return U * (rows / 64 + 68) * terms.abs().sum(0)
