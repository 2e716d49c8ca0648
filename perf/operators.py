"""What is timed of the residual-block operators on channel-last rows: the norm at a block's entry (`rownorm`), its exit (norm, gate,
residual scale and add: `gated_residual`), the 8-bit activation checkpoints (`act8`) and the filter gradient that reads them
(`linear_wgrad8`).  `run` computes a case in its plain form from elementary torch operations, or, where `own` is true, through
dpig_amd.hip_ops.

An 8-bit checkpoint is two uint8 tensors: codes [rows, ld] (ld = channels rounded up to 32) and scales [rows, ld / 32], the biased
exponent (e + 127) of the power of two that a group of 32 channels shares; 255 marks a group that held a value that was not finite.
'e4m3' codes are OCP 8-bit floats, 'int8' codes are excess-128 integers."""
import math

import torch

own = False

GROUP = 32
EPS = 1e-5
F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": F32, "bf16": BF16}
MOST = {"e4m3": 448.0, "int8": 127.0}
LEAST = {"e4m3": 2.0 ** -9, "int8": 1.0}
EXP_MIN, EXP_MAX = -116, {"e4m3": 119, "int8": 121}
BUDGET = 1 << 26            # elements of the largest row tensors
WORK = 2.0 * 131072 * 512 * 512


# ---- cases -------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the fully connected residual nets of the embedding GAN: batch 64, 512 features, where a call's latency is all there is
        dict(name="norm_fwd_fc", op="norm_fwd", rows=64, c=512, dtype="f32", kind="layer", save="no"),
        # entry of a block on the 128 x 64 map of a batch of 16 in bf16, leaving its 8-bit checkpoint
        dict(name="norm_fwd_map_save", op="norm_fwd", rows=131072, c=256, dtype="bf16", kind="rms", save="e4m3"),
        # its backward pass on the 64 x 32 map, from the saved input and with the skip's gradient added
        dict(name="norm_bwd_map", op="norm_bwd", rows=32768, c=384, dtype="f32", kind="layer", save="no", accum=True),
        # ... and from the checkpoint on a ragged number of crops (37 x 37 regions of 5 images, 7 parts)
        dict(name="norm_bwd_saved_odd", op="norm_bwd", rows=47915, c=250, dtype="bf16", kind="layer", save="int8", accum=False),
        # exit of a block, one gate per sample, with the next block's entry norm: 16 samples of 128 x 64
        dict(name="exit_fwd_map_next", op="exit_fwd", rows=131072, c=128, groups=16, dtype="bf16", kind="layer", save="no", next=True),
        # the same at one gate per row, no next norm, rows of 333 channels
        dict(name="exit_fwd_rowgate_odd", op="exit_fwd", rows=9001, c=333, groups=9001, dtype="f32", kind="rms", save="no", next=False),
        # backward of the exit from the checkpoint: 8 samples of 64 x 64
        dict(name="exit_bwd_saved", op="exit_bwd", rows=32768, c=640, groups=8, dtype="bf16", kind="layer", save="e4m3"),
        # ... and for the fully connected nets, each row its own gate
        dict(name="exit_bwd_fc", op="exit_bwd", rows=64, c=512, groups=64, dtype="f32", kind="rms", save="no"),
        # a ReLU output of a 128-channel layer at 256 x 256, batch 8: stored and read back
        dict(name="act8_round_map", op="act8_round", rows=524288, c=128, dtype="bf16", fmt="e4m3"),
        # the activation's gradient from the checkpoint
        dict(name="act8_mask_map", op="act8_mask", rows=131072, c=256, dtype="f32", fmt="int8", act="lrelu"),
        # filter gradient of a 512 -> 512 layer on the rows of the 128 x 64 map, bf16 gradients, the norm's affine part folded in
        dict(name="wgrad8_map", op="wgrad8", rows=131072, c=512, k=512, dtype="bf16", fmt="e4m3", affine=True),
        # the same of a narrower, ragged layer with fp32 gradients
        dict(name="wgrad8_f32_odd", op="wgrad8", rows=20011, c=250, k=390, dtype="f32", fmt="int8", affine=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "exit_fwd", "exit_bwd", "act8_round", "act8_mask", "wgrad8", "wgrad8"])
    c = rng.choice([_log(rng, 16, 2048), 8 * _log(rng, 4, 128), 64 * rng.randint(1, 12)])
    case = dict(op=op, c=c, dtype=rng.choice(["f32", "bf16"]))
    if op == "wgrad8":
        k = rng.choice([_log(rng, 16, 1024), 64 * rng.randint(1, 12)])
        c = case["c"] = min(c, 1024)
        most = min(WORK / (2.0 * c * k) / (4 if case["dtype"] == "f32" else 1), BUDGET / max(c, k))
        case.update(rows=_log(rng, 1, max(2, most)), k=k, fmt=rng.choice(["e4m3", "int8"]), affine=rng.random() < 0.5)
        return case
    rows = _log(rng, 1, max(2, (BUDGET // 2) // c))
    if op.startswith("act8"):
        case.update(rows=rows, fmt=rng.choice(["e4m3", "int8"]))
        if op == "act8_mask":
            case["act"] = rng.choice(["relu", "lrelu"])
        return case
    case.update(kind=rng.choice(["layer", "rms"]), save=rng.choice(["no", "no", "e4m3", "int8"]))
    if op == "norm_fwd" or op == "norm_bwd":
        case["rows"] = rows
        if op == "norm_bwd":
            case["accum"] = rng.random() < 0.5
        return case
    how = rng.choice(["sample", "row", "all"])
    if how == "sample":
        g = rng.randint(1, min(64, rows))
        case.update(rows=rows // g * g, groups=g)
    else:
        case.update(rows=rows, groups=rows if how == "row" else 1)
    if op == "exit_fwd":
        case["next"] = rng.random() < 0.5
        case["save"] = "no" if not case["next"] else case["save"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    rows, c, dtype = case["rows"], case["c"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=F32)

    spread = torch.exp(0.5 * normal(c))                       # channels differ in size, as activations do
    s = dict(case=dict(case))
    op = case["op"]
    if op in ("norm_fwd", "norm_bwd", "exit_fwd", "exit_bwd"):
        s["scale"] = 1 + 0.1 * normal(c)
        s["offset"] = 0.1 * normal(c)
    if op in ("exit_fwd", "exit_bwd"):
        s["gate"] = 1 + 0.3 * normal(case["groups"], c)
        s["res_scale"] = 0.3 + 0.05 * normal(c)
    if op == "norm_fwd":
        s["x"] = (normal(rows, c) * spread + 0.3 * normal(c)).to(dtype)
    elif op == "exit_fwd":
        s["x"] = (normal(rows, c) * spread).to(dtype)
        s["f"] = (normal(rows, c) * spread.flip(0) + 0.2).to(dtype)
        if case["next"]:
            s["scale2"] = 1 + 0.1 * normal(c)
            s["offset2"] = 0.1 * normal(c)
    elif op in ("norm_bwd", "exit_bwd"):
        x = (normal(rows, c) * spread + 0.3 * normal(c)).to(dtype)
        x32 = x.to(F32)
        mean = x32.mean(1) if case["kind"] == "layer" else torch.zeros(rows, device=dev)
        s["rstd"] = torch.rsqrt((x32 - mean[:, None]).square().mean(1) + EPS)
        s["mean"] = mean
        s["dy"] = (1e-2 * normal(rows, c)).to(dtype)
        if case["save"] == "no":
            s["x"] = x
        else:
            s["codes"], s["scales"] = _store((x32 - mean[:, None]) * s["rstd"][:, None], case["save"])
        if case.get("accum"):
            s["accum"] = (1e-2 * normal(rows, c)).to(dtype)
    else:
        x = (torch.relu(normal(rows, c)) * spread).to(dtype)
        if op == "act8_round":
            s["x"] = x
        else:
            s["codes"], s["scales"] = _store(x.to(F32), case["fmt"])
            s["dy"] = (1e-2 * normal(rows, case["k"] if op == "wgrad8" else c)).to(dtype)
            if case.get("affine"):
                s["scale"] = 1 + 0.1 * normal(c)
                s["offset"] = 0.1 * normal(c)
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------------------
def _store(x, fmt):
    """fp32 [rows, c] -> (codes [rows, ld], scales [rows, ld / 32])."""
    rows, c = x.shape
    ld = -(-c // GROUP) * GROUP
    xp = torch.nn.functional.pad(x, (0, ld - c)).reshape(rows, ld // GROUP, GROUP)
    finite = torch.isfinite(xp).all(-1)
    amax = torch.where(finite[..., None], xp, torch.zeros_like(xp)).abs().amax(-1)
    m, ex = torch.frexp(amax)
    e = (ex - 9 + (m > 0.875)) if fmt == "e4m3" else (ex - 7 + (m > 127.0 / 128.0))
    e = torch.where(amax > 0, e, torch.full_like(e, EXP_MIN)).clamp(EXP_MIN, EXP_MAX[fmt])
    v = torch.ldexp(xp, -e[..., None]).clamp(-MOST[fmt], MOST[fmt])
    v = torch.nan_to_num(v, nan=0.0)
    r = v.to(torch.float8_e4m3fn).to(F32) if fmt == "e4m3" else torch.round(v)
    r = torch.where((r == 0) & (xp != 0) & ~torch.isnan(xp), torch.copysign(torch.full_like(r, LEAST[fmt]), xp), r)
    codes = r.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "e4m3" else (r + 128).to(torch.uint8)
    scales = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return codes.reshape(rows, ld), scales


def _load(codes, scales, c, fmt):
    """The fp32 values that a checkpoint stands for."""
    rows, ld = codes.shape
    v = codes.view(torch.float8_e4m3fn).to(F32) if fmt == "e4m3" else codes.to(F32) - 128.0
    e = scales.to(torch.int32)
    s = torch.where(e == 255, torch.full(e.shape, float("nan"), device=e.device), torch.ldexp(torch.ones_like(e, dtype=F32), e - 127))
    return (v.reshape(rows, ld // GROUP, GROUP) * s[..., None]).reshape(rows, ld)[:, :c]


def _norm(x, kind):
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    d = x - mean
    rstd = torch.rsqrt(d.square().mean(1, keepdim=True) + EPS)
    return d * rstd, mean[:, 0], rstd[:, 0]


def _norm_bwd(g, xh, rstd, kind):
    m1 = g.mean(1, keepdim=True) if kind == "layer" else 0.0
    return rstd[:, None] * (g - m1 - xh * (g * xh).mean(1, keepdim=True))


def _saved(s):
    """xh in fp32 from what a backward case holds."""
    case = s["case"]
    if case["save"] == "no":
        return (s["x"].to(F32) - s["mean"][:, None]) * s["rstd"][:, None]
    return _load(s["codes"], s["scales"], case["c"], case["save"])


def _plain(s):
    case = s["case"]
    op, c, kind = case["op"], case["c"], case.get("kind")
    if op == "norm_fwd":
        x = s["x"]
        xh, mean, rstd = _norm(x.to(F32), kind)
        out = dict(y=(xh * s["scale"] + s["offset"]).to(x.dtype), rstd=rstd)
        if kind == "layer":
            out["mean"] = mean
        if case["save"] != "no":
            out["saved"] = _load(*_store(xh, case["save"]), c, case["save"]).to(BF16)
        return out
    if op == "norm_bwd":
        dy = s["dy"].to(F32)
        xh = _saved(s)
        dx = _norm_bwd(dy * s["scale"], xh, s["rstd"], kind)
        if case["accum"]:
            dx = dx + s["accum"].to(F32)
        return dict(dx=dx.to(s["dy"].dtype), dscale=(dy * xh).sum(0), doffset=dy.sum(0))
    if op == "exit_fwd":
        x, f = s["x"].to(F32), s["f"].to(F32)
        xh, mean, rstd = _norm(f, kind)
        gate = s["gate"].repeat_interleave(case["rows"] // case["groups"], 0)
        y = (x + s["res_scale"] * gate * (xh * s["scale"] + s["offset"])).to(s["x"].dtype)
        out = dict(out=y, rstd=rstd)
        if case["next"]:
            xh2, _, rstd2 = _norm(y.to(F32), kind)
            out["next"] = (xh2 * s["scale2"] + s["offset2"]).to(y.dtype)
            out["next_rstd"] = rstd2
            if case["save"] != "no":
                out["saved"] = _load(*_store(xh2, case["save"]), c, case["save"]).to(BF16)
        return out
    if op == "exit_bwd":
        dy = s["dy"].to(F32)
        xh = _saved(s)
        g, per = case["groups"], case["rows"] // case["groups"]
        n = xh * s["scale"] + s["offset"]
        gate = s["gate"].repeat_interleave(per, 0)
        dn = dy * s["res_scale"] * gate
        df = _norm_bwd(dn * s["scale"], xh, s["rstd"], kind)
        return dict(df=df.to(s["dy"].dtype), dscale=(dn * xh).sum(0), doffset=dn.sum(0),
                    dgate=(dy * s["res_scale"] * n).reshape(g, per, c).sum(1), dres_scale=(dy * gate * n).sum(0))
    if op == "act8_round":
        return _load(*_store(s["x"].to(F32), case["fmt"]), c, case["fmt"]).to(s["x"].dtype)
    if op == "act8_mask":
        v = _load(s["codes"], s["scales"], c, case["fmt"])
        dy = s["dy"].to(F32)
        return torch.where(v > 0, dy, dy * (0.2 if case["act"] == "lrelu" else 0.0)).to(s["dy"].dtype)
    v = _load(s["codes"], s["scales"], c, case["fmt"])
    if case["affine"]:
        v = v * s["scale"] + s["offset"]
    dy = s["dy"].to(F32)
    return dict(dw=v.t() @ dy, db=dy.sum(0))


# ---- the framework's calls -----------------------------------------------------------------------------------------------------------
def _own(s):
    import dpig_amd.hip_ops as H
    from dpig_amd._lib import ACT_LRELU, ACT_RELU
    case = s["case"]
    op, kind = case["op"], case.get("kind")
    save = None if case.get("save", "no") == "no" else case["save"]
    if op == "norm_fwd":
        y, mean, rstd, saved = H.rownorm_fwd(s["x"], s["scale"], s["offset"], EPS, kind, save8=save)
        out = dict(y=y, rstd=rstd)
        if kind == "layer":
            out["mean"] = mean
        if save:
            out["saved"] = H.act8_load(saved, BF16)
        return out
    if op in ("norm_bwd", "exit_bwd"):
        held = s["x"] if save is None else H.Act8(s["codes"], s["scales"], (case["rows"], case["c"]), save)
        mean = s["mean"] if kind == "layer" else None
    if op == "norm_bwd":
        dx, dscale, doffset = H.rownorm_bwd(s["dy"], held, s["scale"], mean, s["rstd"], kind, accum=s.get("accum"))
        return dict(dx=dx, dscale=dscale, doffset=doffset)
    if op == "exit_fwd":
        nxt = (s["scale2"], s["offset2"], EPS, kind) if case["next"] else None
        out, _, rstd, _, after = H.gated_residual_fwd(s["x"], s["f"], s["scale"], s["offset"], s["gate"], s["res_scale"], EPS, kind,
                                                      next_norm=nxt, next_save8=save)
        r = dict(out=out, rstd=rstd)
        if nxt is not None:
            h, _, rstd2, saved = after
            r["next"], r["next_rstd"] = h, rstd2
            if save:
                r["saved"] = H.act8_load(saved, BF16)
        return r
    if op == "exit_bwd":
        df, dscale, doffset, dgate, dres = H.gated_residual_bwd(s["dy"], held, s["scale"], s["offset"], s["gate"], s["res_scale"],
                                                                mean, s["rstd"], kind)
        return dict(df=df, dscale=dscale, doffset=doffset, dgate=dgate, dres_scale=dres)
    if op == "act8_round":
        return H.act8_load(H.act8_store(s["x"], case["fmt"]), s["x"].dtype)
    a = H.Act8(s["codes"], s["scales"], (case["rows"], case["c"]), case["fmt"])
    if op == "act8_mask":
        return H.act8_act_bwd(s["dy"], a, ACT_LRELU if case["act"] == "lrelu" else ACT_RELU, 0.2)
    dw, db = H.linear_wgrad8(a, s["dy"], scale=s.get("scale"), offset=s.get("offset"), want_bias=True)
    return dict(dw=dw, db=db)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------
def work(case):
    op, n, r, c = case["op"], case["rows"] * case["c"], case["rows"], case["c"]
    w = 4 if case["dtype"] == "f32" else 2
    code = r * (-(-c // GROUP)) * (GROUP + 1)
    held = n * w if case.get("save", "no") == "no" else code
    extra = 0 if case.get("save", "no") == "no" else code + 2 * n          # the checkpoint, and the values it stands for
    if op == "norm_fwd":
        return {"bytes": 2 * n * w + 8 * r + 8 * c + extra, "flops": 8.0 * n}
    if op == "norm_bwd":
        return {"bytes": n * w * (3 if case["accum"] else 2) + held + 8 * r + 12 * c, "flops": 11.0 * n}
    if op == "exit_fwd":
        return {"bytes": n * w * (4 if case["next"] else 3) + 8 * r + 4 * case["groups"] * c + 20 * c + extra, "flops": (19.0 if case["next"] else 11.0) * n}
    if op == "exit_bwd":
        return {"bytes": 2 * n * w + held + 8 * r + 8 * case["groups"] * c + 24 * c, "flops": 14.0 * n}
    if op == "act8_round":
        return {"bytes": 2 * n * w + 2 * code, "flops": 6.0 * n}
    if op == "act8_mask":
        return {"bytes": 2 * n * w + r * c, "flops": 2.0 * n}
    k = case["k"]
    return {"bytes": code + r * k * w + 4 * c * k + 4 * k, "flops": 2.0 * r * c * k + r * k}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------------
def _grid(v, fmt):
    """Nearest value of the format's grid, ties to even, for |v| at most its largest value."""
    if fmt == "int8":
        r = torch.floor(v)
        d = v - r
        return torch.where((d > 0.5) | ((d == 0.5) & (torch.remainder(r, 2) == 1)), r + 1, r)
    p = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(p.clamp(min=-6.0) - 3)
    return torch.round(v / step) * step


def _held(x, fmt):
    """fp64 [rows, c] -> the values that its checkpoint stands for."""
    rows, c = x.shape
    width = -(-c // GROUP)
    wide = torch.zeros(rows, width * GROUP, dtype=x.dtype, device=x.device)
    wide[:, :c] = x
    part = wide.reshape(rows * width, GROUP)
    big = part.abs().amax(1, keepdim=True)
    e = torch.ceil(torch.log2(big.clamp(min=1e-300) / MOST[fmt]))
    e = torch.where(big > MOST[fmt] * torch.exp2(e), e + 1, torch.where(big <= MOST[fmt] * torch.exp2(e - 1), e - 1, e))
    unit = torch.exp2(e.clamp(EXP_MIN, EXP_MAX[fmt]))
    q = _grid(part / unit, fmt)
    q = torch.where((q == 0) & (part != 0), torch.sign(part) * LEAST[fmt], q)
    return (q * unit).reshape(rows, -1)[:, :c]


def _values(s, fmt):
    """fp64 values of a given checkpoint, from the bits of its codes."""
    codes, c = s["codes"].to(torch.int64)[:, :s["case"]["c"]], s["case"]["c"]
    if fmt == "int8":
        v = (codes - 128).double()
    else:
        ex, man = (codes >> 3) & 15, codes & 7
        v = torch.where(ex == 0, man.double() * 2.0 ** -9, (8 + man).double() * torch.exp2(ex.double() - 10))
        v = torch.where(codes >= 128, -v, v)
    unit = torch.exp2(s["scales"].double() - 127).repeat_interleave(GROUP, 1)[:, :c]
    return v * unit


def exact(case, seed):
    s = prepare(case, seed)
    op, kind = case["op"], case.get("kind")
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.dtype in (F32, BF16)}

    def whiten(t):
        mu = t.sum(1, keepdim=True) / t.shape[1] if kind == "layer" else 0.0 * t[:, :1]
        var = ((t - mu) ** 2).sum(1, keepdim=True) / t.shape[1]
        return (t - mu) / (var + EPS) ** 0.5, mu[:, 0], (var[:, 0] + EPS) ** -0.5

    if op == "norm_fwd":
        xh, mu, r = whiten(d["x"])
        out = dict(y=d["scale"] * xh + d["offset"], rstd=r)
        if kind == "layer":
            out["mean"] = mu
        if case["save"] != "no":
            out["saved"] = _held(xh, case["save"])
        return out
    if op == "exit_fwd":
        xh, _, r = whiten(d["f"])
        per = case["rows"] // case["groups"]
        branch = (d["scale"] * xh + d["offset"]).reshape(case["groups"], per, -1) * d["gate"][:, None] * d["res_scale"]
        y = d["x"] + branch.reshape(case["rows"], -1)
        out = dict(out=y, rstd=r)
        if case["next"]:
            xh2, _, r2 = whiten(y.to(TYPES[case["dtype"]]).double())
            out["next"], out["next_rstd"] = d["scale2"] * xh2 + d["offset2"], r2
            if case["save"] != "no":
                out["saved"] = _held(xh2, case["save"])
        return out
    if op in ("norm_bwd", "exit_bwd"):
        xh = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None] if case["save"] == "no" else _values(s, case["save"])
        weight = d["scale"].expand_as(xh)
        if op == "exit_bwd":
            gate = d["gate"][:, None].expand(-1, case["rows"] // case["groups"], -1).reshape(xh.shape)
            weight = weight * d["res_scale"] * gate
        g = weight * d["dy"]
        grad = g - xh * ((g * xh).sum(1, keepdim=True) / case["c"])
        if kind == "layer":
            grad = grad - g.sum(1, keepdim=True) / case["c"]
        grad = grad * d["rstd"][:, None]
        if op == "norm_bwd":
            return dict(dx=grad + d["accum"] if case["accum"] else grad, dscale=(d["dy"] * xh).sum(0), doffset=d["dy"].sum(0))
        shape = (case["groups"], -1, case["c"])
        a, b = (d["dy"] * xh).reshape(shape).sum(1), d["dy"].reshape(shape).sum(1)
        t = d["scale"] * a + d["offset"] * b
        return dict(df=grad, dscale=d["res_scale"] * (d["gate"] * a).sum(0), doffset=d["res_scale"] * (d["gate"] * b).sum(0),
                    dgate=d["res_scale"] * t, dres_scale=(d["gate"] * t).sum(0))
    if op == "act8_round":
        return _held(d["x"], case["fmt"])
    v = _values(s, case["fmt"])
    if op == "act8_mask":
        return d["dy"] * torch.where(v > 0, 1.0, 0.2 if case["act"] == "lrelu" else 0.0).double()
    if case["affine"]:
        v = v * d["scale"] + d["offset"]
    dw = torch.zeros(case["c"], case["k"], dtype=torch.float64, device=v.device)
    for lo in range(0, case["rows"], 16384):
        dw += v[lo:lo + 16384].t().contiguous() @ d["dy"][lo:lo + 16384]
    return dict(dw=dw, db=d["dy"].sum(0))
