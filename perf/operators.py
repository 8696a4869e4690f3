"""What the training operators are measured on: layer norm with its gradients, a linear layer with its epilogue and gradients, AdamW.

Sizes are those of the networks in this repository: token counts and widths of the two UNet stages (320 / 640 / 1280 channels; 16 frames
of 16^2 ... 128^2 tokens), the time embedding, the CLIP image tower's feed-forward, and odd ones that no tile divides.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


@functools.lru_cache(maxsize=None)
def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hi3d-official_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from hi3d_hip import torch_ops
    return torch_ops.load()


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one context token per frame of a clip: the smallest norm, nothing but latency
        dict(name="norm context tokens", op="norm", rows=16, width=1024, dtype="bf16", wdtype="fp32", residual=False),
        # the residual stream of the 1024^2 stage's widest level (16 frames of 128 x 128 tokens): sum, norm and statistics in one pass
        dict(name="residual norm 128x128", op="norm", rows=262144, width=320, dtype="bf16", wdtype="fp32", residual=True),
        # the backward pass one level down, the gradient of the residual stream joining it
        dict(name="norm gradients 64x64", op="norm_grad", rows=65536, width=640, dtype="bf16", wdtype="fp32", residual=True),
        # a width that no vector divides, half precision throughout
        dict(name="norm gradients odd", op="norm_grad", rows=7013, width=1285, dtype="fp16", wdtype="fp16", residual=False),
        # the time embedding's second layer over a clip's frames: few rows, the weights are all there is to read
        dict(name="linear time embedding", op="linear", rows=16, inner=1280, outer=1280, dtype="bf16", act="silu", residual=False, save=False),
        # one token, from the wide side of a feed-forward back into the residual stream
        dict(name="linear one token", op="linear", rows=1, inner=5120, outer=1280, dtype="bf16", act="none", residual=True, save=False),
        # the image tower's feed-forward over 16 frames of 257 tokens, its activation's argument kept for the backward pass
        dict(name="linear image tower", op="linear", rows=4112, inner=1280, outer=5120, dtype="bf16", act="gelu", residual=False, save=True),
        # the output side of a feed-forward at 64 x 64 tokens, added to the residual stream
        dict(name="linear residual 64x64", op="linear", rows=65536, inner=2560, outer=640, dtype="bf16", act="none", residual=True, save=False),
        # the backward pass of a feed-forward's input side at 32 x 32 tokens: both products and the bias
        dict(name="linear gradients 32x32", op="linear_grad", rows=16384, inner=1280, outer=5120, dtype="bf16", act="gelu"),
        # sizes that no tile and no vector divides
        dict(name="linear gradients odd", op="linear_grad", rows=3083, inner=650, outer=1290, dtype="fp16", act="silu"),
        # the norms and biases of a level: many short tensors
        dict(name="adamw norms and biases", op="adamw", tensors=60, size=960, odd=False, dtype="fp32", gdtype="fp32", copy=False),
        # a level's weights: 32-bit parameters, gradients and the working copy in 16 bits
        dict(name="adamw weights", op="adamw", tensors=20, size=6553600, odd=False, dtype="fp32", gdtype="bf16", copy=True),
    ]


def _log(rng, lo, hi, odd=0.5):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() >= odd:
        n = max(lo, n // 32 * 32)
    return min(hi, max(lo, n))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "linear", "linear", "linear_grad", "linear_grad", "adamw"])
    if op in ("norm", "norm_grad"):
        width = _log(rng, 64, 5120)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return dict(op=op, rows=_log(rng, 1, 80_000_000 // width, 0.8), width=width, dtype=dtype,
                    wdtype=rng.choice(["fp32", dtype]), residual=rng.random() < 0.5)
    if op in ("linear", "linear_grad"):
        inner, outer = _log(rng, 64, 5120), _log(rng, 64, 5120)
        case = dict(op=op, rows=_log(rng, 1, min(65536, 100_000_000_000 // (inner * outer)), 0.7), inner=inner, outer=outer,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), act=rng.choice(["none", "gelu", "quick_gelu", "silu", "relu"]))
        return case if op == "linear_grad" else dict(case, residual=rng.random() < 0.5, save=rng.random() < 0.5)
    tensors = _log(rng, 1, 200, 1.0)
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    return dict(op=op, tensors=tensors, size=_log(rng, 64, 120_000_000 // tensors), odd=rng.random() < 0.5, dtype=dtype,
                gdtype=rng.choice(["fp32", "bf16", "fp16"]) if dtype == "fp32" else dtype, copy=dtype == "fp32" and rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------------- their inputs
ADAM = dict(lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-8, decay=0.01, step=1000)


def _sizes(case):
    """Numbers of elements of the tensors of an optimiser's list: around `size`, a quarter of them a quarter of it."""
    n, k = case["size"], case["tensors"]
    return [max(1, (n if i % 4 else n // 4) + (i * 37 % 61 if case["odd"] else 0)) for i in range(k)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, dtype="fp32", scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(DTYPES[dtype])

    if case["op"] in ("norm", "norm_grad"):
        r, c, d, w = case["rows"], case["width"], case["dtype"], case["wdtype"]
        s = dict(case=case, weight=rnd(c, dtype=w, scale=0.2, shift=1.0), bias=rnd(c, dtype=w, scale=0.2))
        if case["op"] == "norm":
            # a residual stream: a mean of its own in each channel
            s.update(x=rnd(r, c, dtype=d), residual=(rnd(r, c) * 2 + rnd(c)).to(DTYPES[d]) if case["residual"] else None)
            return s
        z = (rnd(r, c) * 2 + rnd(c)).to(DTYPES[d])
        zf = z.float()
        mean = zf.mean(1)
        rstd = torch.rsqrt((zf - mean[:, None]).square().mean(1) + EPS)
        s.update(z=z, mean=mean, rstd=rstd, dy=rnd(r, c, dtype=d), dz=rnd(r, c, dtype=d) if case["residual"] else None)
        return s
    if case["op"] in ("linear", "linear_grad"):
        m, k, n, d = case["rows"], case["inner"], case["outer"], case["dtype"]
        s = dict(case=case, x=rnd(m, k, dtype=d), w=rnd(n, k, dtype=d, scale=k ** -0.5), bias=rnd(n, dtype="fp32", scale=0.2))
        if case["op"] == "linear":
            s["residual"] = rnd(m, n, dtype=d) if case["residual"] else None
        else:
            s.update(dy=rnd(m, n, dtype=d), z=rnd(m, n, dtype=d) if case["act"] != "none" else None)
        return s
    sizes = _sizes(case)
    total, d = sum(sizes), case["dtype"]

    def parts(flat):
        return list(flat.split(sizes)) if flat is not None else []

    p = rnd(total, dtype=d, scale=0.03)
    # a trained network's state: first moments of the gradients' own size, second moments above them
    m = rnd(total, scale=3e-4)
    v = (rnd(total, scale=1e-3).square() + 1e-9)
    grad = rnd(total, dtype=case["gdtype"], scale=1e-3)
    copy = torch.zeros(total, device="cuda", dtype=torch.bfloat16) if case["copy"] else None
    return dict(case=case, p=p, m=m, v=v, copy=copy, params=parts(p), exp_avg=parts(m), exp_avg_sq=parts(v), grads=parts(grad), copies=parts(copy))


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return torch.clamp_min(z, 0) if act == "relu" else z


def _act_slope(z, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    if act in ("quick_gelu", "silu"):
        a = 1.702 if act == "quick_gelu" else 1.0
        s = torch.sigmoid(a * z)
        return s * (1 + a * z * (1 - s))
    return (z > 0).float()


def _plain_norm(s):
    x = s["x"]
    z = (x.float() + s["residual"].float()).to(x.dtype) if s["residual"] is not None else x
    zf = z.float()
    mean = zf.mean(1)
    d = zf - mean[:, None]
    rstd = torch.rsqrt(d.square().mean(1) + EPS)
    y = (d * rstd[:, None] * s["weight"].float() + s["bias"].float()).to(x.dtype)
    return [y, mean, rstd] + ([z] if s["residual"] is not None else [])


def _plain_norm_grad(s):
    dy, w = s["dy"].float(), s["weight"].float()
    xhat = (s["z"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    wdy = dy * w
    dx = (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
    if s["dz"] is not None:
        dx = dx + s["dz"].float()
    return [dx.to(s["dy"].dtype), (dy * xhat).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["weight"].dtype)]


def _plain_linear(s):
    x, case = s["x"], s["case"]
    z = x.float() @ s["w"].float().t() + s["bias"]
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return [y.to(x.dtype)] + ([z.to(x.dtype)] if case["save"] and case["act"] != "none" else [])


def _plain_linear_grad(s):
    dt, act = s["x"].dtype, s["case"]["act"]
    dz = s["dy"].float()
    if act != "none":
        dz = dz * _act_slope(s["z"].float(), act)
    return [(dz @ s["w"].float()).to(dt), (dz.t() @ s["x"].float()).to(dt), dz.sum(0)]


def _plain_adamw(s):
    a = ADAM
    g = [t.float() for t in s["grads"]]
    torch._foreach_mul_(s["exp_avg"], a["beta1"])
    torch._foreach_add_(s["exp_avg"], torch._foreach_mul(g, 1 - a["beta1"]))
    torch._foreach_mul_(s["exp_avg_sq"], a["beta2"])
    torch._foreach_add_(s["exp_avg_sq"], torch._foreach_mul(torch._foreach_mul(g, g), 1 - a["beta2"]))
    den = torch._foreach_sqrt(s["exp_avg_sq"])
    torch._foreach_div_(den, math.sqrt(1 - a["beta2"] ** a["step"]))
    torch._foreach_add_(den, a["eps"])
    p = torch._foreach_mul([t.float() for t in s["params"]], 1 - a["lr"] * a["decay"])
    change = torch._foreach_div(s["exp_avg"], den)
    torch._foreach_mul_(change, -a["lr"] / (1 - a["beta1"] ** a["step"]))
    torch._foreach_add_(p, change)
    torch._foreach_copy_(s["params"], p)
    if s["copies"]:
        torch._foreach_copy_(s["copies"], p)


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        if not own:
            return _plain_norm(s)
        if s["residual"] is None:
            return list(_ops().layernorm_fwd(s["x"], s["weight"], s["bias"], EPS))
        y, z, mean, rstd = _ops().add_layernorm_fwd(s["x"], s["residual"], s["weight"], s["bias"], EPS)
        return [y, mean, rstd, z]
    if op == "norm_grad":
        if not own:
            return _plain_norm_grad(s)
        return list(_ops().layernorm_bwd(s["dy"], s["z"], s["mean"], s["rstd"], s["weight"], s["bias"], s["dz"]))
    if op == "linear":
        if not own:
            return _plain_linear(s)
        save = case["save"] and case["act"] != "none"
        y, z = _ops().linear_act(s["x"], s["w"], s["bias"], s["residual"], case["act"], save)
        return [y, z] if save else [y]
    if op == "linear_grad":
        if not own:
            return _plain_linear_grad(s)
        return list(_ops().linear_act_bwd(s["dy"], s["x"], s["w"], s["z"], s["bias"], case["act"], True, True))
    if own:
        a = ADAM
        _ops().adamw_(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["copies"], a["lr"], a["beta1"], a["beta2"], a["eps"],
                      a["decay"], a["step"], None, None, None, None)
    else:
        _plain_adamw(s)
    return [s["p"], s["m"], s["v"]] + ([s["copy"]] if s["copy"] is not None else [])


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n, e, w = case["rows"] * case["width"], SIZE[case["dtype"]], SIZE[case["wdtype"]]
        if op == "norm":       # x (, residual) in; y (, their sum) out; weight and bias; two statistics a row
            return dict(bytes=n * e * (4 if case["residual"] else 2) + 2 * case["width"] * w + 8 * case["rows"], flops=8 * n)
        # dy, the norm's argument (, the other gradient) in; dx out; weight in, two gradients out; two statistics a row
        return dict(bytes=n * e * (4 if case["residual"] else 3) + 3 * case["width"] * w + 8 * case["rows"], flops=14 * n)
    if op in ("linear", "linear_grad"):
        m, k, n, e = case["rows"], case["inner"], case["outer"], SIZE[case["dtype"]]
        if op == "linear":
            outs = 1 + case["residual"] + (case["save"] and case["act"] != "none")
            return dict(bytes=e * (m * k + n * k + m * n * outs) + 4 * n, flops=2 * m * n * k)
        outs = 2 if case["act"] != "none" else 1
        return dict(bytes=e * (2 * m * k + 2 * n * k + m * n * outs) + 4 * n, flops=4 * m * n * k)
    n = sum(_sizes(case))
    return dict(bytes=n * (2 * SIZE[case["dtype"]] + SIZE[case["gdtype"]] + 16 + (2 if case["copy"] else 0)), flops=14 * n)


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    F = torch.nn.functional
    acts = {"none": lambda t: t, "gelu": F.gelu, "quick_gelu": lambda t: t / (1 + torch.exp(-1.702 * t)), "silu": F.silu, "relu": F.relu}
    if op == "norm":
        z = s["x"].double()
        if s["residual"] is not None:
            z = (z + s["residual"].double()).to(s["x"].dtype).double()      # the sum is held in the stream's own type
        y = F.layer_norm(z, z.shape[1:], s["weight"].double(), s["bias"].double(), EPS)
        var, mean = torch.var_mean(z, 1, correction=0)
        return [y, mean, 1 / torch.sqrt(var + EPS)] + ([z] if s["residual"] is not None else [])
    if op == "norm_grad":
        z, w, b = (s[k].double().requires_grad_() for k in ("z", "weight", "bias"))
        y = F.layer_norm(z, z.shape[1:], w, b, EPS)
        dx, dw, db = torch.autograd.grad(y, [z, w, b], s["dy"].double())
        return [dx + s["dz"].double() if s["dz"] is not None else dx, dw, db]
    if op == "linear":
        z = torch.addmm(s["bias"].double(), s["x"].double(), s["w"].double().t())
        y = acts[case["act"]](z)
        y = y + s["residual"].double() if s["residual"] is not None else y
        return [y] + ([z] if case["save"] and case["act"] != "none" else [])
    if op == "linear_grad":
        dz = s["dy"].double()
        if case["act"] != "none":
            z = s["z"].double().requires_grad_()
            dz = torch.autograd.grad(acts[case["act"]](z), z, dz)[0]
        return [torch.mm(dz, s["w"].double()), torch.mm(dz.t(), s["x"].double()), dz.sum(0)]
    a = ADAM
    g = torch.cat(s["grads"]).double()
    m = torch.lerp(g, s["m"].double(), a["beta1"])
    v = torch.lerp(g * g, s["v"].double(), a["beta2"])
    mhat, vhat = m / (1 - a["beta1"] ** a["step"]), v / (1 - a["beta2"] ** a["step"])
    p = s["p"].double()
    p = p - a["lr"] * (mhat / (vhat.sqrt() + a["eps"]) + a["decay"] * p)
    return [p, m, v] + ([p] if s["copy"] is not None else [])
