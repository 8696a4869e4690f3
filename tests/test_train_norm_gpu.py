"""Layer norm for training (torch.ops.hi3d.layernorm_fwd / add_layernorm_fwd / layernorm_bwd, hi3d_hip.train.layer_norm) against
the formula in 64 bits on the same inputs.

Tolerances, element by element: the one rounding of a stored value, eps / 2 of its type relative to it, plus what fp32 arithmetic can
lose on the way: DEPTH roundings of 2^-24 each, relative to the sums of absolute values that enter the element.  DEPTH = 128 covers the
longest chain here: a sum of 8192 values in 256 lanes of 32 (32 additions), the tree over the lanes (8), products and the second
sum, or for the columns' sums the rows of one lane, the tree, 4 waves, and 64 partial sums a slice of 8.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U32, DEPTH = 2.0 ** -24, 128


@pytest.fixture(scope="module")
def ns():
    from hi3d_hip import torch_ops
    return torch_ops.load()


def rnd(shape, seed, dt="fp32", scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(DT[dt])


def near(got, want, slack, what):
    """got within its type's half step of want, plus slack (both 64-bit); what is not finite has to be so alike."""
    got, u = got.detach().cpu(), torch.finfo(got.dtype).eps / 2
    g = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(g), fine), what
    # smallest: half a step of the type's subnormals
    tol = u * want.abs() + slack * (1 + u) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bad = fine & ((g - want).abs() > tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((g - want).abs() / tol)[bad].max().item():.2f} of its tolerance"


def norm64(z, w, b, eps):
    """(y, mean, rstd, h, slack of y, of mean, of rstd) of rows z in 64 bits."""
    z = z.double()
    mean = z.mean(-1, keepdim=True)
    d = z - mean
    var = d.square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = d * rstd
    w = w.double() if w is not None else torch.ones(z.shape[-1], dtype=torch.float64)
    b = b.double() if b is not None else torch.zeros(z.shape[-1], dtype=torch.float64)
    y = h * w + b
    s_mean = DEPTH * U32 * z.abs().mean(-1, keepdim=True)
    # the mean's error moves every difference alike; its effect on the variance is of second order (the differences' sum is zero)
    s_rstd = rstd * (DEPTH * U32 + (s_mean * rstd).square())
    s_y = (s_mean * rstd + h.abs() * (DEPTH * U32 + (s_mean * rstd).square())) * w.abs() + 4 * U32 * (b.abs() + (h * w).abs())
    return y, mean[..., 0], rstd[..., 0], h, s_y, s_mean[..., 0], s_rstd[..., 0]


SHAPES = [(1, 1), (3, 2), (3, 7), (5, 8), (1, 40), (17, 63), (33, 320), (1000, 640), (77, 1285), (9, 1280), (6, 1281), (4, 2561), (3, 5120),
          (2, 8192), (1030, 40), (260, 65)]


@pytest.mark.parametrize("dt,wdt", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("R,C", SHAPES)
def test_forward_and_gradients(dev, ns, R, C, dt, wdt):
    eps = 1e-5
    x, r = rnd((R, C), 1, dt, 2.0, 0.5), rnd((R, C), 2, dt)
    w, b = rnd((C,), 3, wdt, 0.2, 1.0), rnd((C,), 4, wdt, 0.2)
    y, mean, rstd = ns.layernorm_fwd(x.to(dev), w.to(dev), b.to(dev), eps)
    yr, z, mean_r, rstd_r = ns.add_layernorm_fwd(x.to(dev), r.to(dev), w.to(dev), b.to(dev), eps)
    zc = (x.float() + r.float()).to(DT[dt])
    assert torch.equal(z.cpu(), zc)                                   # one fp32 addition, one rounding
    for got, src in (((y, mean, rstd), x), ((yr, mean_r, rstd_r), zc)):
        y64, m64, s64, _, sy, sm, ss = norm64(src, w, b, eps)
        assert got[0].dtype == DT[dt] and got[1].shape == (R,)
        near(got[0], y64, sy, "y")
        near(got[1], m64, sm, "mean")
        near(got[2], s64, ss, "rstd")
    # gradients: of the statistics as they are given
    dy, dz = rnd((R, C), 5, dt), rnd((R, C), 6, dt)
    m64, s64 = mean_r.double().cpu()[:, None], rstd_r.double().cpu()[:, None]
    h = (zc.double() - m64) * s64
    d, wd = dy.double(), dy.double() * w.double()
    s1, s2 = wd.mean(-1, keepdim=True), (wd * h).mean(-1, keepdim=True)
    dx64 = s64 * (wd - s1 - h * s2)
    h_abs = h.abs() + zc.double().abs() * s64                          # (z - mean is exact to one rounding; h carries two)
    slack = DEPTH * U32 * s64 * (wd.abs() + wd.abs().mean(-1, keepdim=True) + h.abs() * (wd.abs() * h_abs).mean(-1, keepdim=True))
    for extra in (None, dz):
        dx, dw, db = ns.layernorm_bwd(dy.to(dev), z, mean_r, rstd_r, w.to(dev), b.to(dev), extra.to(dev) if extra is not None else None)
        want = dx64 + extra.double() if extra is not None else dx64
        near(dx, want, slack + 2 * U32 * want.abs(), "dx")
        near(dw, (d * h).sum(0), DEPTH * U32 * (d.abs() * h_abs).sum(0), "dweight")
        near(db, d.sum(0), DEPTH * U32 * d.abs().sum(0), "dbias")
        assert dw.dtype == db.dtype == DT[wdt]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_many_rows_take_every_block_and_give_the_same_bits_twice(dev, ns, dt):
    R, C = 40011, 320
    z, dy, w = rnd((R, C), 1, dt).to(dev), rnd((R, C), 2, dt).to(dev), rnd((C,), 3, "fp32", 0.2, 1.0).to(dev)
    y, mean, rstd = ns.layernorm_fwd(z, w, None, 1e-5)
    y64, _, _, _, sy, _, _ = norm64(z.cpu(), w.cpu(), None, 1e-5)
    near(y, y64, sy, "y")
    a = ns.layernorm_bwd(dy, z, mean, rstd, w, w, None)
    b = ns.layernorm_bwd(dy, z, mean, rstd, w, w, None)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    h = (z.double().cpu() - mean.double().cpu()[:, None]) * rstd.double().cpu()[:, None]
    d = dy.double().cpu()
    near(a[1], (d * h).sum(0), DEPTH * U32 * (d * h).abs().sum(0), "dweight")
    near(a[2], d.sum(0), DEPTH * U32 * d.abs().sum(0), "dbias")


def test_without_weight_or_bias_and_without_rows(dev, ns):
    x, dy = rnd((5, 33), 1).to(dev), rnd((5, 33), 2).to(dev)
    y, mean, rstd = ns.layernorm_fwd(x, None, None, 1e-5)
    near(y, *[norm64(x.cpu(), None, None, 1e-5)[i] for i in (0, 4)], "y")
    dx, dw, db = ns.layernorm_bwd(dy, x, mean, rstd, None, None, None)
    assert dw is None and db is None and torch.isfinite(dx).all()
    b = rnd((33,), 3).to(dev)
    _, dw, db = ns.layernorm_bwd(dy, x, mean, rstd, None, b, None)
    assert dw is None
    near(db, dy.double().cpu().sum(0), DEPTH * U32 * dy.double().cpu().abs().sum(0), "dbias")
    e = x[:0]
    y, mean, rstd = ns.layernorm_fwd(e, b, b, 1e-5)
    assert y.shape == (0, 33) and mean.shape == (0,)
    dx, dw, db = ns.layernorm_bwd(e, e, mean, rstd, b, b, None)
    assert dx.shape == (0, 33) and not dw.any() and not db.any()


def test_rows_at_any_pitch_offset_and_order(dev, ns):
    """Slices of wider tensors, views at odd element offsets, more than two dimensions, transposed and broadcast tensors."""
    for dt in ("bf16", "fp32"):
        C = 77
        wide = rnd((12, 200), 1, dt).to(dev)
        w, b = rnd((C + 1,), 2, dt, 0.2, 1.0).to(dev)[1:], rnd((2 * C,), 3, dt).to(dev)[::2]
        views = [wide[:, 3:3 + C], wide.reshape(-1)[5:5 + 4 * C].reshape(4, C), wide[::3, 100:100 + C], wide[:, :C].reshape(3, 4, C).transpose(0, 1),
                 wide[:C].t()[:, :12].reshape(-1)[:C].expand(6, C), wide[0, :C]]
        for v in views:
            ref = v.contiguous()
            a, m, s = ns.layernorm_fwd(v, w, b, 1e-5)
            a2, m2, s2 = ns.layernorm_fwd(ref, w.contiguous(), b.contiguous(), 1e-5)
            assert torch.equal(a, a2) and torch.equal(m, m2) and torch.equal(s, s2)
            dy = rnd(v.shape, 4, dt).to(dev)
            g = ns.layernorm_bwd(dy.transpose(0, -1).contiguous().transpose(0, -1), v, m, s, w, b, v)
            g2 = ns.layernorm_bwd(dy, ref, m, s, w.contiguous(), b.contiguous(), ref)
            assert all(torch.equal(p, q) for p, q in zip(g, g2))
        assert torch.equal(wide, rnd((12, 200), 1, dt).to(dev))       # inputs are left as they were


def test_rows_that_are_flat_far_from_zero_or_not_finite(dev, ns):
    C = 320
    x = rnd((6, C), 1, "fp32")
    x[0] = 3.25                                  # no spread at all: rstd = eps^-1/2, y = bias
    x[1] += 4096.0                               # the mean is 4000 times the spread
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 0.0
    w, b = rnd((C,), 2, "fp32", 0.2, 1.0), rnd((C,), 3)
    y, mean, rstd = (t.cpu() for t in ns.layernorm_fwd(x.to(dev), w.to(dev), b.to(dev), 1e-5))
    assert torch.equal(y[0], b) and torch.equal(y[4], b)
    y64, _, _, _, sy, _, _ = norm64(x, w, b, 1e-5)
    near(y[1], y64[1], sy[1], "far mean")
    near(y[5], y64[5], sy[5], "the row behind")
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    # a gradient of such rows reaches its own row's dx alone
    g = ns.layernorm_bwd(torch.ones_like(x).to(dev), x.to(dev), mean.to(dev), rstd.to(dev), w.to(dev), None, None)[0].cpu()
    assert torch.isnan(g[2]).all() and torch.isnan(g[3]).all() and torch.isfinite(g[[0, 1, 4, 5]]).all()


def test_offsets_beyond_32_bits(dev, ns):
    """Rows at a pitch that puts the last ones over 2^31 elements (and 2^32 bytes) from the first."""
    C, R, ld = 64, 9, 300_000_000
    flat = torch.zeros((R - 1) * ld + C, dtype=torch.bfloat16, device=dev)
    v = flat.as_strided((R, C), (ld, 1))
    src = rnd((R, C), 1, "bf16").to(dev)
    v.copy_(src)
    y, mean, rstd = ns.layernorm_fwd(v, None, None, 1e-5)
    y2, _, _ = ns.layernorm_fwd(src, None, None, 1e-5)
    assert torch.equal(y, y2)
    assert torch.equal(ns.layernorm_bwd(src, v, mean, rstd, None, None, v)[0], ns.layernorm_bwd(src, src, mean, rstd, None, None, src)[0])


def test_refusals(dev, ns):
    x, w = rnd((4, 16), 1).to(dev), rnd((16,), 2).to(dev)
    y, mean, rstd = ns.layernorm_fwd(x, w, w, 1e-5)
    bad = [lambda: ns.layernorm_fwd(x.double(), w, w, 1e-5), lambda: ns.layernorm_fwd(x, w[:8], w, 1e-5), lambda: ns.layernorm_fwd(x, w, w.bfloat16(), 1e-5),
           lambda: ns.layernorm_fwd(x, w, w, -1.0), lambda: ns.layernorm_fwd(x, w, w, float("nan")), lambda: ns.layernorm_fwd(x, w.cpu(), w, 1e-5),
           lambda: ns.layernorm_fwd(x[:, :0], None, None, 1e-5), lambda: ns.layernorm_fwd(torch.zeros(2, 8193, device=dev), None, None, 1e-5),
           lambda: ns.layernorm_fwd(x.cpu(), w, w, 1e-5), lambda: ns.add_layernorm_fwd(x, x[:1], w, w, 1e-5), lambda: ns.add_layernorm_fwd(x, x.bfloat16(), w, w, 1e-5),
           lambda: ns.layernorm_bwd(x[:2], x, mean, rstd, w, w, None), lambda: ns.layernorm_bwd(x, x, mean[:2], rstd, w, w, None),
           lambda: ns.layernorm_bwd(x, x, mean.double(), rstd, w, w, None), lambda: ns.layernorm_bwd(x, x, mean, rstd, w, w, x.bfloat16())]
    for f in bad:
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_differentiable_form(dev, ns, dt):
    """train.layer_norm: its gradients are the operator's, in every combination of what is asked for, and agree with differences of
    the formula in 64 bits."""
    from hi3d_hip import train
    B, S, C = 3, 5, 48
    x, r, w, b = (t.to(dev).requires_grad_() for t in (rnd((B, S, C), 1, dt), rnd((B, S, C), 2, dt), rnd((C,), 3, "fp32", 0.2, 1.0), rnd((C,), 4)))
    gy, gz = rnd((B, S, C), 5, dt).to(dev), rnd((B, S, C), 6, dt).to(dev)
    y, z = train.layer_norm(x, w, b, residual=r)
    got = torch.autograd.grad([y, z], [x, r, w, b], [gy, gz])
    _, _, mean, rstd = ns.add_layernorm_fwd(x.detach(), r.detach(), w.detach(), b.detach(), 1e-5)
    dx, dw, db = ns.layernorm_bwd(gy, z.detach(), mean, rstd, w.detach(), b.detach(), gz)
    for p, q in zip(got, (dx, dx, dw, db)):
        assert torch.equal(p, q)
    y, z = train.layer_norm(x, w, b, residual=r)
    assert torch.equal(torch.autograd.grad(z.sum(), x)[0], torch.ones_like(x))                # y unused
    y, z = train.layer_norm(x, w, b, residual=r)
    assert torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()                          # z unused, dy a broadcast one
    y = train.layer_norm(x, w, None)
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    if dt == "fp32":     # along a direction: (f(x + t v) - f(x - t v)) / 2 t in 64 bits; error O(t^2) + 2^-52 / t, both far below the fp32 slack
        x64, w64, v, vw, t = x.detach().double().cpu(), w.detach().double().cpu(), rnd((B, S, C), 8).double(), rnd((C,), 9).double(), 1e-5
        f = lambda a, c: (norm64(a, c, None, 1e-5)[0] * gy.double().cpu()).sum()
        diff = (f(x64 + t * v, w64 + t * vw) - f(x64 - t * v, w64 - t * vw)) / (2 * t)
        mine = (gx.double().cpu() * v).sum() + (gw.double().cpu() * vw).sum()
        scale = (gx.double().cpu() * v).abs().sum() + (gw.double().cpu() * vw).abs().sum()
        assert (mine - diff).abs() < 2 * DEPTH * U32 * scale * 4


def test_on_another_stream_and_replayed(dev, ns):
    """The launch goes to the current stream, and a captured forward and backward replay on new values."""
    x, dy, w = rnd((300, 640), 1, "bf16").to(dev), rnd((300, 640), 2, "bf16").to(dev), rnd((640,), 3, "fp32", 0.2, 1.0).to(dev)

    def both():
        y, z, m, s = ns.add_layernorm_fwd(x, dy, w, w, 1e-5)
        return (y, z, m, s) + ns.layernorm_bwd(dy, z, m, s, w, w, x)
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    for seed in (4, 5, 6):
        x.copy_(rnd((300, 640), seed, "bf16"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, both()))


@pytest.mark.parametrize("R,C,dt", [(7, 40, "bf16"), (1030, 320, "fp16"), (300, 5120, "fp32")])
def test_frozen_weight_and_bias_cost_nothing(dev, ns, monkeypatch, R, C, dt):
    """Sums that nobody asks for are not taken, and the others keep their bits."""
    from hi3d_hip import train
    z, dy, w, b = rnd((R, C), 1, dt).to(dev), rnd((R, C), 2, dt).to(dev), rnd((C,), 3, "fp32", 0.2, 1.0).to(dev), rnd((C,), 4).to(dev)
    _, mean, rstd = ns.layernorm_fwd(z, w, b, 1e-5)
    dx, dw, db = ns.layernorm_bwd(dy, z, mean, rstd, w, b, z)
    for nw, nb in ((True, True), (True, False), (False, True), (False, False)):
        got = ns.layernorm_bwd(dy, z, mean, rstd, w, b, z, nw, nb)
        assert torch.equal(got[0], dx)
        assert torch.equal(got[1], dw) if nw else got[1] is None
        assert torch.equal(got[2], db) if nb else got[2] is None
    asked = []

    class Spy:
        def __getattr__(self, name):
            f = getattr(ns, name)
            def call(*a):
                out = f(*a)
                if name == "layernorm_bwd":
                    asked.append([t is not None for t in out])
                return out
            return call
    monkeypatch.setattr(train.torch_ops, "load", lambda: Spy())
    for nw, nb in ((True, False), (False, True), (False, False)):
        x, wp, bp = z.clone().requires_grad_(), w.clone().requires_grad_(nw), b.clone().requires_grad_(nb)
        train.layer_norm(x, wp, bp).backward(dy)
        plain = ns.layernorm_bwd(dy, z, mean, rstd, w, b, None)
        assert asked.pop() == [True, nw, nb] and torch.equal(x.grad, plain[0])
        assert torch.equal(wp.grad, plain[1]) if nw else wp.grad is None
        assert torch.equal(bp.grad, plain[2]) if nb else bp.grad is None
