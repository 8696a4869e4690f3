"""The linear layer with its epilogue and gradients (torch.ops.hi3d.linear_act / linear_act_bwd, hi3d_hip.train.linear) against the
formula in 64 bits on the same inputs.

Tolerances, element by element.  A stored value is rounded once: eps / 2 of its type.  A product's fp32 sum of K terms is a chain of one
matrix instruction for each 32 of them, which adds 32 terms in some order, and at most 32 partial sums joined: (K / 32 + 64) roundings of
2^-24 relative to the sum of the terms' absolute values.  The activations and their slopes are within 1e-5 of their value, or of 1 where
they are a difference from it.  With an activation, dz is rounded to the operands' type for the products: eps / 2 of every |dz| that enters a
sum.
"""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = {"none": lambda z: z, "gelu": F.gelu, "quick_gelu": lambda z: z * torch.sigmoid(1.702 * z), "silu": F.silu, "relu": F.relu}
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ns():
    from hi3d_hip import torch_ops
    return torch_ops.load()


def rnd(shape, seed, dt="fp32", scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(DT[dt])


def near(got, want, slack, what):
    u = torch.finfo(got.dtype).eps / 2
    tol = u * want.abs() + slack * (1 + u) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / tol).max().item():.2f} of its tolerance"


def chain(k):
    return (k / 32 + 64) * U32


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    z = z.clone().requires_grad_()
    return torch.autograd.grad(ACTS[act](z).sum(), z)[0]


def check_fwd(ns, x, w, b, r, act):
    z64 = x.double() @ w.double().t() + (b.double() if b is not None else 0)
    s = chain(x.shape[1]) * (x.double().abs() @ w.double().abs().t()) + 4 * U32 * z64.abs()
    y64 = ACTS[act](z64)
    sy = 1.13 * s + 1e-5 * y64.abs()
    if r is not None:
        y64 = y64 + r.double()
        sy = sy + 2 * U32 * y64.abs()
    y, z = ns.linear_act(x, w, b, r, act, True)
    near(z, z64, s, "z")
    near(y, y64, sy, "y")
    y2, none = ns.linear_act(x, w, b, r, act, False)
    assert none is None and torch.equal(y, y2) and y.dtype == x.dtype


def check_bwd(ns, dy, x, w, z, b, act):
    m, n, k = x.shape[0], w.shape[0], x.shape[1]
    d64 = dy.double() * (slope64(z.double(), act) if act != "none" else 1)
    # what a rounded dz may be off by: eps / 2 of it and the slope's own error; nothing where dz is dy
    sd = torch.zeros_like(d64) if act == "none" else torch.finfo(x.dtype).eps / 2 * d64.abs() + 2e-5 * dy.double().abs()
    s_db = torch.zeros_like(d64) if act == "none" else 2e-5 * dy.double().abs()
    want = (d64 @ w.double(), d64.t() @ x.double(), d64.sum(0))
    slack = ((sd + chain(n) * d64.abs()) @ w.double().abs(), (sd + chain(m) * d64.abs()).t() @ x.double().abs(), (s_db + 512 * U32 * d64.abs()).sum(0))
    # (the order of a sum goes by the sizes and by what is asked for: each combination is held to the formula, the bias' gradient to the same bits)
    db = None
    for nx, nw, nb in ((True, True, True), (True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        got = ns.linear_act_bwd(dy, x, w, z, b if nb else None, act, nx, nw)
        for asked, g, f, s, name in zip((nx, nw, nb and b is not None), got, want, slack, ("dx", "dw", "db")):
            if asked:
                near(g, f, s, name)
            else:
                assert g is None
        if got[2] is not None:
            assert got[2].dtype == b.dtype and (db is None or torch.equal(got[2], db))
            db = got[2]


SIZES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (7, 64, 64), (16, 1280, 320), (33, 40, 72), (64, 64, 129), (100, 130, 70), (128, 66, 24), (129, 257, 65), (257, 321, 193), (300, 320, 640),
         (513, 640, 136), (1, 1280, 5120), (4, 37, 4101), (7, 50, 2055), (8, 24, 4999), (17, 1290, 650), (32, 33, 1029)]


@pytest.mark.parametrize("dt,bdt,act", [("bf16", "fp32", "none"), ("bf16", "bf16", "gelu"), ("fp16", "fp32", "silu"), ("fp16", "fp16", "quick_gelu"), ("bf16", "fp32", "relu")])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes_types_and_activations(dev, ns, M, N, K, dt, bdt, act):
    x, w, b = rnd((M, K), 1, dt).to(dev), rnd((N, K), 2, dt, K ** -0.5).to(dev), rnd((N,), 3, bdt, 0.3).to(dev)
    r, dy, z = rnd((M, N), 4, dt).to(dev), rnd((M, N), 5, dt).to(dev), rnd((M, N), 6, dt, 2.0).to(dev)
    check_fwd(ns, x, w, b, r, act)
    check_fwd(ns, x, w, None, None, act)
    check_bwd(ns, dy, x, w, z if act != "none" else None, b, act)


@pytest.mark.parametrize("M,N,K,act", [(4112, 5120, 1280, "gelu"), (8192, 640, 2560, "none"), (3083, 1290, 650, "silu"), (2048, 1024, 1024, "none"), (20000, 320, 320, "gelu"),
                                       (5000, 1288, 4096, "none"), (4097, 5120, 1280, "relu"), (4127, 5117, 1283, "quick_gelu")])
def test_large_products_and_the_same_bits_twice(dev, ns, M, N, K, act):
    x, w, b = rnd((M, K), 1, "bf16").to(dev), rnd((N, K), 2, "bf16", K ** -0.5).to(dev), rnd((N,), 3, "fp32", 0.3).to(dev)
    dy, z = rnd((M, N), 5, "bf16").to(dev), rnd((M, N), 6, "bf16").to(dev)
    check_fwd(ns, x, w, b, dy, act)
    check_bwd(ns, dy, x, w, z if act != "none" else None, b, act)
    one = ns.linear_act(x, w, b, dy, act, True) + ns.linear_act_bwd(dy, x, w, z, b, act, True, True)
    two = ns.linear_act(x, w, b, dy, act, True) + ns.linear_act_bwd(dy, x, w, z, b, act, True, True)
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_places_are_not_exchanged(dev, ns):
    """Selections: every product of whole numbers is exact, so that an element in a wrong place is a wrong value."""
    M, N, K = 300, 340, 200
    x = torch.zeros(M, K).bfloat16()
    x[torch.arange(M), torch.arange(M) % K] = 1.0
    w = (torch.arange(N * K).reshape(N, K) % 251 - 125.0).bfloat16()
    dy = torch.zeros(M, N).bfloat16()
    dy[torch.arange(M), (torch.arange(M) * 7) % N] = 1.0
    y, _ = ns.linear_act(x.to(dev), w.to(dev), None, None, "none", False)
    assert torch.equal(y.cpu().float(), x.float() @ w.float().t())
    xx = (torch.arange(M * K).reshape(M, K) % 249 - 124.0).bfloat16()
    dx, dw, _ = ns.linear_act_bwd(dy.to(dev), xx.to(dev), w.to(dev), None, None, "none", True, True)
    assert torch.equal(dx.cpu().float(), dy.float() @ w.float())
    assert torch.equal(dw.cpu().float(), (dy.float().t() @ xx.float()).bfloat16().float())


def test_activation_tails(dev, ns):
    """Through an identity: gelu and its slope keep their digits where they are tiny, and the limits are the formula's."""
    v = torch.linspace(-14, 14, 4096).reshape(64, 64).half()
    eye = torch.eye(64, dtype=torch.float16)
    for act in ("gelu", "quick_gelu", "silu", "relu"):
        y, z = (t.cpu() for t in ns.linear_act(v.to(dev), eye.to(dev), None, None, act, True))
        assert torch.equal(z, v)
        near(y, ACTS[act](v.double()), 1e-5 * ACTS[act](v.double()).abs(), act)
        db = ns.linear_act_bwd(torch.ones_like(v).to(dev), v.to(dev), eye.to(dev), v.to(dev), None, act, True, False)[0].cpu()
        near(db, slope64(v.double(), act), 2e-5 * torch.ones(64, 64, dtype=torch.float64), act + "'")
    odd = torch.tensor([[float("inf"), float("nan"), 0.5, -3.0, 0.0, 0.0, 0.0, 0.0]]).half()
    for act in ("gelu", "quick_gelu", "silu", "relu"):                # one such value makes its whole row's sums of it: row by row, through a column of ones
        for v0 in (odd[0, 0], odd[0, 1], -odd[0, 0]):
            x1 = torch.zeros(1, 8, dtype=torch.float16)
            x1[0, 0] = v0
            y, z = (t.cpu() for t in ns.linear_act(x1.to(dev), torch.ones(8, 8, dtype=torch.float16, device=dev), None, None, act, True))
            assert torch.equal(torch.isnan(z), torch.isnan(v0).expand(1, 8)) and (torch.isnan(v0) or (z == v0).all())
            assert (torch.isnan(y) if torch.isnan(v0) else (y == v0) if v0 > 0 else (torch.isnan(y) | (y == 0))).all()
    big = torch.tensor([[1000.0, -1000.0, 60000.0, -60000.0, 0.0, -0.0, 1e-7, -1e-7]]).half()
    for act in ("gelu", "quick_gelu", "silu", "relu"):
        y, _ = ns.linear_act(big.to(dev), torch.eye(8, dtype=torch.float16, device=dev), None, None, act, False)
        near(y.cpu(), ACTS[act](big.double()), torch.full((1, 8), 1e-30, dtype=torch.float64), act)


def test_nan_and_infinity_stay_in_their_rows_and_columns(dev, ns):
    M, N, K = 70, 72, 96
    x, w, dy = rnd((M, K), 1, "bf16"), rnd((N, K), 2, "bf16"), rnd((M, N), 3, "bf16")
    x[5, 3], w[9, 4], dy[11, 20] = float("nan"), float("inf"), float("nan")
    y, _ = ns.linear_act(x.to(dev), w.to(dev), None, None, "none", False)
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[5] = bad[:, 9] = True
    assert torch.equal(~torch.isfinite(y.cpu()), bad)
    dx, dw, db = ns.linear_act_bwd(dy.to(dev), x.to(dev), w.to(dev), None, torch.zeros(N, device=dev), "none", True, True)
    bx = torch.zeros(M, K, dtype=torch.bool); bx[11] = True; bx[:, 4] = True
    bw = torch.zeros(N, K, dtype=torch.bool); bw[20] = True; bw[:, 3] = True
    assert torch.equal(~torch.isfinite(dx.cpu()), bx) and torch.equal(~torch.isfinite(dw.cpu()), bw)
    assert torch.equal(~torch.isfinite(db.cpu()), torch.arange(N) == 20)


def test_what_lies_around_the_operands_is_not_read_into_results(dev, ns):
    """Operands, bias and residual as windows of tensors that hold NaN elsewhere: every pitch, odd offsets, transposed ones; inputs stay as they were."""
    for M, N, K, at in ((70, 72, 104, 8), (70, 72, 104, 3), (65, 71, 99, 5), (300, 328, 136, 16)):
        def window(rows, cols, seed):
            t = torch.full((rows + 3, cols + 2 * at + 5), float("nan"), dtype=torch.bfloat16, device=dev)
            v = t[2:2 + rows, at:at + cols]
            v.copy_(rnd((rows, cols), seed, "bf16"))
            return v
        x, w, r, dy, z = window(M, K, 1), window(N, K, 2), window(M, N, 3), window(M, N, 4), window(M, N, 5)
        b = window(1, N, 6)[0]
        c = [t.contiguous() for t in (x, w, r, dy, z, b)]
        got = ns.linear_act(x, w, b, r, "silu", True) + ns.linear_act_bwd(dy, x, w, z, b, "silu", True, True) + ns.linear_act_bwd(dy, x, w, None, b, "none", True, True)
        want = ns.linear_act(c[0], c[1], c[5], c[2], "silu", True) + ns.linear_act_bwd(c[3], c[0], c[1], c[4], c[5], "silu", True, True) + \
            ns.linear_act_bwd(c[3], c[0], c[1], None, c[5], "none", True, True)
        assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(got, want))
        assert torch.equal(x, c[0]) and torch.equal(dy, c[3])
        xt = c[0].t().contiguous().t()                                            # [M, K] with unit stride along M
        assert torch.equal(ns.linear_act(xt, w, b, r, "silu", False)[0], want[0])
        e = ns.linear_act_bwd(dy[:1].expand(M, N), x, w, None, b, "none", True, True)          # a broadcast gradient
        f = ns.linear_act_bwd(c[3][:1].repeat(M, 1), c[0], c[1], None, c[5], "none", True, True)
        assert all(torch.equal(p, q) for p, q in zip(e, f))


def test_results_at_any_alignment(dev, ns):
    """The C entries' outputs (torch allocates aligned ones): one element off, and nothing around them is written."""
    import ctypes as C
    from hi3d_hip import lib as l
    lib = l.load()

    class Desc(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("x", "w", "bias", "residual", "y", "z", "dy", "dx", "dw", "db")] + \
                   [(n, C.c_int64) for n in ("M", "ldx", "ldw", "ldr", "lddy", "ldz")] + [(n, C.c_int32) for n in ("N", "K", "dtype", "bias_dtype", "act")] + \
                   [("ws", C.c_void_p), ("ws_bytes", C.c_int64)]
    M, N, K = 200, 136, 72
    x, w, b, dy, z = rnd((M, K), 1, "bf16").to(dev), rnd((N, K), 2, "bf16").to(dev), rnd((N,), 3).to(dev), rnd((M, N), 4, "bf16").to(dev), rnd((M, N), 5, "bf16").to(dev)
    y0, z0 = ns.linear_act(x, w, b, None, "gelu", True)
    g0 = ns.linear_act_bwd(dy, x, w, z, b, "gelu", True, True)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device=dev)
    off = [torch.full((n + 9,), 7.0, dtype=torch.bfloat16, device=dev) for n in (M * N, M * N, M * K, N * K)]
    p = [t.data_ptr() + 2 for t in off]
    db = torch.empty(N, device=dev)
    d = Desc(x=x.data_ptr(), w=w.data_ptr(), bias=b.data_ptr(), y=p[0], z=p[1], M=M, ldx=K, ldw=K, N=N, K=K, dtype=1, bias_dtype=0, act=1, ws=ws.data_ptr(), ws_bytes=ws.numel())
    st = torch.cuda.current_stream().cuda_stream
    assert lib.hi3d_linear_fwd(C.addressof(d), st) == 0
    e = Desc(x=x.data_ptr(), w=w.data_ptr(), dy=dy.data_ptr(), z=z.data_ptr(), dx=p[2], dw=p[3], db=db.data_ptr(), M=M, ldx=K, ldw=K, lddy=N, ldz=N, N=N, K=K, dtype=1, bias_dtype=0,
             act=1, ws=ws.data_ptr(), ws_bytes=ws.numel())
    assert lib.hi3d_linear_bwd(C.addressof(e), st) == 0
    torch.cuda.synchronize()
    for t, want in zip(off, (y0, z0, g0[0], g0[1])):
        n = want.numel()
        assert torch.equal(t[1:1 + n].reshape(want.shape), want) and t[0] == 7 and (t[1 + n:] == 7).all()
    assert torch.equal(db, g0[2])


def test_rows_far_apart(dev, ns):
    """Pitches that a tile's 32-bit offsets do not reach, for every operand."""
    M, N, K, ld = 65, 72, 96, 3_000_000
    c = [rnd((M, K), 1, "bf16"), rnd((N, K), 2, "bf16"), rnd((M, N), 3, "bf16"), rnd((M, N), 4, "bf16"), rnd((M, N), 5, "bf16")]
    flat = torch.zeros((N - 1) * ld + N * 5 + K, dtype=torch.bfloat16, device=dev)
    far, at = [], 0
    for t in c:                                    # all in one buffer, side by side
        v = flat.as_strided(t.shape, (ld, 1), at)
        v.copy_(t)
        far.append(v)
        at += (t.shape[1] + 7) // 8 * 8
    b = rnd((N,), 6).to(dev)
    c = [t.to(dev) for t in c]

    def run(x, w, r, dy, z):
        return ns.linear_act(x, w, b, r, "gelu", True) + ns.linear_act_bwd(dy, x, w, z, b, "gelu", True, True) + ns.linear_act_bwd(dy, x, w, None, b, "none", True, True)
    assert all(torch.equal(p, q) for p, q in zip(run(*far), run(*c)))


def test_no_rows(dev, ns):
    x, w, b = torch.zeros(0, 40, device=dev).bfloat16(), rnd((24, 40), 1, "bf16").to(dev), rnd((24,), 2).to(dev)
    y, z = ns.linear_act(x, w, b, x.new_zeros(0, 24), "gelu", True)
    assert y.shape == z.shape == (0, 24)
    dx, dw, db = ns.linear_act_bwd(y, x, w, z, b, "gelu", True, True)
    assert dx.shape == (0, 40) and dw.shape == (24, 40) and not dw.any() and not db.any()


def test_offsets_beyond_32_bits(dev, ns):
    """More than 2^31 elements of x and of y; the last rows are those of a product by themselves."""
    K, N = 64, 64
    M = (1 << 31) // 64 + 515
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=dev)
    w, tail = rnd((N, K), 2, "bf16").to(dev), rnd((700, K), 1, "bf16").to(dev)
    x[-700:] = tail
    y, _ = ns.linear_act(x, w, None, None, "none", False)
    ref, _ = ns.linear_act(tail, w, None, None, "none", False)
    assert torch.equal(y[-700:], ref) and not y[:1000].any()
    dx, dw, _ = ns.linear_act_bwd(y, x, w, None, None, "none", True, True)
    rx, rw, _ = ns.linear_act_bwd(ref, tail, w, None, None, "none", True, True)
    assert torch.equal(dx[-700:], rx)
    near(dw, rw.double(), torch.finfo(torch.bfloat16).eps / 2 * rw.double().abs() + 2 * chain(1024) * (ref.double().abs().t() @ tail.double().abs()), "dw")


def test_refusals(dev, ns):
    x, w, b, r = rnd((8, 16), 1, "bf16").to(dev), rnd((24, 16), 2, "bf16").to(dev), rnd((24,), 3).to(dev), rnd((8, 24), 4, "bf16").to(dev)
    f = lambda x=x, w=w, b=b, r=r, act="none": ns.linear_act(x, w, b, r, act, False)
    g = lambda dy=r, x=x, w=w, z=r, b=b, act="gelu": ns.linear_act_bwd(dy, x, w, z, b, act, True, True)
    f(), g()
    for bad in (dict(x=x.float()), dict(x=x.half()), dict(w=w.float()), dict(w=w[:, :8]), dict(b=b[:8]), dict(b=b.half()), dict(b=b.double()), dict(r=r[:4]), dict(r=r.float()),
                dict(act="tanh"), dict(x=x[0]), dict(w=w.cpu()), dict(x=x.cpu()), dict(x=x[:, :0], w=w[:, :0]), dict(w=w[:0], b=None, r=None)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(**bad)
    for bad in (dict(dy=r[:4]), dict(dy=r.float()), dict(z=None), dict(z=r[:, :8]), dict(x=x[:4]), dict(w=w[:8]), dict(act=""), dict(b=b[:3])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            g(**bad)
    with pytest.raises(RuntimeError):
        ns.linear_act(torch.zeros(1, 1, device=dev).bfloat16().expand(2, 2_200_000), torch.zeros(1, 1, device=dev).bfloat16().expand(2, 2_200_000), None, None, "none", False)


def test_differentiable_form(dev, ns):
    from hi3d_hip import train
    B, S, K, N = 2, 9, 40, 24
    x, w, b, r = (t.to(dev).requires_grad_() for t in (rnd((B, S, K), 1, "bf16"), rnd((N, K), 2, "bf16", 0.2), rnd((N,), 3), rnd((B, S, N), 4, "bf16")))
    g = rnd((B, S, N), 5, "bf16").to(dev)
    for act in ACTS:
        y = train.linear(x, w, b, residual=r, act=act)
        got = torch.autograd.grad(y, [x, w, b, r], g)
        _, z = ns.linear_act(x.detach().reshape(-1, K), w.detach(), b.detach(), None, act, True)
        dx, dw, db = ns.linear_act_bwd(g.reshape(-1, N), x.detach().reshape(-1, K), w.detach(), z, b.detach(), act, True, True)
        assert torch.equal(got[0].reshape(-1, K), dx) and torch.equal(got[1], dw) and torch.equal(got[2], db) and torch.equal(got[3], g)
        y = train.linear(x.detach(), w, None, act=act)                  # a frozen input: nothing is computed for it
        none = ns.linear_act_bwd(g.reshape(-1, N), x.detach().reshape(-1, K), w.detach(), ns.linear_act(x.detach().reshape(-1, K), w.detach(), None, None, act, True)[1],
                                 None, act, False, True)
        assert none[0] is None and torch.equal(torch.autograd.grad(y, w, g)[0], none[1])
        # differences of the formula in 64 bits along a direction of the weights
        v, t, W, X = rnd((N, K), 7).double().to(dev), 1e-6, w.detach().double(), x.detach().double()
        if act != "relu":                                               # (its kinks are not differentiable)
            fn = lambda a: (ACTS[act](X @ a.t() + b.detach().double()) * g.double()).sum()
            diff = (fn(W + t * v) - fn(W - t * v)) / (2 * t)
            z64 = X @ W.t() + b.detach().double()
            d = (g.double().abs() * 1.13).reshape(-1, N)
            # dz: z and dz are each rounded to bf16 (2^-8; the slope changes by less than z's change), dw once more
            bound = ((3 * 2.0 ** -8 * d * (1 + z64.reshape(-1, N).abs())).t() @ X.reshape(-1, K).abs() * v.abs()).sum()
            assert ((got[1].double() * v).sum() - diff).abs() < bound
    with pytest.raises(RuntimeError):
        train.linear(x, w, b, residual=r[:, :1])


def test_on_another_stream_and_replayed(dev, ns):
    x, w, b, dy = rnd((300, 640), 1, "bf16").to(dev), rnd((321, 640), 2, "bf16", 0.04).to(dev), rnd((321,), 3).to(dev), rnd((300, 321), 4, "bf16").to(dev)

    def both():
        y, z = ns.linear_act(x, w, b, dy, "gelu", True)
        return (y, z) + ns.linear_act_bwd(dy, x, w, z, b, "gelu", True, True)
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    with torch.cuda.graph(h):                           # a second graph: its workspaces are its own
        out2 = both()
    for seed in (5, 6, 7):
        x.copy_(rnd((300, 640), seed, "bf16"))
        g.replay(); h.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(p, q) and torch.equal(p2, q) for p, p2, q in zip(out, out2, want))


def test_a_training_step_of_a_feed_forward_block(dev):
    """The operators together, as a module tree that is trained uses them: x + W2 gelu(W1 norm(x)), its gradients, and an AdamW step with
    fp32 parameters and bf16 working copies -- against the same step in 64 bits from the same bf16 weights."""
    from hi3d_hip import train
    T, C, H = 200, 80, 320
    init = dict(g=rnd((C,), 1, "fp32", 0.2, 1.0), b=rnd((C,), 2, "fp32", 0.2), w1=rnd((H, C), 3, "fp32", C ** -0.5), b1=rnd((H,), 4, "fp32", 0.2),
                w2=rnd((C, H), 5, "fp32", H ** -0.5), b2=rnd((C,), 6, "fp32", 0.2))
    x, r, gy = rnd((T, C), 7, "bf16").to(dev), rnd((T, C), 8, "bf16").to(dev), rnd((T, C), 9, "bf16").to(dev)
    p = {k: torch.nn.Parameter(v.to(dev)) for k, v in init.items()}
    opt = train.AdamW(list(p.values()), lr=1e-2, weight_decay=0.05, working_dtype=torch.bfloat16)
    lo = {k: opt.working_copy(p[k]) if k in ("w1", "w2") else p[k] for k in p}
    y, z = train.layer_norm(x, lo["g"], lo["b"], residual=r)
    out = train.linear(train.linear(y, lo["w1"], lo["b1"], act="gelu"), lo["w2"], lo["b2"], residual=z)
    out.backward(gy)
    grads = {k: v.grad for k, v in lo.items()}
    assert p["w1"].grad is None and grads["w1"].dtype == torch.bfloat16
    q = {k: v.detach().double().requires_grad_() for k, v in lo.items()}
    zz = (x.float() + r.float()).bfloat16().double()
    h = F.linear(F.layer_norm(zz, (C,), q["g"], q["b"], 1e-5), q["w1"], q["b1"])
    ref = F.linear(F.gelu(h), q["w2"], q["b2"]) + zz
    assert ((out.double() - ref).norm() / ref.norm()).item() < 3 * 2.0 ** -8            # y, gelu(h) and out: three roundings
    for k, want in zip(q, torch.autograd.grad(ref, list(q.values()), gy.double())):
        # roundings on the way back: y, z1, gelu, dz1, the gradient that leaves the second layer, the stored one; each 2^-8 at most
        assert ((grads[k].double() - want).norm() / want.norm()).item() < 6 * 2.0 ** -8, k
    before = {k: v.detach().clone() for k, v in p.items()}
    opt.step()
    for k in p:
        g64 = grads[k].double()
        want = before[k].double() * (1 - 1e-2 * 0.05) - 1e-2 * g64 / (g64.abs() + 1e-8)     # the first step: m / sqrt(v) is the gradient's sign, but for eps
        assert ((p[k].double() - want).abs() <= 32 * U32 * (before[k].double().abs() + 1e-2) + 1e-2 * 1e-6).all(), k
        assert torch.equal(opt.working_copy(p[k]).detach(), p[k].detach().bfloat16())
    y, z = train.layer_norm(x, lo["g"], lo["b"], residual=r)
    stale = train.linear(y, lo["w1"], lo["b1"])
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        stale.sum().backward()
    opt.zero_grad()
    assert all(v.grad is None for v in lo.values())


@pytest.mark.parametrize("pitch", [0, 1, 8, 40, 1 << 40])
@pytest.mark.parametrize("M,N,K,act", [(1, 64, 72, "none"), (1, 136, 64, "gelu"), (1, 63, 65, "none"), (40, 1, 64, "none"), (40, 1, 65, "silu"), (1, 1, 8, "none")])
def test_a_single_row_has_no_pitch(dev, ns, M, N, K, act, pitch):
    """The C entries take any pitch for an operand of one row and never use it: the same bits as at its width.  dw's contraction runs over the rows of
    dy and x, dx's over those of w: a row that was read again would be counted again (an infinity times the zeros beside it as NaN)."""
    import ctypes as C
    from hi3d_hip import lib as l
    lib = l.load()

    class Desc(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("x", "w", "bias", "residual", "y", "z", "dy", "dx", "dw", "db")] + \
                   [(n, C.c_int64) for n in ("M", "ldx", "ldw", "ldr", "lddy", "ldz")] + [(n, C.c_int32) for n in ("N", "K", "dtype", "bias_dtype", "act")] + \
                   [("ws", C.c_void_p), ("ws_bytes", C.c_int64)]
    x, w, r, dy, z = (rnd(s, i, "bf16").to(dev) for i, s in enumerate(((M, K), (N, K), (M, N), (M, N), (M, N))))
    if N == 1:
        w[0, 3] = float("inf")
    b = rnd((N,), 9).to(dev)
    code = {"none": 0, "gelu": 1, "silu": 3}[act]
    y, kept = ns.linear_act(x, w, b, r, act, True)
    want = ns.linear_act_bwd(dy, x, w, z, b, act, True, True)
    if N == 1:
        assert torch.isinf(want[0][:, 3]).all() and torch.isfinite(want[0][:, :3]).all()
    out = [torch.zeros_like(t) for t in (y, kept, *want)]
    m1 = lambda width: pitch if M == 1 else width
    d = Desc(x=x.data_ptr(), w=w.data_ptr(), bias=b.data_ptr(), residual=r.data_ptr(), y=out[0].data_ptr(), z=out[1].data_ptr(), M=M, ldx=m1(K), ldr=m1(N),
             ldw=pitch if N == 1 else K, N=N, K=K, dtype=1, bias_dtype=0, act=code)
    e = Desc(x=x.data_ptr(), w=w.data_ptr(), dy=dy.data_ptr(), z=z.data_ptr(), dx=out[2].data_ptr(), dw=out[3].data_ptr(), db=out[4].data_ptr(), M=M, ldx=m1(K),
             ldw=pitch if N == 1 else K, lddy=m1(N), ldz=m1(N), N=N, K=K, dtype=1, bias_dtype=0, act=code)
    st = torch.cuda.current_stream().cuda_stream
    for desc, size, entry in ((d, lib.hi3d_linear_fwd_workspace_bytes, lib.hi3d_linear_fwd), (e, lib.hi3d_linear_bwd_workspace_bytes, lib.hi3d_linear_bwd)):
        ws = torch.empty(max(size(C.addressof(desc)), 1), dtype=torch.uint8, device=dev)
        desc.ws, desc.ws_bytes = ws.data_ptr(), ws.numel()
        assert entry(C.addressof(desc), st) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(p.view(torch.int16) if p.dtype == torch.bfloat16 else p, q.view(torch.int16) if q.dtype == torch.bfloat16 else q)
               for p, q in zip(out, (y, kept, *want)))


def test_gelus_slope_keeps_its_digits_in_32_bits(dev, ns):
    """The bias' gradient of one row of ones is the slope itself, not rounded to 16 bits: Phi(z) + z phi(z), |z| <= 13 (beyond, Phi(-|z|) leaves fp32's
    normal numbers).  Phi(-a): 1.5e-7 of the fit, a^2 2^-24 of the exponent's two roundings (a^2 / 2 each), and 24 roundings for the reciprocal, the
    exponential (a unit in the last place is two) and 16 steps; a phi(a): the exponent's again and 8; the sum of the two: 2."""
    z = torch.cat([torch.linspace(-13, 13, 8001), torch.linspace(-1e-2, 1e-2, 99), torch.zeros(1)]).bfloat16()[None]
    n = z.shape[1]
    one, w = torch.ones(1, n).bfloat16().to(dev), torch.zeros(n, 8).bfloat16().to(dev)
    got = ns.linear_act_bwd(one, torch.zeros(1, 8).bfloat16().to(dev), w, z.to(dev), torch.zeros(n, device=dev), "gelu", False, False)[2].double().cpu()
    z = z[0].double()
    a = z.abs()
    tail, bell = torch.special.log_ndtr(-a).exp(), torch.exp(-a * a / 2) * (0.5 / torch.pi) ** 0.5
    want = torch.where(z < 0, tail, 1 - tail) + z * bell
    slack = (1.5e-7 + (a * a + 24) * U32) * tail + (a * a + 8) * U32 * a * bell + 2 * U32 * want.abs()
    off = (got - want).abs() / slack
    assert (off <= 1).all(), f"worst {off.max().item():.2f} of its tolerance at {z[off.argmax()].item()}"


def test_a_gated_feed_forward_as_the_unets_have_it(dev):
    """Linear(C -> 8 C), split, a gelu(g), Linear(4 C -> C) and the residual (attention.py:87-113): both linear layers on the operators, the gate in torch.
    Result and gradients against 64 bits from the same bf16 weights, relative to their norm, 2^-8 for each bf16 rounding on the way."""
    from hi3d_hip import train
    T, C = 154, 80
    init = dict(w=rnd((8 * C, C), 3, "bf16", C ** -0.5), b=rnd((8 * C,), 4, "fp32", 0.2), v=rnd((C, 4 * C), 5, "bf16", (4 * C) ** -0.5), c=rnd((C,), 6, "fp32", 0.2),
                y=rnd((2, T // 2, C), 7, "bf16"), z=rnd((2, T // 2, C), 8, "bf16"))
    p = {k: t.to(dev).requires_grad_() for k, t in init.items()}
    q = {k: t.to(dev).double().requires_grad_() for k, t in init.items()}
    gy = rnd((2, T // 2, C), 9, "bf16").to(dev)
    a, g = train.linear(p["y"], p["w"], p["b"]).chunk(2, dim=-1)
    out = train.linear(a * F.gelu(g), p["v"], p["c"], residual=p["z"])
    out.backward(gy)
    a, g = F.linear(q["y"], q["w"], q["b"]).chunk(2, dim=-1)
    ref = F.linear(a * F.gelu(g), q["v"], q["c"]) + q["z"]
    ref.backward(gy.double())
    assert ((out.double() - ref).norm() / ref.norm()).item() < 4 * 2.0 ** -8              # a and g, gelu(g), the product, the result
    for k in p:
        # those, and on the way back the product's gradient, the two that the gate sends (through a product each), and the stored one
        assert ((p[k].grad.double() - q[k].grad).norm() / q[k].grad.norm()).item() < 9 * 2.0 ** -8, k
