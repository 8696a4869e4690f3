"""AdamW over many tensors (torch.ops.hi3d.adamw_, hi3d_hip.train.AdamW) against the formula in 64 bits.

Tolerances: a stored value's one rounding (eps / 2 of its type), plus fp32 arithmetic: m and v are two products and a sum (4 roundings of
2^-24 on the sum of absolute values), the parameter's change is those through sqrt, division and three products (16 roundings of
itself), and the coefficients are rounded to fp32 once (counted among them).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U32 = 2.0 ** -24
H = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.02)


@pytest.fixture(scope="module")
def ns():
    from hi3d_hip import torch_ops
    return torch_ops.load()


def tensors(sizes, dt, gdt, seed, dev, copy=None):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, s, d: (torch.randn(n, generator=g) * s).to(d)
    p, gr = [mk(n, 0.03, DT[dt]) for n in sizes], [mk(n, 1e-3, DT[gdt]) for n in sizes]
    m, v = [mk(n, 1e-3, torch.float32) for n in sizes], [mk(n, 1e-3, torch.float32).square() for n in sizes]
    c = [torch.zeros(n, dtype=DT[copy]) for n in sizes] if copy else []
    return [[t.to(dev) for t in l] for l in (p, gr, m, v, c)]


def step64(p, g, m, v, step, scale=1.0, lr=None):
    """One step in 64 bits, with the slack of each result."""
    p, m, v, g = p.double(), m.double(), v.double(), g.double() / scale
    lr = H["lr"] if lr is None else lr
    m1, v1 = H["b1"] * m + (1 - H["b1"]) * g, H["b2"] * v + (1 - H["b2"]) * g * g
    sm, sv = 4 * U32 * (m.abs() + g.abs()), 4 * U32 * (v + g * g)
    den = v1.sqrt() / math.sqrt(1 - H["b2"] ** step) + H["eps"]
    size = lr / (1 - H["b1"] ** step)
    change = size * m1 / den
    # v's own error is within 4 roundings of v1 or so: v1 >= b2 v + (1 - b2) g^2 >= 1e-3 (v + g^2), and sqrt halves it
    s_change = 16 * U32 * change.abs() + size * sm / den + change.abs() * sv / (2 * v1.clamp_min(1e-300))
    p1 = p * (1 - lr * H["wd"]) - change
    return (p1, 4 * U32 * p.abs() + s_change), (m1, sm), (v1, sv)


def near(got, want, slack, what):
    u = torch.finfo(got.dtype).eps / 2
    g = got.double().cpu()
    tol = u * want.abs() + slack * (1 + u) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bad = (g - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((g - want).abs() / tol).max().item():.2f} of its tolerance"


def call(ns, t, step=7, lr=None, **dev):
    ns.adamw_(*t, H["lr"] if lr is None else lr, H["b1"], H["b2"], H["eps"], H["wd"], step, dev.get("step_t"), dev.get("lr_t"), dev.get("scale"), dev.get("found"))


def check(t, before, step, scale=1.0, lr=None):
    for i in range(len(t[0])):
        want = step64(*[before[k][i].cpu() for k in (0, 1, 2, 3)], step, scale, lr)
        for k, (w, s) in zip((0, 2, 3), want):
            near(t[k][i], w, s, f"tensor {i} of {t[0][i].numel()}, list {k}")
        if t[4]:     # the copy is of the 32-bit value before its rounding to storage, which is exact: two roundings at most
            near(t[4][i], want[0][0], want[0][1], f"copy {i}")
        assert torch.equal(t[1][i], before[1][i])


@pytest.mark.parametrize("dt,gdt,copy", [("fp32", "fp32", None), ("fp32", "bf16", "bf16"), ("fp32", "fp16", "fp16"), ("bf16", "bf16", None),
                                         ("fp16", "fp16", None), ("bf16", "fp32", None)])
@pytest.mark.parametrize("step", [1, 1000])
def test_step(dev, ns, dt, gdt, copy, step):
    sizes = [0, 1, 2, 3, 5, 4095, 4096, 4097, 64, 100003, 1]
    t = tensors(sizes, dt, gdt, step, dev, copy)
    before = [[x.clone() for x in l] for l in t]
    call(ns, t, step)
    check(t, before, step)


def test_more_tensors_than_one_launch_takes_and_mixed_types(dev, ns):
    a, b = tensors([13 + i for i in range(150)], "fp32", "bf16", 1, dev), tensors([7 * i + 1 for i in range(100)], "bf16", "bf16", 2, dev)
    t = [[x for pair in zip(p, q) for x in pair] + p[len(q):] for p, q in zip(a, b)]
    before = [[x.clone() for x in l] for l in t]
    call(ns, t)
    check(t, before, 7)
    again = [[x.clone() for x in l] for l in before]
    call(ns, again)
    assert all(torch.equal(x, y) for l, k in zip(t, again) for x, y in zip(l, k))


def test_views_at_odd_offsets_touch_nothing_else(dev, ns):
    sizes = [5, 1, 4099, 33, 7, 8192]
    t = tensors([sum(sizes) + 9], "fp32", "fp16", 3, dev, "bf16")
    flat = [l[0] for l in t]
    before = [f.clone() for f in flat]
    parts = [list(f[1:1 + sum(sizes)].split(sizes)) for f in flat]
    olds = [list(f[1:1 + sum(sizes)].split(sizes)) for f in before]
    call(ns, parts)
    check(parts, olds, 7)
    for f, o in zip(flat, before):
        assert torch.equal(f[:1], o[:1]) and torch.equal(f[1 + sum(sizes):], o[1 + sum(sizes):])


def test_dense_tensors_in_any_order_of_dimensions(dev, ns):
    mk = lambda s: torch.randn((6, 5, 3, 3), generator=torch.Generator().manual_seed(s)).to(dev).to(memory_format=torch.channels_last)
    t = [[mk(1)], [mk(2)], [mk(3)], [mk(4).square()], []]
    ref = [[x.permute(0, 2, 3, 1).reshape(-1).clone() for x in l] for l in t]
    call(ns, t)
    call(ns, ref)
    for l, k in zip(t, ref):
        for x, y in zip(l, k):
            assert torch.equal(x.permute(0, 2, 3, 1).reshape(-1), y)


def test_step_count_rate_scale_and_overflow_on_the_device(dev, ns):
    sizes = [100, 4097]
    t = tensors(sizes, "fp32", "fp16", 5, dev, "fp16")
    one = lambda v: torch.full((1,), v, device=dev)
    step, lr, scale, found = one(41.0), one(2e-3), one(1024.0), one(0.0)
    before = [[x.clone() for x in l] for l in t]
    call(ns, t, step=1, step_t=step, lr_t=lr, scale=scale, found=found)
    assert step.item() == 42
    check(t, before, 42, 1024.0, float(lr))          # the rate as fp32 holds it
    before = [[x.clone() for x in l] for l in t]
    found.fill_(1.0)
    t[1][0][3] = float("inf")
    call(ns, t, step=1, step_t=step, lr_t=lr, scale=scale, found=found)
    assert step.item() == 42 and all(torch.equal(x, y) for k in (0, 2, 3, 4) for x, y in zip(t[k], before[k]))
    found.fill_(0.0)
    t[1][0][3] = 0.0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(ns, t, step=1, step_t=step, lr_t=lr, scale=scale, found=found)
    for k in range(3):
        before = [[x.clone() for x in l] for l in t]
        g.replay()
        torch.cuda.synchronize()
        assert step.item() == 43 + k
        check(t, before, 43 + k, 1024.0, float(lr))
        lr.mul_(0.5)


def test_zero_and_non_finite_gradients_stay_in_their_elements(dev, ns):
    t = tensors([64], "fp32", "fp32", 6, dev)
    t[1][0].zero_(); t[2][0].zero_(); t[3][0].zero_()
    p = t[0][0].clone()
    t[1][0][5], t[1][0][9] = float("nan"), float("inf")
    call(ns, t, 1)
    bad = torch.tensor([i in (5, 9) for i in range(64)], device=dev)
    assert torch.isnan(t[0][0][bad]).all()
    near(t[0][0][~bad], (p.double().cpu() * (1 - H["lr"] * H["wd"]))[~bad.cpu()], 2 * U32 * p.double().cpu().abs()[~bad.cpu()], "decay alone")


def test_refusals(dev, ns):
    def fresh():
        return tensors([32, 64], "fp32", "fp32", 7, dev)
    def expect(change, **kw):
        t = fresh()
        t = change(t) or t
        before = [[x.clone() for x in l] for l in t]
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(ns, t, **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for l, k in zip(t, before) for x, y in zip(l, k))
    expect(lambda t: [t[0][:1]] + t[1:])                                              # lists of different lengths
    expect(lambda t: [[t[0][0], t[0][0]], [t[1][0]] * 2, [t[2][0], t[2][0].clone()], [t[3][0], t[3][0].clone()], []])      # a parameter twice
    expect(lambda t: [t[0], t[1], [t[3][0], t[2][1]], t[3], []])                      # m is v
    expect(lambda t: [t[0], [t[0][0], t[1][1]], t[2], t[3], []])                      # the gradient is the parameter
    expect(lambda t: [[t[0][0].bfloat16(), t[0][1]], t[1], t[2], t[3], [t[0][0].half(), t[0][1].half()]])    # a copy of a 16-bit parameter
    expect(lambda t: [t[0], t[1], [t[2][0].half(), t[2][1]], t[3], []])
    expect(lambda t: [[t[0][0].double(), t[0][1]], t[1], t[2], t[3], []])
    expect(lambda t: [[t[0][0][::2], t[0][1]], [t[1][0][::2], t[1][1]], [t[2][0][::2], t[2][1]], [t[3][0][::2], t[3][1]], []])   # holes
    expect(lambda t: [t[0], [t[1][0][:16], t[1][1]], t[2], t[3], []])
    expect(lambda t: [t[0], [t[1][0].cpu(), t[1][1]], t[2], t[3], []])
    expect(lambda t: None, step=0)
    expect(lambda t: None, lr=-1.0)
    expect(lambda t: None, lr=float("nan"))
    expect(lambda t: None, found=torch.zeros(1, device=dev))                          # without the step on the device
    expect(lambda t: None, step_t=torch.zeros(1, device=dev, dtype=torch.float64))


def test_optimiser_is_torchs(dev):
    """train.AdamW against torch.optim.AdamW's single-tensor form in 64 bits: several steps, a parameter without a gradient at first, two groups, and a
    state that is saved and loaded half way (moments of bf16 parameters stay fp32)."""
    from hi3d_hip import train
    shapes = [(33,), (16, 8), (4, 3, 3, 3), (1,)]
    gen = torch.Generator().manual_seed(3)
    init = [torch.randn(s, generator=gen) * 0.1 for s in shapes]
    mine = [torch.nn.Parameter(t.clone().to(dev)) for t in init]
    mine[2] = torch.nn.Parameter(init[2].to(dev).to(memory_format=torch.channels_last))
    ref = [torch.nn.Parameter(t.double()) for t in init]
    groups = lambda p: [dict(params=p[:2], lr=1e-2), dict(params=p[2:], lr=3e-3, weight_decay=0.1, betas=(0.8, 0.95))]
    opt, ropt = train.AdamW(groups(mine)), torch.optim.AdamW(groups(ref), foreach=False)
    steps = 6
    for k in range(steps):
        for i, (p, q) in enumerate(zip(mine, ref)):
            if i == 1 and k < 2:
                continue
            g = torch.randn(p.shape, generator=gen)
            p.grad, q.grad = g.to(dev), g.double()          # (parameter 2's gradient has other strides than it)
        opt.step(); ropt.step()
        if k == 3:
            sd = opt.state_dict()
            opt = train.AdamW(groups(mine))
            opt.load_state_dict(sd)
    for p, q in zip(mine, ref):
        # a step's slack (above) is under 40 U of its change plus 4 U of p; m and v carry theirs along
        want = q.detach()
        assert ((p.detach().double().cpu() - want).abs() <= steps * 64 * U32 * (want.abs() + steps * 1e-2 * 3)).all()
    b = torch.nn.Parameter(torch.randn(10, device=dev).bfloat16())
    o = train.AdamW([b])
    b.grad = torch.ones_like(b)
    o.step()
    o2 = train.AdamW([b])
    o2.load_state_dict(o.state_dict())
    t = torch.nn.Parameter(b.detach().float())                    # a state that torch's optimiser saved
    ot = torch.optim.AdamW([t], lr=0.5, weight_decay=0.0)
    t.grad = torch.ones_like(t)
    ot.step()
    u = torch.nn.Parameter(t.detach().clone())
    o5 = train.AdamW([u])
    o5.load_state_dict(ot.state_dict())
    with pytest.raises(RuntimeError):
        train.AdamW([u]).load_state_dict(torch.optim.AdamW([u], amsgrad=True).state_dict())
    t.grad = u.grad = torch.full_like(t, 0.5)
    ot.step(); o5.step()
    assert o5.state[u]["step"] == 2 and o5.param_groups[0]["lr"] == 0.5
    assert ((t - u).abs() <= 64 * U32 * (t.detach().abs() + 1)).all()          # (both in fp32: a step's roundings, above, on each side)
    w = torch.nn.Parameter(torch.randn(10, device=dev))
    o3, o4 = train.AdamW([w], working_dtype=torch.bfloat16), train.AdamW([w], working_dtype=torch.bfloat16)
    held = o4.working_copy(w)
    o3.working_copy(w).grad = torch.ones(10, device=dev).bfloat16()
    o3.step()
    o4.load_state_dict(o3.state_dict())
    assert o4.working_copy(w) is held and torch.equal(held, w.bfloat16()) and held.requires_grad and held.is_leaf
    assert o2.state[b]["exp_avg"].dtype == torch.float32 and torch.equal(o2.state[b]["exp_avg"], o.state[b]["exp_avg"]) and o2.state[b]["step"] == 1


def test_optimiser_state_between_its_modes(dev):
    """A state goes from host to device counts and back with its step count, and what the optimiser has handed out stays in use."""
    from hi3d_hip import train
    gen = torch.Generator().manual_seed(29)
    start = torch.randn(300, generator=gen).to(dev)
    grads = [torch.randn(300, generator=gen).to(dev) for _ in range(6)]

    def take(opt, p, i):
        p.grad = grads[i].clone()
        opt.step()

    a = torch.nn.Parameter(start.clone())                  # six steps without a break
    whole = train.AdamW([a], lr=1e-2)
    for i in range(6):
        take(whole, a, i)

    b = torch.nn.Parameter(start.clone())                  # host counts, device counts, host counts: two steps each
    first = train.AdamW([b], lr=1e-2)
    take(first, b, 0); take(first, b, 1)
    second = train.AdamW([b], lr=torch.full((1,), 0.5, device=dev), capturable=True)
    lr = second.param_groups[0]["lr"]
    second.load_state_dict(first.state_dict())
    group = second.param_groups[0]
    assert group["capturable"] and group["lr"] is lr and abs(float(lr) - 1e-2) < 1e-8 and int(group["step_t"]) == 2
    take(second, b, 2); take(second, b, 3)
    third = train.AdamW([b], lr=0.5)
    third.load_state_dict(second.state_dict())
    assert not third.param_groups[0]["capturable"] and third.state[b]["step"] == 4
    take(third, b, 4); take(third, b, 5)
    # lr from fp32 device memory is off by half a step, relative: the rest is a step's roundings, 40 U of its change and 4 U of p
    assert ((a - b).detach().abs() <= 6 * 128 * U32 * (a.detach().abs() + 6e-2 * 3)).all()

    # buffers that are held are filled, not replaced; a state without copies gives the parameter, rounded
    c = torch.nn.Parameter(start.clone())
    opt = train.AdamW([c], working_dtype=torch.bfloat16, capturable=True)
    copy = opt.working_copy(c)
    copy.grad = grads[0].bfloat16()
    opt.step()
    state, count = dict(opt.state[c]), opt.param_groups[0]["step_t"]
    with torch.no_grad():
        c.copy_(b)
    opt.load_state_dict(third.state_dict())
    assert opt.working_copy(c) is copy and torch.equal(copy, b.bfloat16()) and opt.param_groups[0]["step_t"] is count and int(count) == 6
    for k in ("exp_avg", "exp_avg_sq"):
        assert opt.state[c][k] is state[k] and torch.equal(state[k], third.state[b][k])

    # different counts cannot be kept as one on the device
    p = [torch.nn.Parameter(start.clone()) for _ in range(2)]
    uneven = train.AdamW(p)
    take(uneven, p[0], 0)
    with pytest.raises(RuntimeError):
        train.AdamW(p, capturable=True).load_state_dict(uneven.state_dict())


def test_optimiser_with_working_copies_captured(dev):
    from hi3d_hip import train
    p = [torch.nn.Parameter(torch.randn(n, device=dev)) for n in (10, 4100)]
    lr = torch.full((1,), 1e-2, device=dev)
    opt = train.AdamW(p, lr=lr, working_dtype=torch.bfloat16, capturable=True)
    for q in p:
        assert torch.equal(opt.working_copy(q), q.detach().bfloat16())
        q.grad = torch.randn_like(q)
    opt.step()                                           # eager first: the states exist
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    q = [torch.nn.Parameter(t.detach().clone()) for t in p]
    plain = train.AdamW(q, lr=1e-2)
    for a, b in zip(q, p):
        plain._state_of(a, plain.param_groups[0]).update(step=1, exp_avg=opt.state[b]["exp_avg"].clone(), exp_avg_sq=opt.state[b]["exp_avg_sq"].clone())
    for k in range(3):
        for a, b in zip(q, p):
            b.grad.copy_(torch.randn_like(b))
            a.grad = b.grad.clone()
        lr.fill_(1e-2 / (k + 1))
        plain.param_groups[0]["lr"] = float(lr)
        g.replay()
        plain.step()
        torch.cuda.synchronize()
        for a, b in zip(q, p):
            assert torch.equal(a, b) and torch.equal(opt.working_copy(b), b.detach().bfloat16())
    p[0].grad = None
    with pytest.raises(RuntimeError):
        opt.step()
    with pytest.raises(ValueError):
        train.AdamW(p, lr=lr)
    with pytest.raises(ValueError):
        train.AdamW(p, betas=(1.0, 0.9))


def test_a_step_that_counts_on_the_host_is_not_captured(dev):
    from hi3d_hip import train
    p = torch.nn.Parameter(torch.randn(100, device=dev))
    p.grad = torch.randn_like(p)
    opt = train.AdamW([p], lr=1e-2)
    opt.step()
    before, state = p.detach().clone(), {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state[p].items()}
    other = torch.zeros(1, device=dev)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        other += 1
        with pytest.raises(RuntimeError, match="capturable"):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, before) and all(torch.equal(v, opt.state[p][k]) if torch.is_tensor(v) else v == opt.state[p][k] for k, v in state.items())
    opt.step()                                   # and goes on outside of it
    assert opt.state[p]["step"] == 2 and not torch.equal(p, before)


def test_the_first_step_captured(dev):
    """With the working copies taken beforehand everything that a step keeps is there: replays of a captured first step are the eager steps, and the
    count goes on from replay to replay.  Without them the capture is refused."""
    from hi3d_hip import train
    start = [torch.randn(n, device=dev) for n in (10, 4100)]
    grads = [[torch.randn_like(t) for t in start] for _ in range(4)]
    p, q = ([torch.nn.Parameter(t.clone()) for t in start] for _ in range(2))
    make = lambda params: train.AdamW(params, lr=torch.full((1,), 1e-2, device=dev), working_dtype=torch.bfloat16, capturable=True)
    opt, eager = make(p), make(q)
    for a, g in zip(p, grads[0]):
        a.grad = g.clone()
    other = torch.zeros(1, device=dev)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        other += 1
        with pytest.raises(RuntimeError, match="captur"):
            opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, t) for a, t in zip(p, start))
    copies = [opt.working_copy(a) for a in p]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for k in range(4):
        for a, b, t in zip(p, q, grads[k]):
            a.grad.copy_(t)
            b.grad = t.clone()
        g.replay()
        eager.step()
        torch.cuda.synchronize()
        assert opt.param_groups[0]["step_t"].item() == k + 1
        for a, b, c in zip(p, q, copies):
            assert torch.equal(a, b) and torch.equal(c, b.detach().bfloat16())
            assert all(torch.equal(opt.state[a][n], eager.state[b][n]) for n in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("modes", [(True, True), (True, False), (False, True), (False, False)])
def test_with_a_loss_scale(dev, modes):
    """torch.amp.GradScaler over groups that count on the device and on the host, the second added later: the steps of unscaled gradients, and an
    overflow is a step that nobody takes.  The scale is a power of two: scaled and unscaled gradients have the same digits."""
    from hi3d_hip import train
    start = [torch.randn(n, device=dev) for n in (33, 4100)]
    def make():
        p = [torch.nn.Parameter(t.clone()) for t in start]
        opt = train.AdamW([p[0]], lr=1e-2, capturable=modes[0])
        opt.add_param_group(dict(params=[p[1]], capturable=modes[1]))
        return p, opt
    (p, opt), (q, plain) = make(), make()
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    for k in range(4):
        scaled = scaler.scale(torch.ones(1, device=dev)).item()
        grads = [torch.randn_like(t) for t in start]
        for a, b, g in zip(p, q, grads):
            a.grad, b.grad = g * scaled, g.clone()
        before = [a.detach().clone() for a in p]
        if k == 2:
            p[1].grad[7] = float("inf")
        scaler.step(opt)
        scaler.update()
        if k == 2:
            assert all(torch.equal(a, t) for a, t in zip(p, before)) and scaler.get_scale() == 512.0
            continue
        plain.step()
        assert all(torch.equal(a, b) for a, b in zip(p, q)), k
