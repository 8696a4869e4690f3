"""The training kernels' entry points without a GPU: what they refuse before anything is launched, and that they are there."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from hi3d_hip import lib as l
    return l.load()


BAD_TYPE, F32, BF16 = 9, 0, 1
P = 4096          # a pointer that is never followed


def norm_fwd(lib, **k):
    a = dict(x=P, r=0, w=P, b=P, y=P, z=0, mean=P, rstd=P, R=4, C=8, ldx=8, ldr=0, dt=F32, wdt=F32, eps=1e-5) | k
    return lib.hi3d_layernorm_fwd(a["x"], a["r"], a["w"], a["b"], a["y"], a["z"], a["mean"], a["rstd"], a["R"], a["C"], a["ldx"], a["ldr"], a["dt"], a["wdt"], a["eps"], 0)


@pytest.mark.parametrize("k", [dict(x=0), dict(y=0), dict(mean=0), dict(rstd=0), dict(r=P), dict(R=-1), dict(C=0), dict(C=8193), dict(dt=BAD_TYPE), dict(wdt=BAD_TYPE),
                               dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(ldx=7), dict(r=P, z=P, ldr=7)])
def test_layernorm_fwd_refuses(lib, k):
    assert norm_fwd(lib, **k) < 0 and lib.hi3d_last_error()


def test_layernorm_of_no_rows_is_nothing(lib):
    assert norm_fwd(lib, R=0, x=0, y=0, mean=0, rstd=0) == 0
    assert lib.hi3d_layernorm_bwd(*[0] * 10, 0, 8, 8, 8, 8, F32, F32, 0) == 0


def test_layernorm_bwd_refuses(lib):
    def bwd(**k):
        a = dict(dy=P, z=P, dz=0, w=P, mean=P, rstd=P, dx=P, dw=P, db=P, ws=P, R=100000, C=8, lddy=8, ldz=8, lddz=8, dt=F32, wdt=F32) | k
        return lib.hi3d_layernorm_bwd(*[a[n] for n in ("dy", "z", "dz", "w", "mean", "rstd", "dx", "dw", "db", "ws", "R", "C", "lddy", "ldz", "lddz", "dt", "wdt")], 0)
    for k in (dict(dy=0), dict(z=0), dict(mean=0), dict(rstd=0), dict(dx=0), dict(ws=0), dict(R=-1), dict(C=0), dict(C=8193), dict(dt=BAD_TYPE), dict(wdt=-1),
              dict(lddy=7), dict(ldz=0), dict(dz=P, lddz=7)):
        assert bwd(**k) < 0, k
    assert lib.hi3d_layernorm_bwd_workspace_floats(1, 8, F32) == 0 and lib.hi3d_layernorm_bwd_workspace_floats(-1, 8, F32) == 0
    assert lib.hi3d_layernorm_bwd_workspace_floats(1 << 40, 640, BF16) == 512 * 2 * 640


def test_adamw_refuses(lib):
    class T(C.Structure):
        _fields_ = [("p", C.c_void_p), ("g", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p), ("copy", C.c_void_p), ("n", C.c_int64)]
    coefs = (C.c_float * 9)()
    step = lambda t, n, pd=F32, gd=F32, cd=BF16, c=coefs: lib.hi3d_adamw_step(C.addressof(t) if t is not None else 0, n, pd, gd, cd, C.addressof(c) if c is not None else 0, 0, 0)
    ok = T(P, P, P, P, 0, 0)
    assert step(ok, 1) == 0 and step(None, 0) == 0                    # no elements, no tensors: nothing is launched
    for t, n, kw in ((None, 1, {}), (ok, -1, {}), (ok, 1, dict(pd=BAD_TYPE)), (ok, 1, dict(gd=BAD_TYPE)), (ok, 1, dict(cd=F32)), (ok, 1, dict(c=None)),
                     (T(0, P, P, P, 0, 4), 1, {}), (T(P, 0, P, P, 0, 4), 1, {}), (T(P, P, 0, P, 0, 4), 1, {}), (T(P, P, P, 0, 0, 4), 1, {}), (T(P, P, P, P, 0, -4), 1, {})):
        assert step(t, n, **kw) < 0
    for k in (0, 1, 5):
        assert lib.hi3d_adamw_coefs(*[0 if i == k else P if i in (0, 1, 5) else 0 for i in range(6)], 0) < 0


class Linear(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("x", "w", "bias", "residual", "y", "z", "dy", "dx", "dw", "db")] + \
               [(n, C.c_int64) for n in ("M", "ldx", "ldw", "ldr", "lddy", "ldz")] + [(n, C.c_int32) for n in ("N", "K", "dtype", "bias_dtype", "act")] + \
               [("ws", C.c_void_p), ("ws_bytes", C.c_int64)]


def linear(**k):
    a = dict(x=P, w=P, bias=P, residual=0, y=P, z=0, dy=P, dx=P, dw=P, db=P, M=64, ldx=64, ldw=64, ldr=64, lddy=64, ldz=64, N=64, K=64, dtype=BF16, bias_dtype=F32, act=0,
             ws=P, ws_bytes=1 << 40) | k
    return Linear(**{n: (a[n] or None) if t is C.c_void_p else a[n] for n, t in Linear._fields_})


@pytest.mark.parametrize("k", [dict(x=0), dict(w=0), dict(M=-1), dict(N=0), dict(K=0), dict(dtype=F32), dict(dtype=BAD_TYPE), dict(bias_dtype=2), dict(act=5), dict(act=-1),
                               dict(ldw=63), dict(ldx=63), dict(M=65, K=63, ws=0), dict(M=65, K=63, ws_bytes=10), dict(M=65, K=63, ws=P + 8), dict(K=1 << 22, ldx=1 << 22, ldw=1 << 22),
                               dict(N=1 << 22), dict(M=1 << 31)])
def test_linear_refuses(lib, k):
    d = linear(**k)
    assert lib.hi3d_linear_fwd(C.addressof(d), 0) < 0 and lib.hi3d_last_error()


@pytest.mark.parametrize("k", [dict(dy=0), dict(x=0), dict(w=0), dict(act=1), dict(act=1, z=P, ldz=63), dict(lddy=63), dict(ldx=63), dict(ldw=63), dict(M=129, db=P, ws=0), dict(M=1 << 31),
                               dict(act=1, z=P, ws_bytes=64 * 64 * 2 - 1)])
def test_linear_bwd_refuses(lib, k):
    d = linear(**k)
    assert lib.hi3d_linear_bwd(C.addressof(d), 0) < 0 and lib.hi3d_last_error()


def test_linear_null_and_empty(lib):
    assert lib.hi3d_linear_fwd(0, 0) < 0 and lib.hi3d_linear_bwd(0, 0) < 0
    assert lib.hi3d_linear_fwd_workspace_bytes(0) == 0 and lib.hi3d_linear_bwd_workspace_bytes(0) == 0
    assert lib.hi3d_linear_fwd(C.addressof(linear(M=0, x=0, y=0)), 0) == 0
    assert lib.hi3d_linear_bwd(C.addressof(linear(M=0, dy=0, dw=0, db=0)), 0) == 0
    # rows of 63 elements cannot be read in place: both operands are copied; 64 can
    assert lib.hi3d_linear_fwd_workspace_bytes(C.addressof(linear(M=1024, N=1024, K=64))) == 0
    assert lib.hi3d_linear_fwd_workspace_bytes(C.addressof(linear(M=1024, N=1024, K=63))) == 2 * 1024 * 64 * 2


def test_cpu_tensors_are_refused():
    from hi3d_hip import torch_ops, train
    ns = torch_ops.load()
    x = torch.zeros(2, 4)
    for f in (lambda: ns.layernorm_fwd(x, None, None, 1e-5), lambda: ns.add_layernorm_fwd(x, x, None, None, 1e-5), lambda: train.layer_norm(x),
              lambda: ns.linear_act(x, x, None, None, "none", False), lambda: ns.linear_act_bwd(x[:, :2], x, x, None, None, "none", True, True),
              lambda: ns.adamw_([x], [x], [x], [x], [], 0.1, 0.9, 0.99, 1e-8, 0.0, 1, None, None, None, None)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()
    opt = train.AdamW([torch.nn.Parameter(x)])
    opt.param_groups[0]["params"][0].grad = x.clone()
    with pytest.raises((RuntimeError, NotImplementedError)):
        opt.step()


def test_linear_of_one_row_takes_no_notice_of_its_pitch(lib):
    """An operand of one row is read where it lies, whatever pitch stands beside it: the same workspace as at its width."""
    size = lambda **k: lib.hi3d_linear_bwd_workspace_bytes(C.addressof(linear(db=0, z=P, **k)))
    for act in (0, 1):
        assert size(M=1, ldx=3, lddy=0, ldz=1, act=act) == size(M=1, ldx=1 << 40, lddy=8, act=act) == size(M=1, act=act)
        assert size(M=1, K=63, ldx=0, ldw=63, act=act) == size(M=1, K=63, ldx=63, ldw=63, act=act)
        assert size(N=1, ldw=3, lddy=1, ldz=1, act=act) == size(N=1, lddy=1, ldz=1, act=act)
    fwd = lambda **k: lib.hi3d_linear_fwd_workspace_bytes(C.addressof(linear(**k)))
    assert fwd(N=1, ldw=3, ldr=1) == fwd(N=1, ldr=1) == 0


def leaf(n=4, dtype=torch.float32, grad=True):
    p = torch.nn.Parameter(torch.ones(n, dtype=dtype))
    if grad:
        p.grad = torch.ones(n, dtype=dtype)
    return p


class Launches:
    """In the operators' place: takes what AdamW.step() hands over, refuses where it is told to."""
    def __init__(self, refuse=()):
        self.calls, self.refuse = [], list(refuse)

    def adamw_(self, *a):
        if self.refuse and self.refuse.pop(0):
            raise RuntimeError("refused")
        self.calls.append(a)


@pytest.fixture
def launches(monkeypatch):
    from hi3d_hip import train
    def put(**k):
        l = Launches(**k)
        monkeypatch.setattr(train.torch_ops, "load", lambda: l)
        return l
    return put


@pytest.fixture
def capturing(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)


def test_a_step_that_counts_on_the_host_is_not_captured(launches, capturing):
    """A replay would take the same step number and rate for ever."""
    from hi3d_hip import train
    ops = launches()
    p, q = leaf(), leaf()
    for opt in (train.AdamW([p, q]), train.AdamW([dict(params=[p], capturable=True), dict(params=[q])])):
        with pytest.raises(RuntimeError, match="capturable"):
            opt.step()
        assert not ops.calls and not opt.state


def test_state_is_not_made_in_a_capture(launches, monkeypatch):
    """What is made in a capture is made again, as zeros, by every replay: the moments, the working copies and the step count have to be there."""
    from hi3d_hip import train
    ops = launches()
    p, q = leaf(), leaf()
    opt = train.AdamW([p, q], working_dtype=torch.bfloat16, capturable=True)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_initialized", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for f in (opt.step, lambda: opt.working_copy(p)):
            with pytest.raises(RuntimeError, match="captur"):
                f()
            assert not ops.calls and not any(opt.state.values()) and opt.param_groups[0]["step_t"] is None
    opt.working_copy(p)                              # q has no state yet
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_initialized", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captur"):
            opt.step()
        assert not ops.calls and not opt.state.get(q)
    opt.working_copy(q)
    count = opt.param_groups[0]["step_t"]
    assert count is not None and count.item() == 0
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_initialized", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        opt.step()
    assert len(ops.calls) == 1 and ops.calls[0][11] is count


def test_a_group_without_gradients_needs_no_state_in_a_capture(launches, capturing):
    from hi3d_hip import train
    ops = launches()
    train.AdamW([leaf(grad=False)], capturable=True).step()
    assert not ops.calls


def test_a_group_that_is_added_later_decides_about_the_loss_scale(launches):
    """Scaled gradients reach step() only where every group reads the scale on the device; a group that counts on the host would not."""
    from hi3d_hip import train
    opt = train.AdamW([leaf()], capturable=True)
    assert opt._step_supports_amp_scaling
    opt.add_param_group(dict(params=[leaf()], capturable=False))
    assert not opt._step_supports_amp_scaling
    opt = train.AdamW([leaf()])
    assert not opt._step_supports_amp_scaling
    opt.param_groups[0]["capturable"] = True
    opt.add_param_group(dict(params=[leaf()], capturable=True))
    assert opt._step_supports_amp_scaling
    import copy
    assert copy.deepcopy(opt)._step_supports_amp_scaling


def test_a_refused_step_is_not_counted(launches):
    from hi3d_hip import train
    p, q, r = leaf(), leaf(), leaf(grad=False)
    opt = train.AdamW([p, q, r])
    ops = launches(refuse=[True])
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    assert [opt.state[t]["step"] for t in (p, q)] == [0, 0]
    opt.step()
    assert [opt.state[t]["step"] for t in (p, q)] == [1, 1] and ops.calls[-1][10] == 1
    r.grad = torch.ones(4)                            # two launches: steps 2 and 1, the second refused
    ops.refuse = [False, True]
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    assert [opt.state[t]["step"] for t in (p, q, r)] == [2, 2, 0]
    q.grad = q.grad.to_sparse()                       # found among the gradients, before anything is launched
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    assert [opt.state[t]["step"] for t in (p, q, r)] == [2, 2, 0]


def test_a_copy_that_cannot_be_kept_is_refused_every_time(launches):
    """A working copy is of an fp32 parameter: the second step is refused like the first, and no half of the state is left."""
    from hi3d_hip import train
    ops = launches()
    p, q = leaf(dtype=torch.bfloat16), leaf()
    opt = train.AdamW([p, q], working_dtype=torch.bfloat16)
    for f in (opt.step, opt.step, lambda: opt.working_copy(p), lambda: opt.working_copy(p)):
        with pytest.raises(RuntimeError, match="fp32"):
            f()
    assert not ops.calls and not opt.state.get(p)
    assert opt.working_copy(q).dtype == torch.bfloat16


def test_z_is_kept_only_for_a_backward_pass(monkeypatch):
    """Without gradients to come -- no_grad, inference, frozen operands, a gradient for the residual alone -- the activation's argument is not written."""
    from hi3d_hip import train
    kept = []

    class Ops:
        def linear_act(self, x, w, bias, residual, act, save):
            kept.append(save)
            return x @ w.t(), x @ w.t() if save else None
    monkeypatch.setattr(train.torch_ops, "load", lambda: Ops())
    x, w = torch.ones(2, 3), torch.ones(4, 3, requires_grad=True)
    r = torch.zeros(2, 4, requires_grad=True)
    train.linear(x, w, act="gelu")
    train.linear(x, w, act="none")
    train.linear(x, w.detach(), residual=r, act="gelu")
    with torch.no_grad():
        y = train.linear(x, w, residual=r, act="gelu")
    with torch.inference_mode():
        train.linear(x, w, act="silu")
    assert kept == [True, False, False, False, False] and not y.requires_grad


def test_a_count_on_one_device_is_not_taken_for_parameters_on_another(launches):
    """Refused before the first of the devices has taken the step; counts on the host go by device."""
    from hi3d_hip import train
    ops = launches()
    p, q = leaf(), torch.nn.Parameter(torch.ones(4, device="meta"))
    q.grad = torch.ones(4, device="meta")
    opt = train.AdamW([p, q], capturable=True)
    with pytest.raises(RuntimeError, match="device"):
        opt.step()
    assert not ops.calls
    train.AdamW([p, q]).step()
    assert len(ops.calls) == 2
