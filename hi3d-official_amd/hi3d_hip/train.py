"""Training with the gfx950 kernels: operators with gradients, and the optimiser.

The sampler's operators (hi3d_hip.ops, torch.ops.hi3d.layernorm / linear) have no gradients.  These do, for a module tree that is
trained through the operator binding:

    from hi3d_hip import train
    y = train.layer_norm(x, weight, bias)                       # nn.LayerNorm
    y, z = train.layer_norm(x, weight, bias, residual=r)        # z = x + r, y = LayerNorm(z)
    y = train.linear(x, w, bias, residual=r, act="gelu")        # act(x w^T + bias) + r
    opt = train.AdamW(model.parameters(), lr=1e-5)              # torch.optim.AdamW

`AdamW` is a torch.optim.Optimizer and so a `target:` of the reference's YAML (`optimizer_config`).  Underneath are
torch.ops.hi3d.layernorm_fwd / add_layernorm_fwd / layernorm_bwd / linear_act /
linear_act_bwd / adamw_, which may be called by themselves (they record no gradients): a step that is
captured into a HIP graph calls these, since a captured autograd backward shares its leaves' gradient nodes -- and the
stream they were made on -- with any eager graph of the same leaves that is still alive.
"""
import torch

from . import lib as _l
from . import torch_ops


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ns = torch_ops.load()
        ctx.set_materialize_grads(False)
        if residual is None:
            y, mean, rstd = ns.layernorm_fwd(x, weight, bias, eps)
            ctx.save_for_backward(x, mean, rstd, weight, bias)
            return y
        y, z, mean, rstd = ns.add_layernorm_fwd(x, residual, weight, bias, eps)
        ctx.save_for_backward(z, mean, rstd, weight, bias)
        return y, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz=None):
        z, mean, rstd, weight, bias = ctx.saved_tensors
        if dy is None:                               # nothing reads y: the gradient passes through the sum alone
            return dz, dz, None, None, None
        dx, dw, db = torch_ops.load().layernorm_bwd(dy, z, mean, rstd, weight, bias, dz, *ctx.needs_input_grad[2:4])
        return dx, dx if ctx.needs_input_grad[1] else None, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """LayerNorm over x's last dimension, differentiable: y, or (y, x + residual) where a residual of x's shape and type is given.
    x: fp32, bf16 or fp16, any strides; weight, bias: [width] of one of these types, or None; width up to 8192.  The sum is
    rounded to x's type before it is normalised (it is what the next layer reads); statistics and sums are fp32."""
    return _LayerNorm.apply(x, residual, weight, bias, float(eps))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act, recorded):
        y, z = torch_ops.load().linear_act(x, w, bias, residual, act, recorded and act != "none" and any(ctx.needs_input_grad[:3]))
        ctx.act = act
        ctx.save_for_backward(x, w, bias, z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, bias, z = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if nx or nw or nb:
            dx, dw, db = torch_ops.load().linear_act_bwd(dy, x, w, z, bias if nb else None, ctx.act, nx, nw)
        return dx, dw, db, dy if nr else None, None, None


def linear(x, w, bias=None, residual=None, act="none"):
    """act(x w^T + bias) (+ residual), differentiable.  x [..., K], w [N, K] (nn.Linear's): both bf16 or both fp16 (nothing is cast, not under autocast
    either: fp32 parameters take part as 16-bit copies, AdamW's `working_dtype`), any strides, widths up to 1048576; bias [N]: fp32 or x's type; residual [..., N] of x's type and exactly the result's shape; act: "none", "gelu" (exact), "quick_gelu", "silu",
    "relu".  Products and sums are fp32; the gradients' products take dy act'(z) rounded to x's type, z being kept in it (bias' gradient: not rounded)."""
    lead = x.shape[:-1]
    if residual is not None:
        if residual.shape != (*lead, w.shape[0]):
            raise _l.Hi3dError(f"linear: residual must be {tuple(lead) + (w.shape[0],)}, got {tuple(residual.shape)}")
        residual = residual.reshape(-1, w.shape[0])
    # (inside forward() the grad mode is off whatever the caller's is, and a leaf needs a gradient under no_grad too)
    return _Linear.apply(x.reshape(-1, x.shape[-1]), w, bias, residual, act, torch.is_grad_enabled()).reshape(*lead, w.shape[0])


def _capturing():
    """Whether the current stream is being captured into a graph."""
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update for all tensors of a group in one launch per 72 of them (torch.ops.hi3d.adamw_).

    Parameters fp32, bf16 or fp16 on one GPU, dense in memory; moments are fp32 whatever the parameter's type.
    working_dtype (torch.bfloat16 / torch.float16): fp32 parameters keep a copy in that type which every step rewrites -- the
    weights that the forward pass reads, `working_copy(p)`, a leaf with a gradient of its own: step() takes that one where p has none.
    capturable: step count on the device (per group: each of its parameters then needs a gradient at every step), so that step() can be
    captured into a HIP graph (one that counts on the host refuses: every replay would be the same step) once the state is there -- after an eager step, or
    after working_copy() of every parameter; `lr` may then be a one-element fp32 device tensor.  torch.amp.GradScaler's scale and
    overflow flag are read on the device in this mode (it looks at the parameters' own gradients: not together with working copies').
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, working_dtype=None, capturable=False):
        if torch.is_tensor(lr):
            if not capturable:
                raise ValueError("lr as a tensor needs capturable=True")
        elif not lr >= 0.0:
            raise ValueError(f"invalid learning rate: {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"invalid betas: {betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"invalid eps or weight_decay: {eps}, {weight_decay}")
        if working_dtype not in (None, torch.bfloat16, torch.float16):
            raise ValueError(f"working_dtype must be torch.bfloat16 or torch.float16, not {working_dtype}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, working_dtype=working_dtype,
                                      capturable=capturable, step_t=None))

    @property
    def _step_supports_amp_scaling(self):
        """GradScaler asks: whether step() divides by its scale, and heeds its overflow flag, by itself (else it does so before the step)."""
        return all(g["capturable"] for g in self.param_groups)

    def working_copy(self, p):
        """The 16-bit copy of parameter p that step() keeps (before the first step: p rounded)."""
        return self._state_of(p, self._group_of(p))["copy"]

    def _group_of(self, p):
        for g in self.param_groups:
            if any(q is p for q in g["params"]):
                if g["working_dtype"] is None:
                    raise ValueError("this parameter's group has no working_dtype")
                return g
        raise KeyError("not a parameter of this optimiser")

    def _state_of(self, p, group):
        s = self.state[p]
        if "exp_avg" not in s or (group["capturable"] and group["step_t"] is None):
            # (made in a capture they would be graph nodes: zeroed again by every replay)
            if _capturing():
                raise _l.Hi3dError("the optimiser's state cannot be made while a graph is captured: take a step, or every parameter's working_copy(), before")
            if group["capturable"] and group["step_t"] is None:
                group["step_t"] = torch.zeros(1, device=p.device)
        if "exp_avg" not in s:
            if group["working_dtype"] is not None and p.dtype != torch.float32:
                raise _l.Hi3dError("a working copy is kept of fp32 parameters only")
            s["step"] = 0
            s["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            s["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            if group["working_dtype"] is not None:
                s["copy"] = p.detach().to(group["working_dtype"]).requires_grad_(p.requires_grad)
        return s

    def _grad(self, p):
        if p.grad is not None or "copy" not in self.state.get(p, ()):
            return p.grad
        return self.state[p]["copy"].grad

    def zero_grad(self, set_to_none=True):
        super().zero_grad(set_to_none)
        for s in self.state.values():
            c = s.get("copy")
            if c is not None and c.grad is not None:
                if set_to_none:
                    c.grad = None
                else:
                    c.grad.zero_()

    @torch.no_grad()
    def step(self, closure=None):
        if _capturing() and not all(g["capturable"] for g in self.param_groups):
            raise _l.Hi3dError("step() is being captured, but a parameter group was not made with capturable=True")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ns = torch_ops.load()
        scale, found_inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        if _capturing():                                     # (all of them, before any is launched)
            for group in self.param_groups:
                for p in group["params"]:
                    if self._grad(p) is not None:
                        self._state_of(p, group)
        for group in self.param_groups:
            with_grad = [p for p in group["params"] if self._grad(p) is not None]
            if group["capturable"] and with_grad and len(with_grad) < len(group["params"]):
                raise _l.Hi3dError("capturable: every parameter of the group needs a gradient at every step")
            if group["capturable"] and len({p.device for p in with_grad}) > 1:
                raise _l.Hi3dError("capturable: the group's step count is on one device, and so must its parameters be")
            by_step = {}                                    # (one list, unless some parameters had no gradient at earlier steps)
            for p in with_grad:
                g = self._grad(p)
                if g.is_sparse:
                    raise _l.Hi3dError("sparse gradients are not supported")
                if g.stride() != p.stride():
                    g = torch.empty_like(p, dtype=g.dtype).copy_(g)
                s = self._state_of(p, group)
                step = 0 if group["capturable"] else s["step"] + 1
                lists, states = by_step.setdefault((p.device, step), (([], [], [], [], []), []))
                for to, t in zip(lists, (p, g, s["exp_avg"], s["exp_avg_sq"], s.get("copy"))):
                    if t is not None:
                        to.append(t)
                states.append(s)
            b1, b2 = group["betas"]
            for (_, step), (lists, states) in by_step.items():
                lr_t = step_t = None
                if group["capturable"]:
                    step_t, lr_t = group["step_t"], group["lr"] if torch.is_tensor(group["lr"]) else None
                ns.adamw_(*lists, 0.0 if lr_t is not None else float(group["lr"]), b1, b2, group["eps"], group["weight_decay"], max(step, 1), step_t, lr_t,
                          scale if step_t is not None else None, found_inf if step_t is not None else None)
                for s in states:                            # (a step that was refused is not counted)
                    s["step"] = step
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep their type (torch casts a state to its parameter's), `working_dtype` and `capturable` stay as
        this optimiser was made with them, and what it holds already -- moments, working copies, step counts and rates on the device -- is
        filled in place: copies that were handed out and a step that was captured go on from the loaded values.  A state of
        torch.optim.AdamW loads too; a copy that the state has not is its parameter, rounded (load the parameters first)."""
        own = [(g["working_dtype"], g["capturable"], g["step_t"], g["lr"]) for g in self.param_groups]
        held = {p: dict(s) for p, s in self.state.items()}
        state, counts = state_dict["state"], []
        for i, g in enumerate(state_dict["param_groups"]):
            if g.get("amsgrad") or g.get("maximize"):
                raise _l.Hi3dError("a state with amsgrad or maximize cannot be continued here")
            if g.get("step_t") is not None:
                steps = [int(g["step_t"])] * len(g["params"])
            else:
                steps = [int(state.get(k, {}).get("step", 0)) for k in g["params"]]
            if i < len(own) and own[i][1] and len(set(steps)) > 1:
                raise _l.Hi3dError("capturable: every parameter of the group needs the same number of steps behind it")
            counts.append(steps)
        super().load_state_dict(state_dict)
        for g, saved_group, steps, (working_dtype, capturable, step_t, lr) in zip(self.param_groups, state_dict["param_groups"], counts, own):
            for k, v in self.defaults.items():               # (a group saved by torch.optim.AdamW has no working_dtype)
                g.setdefault(k, v)
            g["working_dtype"], g["capturable"], g["step_t"] = working_dtype, capturable, None
            g["lr"] = lr.fill_(float(g["lr"])) if torch.is_tensor(lr) else float(g["lr"])
            if capturable and steps and (step_t is not None or steps[0]):
                g["step_t"] = torch.zeros(1, device=g["params"][0].device) if step_t is None else step_t
                g["step_t"].fill_(float(steps[0]))
            for p, k, step in zip(g["params"], saved_group["params"], steps):
                saved, before = state.get(k, {}), held.get(p, {})
                if not saved and not before:
                    continue
                s = self.state[p]
                s["step"] = 0 if capturable else step
                for name in ("exp_avg", "exp_avg_sq"):
                    s[name] = before[name] if name in before else torch.zeros_like(p, dtype=torch.float32)
                    s[name].copy_(saved[name]) if name in saved else s[name].zero_()
                s.pop("copy", None)
                if working_dtype is not None:
                    s["copy"] = before["copy"] if "copy" in before else p.detach().to(working_dtype).requires_grad_(p.requires_grad)
                    with torch.no_grad():
                        s["copy"].copy_(saved["copy"] if "copy" in saved and saved["copy"].dtype == working_dtype else p)
