"""clip_grad_norm_ + AdamW.step() in two kernel launches.

The reference's step is `torch.nn.utils.clip_grad_norm_(model.parameters(), 1.0)` followed by
`optimizer.step()` on a torch.optim.AdamW (utils/train_and_eval.py:115-118, train.py:221-226).
`clip_and_step` does the same arithmetic on the optimizer's own state tensors (`exp_avg`,
`exp_avg_sq`, `step`), so the optimizer object, its `state_dict()` and checkpoints stay
interchangeable with torch's.  Anything it does not recognise — another optimizer class,
amsgrad/maximize/capturable, sparse or non-float32 tensors, an enabled GradScaler — runs
torch's own `clip_grad_norm_` + `optimizer.step()` unchanged.

`AdamW8` is the same update with both moments in 8 bits (2.02 bytes of state per parameter instead of 8);
`clip_and_step` and `CapturedStep` take it as they take torch's AdamW.
"""
import operator

import torch

from .. import functional as F_
from .._lib import call, query

CHUNK = 4096          # MIS_OPT_CHUNK in include/misamd.h


class _Plan:
    """Device table of (param, grad, exp_avg, exp_avg_sq, n) rows and the chunk prefix of one
    optimizer.  Gradients are re-allocated every step (`zero_grad()` drops them), at addresses that
    need not repeat, so the pointer rows are refreshed whenever they changed: written into one of
    a small ring of pinned staging buffers (allocated once; a slot is reused only after the copy
    that last read it has completed) and uploaded on the launch stream — no allocation, no host
    synchronisation.  The chunk prefix depends on the tensor sizes only and is built once."""
    RING = 4

    def __init__(self, sizes, group_chunks, prefix, dev):
        self.sizes = sizes
        self.group_chunks = group_chunks
        self.n_chunks = prefix[-1]
        self.rows = None
        n = len(sizes)
        self.descs = torch.empty((n, 5), dtype=torch.int64, device=dev)
        self.prefix = torch.tensor(prefix, dtype=torch.int32).pin_memory().to(dev, non_blocking=True)
        self.stage = [torch.empty((n, 5), dtype=torch.int64).pin_memory() for _ in range(self.RING)]
        self.done = [None] * self.RING
        self.slot = 0

    def upload(self, rows):
        global PLAN_UPLOADS
        PLAN_UPLOADS += 1
        k = self.slot
        self.slot = (k + 1) % self.RING
        if self.done[k] is not None:
            self.done[k].synchronize()
        self.stage[k].copy_(torch.tensor(rows, dtype=torch.int64))
        self.descs.copy_(self.stage[k], non_blocking=True)
        ev = torch.cuda.Event()
        ev.record()
        self.done[k] = ev
        self.rows = rows


_PLANS = {}           # id(optimizer) -> _Plan
PLAN_BUILDS = 0       # tables allocated / pointer-row uploads so far (diagnostics, tests)
PLAN_UPLOADS = 0


def _fusable(optimizer, params):
    if type(optimizer) is not torch.optim.AdamW:
        return False
    listed = set()
    for g in optimizer.param_groups:
        if g.get("amsgrad") or g.get("maximize") or g.get("capturable") or g.get("differentiable"):
            return False
        if isinstance(g["lr"], torch.Tensor):
            return False
        for p in g["params"]:
            if p.grad is None:
                continue
            if (not p.is_cuda or p.dtype != torch.float32 or p.grad.dtype != torch.float32 or p.grad.is_sparse
                    or not p.is_contiguous() or not p.grad.is_contiguous()):
                return False
            listed.add(id(p))
    # the clip norm must be taken over exactly the tensors being stepped
    clip = {id(p) for p in params if p.grad is not None}
    return clip == listed and len(listed) > 0


class _Fast:
    """What `clip_and_step` established about an (optimizer, params) pair on its first fused call,
    so that later calls only re-check what can change between steps."""

    def __init__(self):
        self.param_ids = None
        self.groups = None        # [(group dict, [params])]
        self.states = None        # [state dict per param], same order as the pointer rows
        self.static = None        # [(p ptr, exp_avg ptr, exp_avg_sq ptr, numel)]
        self.step_tensors = None
        self.step = None          # the value every step tensor holds


_FAST = {}


def _group_ok(g):
    return not (g.get("amsgrad") or g.get("maximize") or g.get("capturable") or g.get("differentiable")
                or isinstance(g["lr"], torch.Tensor))


def _fast_path(optimizer, params):
    """The cached description if nothing structural changed since it was built, else None."""
    f = _FAST.get(id(optimizer))
    if f is None or f.param_ids != [id(p) for p in params]:
        return None
    state = optimizer.state
    for (g, ps) in f.groups:
        if not _group_ok(g):
            return None
    for p, s, (sp, sm, sv, _) in zip((p for _, ps in f.groups for p in ps), f.states, f.static):
        gr = p.grad
        if (gr is None or gr.dtype != torch.float32 or not gr.is_contiguous() or state.get(p) is not s
                or p.data_ptr() != sp or s["exp_avg"].data_ptr() != sm or s["exp_avg_sq"].data_ptr() != sv):
            return None
    if float(f.step_tensors[0]) != f.step:
        return None
    return f


def clip_and_step(optimizer, params, max_norm=1.0):
    """clip_grad_norm_(params, max_norm) + optimizer.step().  Returns the total gradient norm (a
    0-dim tensor), like clip_grad_norm_."""
    params = [p for p in params]
    F_.flush_wgrad_reduces()       # (a no-op after a finished backward pass)
    if isinstance(optimizer, AdamW8):
        held = optimizer._params()
        stepped = [p for p in held if p.grad is not None]
        if len(params) != len(held) or not all(map(operator.is_, params, held)):
            given = [p for p in params if p.grad is not None]
            if len(stepped) != len(given) or {id(p) for p in given} != {id(p) for p in stepped}:
                norm = torch.nn.utils.clip_grad_norm_(params, max_norm=max_norm)   # a norm over other tensors than are stepped
                optimizer.step()
                return norm
        return optimizer._launch(float(max_norm), stepped, held)
    fast = _fast_path(optimizer, params)
    if fast is not None:
        return _launch(optimizer, fast, max_norm)
    _FAST.pop(id(optimizer), None)
    return _clip_and_step_checked(optimizer, params, max_norm)


def _launch(optimizer, f, max_norm):
    dev = f.groups[0][1][0].device
    rows = [(sp, p.grad.data_ptr(), sm, sv, n)
            for p, (sp, sm, sv, n) in zip((p for _, ps in f.groups for p in ps), f.static)]
    plan = _PLANS[id(optimizer)]
    if plan.rows != rows:
        plan.upload(rows)
    st = F_._stream()
    ws = F_.workspace(plan.ws_bytes, dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    n_t = len(rows)
    call("mis_grad_sqsum", plan.descs.data_ptr(), plan.prefix.data_ptr(), n_t, plan.n_chunks, ws.data_ptr(), st)
    step = int(f.step) + 1
    for (g, ps), (c0, c1) in zip(f.groups, plan.group_chunks):
        b1, b2 = g["betas"]
        call("mis_clip_adamw_step", plan.descs.data_ptr(), plan.prefix.data_ptr(), n_t, c0, c1, plan.n_chunks,
             ws.data_ptr(), float(max_norm), float(g["lr"]), float(b1), float(b2), float(g["eps"]),
             float(g["weight_decay"]), step, 1, norm.data_ptr() if c0 == 0 else None, st)
    torch._foreach_add_(f.step_tensors, 1)
    f.step = float(step)
    # the kernels wrote through raw pointers: tell autograd (and anything keyed on tensor versions,
    # e.g. cached operand images of the weights) that these tensors changed
    touched = []
    for _, ps in f.groups:
        touched += ps
        touched += [p.grad for p in ps]
    for s in f.states:
        touched += [s["exp_avg"], s["exp_avg_sq"]]
    torch._C._increment_version(touched)
    return norm


def _clip_and_step_checked(optimizer, params, max_norm):
    """Full validation of the (optimizer, params) pair; on success the first fused step and the
    cached description for the following ones."""
    if not _fusable(optimizer, params):
        norm = torch.nn.utils.clip_grad_norm_(params, max_norm=max_norm)
        optimizer.step()
        return norm
    groups, steps = [], []
    for g in optimizer.param_groups:
        ps = [p for p in g["params"] if p.grad is not None]
        if not ps:
            continue
        st = None
        for p in ps:
            s = optimizer.state[p]
            if len(s) == 0:                 # same lazy initialisation as torch.optim.AdamW
                s["step"] = torch.tensor(0.0, dtype=torch.float32)
                s["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                s["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            k = float(s["step"])
            if st is None:
                st = k
            elif k != st:                   # per-tensor step counts differ: leave it to torch
                norm = torch.nn.utils.clip_grad_norm_(params, max_norm=max_norm)
                optimizer.step()
                return norm
        groups.append((g, ps))
        steps.append(int(st) + 1)
    dev = groups[0][1][0].device
    rows = []
    for g, ps in groups:
        for p in ps:
            s = optimizer.state[p]
            rows.append((p.data_ptr(), p.grad.data_ptr(), s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr(), p.numel()))
    sizes = tuple(r[4] for r in rows)
    plan = _PLANS.get(id(optimizer))
    if plan is None or plan.sizes != sizes or plan.descs.device != dev:
        global PLAN_BUILDS
        PLAN_BUILDS += 1
        prefix, c, group_chunks = [], 0, []
        for g, ps in groups:
            c0 = c
            for p in ps:
                prefix.append(c)
                c += (p.numel() + CHUNK - 1) // CHUNK
            group_chunks.append((c0, c))
        prefix.append(c)
        plan = _PLANS[id(optimizer)] = _Plan(sizes, group_chunks, prefix, dev)
    plan.ws_bytes = query("mis_clip_adamw_workspace_bytes", plan.n_chunks)
    if len(set(steps)) != 1:              # groups at different step counts: torch handles that
        norm = torch.nn.utils.clip_grad_norm_(params, max_norm=max_norm)
        optimizer.step()
        return norm
    f = _Fast()
    f.param_ids = [id(p) for p in params]
    f.groups = groups
    f.states = [optimizer.state[p] for _, ps in groups for p in ps]
    f.static = [(r[0], r[2], r[3], r[4]) for r in rows]
    f.step_tensors = [s_["step"] for s_ in f.states]
    f.step = float(steps[0] - 1)
    _FAST[id(optimizer)] = f
    return _launch(optimizer, f, max_norm)


BLOCK8 = 128          # elements that share a scale in AdamW8's moments


def _blocks(n):
    return (n + BLOCK8 - 1) // BLOCK8


def _dense(t):
    """Whether the elements fill their memory without gaps, in whatever order."""
    if t.is_contiguous():
        return True
    want = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _layout(p):
    """(shape, dimensions by falling stride): which element lies at which place of a dense tensor's memory."""
    shape = tuple(p.shape)
    dims = [d for d, n in enumerate(shape) if n != 1] if 0 not in shape else []
    if len(dims) > 1 and not p.is_contiguous():
        dims.sort(key=lambda d: -p.stride(d))
    return shape, tuple(dims)


def _check_layout(i, p, s):
    """The codes of state `s` follow the memory of the tensor they were made for: they mean nothing in another order.  Without a
    record of it they are taken for row-major."""
    shape, order = now = _layout(p)
    made = s.get("layout") or (shape, sorted(order))
    if made != now and (tuple(made[0]), tuple(made[1])) != now:
        raise RuntimeError(f"AdamW8: parameter {i} is now {shape} with strides {p.stride()}, its moments were made for shape "
                           f"{tuple(made[0])} with the dimensions {tuple(made[1])} by falling stride: convert the model back, or "
                           "delete the parameter's state to begin again")


def _check_codes(i, n, s):
    """Whether state `s` of parameter `i` (n elements) holds moments; raises where it holds something else."""
    held = [k for k in AdamW8._STATE if k in s]
    if not held:
        return False
    for k in AdamW8._STATE:
        if k not in s:
            raise ValueError(f"not an AdamW8 state: parameter {i} has no {k}")
        want = _blocks(n) * (1 if k.endswith("_scale") else BLOCK8)
        if s[k].dtype != torch.uint8 or s[k].numel() != want:
            raise ValueError(f"parameter {i}: {k} should be {want} bytes, got {s[k].numel()} of {s[k].dtype}")
    return True


class AdamW8(torch.optim.Optimizer):
    """AdamW with both moments in 8 bits, one launch for all tensors (two when the gradient norm is clipped).

    The update is torch.optim.AdamW's; what is kept between steps is rounded to codes of one byte with an exponent byte
    per 128 elements (mis_adamw8_step in include/misamd.h gives the formats), stochastically: `seed` and the step number
    decide every rounding, so runs repeat bit for bit.  Parameters float32 or bfloat16 with gradients of the same type, on
    one GPU.  Gradients are read, not changed, when clipping (torch's clip_grad_norm_ scales them in place).  A moment
    that is not finite makes its block of 128 read back as NaN.

    state[p] = {"step": int, "exp_avg", "exp_avg_sq": uint8 codes, padded to a multiple of 128,
                "exp_avg_scale", "exp_avg_sq_scale": uint8, one per 128,
                "layout": (shape, dimensions by falling stride)}; `moments(p)` gives their float32 values.
    The codes follow the elements' order in memory.  A parameter may change its type, device or address between steps
    (Module.bfloat16(), .data = ...), but not its shape or memory order: the step raises then.  A cleared state begins again
    at step 1 with moments of zero, one put in its place is gone on from.  A parameter without a gradient is left alone, as
    in torch.
    """
    _STATE = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
    _plan = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0):
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"Invalid betas: {betas}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if not 0 <= int(seed) < 1 << 64:
            raise ValueError(f"Invalid seed: {seed}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, seed=int(seed)))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if len({id(p) for p in self.param_groups[-1]["params"]}) != len(self.param_groups[-1]["params"]):
            self.param_groups.pop()
            raise ValueError("AdamW8 takes each parameter once: all of them are updated by one launch")
        for p in self.param_groups[-1]["params"]:
            if p.dtype not in F_._DT:
                self.param_groups.pop()
                raise TypeError(f"AdamW8 takes float32 and bfloat16 parameters, got {p.dtype}")
        self._plan = None

    def load_state_dict(self, state_dict):
        names = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(names, self._params()):        # (before anything is replaced; torch checks the groups' lengths)
            s = state_dict["state"].get(i)
            if s is not None:
                if not _check_codes(i, p.numel(), s) or "step" not in s:
                    raise ValueError(f"not an AdamW8 state: parameter {i} has no {'step' if 'exp_avg' in s else 'exp_avg'}")
                _check_layout(i, p, s)
        # (the codes go past torch's loading, which would take them through the parameters' floating-point type)
        states = state_dict["state"]
        past = self._STATE + ("layout",)
        rest = {i: {k: v for k, v in s.items() if k not in past} for i, s in states.items()}
        super().load_state_dict({**state_dict, "state": rest})
        params = self._params()
        for i, p in zip(names, params):
            if i in states:
                self.state[p].update({k: states[i][k] for k in self._STATE}, step=int(states[i]["step"]))
        self._plan = None
        if all(p.is_cuda for p in params) and len({p.device for p in params}) == 1:
            self._flat(params, checked=True)
        else:                                      # nothing of the given tensors is kept
            for s in self.state.values():
                s.update({k: s[k].reshape(-1).clone() for k in self._STATE if k in s})
            for p in params:
                if p in self.state:
                    self.state[p]["layout"] = _layout(p)

    def _params(self):
        return [p for g in self.param_groups for p in g["params"]]

    def _flat(self, params=None, checked=False):
        """The flat moment buffers, laid out over all parameters (`params`, where the caller has their list); state[p] holds
        views of them.  checked: what the state holds has been looked at."""
        params = params or self._params()
        plan = self._plan
        if plan is not None and plan.matches(params) and plan.holds(self.state):
            return plan
        devs = {p.device for p in params}
        if len(devs) != 1 or next(iter(devs)).type != "cuda":
            raise RuntimeError(f"AdamW8 needs all parameters on one GPU, got {sorted(map(str, devs))}")
        for i, p in enumerate(params):
            if not checked and self.state.get(p):
                _check_layout(i, p, self.state[p])
                _check_codes(i, p.numel(), self.state[p])
        plan = _Plan8(params, next(iter(devs)))
        views = [buf.split([(b1 - b0) * w for b0, b1 in plan.spans] + [buf.numel() - plan.blocks * w])
                 for buf, w in zip(plan.buffers, (BLOCK8, 1, BLOCK8, 1))]
        to, given = [], []
        for i, p in enumerate(params):
            s = self.state[p]
            for k, v in zip(self._STATE, views):
                if k in s:                        # (codes behind the last element stay zero)
                    n = p.numel() if v is views[0] or v is views[2] else v[i].numel()
                    to.append(v[i][:n])
                    given.append((s[k] if s[k].dim() == 1 else s[k].reshape(-1))[:n])
        if to:
            torch._foreach_copy_(to, given)
        for i, p in enumerate(params):             # (nothing of the old state is replaced before all of it is copied)
            s = self.state[p]
            s.update({k: v[i] for k, v in zip(self._STATE, views)}, step=int(s.get("step", 0)), layout=_layout(p))
        plan.keep(self.state)
        self._plan = plan
        return plan

    def moments(self, p=None):
        """(exp_avg, exp_avg_sq) of parameter `p` as float32 tensors of its shape; without `p` the flat buffers of all
        parameters in their order, each parameter starting at a multiple of 128 (zeros behind its last element)."""
        plan = self._flat()
        dev = plan.device
        b0, b1 = (0, plan.blocks) if p is None else plan.spans[[id(q) for q in plan.params].index(id(p))]
        out = [torch.empty((b1 - b0) * BLOCK8, dtype=torch.float32, device=dev) for _ in range(2)]
        if b1 > b0:
            m, ms, v, vs = (b.data_ptr() for b in plan.buffers)
            with F_._on_device_of(out[0]):
                call("mis_adamw8_moments", m + b0 * BLOCK8, ms + b0, v + b0 * BLOCK8, vs + b0, b1 - b0, out[0].data_ptr(),
                     out[1].data_ptr(), F_._stream())
        if p is None:
            return out[0], out[1]
        return tuple(torch.as_strided(t, p.shape, p.stride()).clone(memory_format=torch.preserve_format) for t in out)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        held = self._params()
        self._launch(None, [p for p in held if p.grad is not None], held)
        return loss

    def _launch(self, max_norm, params, held):
        """One step of `params`, those with a gradient of all that are `held`; max_norm None: no norm is formed.  Returns the
        total gradient norm otherwise."""
        if not params:
            return torch.zeros(()) if max_norm is not None else None
        if params[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("an AdamW8 step cannot be captured as it is (its step number would be frozen): use "
                               "CapturedStep or GraphedTrainStep")
        table = self._flat(held).table(self.param_groups, self.state, params)
        norm = table.launch(max_norm)
        for states in table.states:
            k = states[0]["step"] + 1
            for s in states:
                s["step"] = k
        torch._C._increment_version(params)
        return norm


class _Plan8:
    """The flat moment buffers of one AdamW8 and the device tables of its launches."""

    def __init__(self, params, device):
        self.params, self.device = params, device
        self.spans, at = [], 0
        for p in params:
            if p.dtype not in F_._DT:
                raise TypeError(f"AdamW8 takes float32 and bfloat16 parameters, got {p.dtype}")
            if not _dense(p):
                raise RuntimeError(f"AdamW8 needs dense parameters, got strides {p.stride()} for {tuple(p.shape)}")
            self.spans.append((at, at + _blocks(p.numel())))
            at = self.spans[-1][1]
        self.blocks = at
        self.buffers = [torch.zeros(max(at, 1) * w, dtype=torch.uint8, device=device) for w in (BLOCK8, 1, BLOCK8, 1)]
        self.norm_ws = torch.empty(query("mis_adamw8_workspace_bytes"), dtype=torch.uint8, device=device)
        self.layouts = F_._native().Layouts(params)
        self.tables = []

    def matches(self, params):
        """Whether these are the parameters that buffers and tables were made for, in type, device, shape and strides too."""
        return len(params) == len(self.params) and all(map(operator.is_, params, self.params)) and self.layouts.hold()

    def keep(self, state):
        """Takes note of the state that the buffers serve: `holds` says whether it is still that one."""
        self.states = list(state.values())
        self.held = [v if k in AdamW8._STATE else None for s in self.states for k, v in s.items()]

    def holds(self, state):
        return F_._native().state_holds(state, self.states, self.held)

    def table(self, groups, state, params):
        """The launch tables for `params`, the parameters that have a gradient now."""
        for t in self.tables:
            if t.serves(params):
                break
        else:
            if len(self.tables) >= 4:             # (a few patterns of missing gradients at most; not a growing cache)
                self.tables.clear()
            t = _Table8(self, groups, state, params)
            self.tables.append(t)
        t.refresh()
        return t


class _Table8:
    """The device tables for one set of parameters with gradients: pointer rows, chunk prefix, and the runs of one group
    and one step number, each of them a launch."""

    def __init__(self, plan, groups, state, params):
        self.plan, self.params = plan, params
        self.runs, self.states, self.order = [], [], []       # (group, first chunk, end chunk); their states; flat
        prefix, idle = [0], []
        stepped = {id(p) for p in params}
        for g in groups:
            by_step = {}
            for p in g["params"]:
                if id(p) in stepped:
                    if p.numel():
                        by_step.setdefault(state[p]["step"], []).append(p)
                    else:
                        idle.append(state[p])
            for ps in by_step.values():
                c0 = prefix[-1]
                for p in ps:
                    prefix.append(prefix[-1] + (p.numel() + CHUNK - 1) // CHUNK)
                self.runs.append((g, c0, prefix[-1]))
                self.states.append([state[p] for p in ps])
                self.order += ps
        self.states += [[s] for s in idle]                     # (empty tensors count steps and nothing else)
        span = {id(p): s for p, s in zip(plan.params, plan.spans)}
        self.fixed = [(span[id(p)][0] * BLOCK8, p.numel(), F_._DT[p.dtype]) for p in self.order]
        self.plain = [p.is_contiguous() for p in self.order]
        self.dtypes = [p.dtype for p in self.order]
        self.pointers = self.keep = None
        self.plan_dev = _Plan([f[1] for f in self.fixed], None, prefix, plan.device) if self.order else None

    def serves(self, params):
        """Whether these are its parameters, and every run still has one step number."""
        if len(params) != len(self.params) or not all(map(operator.is_, params, self.params)):
            return False
        for states in self.states:
            k = states[0]["step"]
            if not all([s["step"] == k for s in states]):
                return False
        return True

    def addresses(self):
        """[parameter, gradient, parameter, ...] pointers; a gradient in another memory order than its parameter is copied
        into the parameter's."""
        dev, keep = self.plan.device.index, []
        out = F_._native().step_pointers(self.order, dev)
        if out:
            return out, keep
        for p, plain, dtype in zip(self.order, self.plain, self.dtypes):
            g = p.grad
            if g.dtype is not dtype or g.is_sparse or g.get_device() != dev or p.get_device() != dev or g.shape != p.shape:
                raise RuntimeError(f"AdamW8 needs dense gradients of the parameter's type, device and shape, got {g.dtype} "
                                   f"{g.layout} {tuple(g.shape)} on {g.device} for {p.dtype} {tuple(p.shape)} on {p.device}")
            if not (plain and g.is_contiguous()) and g.stride() != p.stride():
                g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g.detach())
                keep.append(g)
            out += (p.data_ptr(), g.data_ptr())
        return out, keep

    def rows(self, pointers):
        spans = sorted((pointers[2 * i], pointers[2 * i] + p.nbytes) for i, p in enumerate(self.order))
        if any(end > begin for (_, end), (begin, _) in zip(spans, spans[1:])):
            raise RuntimeError("AdamW8 updates all parameters in one launch: two of them share memory")
        return [(pointers[2 * i], pointers[2 * i + 1], *f) for i, f in enumerate(self.fixed)]

    def refresh(self):
        if not self.order:
            return
        with F_._on_device_of(self.plan.norm_ws):
            pointers, self.keep = self.addresses()              # (kept until the next step's replace them)
            if pointers != self.pointers:
                self.plan_dev.upload(self.rows(pointers))
                self.pointers = pointers

    def launch(self, max_norm, descs=None, norm_ws=None, dyn=None):
        """The launches of a step on the current stream.  dyn: per run, the device constants of a captured step."""
        plan = self.plan
        if not self.order:
            return torch.zeros((), dtype=torch.float32, device=plan.device) if max_norm is not None else None
        with F_._on_device_of(plan.norm_ws):
            st, t = F_._stream(), self.plan_dev
            d, prefix, n = (t.descs if descs is None else descs).data_ptr(), t.prefix.data_ptr(), len(self.order)
            buffers = [b.data_ptr() for b in plan.buffers]
            norm = ws = None
            if max_norm is not None:
                ws = (plan.norm_ws if norm_ws is None else norm_ws).data_ptr()
                call("mis_adamw8_sqsum", d, prefix, n, t.n_chunks, ws, st)
                norm = torch.empty((), dtype=torch.float32, device=plan.device)
            for k, (g, c0, c1) in enumerate(self.runs):
                b1, b2 = g["betas"]
                call("mis_adamw8_step", d, prefix, n, c0, c1, t.n_chunks, *buffers, ws, max_norm or 0.0, float(g["lr"]),
                     float(b1), float(b2), float(g["eps"]), float(g["weight_decay"]), self.states[k][0]["step"] + 1, g["seed"],
                     None if dyn is None else dyn[k].data_ptr(), norm.data_ptr() if norm is not None and k == 0 else None, st)
        return norm


class _CapturedStep8:
    """CapturedStep for an AdamW8: learning rate, weight decay and step number come from a device buffer; the norm's
    partial sums, the pointer table and the constants belong to this object alone."""
    RING, WIDTH = 8, 32           # bytes per run's constants (20 used)

    def __init__(self, optimizer, params, max_norm):
        self.optimizer, self.max_norm = optimizer, float(max_norm)
        self.params = [p for p in optimizer._params() if p.grad is not None]
        if {id(p) for p in params if p.grad is not None} != {id(p) for p in self.params} or not self.params:
            raise RuntimeError("CapturedStep needs the gradients of exactly the tensors that the optimizer steps")
        if any(optimizer.state[p].get("step", 0) < 1 for p in self.params):
            raise RuntimeError("CapturedStep needs an optimizer that has taken at least one eager step with these parameters "
                               "(clip_and_step)")
        self.plan = optimizer._flat()
        self.table = _Table8(self.plan, optimizer.param_groups, optimizer.state, self.params)
        self.addresses = [p.data_ptr() for p in self.table.order]
        self.options = self._options()
        dev, n, r = self.plan.device, len(self.table.order), max(len(self.table.runs), 1)
        self.rows_host = torch.empty((n, 5), dtype=torch.int64).pin_memory()
        self.descs = torch.empty((n, 5), dtype=torch.int64, device=dev)
        self.ws = torch.empty_like(self.plan.norm_ws)
        self.dyn_host = [torch.zeros((r, self.WIDTH), dtype=torch.uint8).pin_memory() for _ in range(self.RING)]
        self.dyn_done = [None] * self.RING
        self.slot = 0
        self.dyn = torch.zeros((r, self.WIDTH), dtype=torch.uint8, device=dev)
        self.norm = None

    def _options(self):
        """What a launch holds fast (learning rate and weight decay come from the device buffer)."""
        return [(tuple(g["betas"]), g["eps"], g["seed"]) for g, _, _ in self.table.runs]

    def prepare(self):
        if self._options() != self.options:
            raise RuntimeError("betas, eps or seed changed after the capture (a scheduler that cycles momentum does that): capture "
                               "the step again")
        if self.optimizer._plan is not self.plan or not self.plan.holds(self.optimizer.state):
            raise RuntimeError("the optimizer's state was replaced after the capture: capture the step again")
        if not self.plan.matches(self.plan.params) or [p.data_ptr() for p in self.table.order] != self.addresses:
            raise RuntimeError("a parameter was converted or its memory replaced after the capture: capture the step again")
        if not self.table.serves(self.params):
            raise RuntimeError("the parameters' step numbers no longer agree: capture the step again")
        i = self.slot
        self.slot = (i + 1) % self.RING
        if self.dyn_done[i] is not None:
            self.dyn_done[i].synchronize()
        host = self.dyn_host[i]
        for k, (g, _, _) in enumerate(self.table.runs):
            b1, b2 = g["betas"]
            call("mis_adamw8_step_constants", float(g["lr"]), float(b1), float(b2), float(g["weight_decay"]),
                 self.table.states[k][0]["step"] + 1, host[k].data_ptr())
        with F_._on_device_of(self.dyn):
            self.dyn.copy_(host, non_blocking=True)
            ev = torch.cuda.Event()
            ev.record()
        self.dyn_done[i] = ev

    def launch(self):
        pointers, self.keep = self.table.addresses()
        self.addresses = pointers[::2]                          # the parameters', which every replay writes to
        self.rows_host.copy_(torch.tensor(self.table.rows(pointers), dtype=torch.int64))
        self.descs.copy_(self.rows_host, non_blocking=True)
        self.norm = self.table.launch(self.max_norm, self.descs, self.ws, self.dyn)
        return self.norm

    def advance(self):
        for states in self.table.states:
            for s in states:
                s["step"] += 1
        torch._C._increment_version(self.params)


def captured_step(optimizer, params, max_norm=1.0):
    """The CapturedStep of this optimizer: prepare(), launch() inside the capture, advance()."""
    if isinstance(optimizer, AdamW8):
        return _CapturedStep8(optimizer, params, max_norm)
    return CapturedStep(optimizer, params, max_norm)


class CapturedStep:
    """clip_grad_norm_ + AdamW.step() in a form that can sit inside a HIP graph: the launches take
    everything that changes from step to step (learning rate, bias corrections) from a small
    device buffer, so one capture serves every replay.

    `launch()` is called once, inside the capture (the gradients exist by then; their addresses
    are those of every replay).  Before each replay `prepare()` forms the step's constants on the
    host — the same double arithmetic the eager path uses, so both give the same bits — and
    copies them in; after it `advance()` moves torch's own step counters, which live on the host.
    Pinned host buffers are private to this object: a captured copy re-reads them at every replay.
    """

    def __init__(self, optimizer, params, max_norm=1.0):
        params = [p for p in params]
        if _fast_path(optimizer, params) is None:
            raise RuntimeError("CapturedStep needs an optimizer that has taken at least one fused eager step "
                               "with these parameters (clip_and_step)")
        self.optimizer, self.params, self.max_norm = optimizer, params, float(max_norm)
        self.f = _FAST[id(optimizer)]
        self.plan = _PLANS[id(optimizer)]
        dev = self.f.groups[0][1][0].device
        n_t, n_g = len(self.f.static), len(self.f.groups)
        self.rows_host = torch.empty((n_t, 5), dtype=torch.int64).pin_memory()
        self.descs = torch.empty((n_t, 5), dtype=torch.int64, device=dev)
        # the host may run several steps ahead of the GPU: a small ring of pinned slots, each reused
        # only after the copy that read it has completed
        self.dyn_host = [torch.zeros((n_g, 4), dtype=torch.float32).pin_memory() for _ in range(8)]
        self.dyn_done = [None] * 8
        self.slot = 0
        self.dyn = torch.zeros((n_g, 4), dtype=torch.float32, device=dev)
        self.norm = None

    def prepare(self):
        """Host side of the next step: constants for step count + 1 and the current learning rates."""
        step = int(self.f.step) + 1
        i = self.slot
        self.slot = (i + 1) % len(self.dyn_host)
        if self.dyn_done[i] is not None:
            self.dyn_done[i].synchronize()
        host = self.dyn_host[i]
        for k, (g, _) in enumerate(self.f.groups):
            if not _group_ok(g):
                raise RuntimeError("optimizer options changed after the capture")
            b1, b2 = g["betas"]
            query("mis_adamw_step_constants", float(g["lr"]), float(b1), float(b2), float(g["weight_decay"]), step,
                  host[k].data_ptr())
        self.dyn.copy_(host, non_blocking=True)
        ev = torch.cuda.Event()
        ev.record()
        self.dyn_done[i] = ev

    def launch(self):
        """The two launches (and the upload of the pointer rows) on the current, capturing stream."""
        f, plan = self.f, self.plan
        dev = self.descs.device
        rows = [(sp, p.grad.data_ptr(), sm, sv, n)
                for p, (sp, sm, sv, n) in zip((p for _, ps in f.groups for p in ps), f.static)]
        self.rows_host.copy_(torch.tensor(rows, dtype=torch.int64))
        self.descs.copy_(self.rows_host, non_blocking=True)
        st = F_._stream()
        ws = F_.workspace(plan.ws_bytes, dev)
        self.norm = torch.empty((), dtype=torch.float32, device=dev)
        n_t = len(rows)
        call("mis_grad_sqsum", self.descs.data_ptr(), plan.prefix.data_ptr(), n_t, plan.n_chunks, ws.data_ptr(), st)
        for k, ((g, ps), (c0, c1)) in enumerate(zip(f.groups, plan.group_chunks)):
            b1, b2 = g["betas"]
            call("mis_clip_adamw_step_dyn", self.descs.data_ptr(), plan.prefix.data_ptr(), n_t, c0, c1, plan.n_chunks,
                 ws.data_ptr(), self.max_norm, float(b1), float(b2), float(g["eps"]), self.dyn[k].data_ptr(), 1,
                 self.norm.data_ptr() if c0 == 0 else None, st)
        return self.norm

    def advance(self):
        """Host bookkeeping after a replay: torch's step counters, tensor versions."""
        f = self.f
        torch._foreach_add_(f.step_tensors, 1)
        f.step = float(int(f.step) + 1)
        touched = []
        for _, ps in f.groups:
            touched += ps
        torch._C._increment_version(touched)
