"""AdamW over all tensors of a model at once, its moments held in 8 bits or in fp32 (``include/cswap_hip.h``, "AdamW").

The reference leaves the optimiser to its framework (CIFAR10/cifar10.py:98); what a step keeps besides activations are the
optimiser's two moments, 8 bytes a parameter in fp32 and 2.06 here:

    optimizer = AdamW8(model.parameters(), lr=1e-3)             # torch.optim.AdamW's arguments and defaults
    loss.backward();  optimizer.step()
    moments = unpack_moments(optimizer)                         # [(exp_avg, exp_avg_sq)] in fp32

A step is one launch for every 64 tensors, of any mixture of types, on the current stream of their device; nothing waits for it.  It goes by
``optimizer.state`` as it then is, whoever cleared, replaced or moved what is in it, and autograd is told what it writes: a backward pass through
weights that a step has moved is refused, as with torch's optimisers.  Steps and conversions refuse to be traced.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import is_

import torch
from torch.autograd.graph import increment_version

from . import q8
from ._lib import AdamwOptions, check, lib

__all__ = ["AdamW8", "unpack_moments"]

GROUP = 32
_OWN = ("bits", "master", "capturable")     # how an optimiser holds its state, whatever it loads


def _dense_order(t: torch.Tensor) -> bool:
    """Whether t fills its memory, in whatever order of its dimensions."""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def _how(group):
    return group["bits"], group["capturable"], group["master"]


class _Plan:
    """The call for some parameters: its table, filled in but for the gradients' addresses, and what it was made from."""
    __slots__ = ("params", "states", "rows", "kinds", "written", "table", "device", "place", "how", "count")

    def __init__(self, optimizer, group, params):
        self.how = bits, *_ = _how(group)
        self.params, self.states = list(params), [optimizer.state[p] for p in params]
        self.device, self.place = params[0].device, params[0].get_device()
        self.count = self.states[0]["step"]
        # rows of cswap_adamw_tensor: seven words, the type in the last
        self.rows, self.kinds, self.table, self.written = [], [], array("Q"), []
        for p, s in zip(params, self.states):
            if p.dtype not in q8._DTYPE:
                raise TypeError(f"AdamW8: float32, bfloat16 or float16, not {p.dtype}")
            m, v, master = s["exp_avg"], s["exp_avg_sq"], s.get("master")
            _check_state(p, s, (m, v, master), bits)
            if not _dense_order(p):
                raise ValueError(f"AdamW8: a parameter {tuple(p.shape)} with strides {p.stride()} does not fill its memory")
            at, n = p.data_ptr(), p.numel()
            m_at, v_at, master_at = m.data_ptr(), v.data_ptr(), 0 if master is None else master.data_ptr()
            strides = None if p.is_contiguous() else p.stride()
            self.rows.append((p, at, n, strides, s, m, v, master, m_at, v_at, master_at))
            self.kinds.append((n, strides, p.dtype))
            self.table.extend((at, 0, m_at, v_at, master_at, n, q8._DTYPE[p.dtype]))
            self.written += (p, m, v) if master is None else (p, m, v, master)
        if group["capturable"]:
            self.written.append(self.count)

        # all tensors of a launch are worked on at once
        ends = sorted((at, at + n * p.element_size()) for p, at, n, *_ in self.rows if n)
        if any(end > start for (_, end), (start, _) in zip(ends, ends[1:])):
            raise ValueError("AdamW8: parameters that share memory")

    def holds(self, params, group) -> bool:
        """Whether the plan is still that of these parameters and of what is in their states (which these are: ``AdamW8._same_states``)."""
        if len(params) != len(self.rows) or self.how != _how(group):
            return False
        count = self.count
        if isinstance(count, torch.Tensor) and count.device != self.device:
            return False
        for p, (mine, at, n, strides, s, m, v, master, m_at, v_at, master_at) in zip(params, self.rows):
            if p is not mine or p.data_ptr() != at or p.numel() != n:
                return False
            if (not p.is_contiguous()) if strides is None else p.stride() != strides:
                return False
            get = s.get
            if get("exp_avg") is not m or get("exp_avg_sq") is not v or get("master") is not master or get("step") is not count:
                return False
            if m.data_ptr() != m_at or v.data_ptr() != v_at or master is not None and master.data_ptr() != master_at:
                return False
        return True

    def moments_hold(self, params, group) -> bool:
        """The same of what a conversion of the moments reads."""
        if len(params) != len(self.rows) or self.how != _how(group):
            return False
        for p, (mine, _, n, strides, s, m, v, _, m_at, v_at, _) in zip(params, self.rows):
            if p is not mine or p.numel() != n or ((not p.is_contiguous()) if strides is None else p.stride() != strides):
                return False
            if s.get("exp_avg") is not m or s.get("exp_avg_sq") is not v or m.data_ptr() != m_at or v.data_ptr() != v_at:
                return False
        return True

    def set_gradients(self, gradients):
        """Fills in the gradients' addresses; gives back what has to live until the launch."""
        copies, addresses = [], []
        place = self.place
        for (n, strides, dtype), g, p in zip(self.kinds, gradients, self.params):
            if g.dtype is not dtype or g.numel() != n:
                raise TypeError(f"AdamW8: a gradient {tuple(g.shape)} {g.dtype} of a parameter {tuple(p.shape)} {dtype}")
            if g.get_device() != place:
                raise ValueError(f"AdamW8: a gradient on {g.device} of a parameter on {p.device}")
            if ((not g.is_contiguous()) if strides is None else g.stride() != strides) or g.is_neg():
                if g.layout is not torch.strided:       # (none of these is contiguous)
                    raise RuntimeError("AdamW8: no sparse gradients")
                g = torch.empty_like(p).copy_(g)
                copies.append(g)
            addresses.append(g.data_ptr())
        self.table[1::7] = array("Q", addresses)
        return copies


def _check_state(p, s, kept, bits):
    """A state that did not come from here, or a parameter that changed under it."""
    if not p.is_cuda:
        raise ValueError("AdamW8: expected parameters in device memory")
    m, v, master = kept
    n = p.numel()
    for t in (m, v):
        if bits == 8:
            fits = t.dtype is torch.uint8 and t.numel() == -(-n // GROUP) * (GROUP + 1) and t.is_contiguous() and t.data_ptr() % 8 == 0
        else:
            fits = t.dtype is torch.float32 and t.numel() == n and (t.stride() == p.stride() or t.is_contiguous() and p.is_contiguous())
        if not fits or t.device != p.device:
            raise ValueError(f"AdamW8: a moment {tuple(t.shape)} {t.dtype} on {t.device} of a parameter {tuple(p.shape)} on {p.device} held in "
                             f"{bits} bits")
    if bits == 8 and tuple(s.get("strides", p.stride())) != p.stride():
        raise RuntimeError(f"AdamW8: moments in 8 bits of a parameter with strides {tuple(s['strides'])}, which now has {p.stride()}")
    if master is not None and (master.dtype is not torch.float32 or master.numel() != n or master.device != p.device or
                               not (master.stride() == p.stride() or master.is_contiguous() and p.is_contiguous())):
        raise ValueError(f"AdamW8: a master copy {tuple(master.shape)} {master.dtype} on {master.device} of a parameter {tuple(p.shape)} on {p.device}")


class AdamW8(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with ``bits=8`` or 32 for its moments, in each parameter group as it says.

    Parameters are float32, bfloat16 or float16 in device memory; the step is computed in fp32 and rounded to the parameter's
    type once, to nearest: 16-bit parameters of steps below their last place keep still, unless ``master=True`` keeps fp32
    copies of them (their ``state[p]["master"]``, from which a step makes the parameter: what is written to the parameter alone is
    lost with the next one).  In 8 bits a moment has three bits of mantissa over 2^14 (the second: 2^30) below the
    largest of 32 neighbours, rounded up and down in turn so that it drifts as it should; a NaN or an infinity in a gradient makes its 32
    neighbours' moments NaN.  ``state[p]`` has "step", "exp_avg" and "exp_avg_sq", as ``torch.optim.AdamW``'s, which
    ``load_state_dict`` also takes.

    ``capturable=True``: steps are counted in device memory, so that ``step()`` can be captured into a graph and counts on at each
    replay; ``lr`` may be an fp32 tensor of one value on the device.  Make one step before capturing.  Parameters that made their
    first step together then have to have gradients together."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, bits: int = 8, master: bool = False,
                 capturable: bool = False):
        self._forget()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, master=master, capturable=capturable))

    def add_param_group(self, param_group):
        group = {**self.defaults, **{k: v for k, v in param_group.items() if k != "params"}}
        _options(group)
        if group["bits"] not in (8, 32):
            raise ValueError(f"AdamW8: moments in 8 or 32 bits, not {group['bits']}")
        super().add_param_group(param_group)
        given = self.param_groups[-1]["params"]
        if len({id(p) for p in given}) != len(given):
            self.param_groups.pop()
            raise ValueError("AdamW8: a parameter twice")
        for p in given:
            if p.dtype not in q8._DTYPE:
                self.param_groups.pop()
                raise TypeError(f"AdamW8: float32, bfloat16 or float16, not {p.dtype}")

    def __setstate__(self, state):
        super().__setstate__(state)
        self._forget()

    def _forget(self):
        """Plans, and what ``state`` held when they were made: parameters and their dictionaries, one by one."""
        self._plans, self._seen = {}, ([], [])

    def _same_states(self) -> bool:
        """Whether ``state`` still has the dictionaries that the plans were made from, whoever cleared or replaced some."""
        state, (params, states) = self.state, self._seen
        return len(state) == len(params) and all(map(is_, state, params)) and all(map(is_, state.values(), states))

    def _new_state(self, p, group, steps, fresh):
        """``fresh``: gets the moments that are to be 0, all of which are filled at once."""
        if not p.is_cuda:
            raise ValueError("AdamW8: expected parameters in device memory")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW8: a parameter's first step cannot be captured")
        if not _dense_order(p):
            raise ValueError(f"AdamW8: a parameter {tuple(p.shape)} with strides {p.stride()} does not fill its memory")
        s = self.state[p]
        if group["bits"] == 8:
            size = lib().cswap_adamw_moment_bytes(p.numel())
            pair = [torch.empty(size, dtype=torch.uint8, device=p.device) for _ in range(2)]
            s["strides"] = p.stride()
        else:
            pair = [torch.empty_like(p, dtype=torch.float32) for _ in range(2)]
        s["exp_avg"], s["exp_avg_sq"] = pair
        fresh += pair
        self._finish_state(p, s, group, 0, steps)

    def _finish_state(self, p, s, group, step, steps):
        if group["master"] and p.dtype is not torch.float32 and "master" not in s:
            s["master"] = p.detach().to(torch.float32)
        if group["capturable"]:      # one counter for those that begin together
            key = (p.device, step)
            if key not in steps:
                steps[key] = torch.full((1,), step, dtype=torch.int64, device=p.device)
            s["step"] = steps[key]
        else:
            s["step"] = step

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if q8._watched():
            given = [p for group in self.param_groups for p in group["params"]]
            q8._refuse_what_torch_would_lose("AdamW8.step", *given, *(p.grad for p in given))
        # whatever one of the groups refuses is refused before a step of any is made
        ready, made = [], False
        if not self._same_states():
            self._forget()
        for number, group in enumerate(self.param_groups):
            params, gradients = group["params"], [p.grad for p in group["params"]]
            given = [g for g in gradients if g is not None]
            if len(given) < len(params):
                params, gradients = [p for p, g in zip(params, gradients) if g is not None], given
            if not given:
                continue
            capturable = group["capturable"]
            options = _options(group)
            plans = self._plans.get(number)
            if plans is None or not all(plan.holds(some, group) for plan, some in zip(plans, _as_split(plans, params))):
                plans, made = self._make_plans(group, params), True
                self._plans[number] = plans
            if not capturable and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW8: a captured step needs capturable=True")
            if capturable:
                _all_together(group, params, self.state)
            lr = group["lr"] if isinstance(group["lr"], torch.Tensor) else None
            for plan, some in zip(plans, _as_split(plans, params, gradients)):
                if lr is not None and lr.device != plan.device:
                    raise ValueError(f"AdamW8: lr on {lr.device}, parameters on {plan.device}")
                ready.append((plan, group, options, lr, plan.set_gradients(some)))
        if made:
            self._seen = list(self.state), list(self.state.values())
        for plan, group, options, lr, _ in ready:
            if q8._stream_of(plan.device) is not None:
                _launch(plan, group, options, lr)
            else:
                with torch.cuda.device(plan.device):
                    _launch(plan, group, options, lr)
        return loss

    def _make_plans(self, group, params):
        """A plan for the parameters of each device that have made as many steps."""
        steps, split, fresh = {}, {}, []
        try:
            for p in params:
                if "exp_avg" not in self.state[p]:
                    self._new_state(p, group, steps, fresh)
        finally:
            if fresh:
                torch._foreach_zero_(fresh)
        for p in params:
            step = self.state[p]["step"]
            if not _counts(step, group, p.device):      # the option changed, or it was set
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW8: make a step with capturable=True before capturing one")
                self._finish_state(p, self.state[p], group, int(step), steps)
                step = self.state[p]["step"]
            if bool(group["master"]) != ("master" in self.state[p]) and p.dtype is not torch.float32:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW8: make a step with this master before capturing one")
                if group["master"]:
                    self.state[p]["master"] = p.detach().to(torch.float32)
                else:
                    del self.state[p]["master"]
            split.setdefault((p.device, id(step) if group["capturable"] else step), []).append(p)
        return [_Plan(self, group, some) for some in split.values()]

    def load_state_dict(self, state_dict):
        """Of an ``AdamW8`` or of a ``torch.optim.AdamW``; this optimiser's own ``bits``, ``master`` and ``capturable`` stay, and moments are
        converted to them (to 8 bits: to nearest), one parameter at a time."""
        own = [{k: group[k] for k in _OWN} for group in self.param_groups]
        given = {}

        def look(_, last):             # what the caller's hooks leave
            for saved in last["param_groups"]:
                if saved.get("amsgrad") or saved.get("maximize"):
                    raise ValueError("AdamW8: no amsgrad and no maximize")
            for kept in last["state"].values():
                if kept and ("step" not in kept or not all(isinstance(kept.get(k), torch.Tensor) for k in ("exp_avg", "exp_avg_sq"))):
                    raise ValueError(f"AdamW8: expected step, exp_avg and exp_avg_sq in a parameter's state, not {sorted(kept)}")
            given.update(last)
            # torch would cast moments to the parameters' types, all of them before the first is converted
            numbers = {number for saved in last["param_groups"] for number in saved["params"]}
            return {**last, "state": {number: kept for number, kept in last["state"].items() if number not in numbers}}

        def convert(_):                 # before they see what was loaded
            for group, mine, saved in zip(self.param_groups, own, given["param_groups"]):
                group.update(mine)
                lr = group["lr"]
                if isinstance(lr, torch.Tensor):
                    group["lr"] = lr.to(next(iter(group["params"]), lr).device, torch.float32) if group["capturable"] else float(lr)
                steps = {}              # each group counts its own
                for p, number in zip(group["params"], saved["params"]):
                    kept = given["state"].get(number)
                    if kept:
                        self._load(p, group, kept, steps)

        hooks = self.register_load_state_dict_pre_hook(look), self.register_load_state_dict_post_hook(convert, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
            self._forget()

    @torch.no_grad()
    def _load(self, p, group, kept, steps):
        if not p.is_cuda:
            raise ValueError("AdamW8: expected parameters in device memory")
        s = self.state[p]
        s.clear()
        strides = tuple(kept.get("strides", p.stride()))
        pair = [kept["exp_avg"], kept["exp_avg_sq"]]
        size = lib().cswap_adamw_moment_bytes(p.numel())
        if pair[0].dtype is torch.uint8:
            if any(t.dtype is not torch.uint8 or t.numel() != size for t in pair):
                raise ValueError(f"AdamW8: {pair[0].numel()} bytes of moments of a parameter of {p.numel()} values")
            pair = [t.detach().to(p.device, copy=True).reshape(-1) for t in pair]
            if group["bits"] != 8 or strides != p.stride():
                values = [torch.empty_strided(p.shape, strides, dtype=torch.float32, device=p.device) for _ in pair]
                _convert(_row(*values, *pair), "cswap_adamw_unpack", p.device)
                pair = values
        if pair[0].dtype is not torch.uint8:
            pair = [torch.empty_like(p, dtype=torch.float32).copy_(t.reshape(p.shape)) for t in pair]
            if group["bits"] == 8:
                packed = [torch.empty(size, dtype=torch.uint8, device=p.device) for _ in pair]
                _convert(_row(*pair, *packed), "cswap_adamw_pack", p.device)
                pair = packed
        s["exp_avg"], s["exp_avg_sq"] = pair
        if group["bits"] == 8:
            s["strides"] = p.stride()
        if group["master"] and p.dtype is not torch.float32 and kept.get("master") is not None:
            s["master"] = torch.empty_like(p, dtype=torch.float32).copy_(kept["master"].reshape(p.shape))
        self._finish_state(p, s, group, int(kept["step"]), steps)


def _launch(plan, group, options, lr):
    table, count, first, stream = plan.table.buffer_info()[0], len(plan.rows), plan.states[0], q8._stream_of(plan.device)
    if group["capturable"]:
        factors = torch.empty(lib().cswap_adamw_factors_bytes(), dtype=torch.uint8, device=plan.device)
        check(lib().cswap_adamw_step_counted(table, count, group["bits"], C.byref(options), first["step"].data_ptr(),
                                             0 if lr is None else lr.data_ptr(), factors.data_ptr(), stream), "cswap_adamw_step_counted")
    else:
        step = first["step"] + 1
        check(lib().cswap_adamw_step(table, count, group["bits"], C.byref(options), step, stream), "cswap_adamw_step")
        plan.count = step
        for s in plan.states:
            s["step"] = step
    increment_version(plan.written)      # or a backward pass that saved a parameter would not be refused


def _counts(step, group, device) -> bool:
    """Whether this is how a group counts its steps."""
    if group["capturable"]:
        return isinstance(step, torch.Tensor) and step.dtype is torch.int64 and step.numel() == 1 and step.device == device
    return isinstance(step, int)


def _options(group) -> AdamwOptions:
    lr, (b1, b2) = group["lr"], group["betas"]
    if isinstance(lr, torch.Tensor):
        if not group["capturable"] or lr.numel() != 1 or lr.dtype is not torch.float32 or not lr.is_cuda:
            raise ValueError("AdamW8: lr is a number, or, with capturable=True, an fp32 tensor of one value in device memory")
        lr = 0.0
    options = AdamwOptions(lr, b1, b2, group["eps"], group["weight_decay"])
    if not (0.0 <= lr < 1e30 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and 1e-30 <= group["eps"] < 1e30 and 0.0 <= group["weight_decay"] < 1e30):
        raise ValueError(f"AdamW8: lr {lr}, betas {(b1, b2)}, eps {group['eps']}, weight_decay {group['weight_decay']}")
    return options


def _as_split(plans, params, given=None):
    """params, or what is given for each of them, in the plans' order, as far as they are the same ones."""
    given = params if given is None else given
    if len(plans) == 1:
        return [given]
    place = {id(p): k for k, plan in enumerate(plans) for p in plan.params}
    split = [[] for _ in plans]
    for p, one in zip(params, given):
        split[place.get(id(p), 0)].append(one)
    return split


def _all_together(group, params, state):
    counters = {id(state[p]["step"]) for p in params}
    there = {id(p) for p in params}
    for p in group["params"]:
        if id(p) not in there and p in state and id(state[p].get("step")) in counters:
            raise RuntimeError("AdamW8: capturable=True, and a parameter without a gradient shares the count of steps with others that have one")


def _row(m, v, m8, v8):
    return array("Q", (m.data_ptr(), v.data_ptr(), m8.data_ptr(), v8.data_ptr(), m.numel()))


def _convert(rows, name, device):
    """``rows``: cswap_adamw_moments as five words each; ``device``: or its number."""
    device = torch.device("cuda", device) if isinstance(device, int) else device
    if q8._watched():
        q8._refuse_what_torch_would_lose(name)
    stream = q8._stream_of(device)
    if stream is None:
        with torch.cuda.device(device):
            return _convert(rows, name, device)
    check(getattr(lib(), name)(rows.buffer_info()[0], len(rows) // 5, stream), name)


def _held(optimizer):
    """Of the parameters that have made a step, in order: the parameter, its group, its state, its number of values, its device's number, whether it is
    contiguous and, where they are held in 8 bits, the two moments' addresses, checked."""
    same = optimizer._same_states()
    for number, group in enumerate(optimizer.param_groups):
        params = [p for p in group["params"] if "exp_avg" in optimizer.state.get(p, ())]
        plans = optimizer._plans.get(number, ()) if same else ()
        if len(plans) == 1 and plans[0].moments_hold(params, group):
            place = plans[0].place
            for p, _, n, strides, s, _, _, _, m8, v8, _ in plans[0].rows:
                yield p, group, s, n, place, strides is None, m8, v8
            continue
        for p in params:
            s = optimizer.state[p]
            _check_state(p, s, (s["exp_avg"], s["exp_avg_sq"], None), group["bits"])
            yield p, group, s, p.numel(), p.get_device(), p.is_contiguous(), s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr()


@torch.no_grad()
def unpack_moments(optimizer: AdamW8, out=None):
    """``[(exp_avg, exp_avg_sq)]`` in fp32 of the parameters that have made a step, in their order and layout; ``out``: such a list to
    write to."""
    if q8._watched():
        q8._refuse_what_torch_would_lose("unpack_moments", *(t for pair in out or () for t in pair))
    held = list(_held(optimizer))
    if out is None:
        out = [tuple(torch.empty_like(p, dtype=torch.float32) for _ in range(2)) for p, *_ in held]
    elif len(out) != len(held):
        raise ValueError(f"unpack_moments: {len(out)} pairs for {len(held)} parameters")
    rows, written, f32 = {}, [], torch.float32
    for (p, group, s, n, place, contiguous, m8, v8), (m, v) in zip(held, out):
        for t in (m, v):
            if t.dtype is not f32 or t.numel() != n or t.get_device() != place or not (contiguous and t.is_contiguous() or t.stride() == p.stride()):
                raise ValueError(f"unpack_moments: {tuple(t.shape)} {t.dtype} on {t.device} for a parameter {tuple(p.shape)} on {p.device}")
        if group["bits"] == 8:
            some = rows.get(place)
            if some is None:
                some = rows[place] = []
            some += (m.data_ptr(), v.data_ptr(), m8, v8, n)
            written += (m, v)
        else:
            m.copy_(s["exp_avg"].view_as(m))
            v.copy_(s["exp_avg_sq"].view_as(v))
    for place, some in rows.items():
        _convert(array("Q", some), "cswap_adamw_unpack", place)
    increment_version(written)
    return out
