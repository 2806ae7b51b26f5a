"""Adam for parameters that lie back to back in memory.

`FlatAdam` is torch.optim.Adam (upstream: run_nerf.py:217-218, stepped at run_nerf.py:868-881) with the same
constructor arguments, `param_groups`, `state` and `state_dict()` / `load_state_dict()` format.  When every parameter of
a step lies in a run of parameters whose storage is contiguous (a NeRF module keeps its parameters as views of one flat
vector) and whose gradients are laid out the same way (the fused MLP's backward returns views of one flat gradient, and
the data-parallel exchange reduces it in place), the whole update is ONE launch of the library's Adam kernel plus one
increment of the step counters, instead of the stock implementation's multi-tensor launches of 64 Ki elements per block
(three under-filled launches, 100 us, for the 1.2 M parameters of a coarse + fine pair).  The moments of a run are views
of one buffer per run, and so are the step counters, which the optimiser creates on first use -- or rebuilds from whatever
`load_state_dict` put in their place.  Anything else -- a parameter without a gradient, amsgrad, maximize, a layout that
is not contiguous -- takes torch.optim.Adam.step() unchanged, on the same state.

The step only enqueues work (learning rate and step count are read on the device when they live there), so it can be
recorded into a HIP graph like the stock capturable optimiser -- after one eager step: the first step on a layout moves the
moments into their buffers and reads one word back from the device.

`AdamW` decouples the weight decay, takes tensors wherever they lie, and holds its states in 32 or in 8 bits.
"""
from __future__ import annotations

import ctypes
import itertools
import operator
from array import array
from typing import List, Optional

import torch

from ._lib import check, lib
from .ops import ELEM_TYPES
from .ops import _launch as _launch_on


class _Run:
    """Parameters [i0, i1) of the flattened parameter list: contiguous storage, moments and step counters of their own."""
    __slots__ = ("params", "numel", "key", "exp_avg", "exp_avg_sq", "steps", "uniform")

    def __init__(self, params):
        self.params = params
        self.numel = sum(p.numel() for p in params)
        self.key = None
        self.exp_avg = self.exp_avg_sq = self.steps = None
        self.uniform = True      # every parameter of the run has taken the same number of steps


def _contiguous_after(a: torch.Tensor, b: torch.Tensor) -> bool:
    return b.data_ptr() == a.data_ptr() + 4 * a.numel()


class FlatAdam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False, *, maximize=False):
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad, maximize=maximize,
                         fused=True, capturable=True)
        self._runs: Optional[List[List[_Run]]] = None      # per parameter group
        self._layout_key = None
        self._static = False
        self.fast_steps = 0                                # steps taken through the library kernel (for tests and logs)
        self._steps_all = {}                               # device -> [buffer of every run's step counters, words handed out]

    # ---- layout ------------------------------------------------------------------------------------
    @staticmethod
    def _static_ok(group) -> bool:
        """What does not change from step to step: the update rule and the parameters' type and placement."""
        if group.get("amsgrad") or group.get("maximize") or group.get("differentiable") or not group["params"]:
            return False
        if group.get("decoupled_weight_decay") and group["weight_decay"]:      # (from a checkpoint of AdamW; the kernel's decay is Adam's)
            return False
        return all(p.is_cuda and p.dtype == torch.float32 and p.is_contiguous() for p in group["params"])

    def _find_runs(self):
        """Cuts every group's parameter list where the storage stops being contiguous."""
        runs = []
        for group in self.param_groups:
            out, cur = [], []
            for p in group["params"]:
                if cur and not _contiguous_after(cur[-1], p):
                    out.append(_Run(cur))
                    cur = []
                cur.append(p)
            if cur:
                out.append(_Run(cur))
            runs.append(out)
        return runs

    def _adopt_state(self, run: _Run) -> None:
        """Moments and step counters of a run as views of one buffer each, keeping the values the state holds already
        (a fresh optimiser: zeros; after load_state_dict: the loaded tensors)."""
        dev = run.params[0].device
        m = torch.zeros(run.numel, dtype=torch.float32, device=dev)
        v = torch.zeros(run.numel, dtype=torch.float32, device=dev)
        steps = self._step_buffer(run, dev)
        off = 0
        for i, p in enumerate(run.params):
            st = self.state[p]
            n = p.numel()
            if "exp_avg" in st:
                m[off:off + n].copy_(st["exp_avg"].reshape(-1))
                v[off:off + n].copy_(st["exp_avg_sq"].reshape(-1))
                steps[i].copy_(torch.as_tensor(st["step"], dtype=torch.float32))
            st["exp_avg"] = m[off:off + n].view_as(p)
            st["exp_avg_sq"] = v[off:off + n].view_as(p)
            st["step"] = steps[i]
            off += n
        run.exp_avg, run.exp_avg_sq, run.steps = m, v, steps
        run.key = tuple(id(self.state[p]["exp_avg"]) for p in run.params)
        run.uniform = bool(steps.min() == steps.max())     # (a host read: adoption happens once, outside any recording)

    def _step_buffer(self, run: _Run, dev) -> torch.Tensor:
        """The step counters of a run: a slice of ONE buffer for every run on this device, so that a step increments
        them all with one launch."""
        n_all = sum(len(r.params) for runs in self._runs for r in runs)
        buf = self._steps_all.get(dev)
        if buf is None or buf[0].numel() != n_all:
            buf = self._steps_all[dev] = [torch.zeros(n_all, dtype=torch.float32, device=dev), 0]
        first = buf[1]
        if first + len(run.params) > n_all:      # a layout adopted anew: start over (the values are copied in by the caller)
            buf = self._steps_all[dev] = [torch.zeros(n_all, dtype=torch.float32, device=dev), 0]
            first = 0
        buf[1] = first + len(run.params)
        return buf[0][first:first + len(run.params)]

    @staticmethod
    def _increment(runs) -> None:
        """steps += 1 for every run: one launch per stretch of runs whose counters are adjacent slices of one buffer."""
        i = 0
        while i < len(runs):
            j, n = i, runs[i].steps.numel()
            while (j + 1 < len(runs) and runs[j + 1].steps.data_ptr() == runs[i].steps.data_ptr() + 4 * n
                   and runs[j + 1].steps.untyped_storage().data_ptr() == runs[i].steps.untyped_storage().data_ptr()):
                j += 1
                n += runs[j].steps.numel()
            (runs[i].steps if j == i else runs[i].steps.as_strided((n,), (1,))).add_(1.0)
            i = j + 1

    def _state_intact(self, run: _Run) -> bool:
        if run.key is None:
            return False
        state = self.state
        for p, k in zip(run.params, run.key):
            st = state.get(p)
            if st is None or id(st.get("exp_avg")) != k:
                return False
        return True

    # ---- the step ----------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        key = tuple(p.data_ptr() for g in self.param_groups for p in g["params"])
        if key != self._layout_key:
            self._runs, self._layout_key = self._find_runs(), key
            self._static = all(self._static_ok(g) for g in self.param_groups)
        max_runs = lib.nerf_adam_max_runs()
        todo = []     # (group, runs of it whose gradients are laid out like the parameters)
        for group, runs in zip(self.param_groups, self._runs):
            for run in runs:
                grads = [p.grad for p in run.params]
                g0 = grads[0]
                if (not self._static or any(g is None for g in grads) or g0.dtype != torch.float32 or g0.is_sparse
                        or g0.device != run.params[0].device or not grads[-1].is_contiguous()
                        or any(not _contiguous_after(a, b) for a, b in zip(grads, grads[1:]))):
                    super().step()      # a gradient layout the kernel cannot walk: the stock step, on the same state
                    return loss
            todo.append((group, runs))
        for group, runs in todo:
            for run in runs:
                if not self._state_intact(run):
                    self._adopt_state(run)
        if not all(run.uniform for _, runs in todo for run in runs):
            super().step()              # parameters of one run at different step counts: the stock step keeps them apart
            return loss
        for group, runs in todo:
            self._increment(runs)
            beta1, beta2 = group["betas"]
            lr = group["lr"]
            lr_dev = lr.data_ptr() if torch.is_tensor(lr) and lr.is_cuda else None
            lr_val = 0.0 if lr_dev is not None else float(lr)
            if torch.is_tensor(lr) and lr_dev is not None and lr.dtype != torch.float32:
                raise TypeError("FlatAdam: a device learning rate must be a float32 tensor")
            dev = runs[0].params[0].device
            with torch.cuda.device(dev):
                stream = torch.cuda.current_stream().cuda_stream
                for a in range(0, len(runs), max_runs):
                    part = runs[a:a + max_runs]
                    n = len(part)
                    counts = (ctypes.c_int64 * n)(*[r.numel for r in part])
                    arr = lambda ptrs: (ctypes.c_void_p * n)(*ptrs)      # noqa: E731
                    check(lib.nerf_adam_step(n, counts, arr([r.params[0].data_ptr() for r in part]),
                                             arr([r.params[0].grad.data_ptr() for r in part]),
                                             arr([r.exp_avg.data_ptr() for r in part]), arr([r.exp_avg_sq.data_ptr() for r in part]),
                                             arr([r.steps.data_ptr() for r in part]), 0.0, lr_dev, lr_val, float(beta1), float(beta2),
                                             float(group["eps"]), float(group["weight_decay"]), stream))
        self.fast_steps += 1
        return loss

    def load_state_dict(self, state_dict):
        """As torch.optim.Adam, for checkpoints of either optimiser (and of upstream's); the groups keep this class's
        fused / capturable settings whatever the checkpoint's were, so that the stock step stays usable on the state.  A checkpoint of
        AdamW goes on with its decoupled weight decay (the stock step has it); one with states in 8 bits is refused."""
        if any("scale" in st for st in state_dict["state"].values()):
            raise ValueError("FlatAdam: a checkpoint of AdamW with states in 8 bits (state_bits = 8)")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            group["fused"], group["capturable"], group["foreach"] = True, True, None
            for p in group["params"]:
                st = self.state.get(p)
                if st and "step" in st and not (torch.is_tensor(st["step"]) and st["step"].is_cuda):
                    st["step"] = torch.as_tensor(float(st["step"]), dtype=torch.float32, device=p.device)
        self._layout_key = None


def _address(values: array) -> int:
    return values.buffer_info()[0]


_data_ptr, _numel, _is_contiguous, _get_device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype, _layout, _grad = operator.attrgetter("dtype"), operator.attrgetter("layout"), operator.attrgetter("grad")


def _all_are(values, one) -> bool:
    return all(map(operator.is_, values, itertools.repeat(one)))


class _Launch:
    """The tensors of a group that share a device and a type, as the kernel takes them: host arrays of addresses and counts."""
    __slots__ = ("device", "dtype", "kind", "index", "params", "counts", "devices", "pointers", "bytes")

    def __init__(self, device, dtype, index, params, states):
        self.device, self.dtype, self.kind = device, dtype, ELEM_TYPES[dtype]
        self.index, self.params = index, params
        self.devices = array("q", [device.index] * len(params))
        self.counts = array("q", map(_numel, params))
        self.pointers = {"params": array("Q", map(_data_ptr, params))}
        self.bytes = 0
        for name in ("exp_avg", "exp_avg_sq", "scale", "master", "step"):
            ts = [st.get(name) for st in states]
            self.pointers[name] = array("Q", [0 if t is None else t.data_ptr() for t in ts])
            self.bytes += sum(0 if t is None else 2 * t.numel() * t.element_size() for t in ts)
        self.bytes += 3 * sum(self.counts) * dtype.itemsize

    def take(self, all_grads):
        """This step's gradients: (addresses, the tensors they belong to)."""
        grads = all_grads if self.index is None else [all_grads[i] for i in self.index]
        if not _all_are(map(_layout, grads), torch.strided):
            raise TypeError("AdamW: sparse gradients are not supported")
        if not _all_are(map(_dtype, grads), self.dtype) or array("q", map(_get_device, grads)) != self.devices:
            raise TypeError(f"AdamW: a gradient is not in {self.dtype} on {self.device}, as its parameter is")
        if array("q", map(_numel, grads)) != self.counts:
            raise ValueError("AdamW: a gradient has another size than its parameter")
        if not all(map(_is_contiguous, grads)):
            grads = [g.contiguous() for g in grads]
        return array("Q", map(_data_ptr, grads)), grads


class _Plan:
    """What a step of a group needs to know and seldom changes: which tensors take part, their states and addresses.  Every step
    looks whether it still stands -- the same tensor objects, at the same addresses, of the same sizes --, with a few passes over lists
    instead of a dozen checks per tensor (for 48 small tensors those cost more than the launch)."""
    __slots__ = ("params", "absent", "states", "held", "pointed", "addresses", "live", "counts", "launches")

    def __init__(self, opt, params, grads):
        self.params, self.absent = list(params), list(map(operator.is_, grads, itertools.repeat(None)))
        lists = {}
        for i, (p, g) in enumerate(zip(params, grads)):
            if g is None:
                continue
            if g.layout != torch.strided:
                raise TypeError("AdamW: sparse gradients are not supported")
            if p.dtype not in ELEM_TYPES or not p.is_cuda:
                raise TypeError(f"AdamW: expected fp32, bf16 or fp16 parameters on a HIP device, got {p.dtype} on {p.device}")
            if not p.is_contiguous():
                raise ValueError(f"AdamW: a parameter of shape {tuple(p.shape)} is not contiguous")
            lists.setdefault((p.device, p.dtype), []).append(i)
        self.live = [p for p, none in zip(params, self.absent) if not none]
        self.states = [opt._checked_state(p) for p in self.live]
        state_of = dict(zip(map(id, self.live), self.states))
        self.held = list(itertools.chain.from_iterable(map(dict.values, self.states)))
        self.pointed = self.live + [t for t in self.held if torch.is_tensor(t)]
        self.addresses = array("Q", map(_data_ptr, self.pointed))
        self.counts = array("q", map(_numel, self.live))
        self.launches = [_Launch(device, dtype, index if len(index) < len(self.params) else None, [params[i] for i in index],
                                 [state_of[id(params[i])] for i in index]) for (device, dtype), index in lists.items()]

    def stands(self, params, grads) -> bool:
        if len(params) != len(self.params) or not all(map(operator.is_, params, self.params)) or list(map(operator.is_, grads, itertools.repeat(None))) != self.absent:
            return False
        held = list(itertools.chain.from_iterable(map(dict.values, self.states)))
        return (len(held) == len(self.held) and all(map(operator.is_, held, self.held))
                and array("Q", map(_data_ptr, self.pointed)) == self.addresses and array("q", map(_numel, self.live)) == self.counts
                and all(map(_is_contiguous, self.live)))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over any tensors, wherever they lie: one launch of the library's kernel per 60 tensors of a
    group, device and type, after a small one that counts the steps -- where FlatAdam needs parameters and gradients back to back.

    Parameters are fp32, bf16 or fp16 and contiguous, on a HIP device when the step is taken.  `state[p]` holds ordinary tensors:
      step         fp32 scalar on the device
      exp_avg, exp_avg_sq   state_bits = 32: fp32, as torch.optim.AdamW's (whose checkpoints of fp32 parameters load, and the reverse);
                   state_bits = 8: float8_e4m3fn and float8_e5m2, relative to `scale` (for this class alone: torch's would take the
                   codes for moments)
      scale        state_bits = 8: fp32 [blocks of 128 consecutive elements, 2]: the largest |exp_avg| / 448 and exp_avg_sq / 57344, at
                   least 1e-38 unless all are 0
      master       16-bit parameters: the fp32 values they are rounded from (an element of the parameter that was written from
                   outside, and so is no longer its master's rounding, is taken as it is)
    8-bit states are rounded stochastically from a hash of (element, step), so a run repeats bit for bit; a gradient that is not
    finite reaches the states of its whole block of 128 (with 32 bits: of its element).  The learning rate may be a float or an fp32
    device scalar, which a captured step reads at every replay; take one eager step before capturing."""

    _MOMENTS = {32: (torch.float32, torch.float32), 8: (torch.float8_e4m3fn, torch.float8_e5m2)}

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32):
        if state_bits not in self._MOMENTS:
            raise ValueError(f"AdamW: state_bits={state_bits} is neither 32 nor 8")
        self._check_hyper(lr, betas, eps, weight_decay)
        self.state_bits = state_bits
        self._plans, self._seen = {}, []      # what the last step looked up: see _Plan
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=True,
                                      decoupled_weight_decay=True))      # (for Adam's classes, should they load a checkpoint of this one)

    @staticmethod
    def _check_hyper(lr, betas, eps, weight_decay):
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError(f"AdamW: lr={lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"AdamW: betas={betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"AdamW: eps={eps}, weight_decay={weight_decay}")

    def add_param_group(self, param_group):
        params = param_group["params"]
        params = [params] if torch.is_tensor(params) else list(params)
        if len({id(p) for p in params}) != len(params):
            raise ValueError("AdamW: a parameter appears twice in one group")
        super().add_param_group({**param_group, "params": params})

    # ---- states --------------------------------------------------------------------------------------
    def _layout(self, p):
        """name -> (type, shape) of the state of `p`."""
        m, v = self._MOMENTS[self.state_bits]
        out = {"step": (torch.float32, torch.Size(())), "exp_avg": (m, p.shape), "exp_avg_sq": (v, p.shape)}
        if self.state_bits == 8:
            out["scale"] = (torch.float32, torch.Size(((p.numel() + 127) // 128, 2)))
        if p.dtype != torch.float32:
            out["master"] = (torch.float32, p.shape)
        return out

    def _new_state(self, p):
        out = {}
        for name, (dtype, shape) in self._layout(p).items():
            if name == "master":
                out[name] = p.detach().to(torch.float32)
            elif dtype.itemsize == 1:
                out[name] = torch.zeros(shape, dtype=torch.uint8, device=p.device).view(dtype)
            else:
                out[name] = torch.zeros(shape, dtype=dtype, device=p.device)
        return out

    def _checked_state(self, p):
        """The state of `p` -- made on first use --, which the kernel will read by address: every tensor of the layout it assumes."""
        st = self.state[p]
        if not st:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: take one eager step before capturing (the states would be made anew by every replay)")
            st.update(self._new_state(p))
        for name, (dtype, shape) in self._layout(p).items():
            t = st.get(name)
            if not torch.is_tensor(t) or t.dtype != dtype or t.shape != shape or t.device != p.device or not t.is_contiguous():
                raise ValueError(f"AdamW: the state's {name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {p.device}, got "
                                 f"{(t.dtype, tuple(t.shape), t.device) if torch.is_tensor(t) else t}")
        return st

    # ---- the step ------------------------------------------------------------------------------------
    def step(self, closure=None):      # (nothing here is recorded by autograd: the library writes through addresses)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        states = list(self.state.values())
        known = len(states) == len(self._seen) and all(map(operator.is_, states, self._seen))
        work, written = [], []
        for group in self.param_groups:      # (everything is checked before anything is launched)
            self._check_hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"])
            grads = list(map(_grad, group["params"]))
            plan = self._plans.get(id(group)) if known else None
            if plan is None or not plan.stands(group["params"], grads):
                plan = self._plans[id(group)] = _Plan(self, group["params"], grads)
            lr = group["lr"]
            if torch.is_tensor(lr) and lr.is_cuda:
                for launch in plan.launches:
                    if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != launch.device:
                        raise TypeError(f"AdamW: a device learning rate must be one fp32 value on {launch.device}, got {lr.dtype} on {lr.device}")
            work += [(group, launch, launch.take(grads)) for launch in plan.launches]
            written += plan.live
        self._seen = list(self.state.values())
        torch.autograd.graph.increment_version(written)      # (a graph that saved a parameter refuses its backward pass from here on)
        for group, launch, (addresses, _) in work:
            self._launch(group, launch, addresses)
        return loss

    def _launch(self, group, launch, grads):
        device, lr, lr_dev = launch.device, group["lr"], None
        if torch.is_tensor(lr) and lr.is_cuda:
            lr_dev, lr = lr.data_ptr(), 0.0
        n = len(launch.params)
        coef = torch.empty((4 * n,), dtype=torch.float32, device=device)
        beta1, beta2 = group["betas"]
        _launch_on(device, "adamw", launch.bytes, lib.nerf_adamw_step, n, _address(launch.counts), launch.kind, self.state_bits,
                   _address(launch.pointers["params"]), _address(grads), _address(launch.pointers["exp_avg"]),
                   _address(launch.pointers["exp_avg_sq"]), _address(launch.pointers["scale"]), _address(launch.pointers["master"]),
                   _address(launch.pointers["step"]), lr_dev, float(lr), float(beta1), float(beta2), float(group["eps"]),
                   float(group["weight_decay"]), coef.data_ptr())

    # ---- checkpoints ---------------------------------------------------------------------------------
    def load_state_dict(self, state_dict):
        """Checkpoints of this class with the same state_bits, and of torch.optim.Adam / AdamW with state_bits = 32, where their rule is this
        one's: no amsgrad, no maximize, no weight decay in Adam's gradient.  The states keep their own types (torch.optim would cast them
        to the parameter's)."""
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize") or (g.get("weight_decay") and g.get("decoupled_weight_decay") is False):
                raise ValueError("AdamW: a checkpoint with amsgrad, maximize or a weight decay that is part of the gradient")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        fresh = {}
        for i, p in zip(ids, params):
            st = state_dict["state"].get(i)
            if st is None:
                continue
            new = {}
            for name, (dtype, shape) in self._layout(p).items():
                t = st.get(name)
                if name == "master" and t is None:
                    new[name] = p.detach().to(torch.float32)
                elif name == "step":
                    new[name] = torch.as_tensor(0.0 if t is None else t, dtype=torch.float32).reshape(()).to(p.device).clone()
                elif not torch.is_tensor(t) or t.dtype != dtype or t.shape != shape:
                    raise ValueError(f"AdamW: with state_bits={self.state_bits} the checkpoint's {name} must be {dtype} of shape {tuple(shape)}, "
                                     f"got {(t.dtype, tuple(t.shape)) if torch.is_tensor(t) else t}")
                else:
                    new[name] = t.detach().to(p.device, copy=True).contiguous()
            fresh[p] = new
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        for group in self.param_groups:
            group["capturable"] = group["decoupled_weight_decay"] = True
        self._plans, self._seen = {}, []
        for p, new in fresh.items():
            self.state[p] = new

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans, self._seen = {}, []
