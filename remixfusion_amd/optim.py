"""Adam for the mapper's two optimizers, stepped by one librfx launch (rfx_adam_step); AdamW over many tensors with its moments in
32 or in 8 bits (rfx_adamw_step) and clipping by the gradients' global norm (rfx_grad_norm, rfx_grad_scale).

Reference: ``optim.Adam(trainable_parameters, betas=(0.9, 0.99))`` / ``optim.Adam(rba_parameter, ...)`` in
mp_slam/slam.py:271-286, stepped in mp_slam/mapper.py:416-418 and :497-499.  This is a ``torch.optim.Adam`` (same
constructor, param groups, ``state_dict`` layout: ``step`` / ``exp_avg`` / ``exp_avg_sq`` per parameter); only
``step()`` differs: fp32 device parameters are updated by librfx, everything else (CPU tensors, other dtypes, amsgrad,
maximize, closures that need grad mode) takes torch's own implementation.
"""
import ctypes as C
import math

import torch
from torch.optim import optimizer as _torch_optimizer

from . import _lib


class Adam(torch.optim.Adam):
    def __init__(self, params, **kw):
        kw.pop("fused", None)
        kw.pop("foreach", None)
        self._views = {}                # parameter -> (its state's `step` tensor, numpy view of it)
        # parameter -> (lo, hi): only the elements [lo, hi) of it are stepped (state tensors stay full-size).  A hash table
        # partitioned by level over several GPUs: each rank steps the levels it keeps (mp_slam/sharded.py).
        self.slices = {}
        super().__init__(params, **kw)

    def _patch_step_function(self) -> None:
        # torch wraps Optimizer.step in a hook dispatcher + profiler range (~25 us per call, a quarter of a pose iteration's
        # host time here).  step() below runs un-wrapped and hands over to the wrapped torch path itself whenever a step
        # hook is registered, so hooks keep firing.
        self._zero_grad_profile_name = f"Optimizer.zero_grad#{self.__class__.__name__}.zero_grad"

    def _hooked(self) -> bool:
        from torch.optim import optimizer as _o
        return bool(self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks
                    or getattr(_o, "_global_optimizer_pre_hooks", None) or getattr(_o, "_global_optimizer_post_hooks", None))

    def _native(self) -> bool:
        if self.slices and not all(p.is_cuda for p in self.slices):
            raise _lib.RfxError("a sliced Adam step needs device parameters (there is no CPU path)")
        for g in self.param_groups:
            if g.get("amsgrad") or g.get("maximize") or g.get("capturable") or g.get("differentiable") or g.get("decoupled_weight_decay"):
                return False
            if isinstance(g["lr"], torch.Tensor):
                return False
            for p in g["params"]:
                if p.grad is None:
                    continue
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous() and p.grad.is_cuda
                        and p.grad.dtype == torch.float32 and p.grad.is_contiguous() and not p.grad.is_sparse):
                    return False
        return True

    def prepare(self):
        """create the state of every parameter now (zeros, step 0: what the first step() would create on its way) -- a stream's
        first mapper step then issues its optimizer steps as fast as every later one.  Parameters the native step cannot take
        (CPU tensors, other dtypes) are left to torch's own lazy initialisation."""
        for g in self.param_groups:
            if g.get("amsgrad") or g.get("capturable") or g.get("differentiable") or isinstance(g["lr"], torch.Tensor):
                continue
            for p in g["params"]:
                if not (p.is_cuda and p.dtype == torch.float32 and p.requires_grad):
                    continue
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                stp = st["step"]
                if not stp.is_cuda and stp.dtype == torch.float32 and p not in self._views:
                    self._views[p] = (stp, stp.numpy())

    def step(self, closure=None):
        if self._hooked():
            return torch.optim.Optimizer.profile_hook_step(type(self)._step_impl)(self, closure)
        out = self._step_impl(closure)
        self._optimizer_step_code()
        return out

    @torch.no_grad()
    def _step_impl(self, closure=None):
        loss = None
        if closure is not None:                 # first: the gradients it produces decide which implementation steps them
            with torch.enable_grad():
                loss = closure()
        if not self._native():
            if self.slices:
                # torch's Adam would step the WHOLE tensor: outside a rank's own range the gradient buffer is never written
                # (nor zeroed), so the other ranks' levels and their moments would be corrupted silently
                raise _lib.RfxError("Adam.slices is set (a level-partitioned table) but the native step is unavailable for this "
                                    "configuration (amsgrad / capturable / tensor lr / non-contiguous gradient): refusing to "
                                    "fall back to a step over the whole tensor")
            torch_step = torch.optim.Adam.step             # un-wrapped: step() above has dealt with the hooks already
            getattr(torch_step, "__wrapped__", torch_step)(self, None)
            return loss
        lib = _lib.load()
        per_device = {}
        for g in self.param_groups:
            b1, b2 = g["betas"]
            for p in g["params"]:
                if p.grad is None:
                    continue
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)         # host counter, like torch's default Adam
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                # `step` stays the host tensor torch's Adam keeps, but is bumped through a numpy view of it: a CPU-tensor
                # `+= 1` costs ~7 us per parameter, which added up to more host time than the launch itself
                stp = st["step"]
                ent = self._views.get(p)
                if ent is None or ent[0] is not stp:                             # fresh state, or one loaded from a checkpoint
                    if stp.is_cuda or stp.dtype != torch.float32:                # (e.g. saved by a fused / capturable Adam)
                        stp = st["step"] = stp.detach().to("cpu", torch.float32)
                    ent = self._views[p] = (stp, stp.numpy())
                k = int(ent[1].item()) + 1
                ent[1][...] = k
                bc1, bc2 = 1.0 - b1 ** k, 1.0 - b2 ** k
                lo, hi = self.slices.get(p, (0, p.numel()))
                o = 4 * lo
                t = _lib.AdamTensor(p.data_ptr() + o, p.grad.data_ptr() + o, st["exp_avg"].data_ptr() + o, st["exp_avg_sq"].data_ptr() + o,
                                    hi - lo, b1, b2, 1.0 - b1, 1.0 - b2, g["eps"], g["weight_decay"], -(g["lr"] / bc1), math.sqrt(bc2))
                per_device.setdefault(p.device, []).append(t)
        for dev, ts in per_device.items():
            stream = _lib.stream_ptr(dev)
            for i in range(0, len(ts), _lib.ADAM_MAX_TENSORS):
                part = ts[i:i + _lib.ADAM_MAX_TENSORS]
                arr = (_lib.AdamTensor * len(part))(*part)
                if torch.cuda.current_device() == dev.index:
                    _lib.check(lib.rfx_adam_step(arr, len(part), stream), "rfx_adam_step")
                else:
                    with torch.cuda.device(dev):
                        _lib.check(lib.rfx_adam_step(arr, len(part), stream), "rfx_adam_step")
        return loss


_capturing = torch._C._cuda_isCurrentStreamCapturing if hasattr(torch._C, "_cuda_isCurrentStreamCapturing") else (lambda: False)


def _same_memory_order(a, b):
    """whether two dense tensors of one shape hold element i of memory for the same place (a size-1 dimension's stride means nothing)"""
    return a.stride() == b.stride() or a.numel() == 0 or all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n != 1)


def _dense(t):
    """no element twice, no gap: any order of dimensions"""
    if t.is_contiguous():
        return True
    n = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != n:
            return False
        n *= size
    return True


def _overlaps_itself(t):
    return any(st == 0 and sz > 1 for st, sz in zip(t.stride(), t.shape))


class _on:
    """the device that a call's launches go to, as the current one"""
    __slots__ = ("guard",)

    def __init__(self, index):
        self.guard = None if torch._C._cuda_getDevice() == index else torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


def _check_grad(g):
    if g.layout is not torch.strided:
        raise _lib.RfxError("sparse gradients are not supported")
    if g.dtype not in _lib.DTYPES:
        raise _lib.RfxError(f"gradients of type {g.dtype} are not supported: float32, bfloat16 or float16")


def _grad_rows(grads):
    """rfx_grad_tensor descriptors of gradients of the known types"""
    return (_lib.GradTensor * len(grads))(*[_lib.GradTensor(g.data_ptr(), g.numel(), _lib.DTYPES[g.dtype], 0) for g in grads])


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ as two passes of librfx kernels: the norm N of all gradients together (2-norm, summed in
    fp64 in an order that depends on sizes only, or the largest magnitude with norm_type=inf), then every gradient times
    min(1, max_norm / (N + 1e-6)) in place -- nothing is written where that is 1.  Returns N, an fp32 scalar on the gradients'
    device; the host does not wait for it unless error_if_nonfinite asks (RuntimeError before anything is scaled).  A factor that is
    not finite is applied as it is: an infinite norm makes zeros (and NaN of what was infinite), a NaN makes NaN.  One device;
    float32 / bfloat16 / float16 gradients, mixed freely.  Gradients on the CPU take torch's own function, and only there does
    `foreach` (torch's choice between its own implementations) make a difference."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm, norm_type = float(max_norm), float(norm_type)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm has to be a number >= 0: {max_norm}")
    if parameters and parameters[0].is_cuda and not error_if_nonfinite and norm_type in (2.0, math.inf):
        index = torch._C._cuda_getDevice()
        out = _lib.host().clip(parameters, 2 if norm_type == 2.0 else 0, max_norm, index, _lib.stream_ptr(index))
        if isinstance(out, torch.Tensor):
            return out
        _lib.check(min(out, 0), "rfx_grad_clip")
    # what is left: no gradient, another device than the current one, gradients with gaps in memory, types and layouts to be refused
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if not any(g.is_cuda for g in grads):
        return torch.nn.utils.clip_grad_norm_(parameters, max_norm, norm_type, error_if_nonfinite, foreach)
    if norm_type not in (2.0, math.inf):
        raise _lib.RfxError(f"norm_type {norm_type}: only 2 and inf are supported")
    dev = grads[0].device
    for g in grads:
        _check_grad(g)
        if _overlaps_itself(g):
            raise _lib.RfxError("a gradient whose elements share memory (an expanded tensor) cannot be scaled in place")
        if g.device != dev:
            raise _lib.RfxError("gradients on different devices: clip them device by device")
    flat = [g if _dense(g) else g.contiguous() for g in grads]
    lib, rows, n, kind = _lib.load(), _grad_rows(flat), len(flat), 2 if norm_type == 2.0 else 0
    with _on(dev.index), torch.no_grad():
        stream = _lib.stream_ptr(dev)
        ws_bytes = lib.rfx_grad_norm_workspace_bytes(n)
        ws = torch.empty(2 + ws_bytes // 8, dtype=torch.float64, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        clip = ws.data_ptr()
        _lib.check(lib.rfx_grad_norm(rows, n, kind, max_norm, clip, norm.data_ptr(), clip + 16, ws_bytes, stream), "rfx_grad_norm")
        if error_if_nonfinite and not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the norm of the gradients is not finite ({float(norm)}), so they cannot be clipped")
        _lib.check(lib.rfx_grad_scale(rows, n, clip, stream), "rfx_grad_scale")
        for g, f in zip(grads, flat):
            if f is not g:
                g.copy_(f)
    return norm


class AdamW(torch.optim.AdamW):
    """torch.optim.AdamW (decoupled weight decay) whose step is one librfx call over all tensors.  Device parameters in float32,
    bfloat16 or float16; on the CPU torch's own step runs (32-bit moments, no clipping).  Moments are fp32 whatever the parameter's
    type: state[p] = {"step", "exp_avg", "exp_avg_sq"}.  Beyond torch's arguments, the first three also per parameter group:

    state_bits      32, or 8: moments of one byte under an exponent per 256 elements (include/rfx.h has the format), a quarter of the
                    memory and 16 instead of 28 bytes of traffic per fp32 parameter; state[p] holds uint8 "exp_avg", "exp_avg_sq" and
                    int8 "exponents" [2, ceil(n / 256)].  Rounded stochastically from a hash of (seed, step, parameter, element): the same
                    run gives the same bits.  A value that is not finite makes its 256 neighbours NaN at the next step.
    master_weights  bfloat16 / float16 parameters are stepped in an fp32 copy, state[p]["master"], and rounded once.  What writes the
                    parameter otherwise has to write that copy, too (or remove it: the next step makes it from the parameter).
    seed            of the 8-bit roundings.
    max_grad_norm   scale the gradients by min(1, max_grad_norm / (N + 1e-6)), N their global 2-norm, on the way into the moments: the
                    gradients themselves stay as they are.  `grad_norm` is N of the last step (fp32 scalar on the device; None where
                    it had no limit or no gradient).
    capturable      the step count lives on the device and lr may be a device scalar: step() can be captured into a graph (after one
                    step or prepare(), which create the state).  Without it a capture is refused.

    moments() gives the moments as fp32 tensors.  amsgrad, differentiable and decoupled_weight_decay=False are refused (ValueError) however
    a group comes by them: on construction, joining, loading, or set in place and stepped."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *, maximize=False,
                 capturable=False, state_bits=32, master_weights=False, seed=0, max_grad_norm=None, differentiable=False,
                 foreach=None, fused=None):
        if amsgrad or differentiable:
            raise ValueError("remixfusion_amd.optim.AdamW has no amsgrad and no differentiable step")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("a tensor lr needs capturable=True")
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError(f"max_grad_norm has to be None or a number >= 0: {max_grad_norm}")
        self._own = {"state_bits": state_bits, "master_weights": master_weights, "seed": seed}
        self._reset()
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize, capturable=capturable)
        self.defaults.update(self._own, max_grad_norm=None if max_grad_norm is None else float(max_grad_norm))

    def _reset(self):
        self._plans, self.grad_norm = {}, None

    _patch_step_function = Adam._patch_step_function

    def _hooked(self):
        o = _torch_optimizer
        return bool(self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks
                    or o._global_optimizer_pre_hooks or o._global_optimizer_post_hooks)

    @property
    def max_grad_norm(self):
        return self.defaults["max_grad_norm"]

    @max_grad_norm.setter
    def max_grad_norm(self, value):
        if value is not None and not float(value) >= 0.0:
            raise ValueError(f"max_grad_norm has to be None or a number >= 0: {value}")
        self.defaults["max_grad_norm"] = None if value is None else float(value)

    @staticmethod
    def _check_group(group):
        for key in ("amsgrad", "differentiable"):
            if group.get(key):
                raise ValueError(f"remixfusion_amd.optim.AdamW has no {key}")
        if not group.get("decoupled_weight_decay", True):
            raise ValueError("remixfusion_amd.optim.AdamW decays weights apart from the gradient only")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits is 32 or 8: {group['state_bits']}")
        if group["seed"] != int(group["seed"]) or not 0 <= group["seed"] < 1 << 32:
            raise ValueError(f"seed is a whole number of 32 bits: {group['seed']}")

    def add_param_group(self, group):
        own = self._own
        for key, value in own.items():
            group.setdefault(key, value)
        self._check_group(group)
        super().add_param_group(group)
        ids = [id(p) for p in self.param_groups[-1]["params"]]
        if len(set(ids)) != len(ids):
            self.param_groups.pop()
            raise ValueError("a parameter stands twice in a group")

    def __setstate__(self, state):
        super().__setstate__(state)
        if "max_grad_norm" in self.defaults:                 # a copy or an unpickled optimizer: only the three dicts came along
            self._own = {k: self.defaults[k] for k in ("state_bits", "master_weights", "seed")}
        self._reset()
        for g in self.param_groups:
            for k, v in self._own.items():
                g.setdefault(k, v)

    # ---- state ------------------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """as torch's, but moments and master weights keep their own types (torch casts them to the parameter's); a dict of
        torch.optim.AdamW fits groups with 32-bit moments"""
        held = ("exp_avg", "exp_avg_sq", "exponents", "master")
        seen, mine = [], [{k: g[k] for k in self._own} for g in self.param_groups]

        def without_held(opt, d):                            # the last of the hooks: what it keeps from torch is put in below
            seen.append(d)
            for g, own in zip(d["param_groups"], mine):
                self._check_group({**own, **g, "decoupled_weight_decay": True})       # (as torch's AdamW: a dict of Adam fits)
            return {**d, "state": {i: {k: v for k, v in st.items() if k not in held} if isinstance(st, dict) else st
                                   for i, st in d["state"].items()}}

        hook = self.register_load_state_dict_pre_hook(without_held)
        before = self.state, self.param_groups, self._plans, self.grad_norm
        try:
            super().load_state_dict(state_dict)
            for g, saved, old in zip(self.param_groups, seen[0]["param_groups"], mine):
                g.update({k: v for k, v in old.items() if k not in saved})
                for i, p in zip(saved["params"], g["params"]):
                    st = seen[0]["state"].get(i)
                    if st:
                        self._take(p, g, {k: st[k] for k in held if k in st})
            parted = set()
            for p in (p for g in self.param_groups for p in g["params"] if p.is_cuda and self.state.get(p)):
                self._part(self.state[p], parted)
        except Exception:                                    # taken whole or not at all
            self.state, self.param_groups, self._plans, self.grad_norm = before
            raise
        finally:
            hook.remove()

    def _take(self, p, g, held):
        """the part of a loaded state that torch's loading was not to see"""
        st = self.state[p]
        st.update({k: t.to(device=p.device) for k, t in held.items()})
        if isinstance(st.get("step"), torch.Tensor):
            st["step"] = st["step"].detach().clone()         # (raised in place: not in the dict that was given)
        if p.is_cuda:
            self._check_state(p, g)
        elif p.is_floating_point():                          # (torch's step on the CPU wants them in the parameter's type)
            st.update({k: held[k].to(p) for k in ("exp_avg", "exp_avg_sq") if k in held and held[k].is_floating_point()})

    def _check_state(self, p, g):
        """brings a state that came from outside to the types and the memory order a step needs, or refuses it"""
        st, eight = self.state[p], g["state_bits"] == 8
        missing = [k for k in ("step", "exp_avg", "exp_avg_sq") + (("exponents",) if eight else ()) if k not in st]
        if missing:
            raise _lib.RfxError(f"the state of a parameter lacks {', '.join(missing)}")
        order = p if _dense(p) else None                     # whose memory order the state has
        for key in ("exp_avg", "exp_avg_sq"):
            t = st[key]
            if tuple(t.shape) != tuple(p.shape) or not t.is_cuda or t.device != p.device:
                raise _lib.RfxError(f"{key} of shape {tuple(t.shape)} on {t.device} for a parameter of shape {tuple(p.shape)} on {p.device}")
            if (t.dtype == torch.uint8) != eight:
                raise _lib.RfxError(f"{key} of type {t.dtype} for a group with state_bits={g['state_bits']}: moments are not converted on the way in")
            if order is None and _dense(t):                  # (8 bits: the exponents are those of its runs)
                order = t
            fits = _dense(t) and (_same_memory_order(t, order) if order is not None else t.is_contiguous())
            if eight:
                if not fits:
                    raise _lib.RfxError(f"8-bit {key} with strides {tuple(t.stride())} for a parameter with {tuple(p.stride())}: its "
                                        "exponents belong to runs of another memory order")
                if t.data_ptr() & 3:
                    st[key] = t.clone()
            elif not fits or t.dtype != torch.float32:
                st[key] = torch.empty_like(t.contiguous() if order is None else order, dtype=torch.float32).copy_(t)
            order = st[key] if order is None else order
        if eight:
            e = st["exponents"]
            if e.dtype != torch.int8 or tuple(e.shape) != (2, -(-p.numel() // _lib.ADAMW_BLOCK)) or e.device != p.device:
                raise _lib.RfxError(f"exponents of type {e.dtype}, shape {tuple(e.shape)} on {e.device}: int8 [2, {-(-p.numel() // _lib.ADAMW_BLOCK)}] is needed")
            st["exponents"] = e.contiguous()
        step, at = st["step"], p.device if g["capturable"] else torch.device("cpu")
        if not isinstance(step, torch.Tensor) or step.device != at or step.dtype != torch.float32 or step.numel() != 1:
            if torch.cuda.is_current_stream_capturing():
                raise _lib.RfxError("the step count is not where a captured step needs it: call step() or prepare() before capturing")
            st["step"] = torch.as_tensor(step, dtype=torch.float32).detach().reshape(()).to(at)
        if g["master_weights"] and p.dtype != torch.float32:
            w = st.get("master")
            if w is None or tuple(w.shape) != tuple(p.shape) or w.dtype != torch.float32 or w.device != p.device or not (
                    _dense(w) and _same_memory_order(w, st["exp_avg"])):
                if w is not None and tuple(w.shape) != tuple(p.shape):
                    raise _lib.RfxError(f"master of shape {tuple(w.shape)} for a parameter of shape {tuple(p.shape)}")
                st["master"] = torch.empty_like(st["exp_avg"], dtype=torch.float32).copy_(p if w is None else w)
        else:
            st.pop("master", None)                           # steps without it leave it behind the parameter

    def _new_state(self, p, g):
        st = self.state[p]
        st["step"] = torch.zeros((), dtype=torch.float32, device=p.device if g["capturable"] else "cpu")
        kind = torch.uint8 if g["state_bits"] == 8 else torch.float32
        st["exp_avg"] = torch.zeros_like(p, dtype=kind, memory_format=torch.preserve_format)
        st["exp_avg_sq"] = torch.zeros_like(st["exp_avg"])
        if g["state_bits"] == 8:                              # the exponent of a run of zeros is the least one
            st["exponents"] = torch.full((2, -(-p.numel() // _lib.ADAMW_BLOCK)), -127, dtype=torch.int8, device=p.device)
        if g["master_weights"] and p.dtype != torch.float32:
            st["master"] = torch.empty_like(st["exp_avg"], dtype=torch.float32).copy_(p)

    @torch.no_grad()
    def prepare(self):
        """create the state of every device parameter now (what the first step() would do on its way); needed before a step is
        captured into a graph"""
        every = [(p, i, gi) for i, (gi, p) in enumerate((gi, p) for gi, g in enumerate(self.param_groups) for p in g["params"])
                 if p.is_cuda and p.requires_grad]
        if every:
            self._build(every)

    def moments(self):
        """(exp_avg, exp_avg_sq) of all parameters, in their order, as fp32 tensors: the state's own tensors where moments are held
        in 32 bits, the values of the codes where in 8 (on a device), zeros where there is no state yet"""
        codes = [st["exp_avg"] for st in self.state.values() if st and st["exp_avg"].dtype is torch.uint8]
        if not codes:                                            # nothing to launch
            return _lib.host().moments(self.param_groups, self.state, -1, 0)
        if not codes[0].is_cuda:
            raise _lib.RfxError("8-bit moments are read on a device: there is no CPU path")
        index = codes[0].get_device()
        with _on(index):
            out = _lib.host().moments(self.param_groups, self.state, index, _lib.stream_ptr(index))
        if isinstance(out, int):
            _lib.check(min(out, 0), "rfx_adamw_moments")
            raise _lib.RfxError("8-bit moments on several devices: one optimizer per device reads its own")
        return out

    # ---- the step ---------------------------------------------------------------------------------------------------------
    @staticmethod
    def _tensors(st):
        """(key, tensor) of what a step writes of a state"""
        return [(k, st[k]) for k in ("step", "exp_avg", "exp_avg_sq", "exponents", "master") if isinstance(st.get(k), torch.Tensor) and st[k].numel()]

    def _part(self, st, held):
        """a state whose tensors are none of those held already: each parameter writes its own"""
        for key, t in self._tensors(st):
            if t.data_ptr() in held:
                st[key] = t = t.clone()
            held.add(t.data_ptr())

    def _as_captured(self, p, g, held):
        """refuses a state that this step would have to make or bring over: every replay would do it again"""
        st = self.state.get(p)
        if not st:
            raise _lib.RfxError("the state is created by the first step() or prepare(): call it before capturing")
        before = dict(st)
        try:
            self._check_state(p, g)
            self._part(st, held)
            if any(t is not before.get(key) for key, t in st.items()):
                raise _lib.RfxError("the state is not as a captured step needs it: call step() or prepare() before capturing")
        except _lib.RfxError:
            st.clear()
            st.update(before)
            raise

    def _build(self, every):
        """plans for (parameter, its place in the optimizer, its group): states made or checked, one plan per device"""
        capturing = torch.cuda.is_current_stream_capturing()
        stepped = {p for p, _, _ in every}
        by_device = {}
        held = {t.data_ptr() for p, st in self.state.items() if p not in stepped and isinstance(st, dict) for _, t in self._tensors(st)}
        for g in self.param_groups:                           # (whose settings may have been changed in place)
            self._check_group(g)
        for entry in every:
            p, _, gi = entry
            g = self.param_groups[gi]
            by_device.setdefault(p.device, []).append(entry)
            if not p.is_cuda:
                raise _lib.RfxError("parameters on the CPU and on a device in one optimizer are not supported")
            if p.dtype not in _lib.DTYPES:
                raise _lib.RfxError(f"parameters of type {p.dtype} are not supported: float32, bfloat16 or float16")
            if p.layout is not torch.strided or _overlaps_itself(p):
                raise _lib.RfxError("a parameter whose elements share memory (an expanded tensor) or that is sparse is not supported")
            if capturing:
                self._as_captured(p, g, held)
                continue
            if self.state.get(p):
                self._check_state(p, g)
            else:
                self._new_state(p, g)
            self._part(self.state[p], held)
        self._plans = {dev: (_lib.host().Plan(part, self.param_groups, self.state), part) for dev, part in by_device.items()}

    def step(self, closure=None):
        if self._hooked():
            return torch.optim.Optimizer.profile_hook_step(type(self)._step_impl)(self, closure)
        out = self._step_impl(closure)
        self._optimizer_step_code()
        return out

    def _step_impl(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        limit = self.defaults["max_grad_norm"]
        other = False
        if len(self._plans) == 1:
            for dev, (plan, _) in self._plans.items():
                with _on(dev.index):
                    if _capturing() and plan.host_counted:
                        raise _lib.RfxError("a step without capturable=True cannot be captured: its step count would stand still")
                    out = plan.step(self.param_groups, self.state, -1.0 if limit is None else limit, _lib.stream_ptr(dev.index))
                if self._took(out):
                    return loss
                other = out == _lib.host().OTHER_ORDER
        params = [p for g in self.param_groups for p in g["params"] if p.grad is not None]
        if not params:
            self.grad_norm = None
            return loss
        if not any(p.is_cuda for p in params):
            self._cpu_step()
            return loss
        # nothing planned yet, or something is not as planned; other devices than the current one; gradients in another memory order
        with torch.no_grad():
            if not other:
                self._build([(p, i, gi) for i, (gi, p) in enumerate((gi, p) for gi, g in enumerate(self.param_groups) for p in g["params"])
                             if p.grad is not None])
            if limit is not None and len(self._plans) > 1:
                raise _lib.RfxError("max_grad_norm needs all parameters on one device")
            for dev, (plan, part) in self._plans.items():
                with _on(dev.index):
                    if _capturing() and plan.host_counted:
                        raise _lib.RfxError("a step without capturable=True cannot be captured: its step count would stand still")
                    stepped, grads = self._in_order([p for p, _, _ in part])
                    self._took(plan.launch(stepped, grads, self.param_groups, -1.0 if limit is None else limit, _lib.stream_ptr(dev)))
                    for (p, _, _), x in zip(part, stepped):
                        if x is not p:
                            p.copy_(x)
        return loss

    def _took(self, out):
        """a plan's answer: the gradients' norm or None, or the number that says why not"""
        if isinstance(out, int):
            _lib.check(min(out, 0), "rfx_adamw_step")
            return False
        self.grad_norm = out
        return True

    def _cpu_step(self):
        for g in self.param_groups:
            self._check_group(g)
        if self.max_grad_norm is not None or any(g["state_bits"] != 32 or g["master_weights"] for g in self.param_groups):
            raise _lib.RfxError("8-bit moments, master weights and max_grad_norm need device parameters: there is no CPU path")
        torch_step = torch.optim.AdamW.step
        with torch.no_grad():
            getattr(torch_step, "__wrapped__", torch_step)(self, None)

    def _in_order(self, params):
        """parameters and gradients in the memory order of their moments: themselves where they are, copies where not"""
        stepped, grads = [], []
        for p in params:
            g, m = p.grad, self.state[p]["exp_avg"]
            _check_grad(g)
            if g.dtype != p.dtype or g.shape != p.shape or g.device != p.device:
                raise _lib.RfxError(f"a gradient of type {g.dtype}, shape {tuple(g.shape)} on {g.device} for a parameter of type {p.dtype}, "
                                    f"shape {tuple(p.shape)} on {p.device}")
            stepped.append(p if _same_memory_order(p, m) else torch.empty_like(m, dtype=p.dtype).copy_(p))
            grads.append(g if _same_memory_order(g, m) else torch.empty_like(m, dtype=g.dtype).copy_(g))
        return stepped, grads
