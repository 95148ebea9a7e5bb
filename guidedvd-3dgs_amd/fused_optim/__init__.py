"""The optimizer step of a training iteration in one launch, beside the fused image losses:

    from fused_optim import FusedAdamW
    optimizer = FusedAdamW(param_groups, lr=0.0, eps=1e-15, weight_decay=0.0)       # where the trainer has torch.optim.Adam(param_groups, ...)

`FusedAdamW` is a `torch.optim.Optimizer` with AdamW's rule (Adam's where weight_decay is 0) over all tensors of a parameter type at once
(csrc/adamw.hip, C-ABI include/gvd_optim.h).  With state_bits=32 its state has the names, shapes and types of torch.optim.Adam's ("step", "exp_avg",
"exp_avg_sq"), so code that edits the moments when Gaussians are added or removed works as it is, and state dicts go both ways.  With
state_bits=8 the moments take 2 bytes an element instead of 8; `moments` / `set_moments` read and write them as floats.  No CPU path: CPU
parameters raise.
"""
import ctypes
import importlib.util
import math
import os

import torch
from torch.optim.optimizer import _global_optimizer_post_hooks as _every_post_hook, _global_optimizer_pre_hooks as _every_pre_hook

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.environ.get("GVD_OPTIM_LIB") or os.path.join(os.path.dirname(_HERE), "lib", "libgvd_optim.so")  # env: A/B builds
_EXT_PATH = os.path.join(os.path.dirname(_HERE), "lib", "_gvd_optim_torch.so")
_LIB = _EXT = None
BLOCK = 256                                 # GVD_ADAMW_BLOCK: elements that share a scale where moments are held in 8 bits
TINY = 2.0 ** -110                          # a block whose largest magnitude is below this is held as zeros (448 over it would overflow), as in the kernel


def lib():
    global _LIB
    if _LIB is None:
        if not os.path.exists(_LIB_PATH):
            raise RuntimeError(f"{_LIB_PATH} is missing: build the HIP extensions first "
                               f"(python -c 'import __graft_entry__ as g; g.build()')")
        L = ctypes.CDLL(_LIB_PATH)
        L.gvd_optim_last_error.restype = ctypes.c_char_p
        L.gvd_adamw_key.restype = ctypes.c_uint
        L.gvd_adamw_key.argtypes = [ctypes.c_uint] * 3
        _LIB = L
    return _LIB


def ext():
    """The compiled host half of the step (csrc/optim_torch_ext.cpp) over the same library instance."""
    global _EXT
    if _EXT is None:
        lib()
        if not os.path.exists(_EXT_PATH):
            raise RuntimeError(f"{_EXT_PATH} is missing: build the extensions first (python -c 'import __graft_entry__ as g; g.build()')")
        spec = importlib.util.spec_from_file_location("_gvd_optim_torch", _EXT_PATH)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.init(_LIB_PATH)
        _EXT = mod
    return _EXT


def _dense(t):
    """Whether t's elements fill one piece of memory, in whatever order."""
    return t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t)


def _like(t, dtype):
    """Zeros in t's shape and memory order."""
    if dtype == torch.float32:
        return torch.zeros_like(t, dtype=dtype, memory_format=torch.preserve_format)
    return torch.zeros_like(t, dtype=torch.uint8, memory_format=torch.preserve_format).view(dtype)


def _same_order(a, b):
    """Whether two tensors of one shape lie in the same memory order: the strides of dimensions of size 1 do not count."""
    return a.numel() <= 1 or all(x == y for n, x, y in zip(a.shape, a.stride(), b.stride()) if n != 1)


def _in_order(t):
    """t's elements as one row, in the order of memory (a view)."""
    return t.as_strided((t.numel(),), (1,))


class FusedAdamW(torch.optim.Optimizer):
    """AdamW over all tensors at once:

        m = m + (1 - beta1) (g - m),   v = beta2 v + (1 - beta2) g^2
        p = (1 - lr weight_decay) p - lr / (1 - beta1^t)  m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    in 32 bits, rounded once to the parameter's type.  Parameters: float32, float16 or bfloat16 on a ROCm device, dense (any memory
    order); gradients of the same type, shape and device (another memory order is copied).  Every argument may differ by parameter group.  Parameters, states
    and gradients must not share memory (a gradient may belong to several parameters, or be its own parameter): step() refuses them.  What it refuses
    it refuses before anything is counted or launched.

    state_bits   32, or 8: m and sqrt(v) as e4m3 with one float scale per 256 elements, rounded stochastically from a hash of (seed, the
                 parameter's place among all of the optimizer's, step, element) -- unbiased, and the same run gives the same result.  State:
                 "exp_avg", "exp_avg_rms" (float8_e4m3fn), "exp_avg_scale", "exp_avg_rms_scale".
    capturable   the count of steps is held on the device ("step": float32 there), and step() may be captured into a graph, where every replay is
                 the next step; lr may be a float32 tensor of one element on the parameters' device, read at each replay.  Run one eager step
                 first: state cannot be set up while capturing.  Without it step() raises in a capture: the count would be frozen.  A replay leaves the
                 parameters' version counters as they are: after replays, `lvdm_amd.conv.invalidate_packed` for modules whose images are cached."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, seed=0, capturable=False):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed,
                                      capturable=capturable))

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_group(g)
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        if torch.is_tensor(lr):
            if not g["capturable"]:
                raise ValueError("FusedAdamW: lr may be a tensor with capturable=True only (reading it would wait for the device)")
            if lr.dtype != torch.float32 or lr.numel() != 1 or not lr.is_cuda:
                raise ValueError("FusedAdamW: a tensor lr is one float32 on the parameters' device")
        elif not (lr >= 0.0 and math.isfinite(lr)):
            raise ValueError(f"FusedAdamW: invalid learning rate {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"FusedAdamW: invalid betas {(b1, b2)}")
        if not (g["eps"] >= 0.0 and math.isfinite(g["eps"])):
            raise ValueError(f"FusedAdamW: invalid eps {g['eps']}")
        if not (g["weight_decay"] >= 0.0 and math.isfinite(g["weight_decay"])):
            raise ValueError(f"FusedAdamW: invalid weight_decay {g['weight_decay']}")
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits must be 8 or 32, not {g['state_bits']}")
        if not 0 <= g["seed"] < 2 ** 32:
            raise ValueError("FusedAdamW: seed is a whole number of 32 bits")
        if len({id(p) for p in g["params"]}) != len(g["params"]):
            raise ValueError("FusedAdamW: a parameter appears twice in a group")

    # ---- state -------------------------------------------------------------------------------------------------------------
    def _new_state(self, p, group):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():      # (zeros that only a replay would write)
            raise RuntimeError("FusedAdamW: run one step before capturing (its state cannot be set up while capturing), with capturable=True")
        st = dict(step=torch.zeros((), dtype=torch.float32, device=p.device if group["capturable"] else "cpu"))
        if group["state_bits"] == 32:
            st.update(exp_avg=_like(p, torch.float32), exp_avg_sq=_like(p, torch.float32))
        else:
            scales = lambda: torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)  # noqa: E731
            st.update(exp_avg=_like(p, torch.float8_e4m3fn), exp_avg_rms=_like(p, torch.float8_e4m3fn),
                      exp_avg_scale=scales(), exp_avg_rms_scale=scales())
        return st

    def _check_state(self, p, st, bits):
        names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "exp_avg_rms")
        dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
        for n in names:
            t = st.get(n)
            if t is None or t.dtype != dtype or t.shape != p.shape or t.device != p.device or not _same_order(t, p):
                raise RuntimeError(f"FusedAdamW: the state {n!r} does not fit its parameter {tuple(p.shape)} (state_bits={bits}): it takes {dtype} in the "
                                   f"parameter's shape, device and memory order; got "
                                   f"{None if t is None else (t.dtype, tuple(t.shape), t.stride(), str(t.device))}")
        if bits == 8:
            for n in ("exp_avg_scale", "exp_avg_rms_scale"):
                t = st.get(n)
                if t is None or t.dtype != torch.float32 or t.shape != (-(-p.numel() // BLOCK),) or t.device != p.device or not t.is_contiguous():
                    raise RuntimeError(f"FusedAdamW: the state {n!r} does not fit its parameter {tuple(p.shape)}")

    def moments(self, p):
        """(first moment, second moment) of a parameter as float32 in its shape: copies, or the state's own tensors with 32-bit state; None before
        its first step."""
        st = self.state.get(p)
        if not st:
            return None
        if "exp_avg_sq" in st:
            return st["exp_avg"], st["exp_avg_sq"]

        def wide(codes, scale):
            x = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            _in_order(x).copy_(_in_order(codes).float() * scale.repeat_interleave(BLOCK)[:p.numel()])
            return x
        return wide(st["exp_avg"], st["exp_avg_scale"]), wide(st["exp_avg_rms"], st["exp_avg_rms_scale"]).square_()

    @torch.no_grad()
    def set_moments(self, p, exp_avg, exp_avg_sq, step=None):
        """Gives a parameter of this optimizer its moments (any floating type, its shape), in the form its group holds them; `step`: the count of steps
        behind them (default: what its state says, or 0).  After rows were added to or removed from a parameter:

            m, v = opt.moments(old);  t = opt.state.pop(old)["step"];  group["params"][i] = new;  opt.set_moments(new, m[keep], v[keep], t)

        Eight-bit moments are rounded to the nearest here."""
        group = next((g for g in self.param_groups if any(q is p for q in g["params"])), None)
        if group is None:
            raise ValueError("FusedAdamW.set_moments: not a parameter of this optimizer")
        if exp_avg.shape != p.shape or exp_avg_sq.shape != p.shape:
            raise ValueError(f"FusedAdamW.set_moments: moments of shape {tuple(exp_avg.shape)}, {tuple(exp_avg_sq.shape)} for a parameter of {tuple(p.shape)}")
        old = self.state.get(p) or {}
        st = self._new_state(p, group)
        if step is None:
            step = old.get("step", 0.0)
        st["step"].copy_(torch.as_tensor(step, dtype=torch.float32))
        if group["state_bits"] == 32:
            st["exp_avg"].copy_(exp_avg)
            st["exp_avg_sq"].copy_(exp_avg_sq)
        else:
            if not _dense(p):
                raise RuntimeError("FusedAdamW: parameters must be dense")
            for x, codes, scales in ((exp_avg.float(), st["exp_avg"], st["exp_avg_scale"]),
                                     (exp_avg_sq.float().sqrt(), st["exp_avg_rms"], st["exp_avg_rms_scale"])):
                row = torch.zeros(scales.numel() * BLOCK, dtype=torch.float32, device=p.device)
                ordered = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(x)
                row[:p.numel()] = _in_order(ordered)
                row = row.view(-1, BLOCK)
                finite = row.isfinite()                   # (what is not is held as e4m3's NaN and leaves its block as it is, as in the kernel)
                big = torch.where(finite, row.abs(), 0.0).amax(1)
                big = torch.where(big < TINY, 0.0, big)
                scales.copy_(big / 448.0)
                q = torch.where(big[:, None] > 0, row * (448.0 / big[:, None]), 0.0).masked_fill(~finite, float("nan"))
                if codes is st["exp_avg_rms"]:
                    q = torch.where(row > 0, q.clamp(min=2.0 ** -9), q)      # a root above 0 is never held as 0
                _in_order(codes.view(torch.uint8)).copy_(q.to(torch.float8_e4m3fn).view(torch.uint8).view(-1)[:p.numel()])
        self.state[p] = st

    def load_state_dict(self, state_dict):
        """Like torch's, but the state keeps the types it was saved with (torch casts it to the parameter's).  A refused one leaves the optimizer as it was."""
        before = self.state, self.param_groups           # (torch puts others in their place)
        try:
            self._load_state_dict(state_dict)
        except Exception:
            self.state, self.param_groups = before
            raise

    def _load_state_dict(self, state_dict):
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        super().load_state_dict(state_dict)
        for g in self.param_groups:
            for k, d in self.defaults.items():      # groups saved by torch.optim.Adam / AdamW lack this optimizer's own entries
                g.setdefault(k, d)
            if g.get("amsgrad") or g.get("maximize") or g["weight_decay"] and g.get("decoupled_weight_decay") is False:
                raise ValueError("FusedAdamW: the saved optimizer has another rule (amsgrad, maximize, or weight decay that is not decoupled)")
            self._check_group(g)
        params = [(p, g) for g in self.param_groups for p in g["params"]]
        for i, (p, g) in zip(saved, params):
            src = state_dict["state"].get(i)
            if src is None:
                continue
            st = self.state[p]
            for k, v in src.items():
                if torch.is_tensor(v) and k != "step":
                    st[k] = v.detach().to(device=p.device, copy=True)
                    if v.dtype == torch.float32 and v.shape == p.shape and not _same_order(st[k], p):
                        st[k] = _like(p, torch.float32).copy_(v)
            step = torch.as_tensor(src["step"], dtype=torch.float32).detach()
            st["step"] = step.to(device=p.device if g["capturable"] else "cpu", copy=True).reshape(())
            self._check_state(p, st, g["state_bits"])

    # ---- the step ----------------------------------------------------------------------------------------------------------
    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ext().step(self, self.param_groups, self.state)
        return loss

    # torch.optim.Optimizer wraps the step of its classes in a profiler's range and the calls of registered hooks: 6 us where there is neither, as much as all else that the
    # host does for four small tensors.  So the wrapped step is called where one of them is there.
    _wrapped_step = torch.optim.Optimizer.profile_hook_step(_step)

    def step(self, closure=None):
        """One step of every parameter that has a gradient, on the current stream of each parameter's device; nothing waits for the device."""
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _every_pre_hook or _every_post_hook or torch.autograd._profiler_enabled()):
            return self._wrapped_step(closure)
        return self._step(closure)

    step.hooked = True      # (the base class leaves it as it is)
