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
import math
import os
import struct

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.environ.get("GVD_OPTIM_LIB") or os.path.join(os.path.dirname(_HERE), "lib", "libgvd_optim.so")  # env: A/B builds
_LIB = None
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TENSOR = struct.Struct("6Qq3fI")          # gvd_adamw_tensor
BLOCK = 256                                 # GVD_ADAMW_BLOCK: elements that share a scale where moments are held in 8 bits


class _Noop:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_NOOP = _Noop()


def _on(dev):
    """Device guard that is free when `dev` is already the current device (torch.cuda.device() costs ~25 us per use)."""
    idx = dev.index
    return _NOOP if idx is None or idx == torch.cuda.current_device() else torch.cuda.device(dev)


_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    if _RAW_STREAM is not None:
        return _RAW_STREAM(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


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
        L.gvd_adamw_step.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.c_int] + [ctypes.c_double] * 3 + [ctypes.c_void_p] * 2
        _LIB = L
    return _LIB


def _check(rc):
    if rc != 0:
        raise RuntimeError(f"gvd_optim error {rc}: {lib().gvd_optim_last_error().decode()}")


def _dense(t):
    """Whether t's elements fill one piece of memory, in whatever order."""
    return t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t)


def _like(t, dtype):
    """Zeros in t's shape and memory order."""
    if dtype == torch.float32:
        return torch.zeros_like(t, dtype=dtype, memory_format=torch.preserve_format)
    return torch.zeros_like(t, dtype=torch.uint8, memory_format=torch.preserve_format).view(dtype)


def _in_order(t):
    """t's elements as one row, in the order of memory (a view)."""
    return t.as_strided((t.numel(),), (1,))


class FusedAdamW(torch.optim.Optimizer):
    """AdamW over all tensors at once:

        m = m + (1 - beta1) (g - m),   v = beta2 v + (1 - beta2) g^2
        p = (1 - lr weight_decay) p - lr / (1 - beta1^t)  m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    in 32 bits, rounded once to the parameter's type.  Parameters: float32, float16 or bfloat16 on a ROCm device, dense (any memory
    order); gradients of the same type, shape and device (another memory order is copied).  Every argument may differ by parameter group.

    state_bits   32, or 8: m and sqrt(v) as e4m3 with one float scale per 256 elements, rounded stochastically from a hash of (seed, the
                 parameter's place among all of the optimizer's, step, element) -- unbiased, and the same run gives the same result.  State:
                 "exp_avg", "exp_avg_rms" (float8_e4m3fn), "exp_avg_scale", "exp_avg_rms_scale".
    capturable   the count of steps is held on the device ("step": float32 there), and step() may be captured into a graph, where every replay is
                 the next step; lr may be a float32 tensor of one element on the parameters' device, read at each replay.  Run one eager step
                 first: state cannot be set up while capturing.  Without it step() raises in a capture: the count would be frozen."""

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
        if group["capturable"] and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: run one step before capturing (its state cannot be set up while capturing)")
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
            if t is None or t.dtype != dtype or t.shape != p.shape or t.device != p.device or t.stride() != p.stride() and p.numel() > 1:
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
                big = row.abs().amax(1)
                scales.copy_(big / 448.0)
                q = torch.where(big[:, None] > 0, row * (448.0 / big[:, None]), 0.0)
                if codes is st["exp_avg_rms"]:
                    q = torch.where(row > 0, q.clamp(min=2.0 ** -9), q)      # a root above 0 is never held as 0
                _in_order(codes.view(torch.uint8)).copy_(q.to(torch.float8_e4m3fn).view(torch.uint8).view(-1)[:p.numel()])
        self.state[p] = st

    def load_state_dict(self, state_dict):
        """Like torch's, but the state keeps the types it was saved with (torch casts it to the parameter's)."""
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        super().load_state_dict(state_dict)
        for g in self.param_groups:
            for k, d in self.defaults.items():      # groups saved by torch.optim.Adam / AdamW lack this optimizer's own entries
                g.setdefault(k, d)
        params = [(p, g) for g in self.param_groups for p in g["params"]]
        for i, (p, g) in zip(saved, params):
            src = state_dict["state"].get(i)
            if src is None:
                continue
            st = self.state[p]
            for k, v in src.items():
                if torch.is_tensor(v) and k != "step":
                    st[k] = v.detach().to(device=p.device, copy=True)
            step = torch.as_tensor(src["step"], dtype=torch.float32).detach()
            st["step"] = step.to(device=p.device if g["capturable"] else "cpu", copy=True).reshape(())
            self._check_state(p, st, g["state_bits"])

    # ---- the step ----------------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter that has a gradient, on the current stream of each parameter's device; nothing waits for the device."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        launches, place = {}, -1
        for g in self.param_groups:
            common = None
            for p in g["params"]:
                place += 1
                if p.grad is None:
                    continue
                grad = self._gradient(p)
                st = self.state[p]
                if not st:
                    st.update(self._new_state(p, g))
                if common is None:
                    (b1, b2), bits, capturable = g["betas"], g["state_bits"], bool(g["capturable"])
                    common = (float(b1), float(b2), float(g["eps"]), bits, capturable, g["seed"] if bits == 8 or capturable else 0)
                self._check_state(p, st, common[3])
                launches.setdefault((p.device, p.dtype) + common, []).append((p, grad, st, g, place))
        for (device, dtype, b1, b2, eps, bits, capturable, seed), items in launches.items():
            with _on(device):
                if torch.cuda.is_current_stream_capturing() and not capturable:
                    raise RuntimeError("FusedAdamW: step() in a graph capture needs capturable=True (the count of steps would be frozen)")
                self._launch(items, device, dtype, b1, b2, eps, bits, capturable, seed)
        return loss

    @staticmethod
    def _gradient(p):
        g = p.grad
        if not p.is_cuda:
            raise RuntimeError(f"FusedAdamW: parameter on {p.device}; this build has no CPU path")
        if p.dtype not in _TYPES:
            raise TypeError(f"FusedAdamW: parameters are float32, float16 or bfloat16, not {p.dtype}")
        if g.layout != torch.strided:
            raise RuntimeError("FusedAdamW: sparse gradients are not supported")
        if g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
            raise RuntimeError(f"FusedAdamW: a gradient of {g.dtype} {tuple(g.shape)} on {g.device} for a parameter of {p.dtype} {tuple(p.shape)} on {p.device}")
        if not _dense(p):
            raise RuntimeError("FusedAdamW: parameters must be dense (no gaps, no element twice)")
        if g.stride() != p.stride() and p.numel() > 1:
            g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)
        return g

    @staticmethod
    def _launch(items, device, dtype, b1, b2, eps, bits, capturable, seed):
        L = lib()
        ptr = torch.Tensor.data_ptr
        buf = bytearray(_TENSOR.size * len(items))
        second = "exp_avg_sq" if bits == 32 else "exp_avg_rms"
        if len({ptr(it[0]) for it in items if it[0].numel()}) != sum(1 for it in items if it[0].numel()):
            raise RuntimeError("FusedAdamW: two parameters share their memory")
        scalars, size, factor, keep, key = None, 0.0, 0.0, 0.0, 0
        if capturable:
            n = len(items)
            scalars = torch.empty(4 * n, dtype=torch.float32, device=device)
            P = ctypes.c_void_p
            for _, _, st, g, _ in items:
                if st["step"].device != device or st["step"].dtype != torch.float32:
                    raise RuntimeError("FusedAdamW: with capturable=True the state's 'step' is a float32 on the parameter's device")
                if torch.is_tensor(g["lr"]) and g["lr"].device != device:
                    raise RuntimeError("FusedAdamW: lr is on another device than its parameters")
            _check(L.gvd_adamw_scalars((P * n)(*[ptr(it[2]["step"]) for it in items]),
                                       (P * n)(*[ptr(it[3]["lr"]) if torch.is_tensor(it[3]["lr"]) else None for it in items]),
                                       (ctypes.c_double * n)(*[0.0 if torch.is_tensor(it[3]["lr"]) else it[3]["lr"] for it in items]),
                                       (ctypes.c_double * n)(*[it[3]["weight_decay"] for it in items]),
                                       (ctypes.c_uint * n)(*[it[4] for it in items]), n, ctypes.c_double(b1), ctypes.c_double(b2),
                                       ctypes.c_uint(seed), P(ptr(scalars)), P(_stream())))
        at = 0
        for p, grad, st, g, place in items:
            if not capturable:
                t = st["step"]
                t += 1
                t = t.item()
                size, factor = g["lr"] / (1.0 - b1 ** t), 1.0 / math.sqrt(1.0 - b2 ** t)
                keep = 1.0 - g["lr"] * g["weight_decay"]
                if bits == 8:
                    key = L.gvd_adamw_key(seed, place, int(t))
            _TENSOR.pack_into(buf, at, ptr(p), ptr(grad), ptr(st["exp_avg"]), ptr(st[second]), ptr(st["exp_avg_scale"]) if bits == 8 else 0,
                              ptr(st["exp_avg_rms_scale"]) if bits == 8 else 0, p.numel(), size, factor, keep, key)
            at += _TENSOR.size
        _check(L.gvd_adamw_step(bytes(buf), len(items), _TYPES[dtype], bits, b1, b2, eps, None if scalars is None else ptr(scalars), _stream()))
