"""FusedAdamW (csrc/adamw.hip) against the formulas in 64 bits: sizes around a vector, a block and a workgroup's chunk, every parameter
type, other memory orders and alignments, more tensors than a launch holds, moments in 8 bits against their exact stochastic rounding,
non-finite gradients, state dicts, graph capture, other streams; and what it refuses."""
import ctypes
import math
import os
import re
import struct

import pytest
import torch
from torch.optim.optimizer import register_optimizer_step_post_hook

import fused_optim
from fused_optim import FusedAdamW

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
TENSOR = struct.Struct("6Qq3fI")     # gvd_adamw_tensor, as a caller without torch binds it
U = 2.0 ** -24      # half a step of float32, relative


# ---- the plain implementation, 64 bits ------------------------------------------------------------------------------------------
def mix(h):
    h = ((h ^ (h >> 16)) * 0x7A2D4F2D) & 0xffffffff
    h = ((h ^ (h >> 15)) * 0x5C8B3B55) & 0xffffffff
    return h ^ (h >> 16)


def draws(seed, place, step, n):
    key = mix(mix(mix((seed + 0x3D1C27A5) & 0xffffffff) ^ place) ^ step)
    return mix((torch.arange(n, dtype=torch.int64) * 0x9D2C5681 + key) & 0xffffffff)


def reference(p, g, m, v, t, lr, b1, b2, eps, wd):
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v2 / (1 - b2 ** t)).sqrt() + eps
    upd = lr / (1 - b1 ** t) * m2 / denom
    # float32: m2 and v2 within 4 U of what enters them; upd: m2's error over denom, sqrt, factor, sum, quotient and product 1 U each
    big_m = b1 * m.abs() + (1 - b1) * g.abs()
    err_m, err_v = 4 * U * big_m, 4 * U * v2
    err_p = 4 * U * p.abs() + lr / (1 - b1 ** t) * (err_m + 12 * U * m2.abs()) / denom
    return p * (1 - lr * wd) - upd, m2, v2, err_p, err_m, err_v


def codes_of(y, u):
    """y >= 0 as the value of e4m3 that its draw u in [0, 1) picks."""
    step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    return (torch.floor(y / step + u) * step).clamp(max=448.0)


def blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)


def make(shapes, dtype=torch.float32, seed=0, scale=1e-3):
    gen = torch.Generator().manual_seed(seed)
    ps = [torch.randn(s, generator=gen).to(dtype).to(DEV) for s in shapes]
    gs = [[(scale * torch.randn(s, generator=gen)).to(dtype).to(DEV) for s in shapes] for _ in range(3)]
    return ps, gs


# ---- on the CPU -----------------------------------------------------------------------------------------------------------------
def test_library_exports_every_declared_symbol():
    import __graft_entry__ as g
    g.build_optim()
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "gvd_optim.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(gvd_[a-z_0-9]+)\s*\(", hdr))
    assert {"gvd_adamw_step", "gvd_adamw_scalars", "gvd_adamw_key", "gvd_optim_last_error"} <= names
    for n in names:
        assert hasattr(fused_optim.lib(), n), n


def test_c_entry_checks_its_arguments_before_any_launch():
    L = fused_optim.lib()
    L.gvd_adamw_step.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.c_int] + [ctypes.c_double] * 3 + [ctypes.c_void_p] * 2
    one = TENSOR.pack(0, 0, 0, 0, 0, 0, 5, 0.1, 1.0, 1.0, 0)
    assert L.gvd_adamw_step(b"", 0, 0, 32, 0.9, 0.999, 1e-8, None, None) == 0
    for args, word in (((one, 1, 0, 32, 0.9, 0.999, 1e-8), b"null"), ((one, 1, 3, 32, 0.9, 0.999, 1e-8), b"param_type"), ((one, 1, 0, 16, 0.9, 0.999, 1e-8), b"state_bits"),
                       ((one, 1, 0, 32, 1.0, 0.999, 1e-8), b"betas"), ((one, 1, 0, 32, 0.9, float("nan"), 1e-8), b"betas"), ((one, 1, 0, 32, 0.9, 0.999, -1.0), b"eps"),
                       ((one, -1, 0, 32, 0.9, 0.999, 1e-8), b"bad")):
        assert L.gvd_adamw_step(*args, None, None) == -1 and word in L.gvd_optim_last_error(), (args, L.gvd_optim_last_error())
    negative = TENSOR.pack(0, 0, 0, 0, 0, 0, -1, 0.1, 1.0, 1.0, 0)
    assert L.gvd_adamw_step(negative, 1, 0, 32, 0.9, 0.999, 1e-8, None, None) == -1 and b"size" in L.gvd_optim_last_error()
    huge = TENSOR.pack(16, 16, 16, 16, 0, 0, 2 ** 34 + 1, 0.1, 1.0, 1.0, 0)
    assert L.gvd_adamw_step(huge, 1, 0, 32, 0.9, 0.999, 1e-8, None, None) == -1 and b"size" in L.gvd_optim_last_error()
    empty = TENSOR.pack(0, 0, 0, 0, 0, 0, 0, 0.1, 1.0, 1.0, 0)
    assert L.gvd_adamw_step(empty, 1, 0, 32, 0.9, 0.999, 1e-8, None, None) == 0      # nothing to do, nothing launched
    assert L.gvd_adamw_scalars(None, None, None, None, None, 1, ctypes.c_double(0.9), ctypes.c_double(0.999), 0, None, None) == -1


def test_key_is_the_documented_hash():
    for seed, place, step in ((0, 0, 1), (5, 3, 77), (2 ** 32 - 1, 1000, 2 ** 24)):
        assert fused_optim.lib().gvd_adamw_key(seed, place, step) == mix(mix(mix((seed + 0x3D1C27A5) & 0xffffffff) ^ place) ^ step)


def test_the_draws_are_even_and_uncorrelated():
    n = 1 << 18
    a, b = draws(1, 0, 10, n), draws(1, 0, 11, n)
    cols = torch.stack([a & 0xffff, a >> 16, b & 0xffff, b >> 16, torch.roll(a & 0xffff, 1), torch.roll(a >> 16, 1)]).double()
    assert float((cols.mean(1) / 65536 - 0.5).abs().max()) < 6 * 12 ** -0.5 / math.sqrt(n)          # 6 standard errors
    assert float((torch.corrcoef(cols) - torch.eye(6, dtype=torch.float64)).abs().max()) < 6 / math.sqrt(n)


def test_refusals_on_the_host():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-9), dict(weight_decay=-1.0),
               dict(state_bits=16), dict(seed=-1), dict(lr=torch.tensor(1e-3)), dict(lr=torch.tensor(1e-3), capturable=True)):
        with pytest.raises(ValueError):
            FusedAdamW([p], **kw)
    with pytest.raises(ValueError):
        FusedAdamW([{"params": [p]}, {"params": [torch.nn.Parameter(torch.zeros(2))], "lr": -1.0}])
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="twice"):
        FusedAdamW([p, p])
    opt = FusedAdamW([p])
    opt.step()                                       # no gradient: nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()
    with pytest.raises(ValueError, match="not a parameter"):
        opt.set_moments(torch.nn.Parameter(torch.zeros(4)), torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="shape"):
        opt.set_moments(p, torch.zeros(3), torch.zeros(3))


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_and_state_dicts_round_trip(bits):
    gen = torch.Generator().manual_seed(0)
    p = torch.nn.Parameter(torch.randn(7, 100, generator=gen).bfloat16())
    m, v = torch.randn(7, 100, generator=gen), torch.rand(7, 100, generator=gen)
    v[0, :50] = 0.0
    opt = FusedAdamW([p], state_bits=bits)
    assert opt.moments(p) is None
    opt.set_moments(p, m, v, step=41)
    gm, gv = opt.moments(p)
    if bits == 32:
        assert torch.equal(gm, m) and torch.equal(gv, v)
    else:                                            # nearest e4m3: half a step of 2^-3, 2^-4 relative, and half of 2^-9 / 448 of the block's largest below
        floor = m.abs().max() * 2.0 ** -10 / 448
        assert bool(((gm - m).abs() <= 2.0 ** -4 * m.abs() + floor).all())
        r = v.sqrt()
        assert bool(((gv.sqrt() - r).abs() <= 2.0 ** -4 * r * (1 + 1e-5) + r.max() * 2.0 ** -9 / 448).all())
        assert bool(((gv == 0) == (v == 0)).all())
    other = FusedAdamW([torch.nn.Parameter(p.detach().clone())], state_bits=bits)
    other.load_state_dict(opt.state_dict())
    q = other.param_groups[0]["params"][0]
    for k, x in opt.state[p].items():
        y = other.state[q][k]
        assert y.dtype == x.dtype and y.shape == x.shape and y.data_ptr() != x.data_ptr()
        assert torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x, y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y)
    wrong = FusedAdamW([torch.nn.Parameter(p.detach().clone())], state_bits=40 - bits)
    sd = opt.state_dict()
    sd["param_groups"][0]["state_bits"] = 40 - bits
    with pytest.raises(RuntimeError, match="does not fit"):
        wrong.load_state_dict(sd)


def test_refuses_the_state_of_another_rule():
    p = torch.nn.Parameter(torch.randn(5, 3))
    for other in (torch.optim.Adam([p], amsgrad=True), torch.optim.Adam([p], maximize=True), torch.optim.Adam([p], weight_decay=0.1)):
        with pytest.raises(ValueError, match="rule"):
            FusedAdamW([p]).load_state_dict(other.state_dict())
    FusedAdamW([p]).load_state_dict(torch.optim.AdamW([p], weight_decay=0.1).state_dict())


def test_state_is_loaded_into_the_parameters_memory_order():
    p, q = torch.nn.Parameter(torch.randn(5, 3)), torch.nn.Parameter(torch.randn(3, 5).t())
    a, b = FusedAdamW([p]), FusedAdamW([q])
    m, v = torch.randn(5, 3), torch.rand(5, 3)
    a.set_moments(p, m, v, 3)
    b.load_state_dict(a.state_dict())
    assert b.state[q]["exp_avg"].stride() == q.stride() and torch.equal(b.state[q]["exp_avg"], m) and torch.equal(b.state[q]["exp_avg_sq"], v)


def test_loads_the_state_of_torchs_adam():
    p = torch.nn.Parameter(torch.randn(5, 3))
    ref = torch.optim.Adam([p], lr=3e-4, eps=1e-15)
    p.grad = torch.randn(5, 3)
    ref.step()
    q = torch.nn.Parameter(p.detach().clone())
    opt = FusedAdamW([q], weight_decay=0.0)
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 3e-4 and opt.param_groups[0]["state_bits"] == 32
    assert torch.equal(opt.state[q]["exp_avg"], ref.state[p]["exp_avg"]) and float(opt.state[q]["step"]) == 1.0


# ---- on the device: 32-bit moments ------------------------------------------------------------------------------------------------
def check_steps(opt, params, grads, lr, betas, eps, wd, steps):
    """`steps` steps, each against the reference from the state before it."""
    b1, b2 = betas
    for s in range(steps):
        before = []
        for i, p in enumerate(params):
            p.grad = grads[s % len(grads)][i]
            mv = opt.moments(p)
            before.append((p.detach().clone(), *((x.clone() for x in mv) if mv else (torch.zeros_like(p, dtype=torch.float32),) * 2)))
        opt.step()
        for i, p in enumerate(params):
            p0, m0, v0 = before[i]
            t = float(opt.state[p]["step"])
            rp, rm, rv, ep, em, ev = reference(p0, p.grad, m0, v0, t, lr, b1, b2, eps, wd)
            half = 0.0 if p.dtype == torch.float32 else torch.finfo(p.dtype).eps / 2
            tiny = 2.0 ** -149 if p.dtype != torch.float16 else 2.0 ** -25
            m, v = opt.moments(p)
            assert bool(((m.double().cpu() - rm).abs() <= em + 2.0 ** -149).all()), (i, s, "m")
            assert bool(((v.double().cpu() - rv).abs() <= ev + 2.0 ** -149).all()), (i, s, "v")
            assert bool(((p.detach().double().cpu() - rp).abs() <= ep * (1 + half) + half * rp.abs() + tiny).all()), (i, s, "p")


SIZES = [(), (1,), (3,), (4,), (0,), (5, 7), (255,), (256,), (1023,), (1025,), (2047,), (2048,), (2049,), (3, 1000, 7), (40000,)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_steps_match_the_formulas_at_every_size(dtype):
    ps, gs = make(SIZES, dtype)
    params = [torch.nn.Parameter(p) for p in ps]
    kw = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
    opt = FusedAdamW(params, **kw)
    check_steps(opt, params, gs, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"], 3)


@gpu
def test_groups_have_their_own_settings_and_parameters_without_gradient_stay():
    ps, gs = make([(300,), (70, 3), (5000,), (8,)])
    params = [torch.nn.Parameter(p) for p in ps]
    opt = FusedAdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:3], betas=(0.5, 0.9), eps=1e-15), dict(params=params[3:])], lr=1e-3, weight_decay=0.0)
    old = [p.detach().clone() for p in params]
    for i in range(3):
        params[i].grad = gs[0][i]
    opt.step()
    zero = torch.zeros
    for i, (lr, b1, b2, eps) in enumerate(((1e-2, 0.9, 0.999, 1e-8), (1e-2, 0.9, 0.999, 1e-8), (1e-3, 0.5, 0.9, 1e-15))):
        rp, _, _, ep, _, _ = reference(old[i], gs[0][i], zero(old[i].shape), zero(old[i].shape), 1, lr, b1, b2, eps, 0.0)
        assert bool(((params[i].detach().double().cpu() - rp).abs() <= ep).all()), i
    assert torch.equal(params[3], old[3]) and params[3] not in opt.state


@gpu
def test_agrees_with_torchs_adamw_over_steps():
    ps, gs = make([(1000, 3), (1000, 1), (1000, 16, 3)], seed=3)
    a, b = [torch.nn.Parameter(p.clone()) for p in ps], [torch.nn.Parameter(p.clone()) for p in ps]
    oa, ob = FusedAdamW(a, lr=1e-3, weight_decay=0.01, eps=1e-15), torch.optim.AdamW(b, lr=1e-3, weight_decay=0.01, eps=1e-15)
    for s in range(6):
        for i in range(3):
            a[i].grad = b[i].grad = gs[s % 3][i]
        oa.step()
        ob.step()
    for x, y in zip(a, b):   # six updates of at most ~lr, each 20 U off; p 6 U
        x, y = x.detach(), y.detach()
        assert float((x - y).abs().max()) <= 6 * (2 * U * float(y.abs().max()) + 40 * U * 1e-3 * 3.2)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_holds(bits):
    shapes = [(1 + 37 * i % 600,) for i in range(131)]
    ps, gs = make(shapes, seed=1)
    params = [torch.nn.Parameter(p) for p in ps]
    old = [p.detach().clone() for p in params]
    opt = FusedAdamW(params, lr=1e-3, weight_decay=0.0, state_bits=bits)
    for i, p in enumerate(params):
        p.grad = gs[0][i]
    opt.step()
    for i, p in enumerate(params):
        z = torch.zeros(shapes[i])
        rp, _, _, ep, _, _ = reference(old[i], gs[0][i], z, z, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0)
        assert bool(((p.detach().double().cpu() - rp).abs() <= ep).all()), i


def odd_layouts(x):
    """The same values with a transposed memory order, and 4 or 2 bytes off a vector's alignment with neighbours that have to stay."""
    flat = torch.full((x.numel() + 2,), 7.0, dtype=x.dtype, device=x.device)
    flat[1:-1] = x.reshape(-1)
    return x.t().contiguous().t(), flat[1:-1].view(x.shape), flat


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_memory_orders_and_alignments(dtype, bits):
    ps, gs = make([(33, 70)], dtype, seed=2)
    turned, shifted, flat = odd_layouts(ps[0])
    old = ps[0].clone()
    params = [torch.nn.Parameter(x) for x in (ps[0].clone(), turned, shifted)]
    assert not params[1].is_contiguous() and params[2].data_ptr() % 16
    opt = FusedAdamW(params, lr=1e-2, weight_decay=0.0, state_bits=bits)
    for p in params:
        p.grad = gs[0][0].clone()                    # row-major: the turned parameter's gradient is copied into its order
    opt.step()
    z = torch.zeros(old.shape)
    rp, rm, _, ep, _, _ = reference(old, gs[0][0], z, z, 1, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    for p in params:
        assert bool(((p.detach().double().cpu() - rp).abs() <= ep * (1 + half) + half * rp.abs()).all())
        m = opt.moments(p)[0].double().cpu()
        assert bool(((m - rm).abs() <= (4 * U * rm.abs() if bits == 32 else 2.0 ** -3 * rm.abs() + rm.abs().max() * 2.0 ** -9 / 448)).all())
    assert float(flat[0]) == 7.0 and float(flat[-1]) == 7.0
    assert opt.state[params[1]]["exp_avg"].stride() == params[1].stride()


@gpu
def test_refusals_on_the_device():
    p = torch.nn.Parameter(torch.zeros(4, 4, device=DEV))
    opt = FusedAdamW([p])
    p.grad = torch.zeros(4, 4, device=DEV)
    opt.step()
    opt.state[p]["exp_avg"] = torch.zeros(5, 4, device=DEV)      # rows added to the parameter's state alone
    with pytest.raises(RuntimeError, match="does not fit"):
        opt.step()
    e = torch.nn.Parameter(torch.zeros(1, 4, device=DEV).expand(4, 4))
    e.grad = torch.zeros(4, 4, device=DEV)
    with pytest.raises(RuntimeError, match="dense"):
        FusedAdamW([e]).step()
    d = torch.nn.Parameter(torch.zeros(4, device=DEV, dtype=torch.float64))
    d.grad = torch.zeros_like(d)
    with pytest.raises(TypeError):
        FusedAdamW([d]).step()
    base = torch.zeros(8, device=DEV)
    a, b = torch.nn.Parameter(base[:4]), torch.nn.Parameter(base[:4])
    a.grad, b.grad = torch.zeros(4, device=DEV), torch.zeros(4, device=DEV)
    with pytest.raises(RuntimeError, match="share"):
        FusedAdamW([a, b]).step()
    b = torch.nn.Parameter(base[2:6])                # overlapping in part
    b.grad = torch.zeros(4, device=DEV)
    with pytest.raises(RuntimeError, match="share"):
        FusedAdamW([b, a]).step()
    b = torch.nn.Parameter(base[4:])                 # side by side
    b.grad = torch.ones(4, device=DEV)
    FusedAdamW([b, a], lr=0.5).step()
    assert bool((base[:4] == 0).all()) and bool((base[4:] < 0).all())
    s = torch.nn.Parameter(torch.zeros(4, 4, device=DEV))
    s.grad = torch.zeros(4, 4, device=DEV).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        FusedAdamW([s]).step()


@gpu
def test_offsets_beyond_32_bits():
    """2^31 elements and some: the last ones as in a small tensor, the first untouched by them."""
    n, tail = 2 ** 31 + 2048 + 5, 5000
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.zeros_like(p)
    gen = torch.Generator(device=DEV).manual_seed(0)
    small = torch.nn.Parameter(torch.randn(tail, device=DEV, generator=gen).bfloat16())
    small.grad = torch.randn(tail, device=DEV, generator=gen).bfloat16()
    with torch.no_grad():
        p[-tail:] = small
        p.grad[-tail:] = small.grad
    big, ref = FusedAdamW([p], lr=1e-2), FusedAdamW([small], lr=1e-2)
    big.step()
    ref.step()
    assert torch.equal(p[-tail:], small) and not bool(p[:tail].any())
    assert torch.equal(big.state[p]["exp_avg"][-tail:], ref.state[small]["exp_avg"])
    assert int(big.state[p]["exp_avg_sq"].count_nonzero()) == int(ref.state[small]["exp_avg_sq"].count_nonzero())   # nothing written elsewhere


# ---- 8-bit moments ----------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1,), (255,), (257,), (2048,), (5, 1111), (30000,)])
def test_eight_bit_moments_are_rounded_by_their_draws(shape, dtype):
    """Every held value is the one that its draw picks for the exact moment; one of float32's errors away from the border it may be the neighbour."""
    lr, b1, b2, eps, seed = 1e-2, 0.9, 0.999, 1e-8, 9
    filler, p = (torch.nn.Parameter(torch.zeros(3, device=DEV, dtype=dtype)), torch.nn.Parameter(make([shape], dtype, seed=4)[0][0]))
    gen = torch.Generator().manual_seed(8)
    n = p.numel()
    opt = FusedAdamW([filler, p], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, state_bits=8, seed=seed)
    for t in range(1, 4):
        p.grad = (torch.randn(shape, generator=gen) * torch.exp(3 * torch.randn(shape, generator=gen)) * 1e-4).to(dtype).to(DEV)
        filler.grad = torch.zeros_like(filler)
        mv = opt.moments(p)
        m0, v0 = mv if mv else (torch.zeros_like(p, dtype=torch.float32),) * 2
        r0 = v0.double().sqrt().float()
        p0 = p.detach().clone()
        opt.step()
        st = opt.state[p]
        rp, rm, rv, ep, em, _ = reference(p0, p.grad, m0, r0.double() ** 2, t, lr, b1, b2, eps, 0.0)
        half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        assert bool(((p.detach().double().cpu() - rp).abs() <= 2 * ep * (1 + half) + half * rp.abs() + 2.0 ** -40).all())
        h = draws(seed, 1, t, n)
        for name, x, bits in (("exp_avg", rm.reshape(-1), h & 0xffff), ("exp_avg_rms", rv.sqrt().reshape(-1), h >> 16)):
            big = blocks(x).abs().amax(1)
            scale = st[name + "_scale"].double().cpu()
            assert bool(((scale - big / 448).abs() <= 16 * U * big / 448).all()), name
            got = st[name].float().double().cpu().reshape(-1)
            y = x.abs() / (big / 448).repeat_interleave(256)[:n]
            slack = 24 * U * y                                       # root and scaled value: below 24 U together
            if name == "exp_avg":                                    # a first moment may cancel: its error is one of its terms'
                slack = slack + em.reshape(-1) / (big / 448).repeat_interleave(256)[:n]
            lo, hi = codes_of((y - slack).clamp(min=0), bits / 65536), codes_of(y + slack, bits / 65536)
            if name == "exp_avg_rms":
                lo, hi = (torch.where(x > 0, c.clamp(min=2.0 ** -9), c) for c in (lo, hi))
            assert bool(((got.abs() >= lo) & (got.abs() <= hi)).all()), (name, t)
            assert bool((torch.sign(got) * torch.sign(x) >= 0).all())
            assert float((lo != hi).double().mean()) < 1e-3      # the check above is sharp


@gpu
def test_eight_bit_second_moment_follows_a_change_it_could_not_follow_by_nearest_rounding():
    """Gradients double: v has to grow from 1 to 4 over 2000 steps though a step moves its root by 0.15 % at most and e4m3's values lie 6 to 12 % apart.
    Over 8192 independent elements: the draws spread the root by about 5 %, so the mean's 6 standard errors are 0.4 % of r, 0.8 % of r^2; the draws'
    variance lifts the mean of r^2 by 1 % (each step adds at most 5e-4 x 0.12 r^2 of it, which decays over 1000 steps, and not all lie that far)."""
    n = 8192
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = FusedAdamW([p], lr=0.0, weight_decay=0.0, state_bits=8)
    opt.set_moments(p, torch.zeros(n, device=DEV), torch.ones(n, device=DEV), step=5000)
    p.grad = torch.full((n,), 2.0, device=DEV)
    p.grad[::256] = 8.0                              # the largest of each block: the others are held below the top of the range
    for _ in range(2000):
        opt.step()
    m, v = opt.moments(p)
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[::256] = False
    want_v = 4.0 - 3.0 * 0.999 ** 2000
    assert abs(float(v[rest].sqrt().mean()) ** 2 / want_v - 1) < 0.03, float(v[rest].sqrt().mean()) ** 2
    assert abs(float(m[rest].mean()) / 2.0 - 1) < 0.01


@gpu
def test_eight_bit_zeros_and_non_finite_gradients_stay_with_their_element():
    p = torch.nn.Parameter(torch.zeros(1000, device=DEV))
    opt = FusedAdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8, eps=1e-15)
    g = torch.zeros(1000, device=DEV)
    p.grad = g
    opt.step()
    assert bool((p == 0).all()) and bool((opt.moments(p)[1] == 0).all())          # nothing moved, nothing divided by nothing
    g[:300] = torch.randn(300, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    g[5], g[260], g[700] = float("inf"), float("nan"), 1e-25
    opt.step()
    bad = torch.zeros(1000, dtype=torch.bool, device=DEV)
    bad[5] = bad[260] = True
    assert bool((torch.isfinite(p) == ~bad).all())
    m, v = opt.moments(p)
    assert bool((torch.isfinite(m) == ~bad).all()) and bool((torch.isfinite(v) == ~bad).all())
    assert bool((v[:300][~bad[:300]] > 0).all())
    # a root far below its block's largest is held above 0: the next update does not divide by eps alone
    q = torch.nn.Parameter(torch.zeros(256, device=DEV))
    opt = FusedAdamW([q], lr=1e-2, weight_decay=0.0, state_bits=8, eps=1e-15)
    q.grad = torch.full((256,), 1e-9, device=DEV)
    q.grad[0] = 1e3
    for _ in range(20):
        opt.step()
    assert bool((opt.state[q]["exp_avg_rms"].float() > 0).all()) and float(q.detach().abs().max()) <= 20 * 1e-2 * 1.1


@gpu
def test_eight_bit_runs_repeat_and_seeds_differ():
    def run(seed):
        ps, gs = make([(5000,), (300, 7)], seed=6)
        params = [torch.nn.Parameter(p) for p in ps]
        opt = FusedAdamW(params, lr=1e-2, state_bits=8, seed=seed)
        for s in range(5):
            for i, p in enumerate(params):
                p.grad = gs[s % 3][i]
            opt.step()
        return torch.cat([p.detach().reshape(-1) for p in params]), opt.state[params[0]]["exp_avg"].view(torch.uint8)
    a, b, c = run(1), run(1), run(2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[1], c[1])


@gpu
def test_hooks_schedulers_and_the_profiler_see_each_step():
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    p.grad = torch.full_like(p, 1e-2)
    seen = []
    opt = FusedAdamW([p], lr=1e-2)
    schedule = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)
    opt.step()
    schedule.step()
    assert opt.param_groups[0]["lr"] == 5e-3 and not seen
    before = opt.register_step_pre_hook(lambda o, args, kwargs: seen.append(("before", o is opt, float(o.state[p]["step"]))))
    after = opt.register_step_post_hook(lambda o, args, kwargs: seen.append(("after", o is opt, float(o.state[p]["step"]))))
    assert opt.step(lambda: 7.0) == 7.0
    assert seen == [("before", True, 1.0), ("after", True, 2.0)]
    before.remove()
    after.remove()
    opt.step()
    assert len(seen) == 2 and float(opt.state[p]["step"]) == 3
    every = register_optimizer_step_post_hook(lambda o, args, kwargs: seen.append("every"))
    opt.step()
    every.remove()
    assert seen[2:] == ["every"]
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step()
    assert any(e.key == "Optimizer.step#FusedAdamW.step" for e in prof.key_averages())
    assert float(opt.state[p]["step"]) == 5


@gpu
def test_nothing_is_counted_where_a_later_launch_is_refused():
    a, b = (torch.nn.Parameter(torch.ones(64, device=DEV, dtype=t)) for t in (torch.float32, torch.bfloat16))
    opt = FusedAdamW([a, b], lr=1e-2)
    for p in (a, b):
        p.grad = torch.ones_like(p)
    opt.step()
    kept = a.detach().clone()
    opt.state[b]["exp_avg"] = torch.zeros(63, device=DEV)
    with pytest.raises(RuntimeError, match="exp_avg"):
        opt.step()
    assert float(opt.state[a]["step"]) == 1 and torch.equal(a, kept)
    opt.state[b]["exp_avg"] = "none"
    with pytest.raises(RuntimeError, match="no tensor"):
        opt.step()
    opt.state[b] = {}                   # set up anew
    opt.step()
    assert float(opt.state[a]["step"]) == 2 and float(opt.state[b]["step"]) == 1 and not torch.equal(a, kept)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_versions_count_each_step(bits):
    """Graphs that saved a parameter refuse it afterwards, and images packed from it are packed anew."""
    from lvdm_amd import gemm
    lin = torch.nn.Linear(320, 320).half().to(DEV)
    x = torch.randn(512, 320, device=DEV).half()
    opt = FusedAdamW(lin.parameters(), lr=0.1, weight_decay=0.0, state_bits=bits)

    def check():
        with torch.no_grad():
            y = gemm.linear(x, lin.weight, lin.bias).double()
        X, W, b = x.double(), lin.weight.detach().double(), lin.bias.detach().double()
        want = X @ W.t() + b
        assert bool(((y - want).abs() <= 2.0 ** -11 * want.abs() + 321 * U * (X.abs() @ W.abs().t() + b.abs())).all())   # rounded once; sums in 32 bits
        return y
    first = check()
    saved = (lin.weight.float() * lin.weight.float()).sum()
    held = (lin.weight * lin.weight).sum()
    before = [p._version for p in lin.parameters()]
    for p in lin.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    assert all(p._version > v for p, v in zip(lin.parameters(), before))
    assert float((check() - first).abs().max()) > 1
    saved.backward()                                    # (its graph saved copies)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.backward()
    state = {k: v._version for k, v in opt.state[lin.weight].items()}
    opt.step()
    assert all(opt.state[lin.weight][k]._version > v for k, v in state.items())


# ---- capture and streams ----------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on_and_read_lr_at_each_replay(bits):
    shapes = [(3000,), (17, 5), (1,)]
    ps, gs = make(shapes, seed=7)
    a, b = [torch.nn.Parameter(p.clone()) for p in ps], [torch.nn.Parameter(p.clone()) for p in ps]
    lr = torch.tensor([1e-3], device=DEV)
    oa = FusedAdamW(a, lr=lr, capturable=True, state_bits=bits, weight_decay=0.01)
    ob = FusedAdamW(b, lr=1e-3, state_bits=bits, weight_decay=0.01)
    for i, p in enumerate(a):
        p.grad = gs[0][i].clone()
    oa.step()                                        # eager first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for s in range(1, 6):
        lr.fill_(1e-3 * s)
        for i, p in enumerate(a):
            p.grad.copy_(gs[s % 3][i])
        if s == 3:
            oa.step()                                # the program's own eager step between replays
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert float(oa.state[a[0]]["step"]) == s + 1
    for s in range(6):
        ob.param_groups[0]["lr"] = 1e-3 * max(s, 1)
        for i, p in enumerate(b):
            p.grad = gs[s % 3][i]
        ob.step()
    for x, y in zip([p.detach() for p in a], [p.detach() for p in b]):   # the same kernel; scalars made in 64 bits on either side, one rounding apart at most
        tol = 6 * (2 * U * float(y.abs().max()) + 40 * U * 5e-3 * 3.2) if bits == 32 else 1e-4
        assert float((x - y).abs().max()) <= tol


@gpu
def test_a_step_in_a_capture_is_refused_where_its_count_would_freeze():
    p = torch.nn.Parameter(torch.zeros(8, device=DEV))
    p.grad = torch.ones(8, device=DEV)
    opt, fresh = FusedAdamW([p]), FusedAdamW([p], capturable=True)
    opt.step()
    x = torch.zeros(4, device=DEV)
    for o, word in ((opt, "capturable=True"), (fresh, "before capturing")):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x += 1
            with pytest.raises(RuntimeError, match=word):
                o.step()
        graph.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 2.0


@gpu
def test_runs_on_the_current_stream():
    ps, gs = make([(200000,)], seed=9)
    p = torch.nn.Parameter(ps[0])
    old = p.detach().clone()
    opt = FusedAdamW([p], lr=1e-2, weight_decay=0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.grad = gs[0][0] * 1.0                      # produced on the side stream: a step on another one could run ahead of it
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    z = torch.zeros(old.shape)
    rp, _, _, ep, _, _ = reference(old, gs[0][0], z, z, 1, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    assert bool(((p.detach().double().cpu() - rp).abs() <= ep).all())


# ---- in the trainer --------------------------------------------------------------------------------------------------------------
def test_the_trainer_names_its_optimizers():
    import guided_schedule as gs
    p = [torch.nn.Parameter(torch.zeros(3))]
    a, f, e = (gs.RasterTrainer._optimizer(k, p, 1e-4) for k in ("adam", "fused", "fused8"))
    assert type(a) is torch.optim.Adam and type(f) is FusedAdamW and f.param_groups[0]["state_bits"] == 32 and e.param_groups[0]["state_bits"] == 8
    for o in (a, f, e):
        assert o.param_groups[0]["eps"] == 1e-15 and o.param_groups[0]["weight_decay"] == 0
    with pytest.raises(ValueError, match="optimizer"):
        gs.RasterTrainer._optimizer("sgd", p, 1e-4)


@gpu
@pytest.mark.parametrize("kind", ["fused", "fused8"])
def test_training_gaussians(kind):
    """One step of the raster trainer from the same start as torch's Adam: the gradients are the same bits, so parameters are equal to the update's float32 (the
    first step is lr times the gradient's sign, 12 U off at most, and sums with p are rounded); then it goes on."""
    import guided_schedule as gs
    import synthetic as syn
    sc = syn.scene_c1()
    ref, got = (gs.RasterTrainer(sc, sc["cameras"], DEV, lr=1e-3, optimizer=k) for k in ("adam", kind))
    ref.train_step(0)
    got.train_step(0)
    for n, x in ref.state().items():
        y = got.state()[n]
        assert bool(((x - y).abs() <= 4 * U * x.abs() + 16 * U * 1e-3).all()), n
    before = got.state()
    for it in range(1, 6):
        got.train_step(it)
    after = got.state()
    assert all(bool(torch.isfinite(x).all()) for x in after.values()) and not torch.equal(before["means3D"], after["means3D"])
