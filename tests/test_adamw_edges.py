"""FusedAdamW in the calls where it can go wrong without a word: moments at the ends of float32's range, spellings of one memory order, groups that change between steps,
states of another rule, arrays that overlap."""
import pytest
import torch

from fused_optim import FusedAdamW

gpu = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = 2.0 ** -4        # half a step of e4m3, relative
LEAST = 2.0 ** -10      # half of its least subnormal


# ---- moments in 8 bits, given as floats ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("least", [1e-45, 1e-39, 1e-37, 1.3e-36, 1e-34, 2.0 ** -110, 1e-30])
def test_tiny_first_moments_are_held_near_zero(least):
    """Blocks whose largest moment is below 2^-110 are held as zeros; from there on e4m3's rounding holds: half a step of the value, or of the block's largest / 448."""
    p = torch.nn.Parameter(torch.zeros(600))
    m = torch.zeros(600)
    m[:10] = least * torch.linspace(-1.0, 1.0, 10)
    m[300:310] = 0.5                                    # another block, which has to stay
    opt = FusedAdamW([p], state_bits=8)
    opt.set_moments(p, m, torch.zeros(600), step=3)
    got, v = opt.moments(p)
    assert bool((v == 0).all())
    assert bool(((got[256:] - m[256:]).abs() <= E4M3 * m[256:].abs()).all())
    if least < 2.0 ** -110:
        assert bool((got[:256] == 0).all())
    else:
        off = (got[:256].double() - m[:256].double()).abs()
        assert bool((off <= (E4M3 + 2.0 ** -22) * m[:256].abs().double() + 1.001 * LEAST * least / 448).all()) and bool((got[:10] != 0).any())


def test_tiny_second_moments_are_not_lost():
    p = torch.nn.Parameter(torch.zeros(300))
    v = torch.full((300,), 1e-45)                       # float32's least: its root is 3.7e-23
    opt = FusedAdamW([p], state_bits=8)
    opt.set_moments(p, torch.zeros(300), v)
    root = opt.moments(p)[1].double()                   # (squares of 3.7e-23 in float32: the least number or 0)
    codes = opt.state[p]["exp_avg_rms"].float()
    assert bool((codes > 0).all()) and bool(torch.isfinite(root).all())


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_moments_that_are_not_finite_stay_with_their_element(value, device):
    gen = torch.Generator().manual_seed(0)
    p = torch.nn.Parameter(torch.zeros(700, device=device))
    m, v = torch.randn(700, generator=gen).to(device), torch.rand(700, generator=gen).to(device) + 0.1
    m[5] = m[300] = v[6] = v[301] = value
    m[600:], m[650] = 0.0, value                        # a block with nothing else in it
    m[512:600] = 0.0
    opt = FusedAdamW([p], state_bits=8)
    opt.set_moments(p, m, v)
    for got, x in zip(opt.moments(p), (m, v)):
        bad = ~torch.isfinite(x)
        assert torch.equal(torch.isfinite(got), ~bad)
        size = x[~bad].abs().max()
        assert bool(((got - x)[~bad].abs() <= 2.2 * E4M3 * x[~bad].abs() + size * LEAST / 448).all())     # (a square: twice the root's half step, and its own square)


# ---- spellings of one memory order -----------------------------------------------------------------------------------------------
def turned(n, device="cpu"):
    """[n, 1, 3] with strides (3, 1, 1): the same memory as a fresh tensor's (3, 3, 1)."""
    x = torch.randn(n, 3, 1, generator=torch.Generator().manual_seed(1)).to(device).transpose(1, 2).contiguous()
    assert x.stride() == (3, 1, 1) and torch.empty_like(x, memory_format=torch.contiguous_format).stride() != x.stride()
    return x


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dicts_go_between_spellings_of_one_order(bits):
    p, q = torch.nn.Parameter(turned(100)), torch.nn.Parameter(turned(100).clone(memory_format=torch.contiguous_format))
    a, b = FusedAdamW([p], state_bits=bits), FusedAdamW([q], state_bits=bits)
    m, v = torch.randn(100, 1, 3), torch.rand(100, 1, 3)
    for x, y, r, s in ((a, b, p, q), (b, a, q, p)):
        x.set_moments(r, m, v, 3)
        y.load_state_dict(x.state_dict())
        assert all(torch.equal(i, j) for i, j in zip(x.moments(r), y.moments(s)))
        m, v = m + 1, v + 1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_states_and_gradients_of_another_spelling_are_taken_as_they_are(bits):
    """A state set by hand has a fresh tensor's strides, and so has a gradient: both are the parameter's order, nothing is copied."""
    fresh = lambda x: x.clone(memory_format=torch.contiguous_format)  # noqa: E731
    p, q = torch.nn.Parameter(turned(1000, DEV)), torch.nn.Parameter(fresh(turned(1000, DEV)))
    g = torch.randn(1000, 1, 3, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    a, b = FusedAdamW([p], lr=1e-2, state_bits=bits), FusedAdamW([q], lr=1e-2, state_bits=bits)
    for step in range(3):
        p.grad, q.grad = g * (step + 1), g * (step + 1)
        assert p.grad.stride() != p.stride()
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        if step:
            a.step()
            assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
        else:
            a.step()
        b.step()
        assert torch.equal(p, q) and all(torch.equal(x, y) for x, y in zip(a.moments(p), b.moments(q)))
        if bits == 32:
            a.state[p].update({k: fresh(a.state[p][k]) for k in ("exp_avg", "exp_avg_sq")})
            assert a.state[p]["exp_avg"].stride() != p.stride()


@gpu
def test_another_order_is_still_another_order():
    p = torch.nn.Parameter(torch.zeros(4, 1, 3, device=DEV))
    p.grad = torch.arange(12.0, device=DEV).view(3, 1, 4).permute(2, 1, 0)
    opt = FusedAdamW([p], lr=1.0, weight_decay=0.0)
    opt.step()
    assert torch.equal(opt.state[p]["exp_avg"], 0.1 * p.grad) or bool(((opt.state[p]["exp_avg"] - 0.1 * p.grad).abs() <= 4 * 2.0 ** -24 * p.grad).all())
    opt.state[p]["exp_avg"] = torch.zeros(3, 1, 4, device=DEV).permute(2, 1, 0)
    with pytest.raises(RuntimeError, match="does not fit"):
        opt.step()


# ---- groups that change between steps ------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("change,error", [(lambda g: g.update(lr=torch.tensor(1e-3, device=DEV, dtype=torch.float64)), ValueError), (lambda g: g.update(lr=torch.zeros(2, device=DEV)), ValueError),
                                          (lambda g: g.update(lr=torch.zeros(0, device=DEV)), ValueError), (lambda g: g.update(lr=torch.tensor(1e-3)), RuntimeError),
                                          (lambda g: g.update(betas=(0.9, 1.0)), ValueError), (lambda g: g.update(betas=(-0.1, 0.9)), ValueError),
                                          (lambda g: g.update(betas=(float("nan"), 0.9)), ValueError), (lambda g: g.update(eps=-1.0), ValueError),
                                          (lambda g: g.update(eps=float("nan")), ValueError), (lambda g: g.update(state_bits=16), ValueError)])
def test_a_group_that_cannot_be_taken_is_refused_before_another_is_stepped(change, error):
    a, b = (torch.nn.Parameter(torch.ones(70, device=DEV)) for _ in range(2))
    opt = FusedAdamW([dict(params=[a]), dict(params=[b], lr=torch.tensor(1e-3, device=DEV), capturable=True)])
    for p in (a, b):
        p.grad = torch.ones_like(p)
    opt.step()
    kept, old = [p.detach().clone() for p in (a, b)], dict(opt.param_groups[1])
    change(opt.param_groups[1])
    with pytest.raises(error):
        opt.step()
    assert torch.equal(a, kept[0]) and torch.equal(b, kept[1]) and float(opt.state[a]["step"]) == 1 == float(opt.state[b]["step"])
    opt.param_groups[1].update(old)
    opt.step()
    assert not torch.equal(a, kept[0]) and not torch.equal(b, kept[1])


# ---- states of another rule or form -----------------------------------------------------------------------------------------------------
def test_a_refused_state_leaves_the_optimizer_as_it_was():
    p = torch.nn.Parameter(torch.randn(5, 3))
    opt = FusedAdamW([p], lr=3e-3, weight_decay=0.0)
    m, v = torch.randn(5, 3), torch.rand(5, 3)
    opt.set_moments(p, m, v, 7)
    p.grad = torch.randn(5, 3)
    others = [torch.optim.Adam([p], lr=1.0, amsgrad=True), torch.optim.Adam([p], lr=1.0, maximize=True), torch.optim.Adam([p], lr=1.0, weight_decay=0.1)]
    for o in others:
        o.step()
    dicts = [o.state_dict() for o in others]
    short = FusedAdamW([p], lr=1.0, state_bits=8)
    short.set_moments(p, m, v, 9)
    dicts.append(short.state_dict())
    dicts[-1]["param_groups"][0]["state_bits"] = 32         # its moments do not fit that
    state, groups = opt.state, opt.param_groups
    for d in dicts:
        with pytest.raises((ValueError, RuntimeError)):
            opt.load_state_dict(d)
        assert opt.state is state and opt.param_groups is groups and opt.param_groups[0]["lr"] == 3e-3 and set(opt.state[p]) == {"step", "exp_avg", "exp_avg_sq"}
        assert float(opt.state[p]["step"]) == 7 and torch.equal(opt.state[p]["exp_avg"], m) and torch.equal(opt.state[p]["exp_avg_sq"], v)


# ---- arrays that overlap ---------------------------------------------------------------------------------------------------------------
def stepped(bits=32, count=3, n=300):
    base = torch.ones(count * n, device=DEV)
    params = [torch.nn.Parameter(base[i * n:(i + 1) * n]) for i in range(count)]       # side by side in one piece of memory
    opt = FusedAdamW(params, lr=1e-2, state_bits=bits)
    for p in params:
        p.grad = torch.ones_like(p)
    opt.step()
    return opt, params, base


def refused(opt, params, word):
    kept, steps = [p.detach().clone() for p in params], [float(opt.state[p]["step"]) for p in params]
    with pytest.raises(RuntimeError, match=word):
        opt.step()
    assert all(torch.equal(p, x) for p, x in zip(params, kept)) and steps == [float(opt.state[p]["step"]) for p in params]


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_share_memory_are_refused(bits):
    for name in ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "exp_avg_rms", "exp_avg_scale", "exp_avg_rms_scale"):
        opt, params, _ = stepped(bits)
        opt.state[params[2]][name] = opt.state[params[0]][name]
        refused(opt, params, "share")
    if bits == 32:
        opt, params, base = stepped()
        opt.state[params[1]]["exp_avg_sq"] = opt.state[params[1]]["exp_avg"]           # of one parameter
        refused(opt, params, "share")
        opt, params, base = stepped()
        opt.state[params[1]]["exp_avg"] = base[:300]                                   # with a parameter
        refused(opt, params, "share")
        opt, params, base = stepped()
        both = torch.zeros(400, device=DEV)
        opt.state[params[0]]["exp_avg"], opt.state[params[2]]["exp_avg"] = both[:300], both[100:]      # in part
        refused(opt, params, "share")


@gpu
@pytest.mark.parametrize("begin", [0, 1, 150, 299, 450, 600])
def test_a_gradient_that_the_step_would_write_is_refused(begin):
    """Three parameters side by side and a gradient over them that belongs to the second: only its own place exactly is taken."""
    opt, params, base = stepped()
    params[1].grad = base[begin:begin + 300]
    refused(opt, params, "gradient shares memory")
    params[1].grad = opt.state[params[0]]["exp_avg"]
    refused(opt, params, "gradient shares memory")


@gpu
def test_gradients_that_nothing_writes_are_taken():
    opt, params, base = stepped()
    others = [torch.nn.Parameter(torch.ones(300, device=DEV)) for _ in params]
    ref = FusedAdamW(others, lr=1e-2)
    one = torch.linspace(-1, 1, 300, device=DEV)
    for p in others:
        p.grad = torch.ones_like(p)
    ref.step()
    for p in (*params, *others):
        p.grad = one                                                                   # the same for all
    opt.step()
    ref.step()
    params[1].grad, others[1].grad = params[1].detach(), others[1].detach().clone()    # the parameter itself, in its own place
    opt.step()
    ref.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others))
