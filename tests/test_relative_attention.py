"""Attention with a learned relative position bias (csrc/relattn_*.hip) against the formulas in 64 bits, forward and gradients: every kernel form, one row to
long ones, odd sizes, masks that leave rows empty, lengths of zero, NaN behind a length, entries of -infinity and of a type's lowest value, strides, shared keys,
another stream, graph replays; what it refuses; and a training run of a table together with the optimizer step."""
import ctypes
import math
import os
import re

import pytest
import torch

from fused_optim import FusedAdamW
from lvdm_amd import ops, relative

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
D = 64


class Problem(ctypes.Structure):       # gvd_relattn_problem, as a caller without torch binds it
    _fields_ = ([(n, ctypes.c_int) for n in ("B", "H", "Nq", "Nk", "D", "is_bf16", "table_type", "buckets", "both", "causal")]
                + [("first", ctypes.POINTER(ctypes.c_int)), ("scale", ctypes.c_float), ("q_start", ctypes.c_int), ("q_starts", ctypes.c_void_p),
                   ("kv_lens", ctypes.c_void_p)]
                + [(n, ctypes.c_longlong) for n in ("q_bs", "q_rs", "kv_bs", "kv_rs", "o_bs", "o_rs")])


def bucket_plain(d, buckets, max_distance, both):
    side = buckets // 2 if both else buckets
    n = abs(d) if both else max(-d, 0)
    exact = side // 2
    if n >= exact and side > 1:
        n = min(side - 1, exact + int(math.log(n / exact) / math.log(max_distance / exact) * (side - exact) + 1e-9)) if exact else min(n, side - 1)
    elif side == 1:
        n = 0
    return n + (side if both and d > 0 else 0)


def heads_of(t, H, fm):
    t = t.transpose(0, 1) if fm else t
    return t.reshape(t.shape[0], t.shape[1], H, D).permute(0, 2, 1, 3).double()


def rows_of(t, fm):
    B, H, N, _ = t.shape
    t = t.permute(0, 2, 1, 3).reshape(B, N, H * D)
    return t.transpose(0, 1) if fm else t


def formula(q, k, v, table, H, g=None, *, max_distance=128, bidirectional=True, causal=False, q_start=0, kv_lens=None, scale=None, frame_major=False):
    """The outputs in 64 bits, and for each how far a kernel may be: u = half a step of the 16-bit type; weights are rounded to it before the second products
    (u of each weight), results once more; scores, exponentials and sums are 32 bits, 2^-15 relative for weights from 64 products of about 1 x 1
    (64 x 2^-24 x sum |q k| scale, and that sum is below 16 here); fp16 weights below 2^-14 are off by up to 2^-25 absolutely."""
    u = torch.finfo(q.dtype).eps / 2
    small = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    d32 = 2.0 ** -15
    fm, scale = frame_major, D ** -0.5 if scale is None else scale
    Q, K, V = (heads_of(t, H, fm) for t in (q, k, v))
    B, _, Nq, _ = Q.shape
    K, V = K.expand(B, -1, -1, -1), V.expand(B, -1, -1, -1)
    Nk = K.shape[2]
    start = q_start.tolist() if torch.is_tensor(q_start) else [q_start] * B
    lens = [min(max(n, 0), Nk) for n in kv_lens.tolist()] if kv_lens is not None else [Nk] * B
    i, j = torch.arange(Nq)[:, None], torch.arange(Nk)[None]
    dist = torch.stack([j - (i + s) for s in start])
    lo, hi = int(dist.min()), int(dist.max())
    lut = torch.tensor([bucket_plain(x, table.shape[0], max_distance, bidirectional) for x in range(lo, hi + 1)])
    bucket = lut[dist - lo].to(q.device)
    dist = dist.to(q.device)
    there = torch.stack([j[0] < n for n in lens]).to(q.device)
    seen = there[:, None, :] & (dist <= 0 if causal else torch.ones_like(dist, dtype=torch.bool))
    K, V = (torch.where(there[:, None, :, None], t, 0.0) for t in (K, V))
    T = table.double().clamp(max=10000.0)
    T = torch.where(T <= -10000.0, -math.inf, T)      # such entries mask their bucket
    a = Q @ K.transpose(-1, -2) * scale + T[bucket].permute(0, 3, 1, 2)
    a = torch.where(seen[:, None], a, -math.inf)
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(top == -math.inf, 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    o = p @ V
    e_p = (u + d32) * p + small * (p > 0)
    e_o = e_p @ V.abs() + u * o.abs() + small
    res, err = dict(out=rows_of(o, fm)), dict(out=rows_of(e_o, fm))
    if g is None:
        return res, err
    G = heads_of(g, H, fm)
    dv = p.transpose(-1, -2) @ G
    dp = G @ V.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # dQ first forms dS with delta from the rounded output, off by up to e_delta, and takes (that) P K off again: only the roundings of both see it
    e_delta = (G.abs() * e_o).sum(-1, keepdim=True) + d32 * (p * dp.abs()).sum(-1, keepdim=True)
    e_ds = u * (ds.abs() + 2 * p * e_delta) + 2 * d32 * p * (dp.abs() + delta.abs()) + small
    dq, dk = ds @ K * scale, ds.transpose(-1, -2) @ Q * scale
    res |= dict(dq=rows_of(dq, fm), dk=rows_of(dk, fm), dv=rows_of(dv, fm))
    err |= dict(dq=rows_of(e_ds @ K.abs() * scale + u * dq.abs() + small, fm), dk=rows_of(e_ds.transpose(-1, -2) @ Q.abs() * scale + u * dk.abs() + small, fm),
                dv=rows_of(e_p.transpose(-1, -2) @ G.abs() + u * dv.abs() + small, fm))
    onto = lambda x: torch.zeros(table.shape, dtype=torch.float64, device=q.device).index_add_(  # noqa: E731
        0, bucket.expand(B, -1, -1).reshape(-1), x.permute(0, 2, 3, 1).reshape(-1, H))
    res["dtable"] = onto(ds)
    u_t = torch.finfo(table.dtype).eps / 2
    err["dtable"] = onto(2 * d32 * p * (dp.abs() + delta.abs())) + u_t * res["dtable"].abs() + (2.0 ** -25 if table.dtype == torch.float16 else 1e-30)
    return res, err


def inputs(B, H, Nq, Nk, dtype=torch.float16, table_dtype=torch.float32, buckets=32, frame_major=False, seed=0, device=DEV):
    gen = torch.Generator().manual_seed(seed)
    rows = (lambda n: (n, B, H * D)) if frame_major else (lambda n: (B, n, H * D))
    mk = lambda n: torch.randn(*rows(n), generator=gen).to(dtype).to(device)  # noqa: E731
    return mk(Nq), mk(Nk), mk(Nk), (0.8 * torch.randn(buckets, H, generator=gen)).to(table_dtype).to(device), mk(Nq)


def close(got, want, err, names=None):
    for n in names or want:
        x, y, e = got[n].double(), want[n], err[n]
        assert x.shape == y.shape, n
        off = (x - y).abs()
        assert bool((off <= e).all()), (n, float((off - e).max()), float((off / e.clamp(min=1e-30)).max()))


def check(q, k, v, table, g, H, train=True, **kw):
    want, err = formula(q, k, v, table, H, g if train else None, **kw)
    with torch.no_grad():
        out = ops.relative_bias_attention(q, k, v, table, H, **kw)
    close(dict(out=out), want, err, ["out"])
    if not train:
        return
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = ops.relative_bias_attention(*leaves, H, **kw)
    got = dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, g)), out=out.detach())
    for n, t in zip(("dq", "dk", "dv", "dtable"), leaves):
        assert got[n].dtype == t.dtype
    close(got, want, err)


# ---- on the CPU -----------------------------------------------------------------------------------------------------------------
def test_library_exports_every_declared_symbol():
    import __graft_entry__ as g
    g.build_relattn()
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "gvd_relattn.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(gvd_relattn_[a-z_0-9]+)\s*\(", hdr))
    assert {"gvd_relattn_fwd", "gvd_relattn_bwd", "gvd_relattn_fwd_workspace", "gvd_relattn_bwd_workspace"} <= names
    for n in names:
        assert hasattr(relative.lib(), n), n
    body = hdr[hdr.index("typedef struct gvd_relattn_problem {"):hdr.index("} gvd_relattn_problem;")]
    members = [m for line in re.findall(r"^\s*(?:const )?(?:int|float|long long)\*? (.*);", body, flags=re.M) for m in re.findall(r"\w+", line)]
    assert members == [n for n, _ in Problem._fields_]


@pytest.mark.parametrize("side,max_distance", [(1, 2), (2, 8), (3, 16), (4, 64), (16, 128), (32, 128), (64, 500), (128, 1024)])
def test_buckets_are_the_formula(side, max_distance):
    first = relative.first_distances(side, max_distance)
    assert len(first) == side and first[0] == 0 and list(first) == sorted(first) and first[-1] <= max_distance
    d = torch.arange(-1100, 1101)
    for both in (True, False):
        got = relative.relative_buckets(d, 2 * side if both else side, max_distance, both)
        assert got.tolist() == [bucket_plain(int(x), 2 * side if both else side, max_distance, both) for x in d]


def problem(**kw):
    first = (ctypes.c_int * 4)(0, 1, 2, 9)
    args = dict(B=1, H=2, Nq=40, Nk=50, D=64, is_bf16=0, table_type=0, buckets=8, both=1, causal=0, first=first, scale=0.125, q_start=0, q_bs=40 * 128, q_rs=128,
                kv_bs=50 * 128, kv_rs=128, o_bs=40 * 128, o_rs=128)
    args.update(kw)
    return Problem(**args), first


def test_c_entry_checks_its_arguments_before_any_launch():
    L = relative.lib()
    p, _ = problem()
    assert L.gvd_relattn_fwd_workspace(ctypes.byref(p)) == 0 and L.gvd_relattn_bwd_workspace(ctypes.byref(p)) > 0
    assert L.gvd_relattn_fwd(ctypes.byref(p), *[None] * 8) == -1 and b"null" in L.gvd_relattn_last_error()
    assert L.gvd_relattn_bwd(ctypes.byref(p), *[None] * 13) == -1 and b"null" in L.gvd_relattn_last_error()
    assert L.gvd_relattn_fwd(ctypes.byref(p), *[ctypes.c_void_p(8)] * 5, None, None, None) == -1 and b"aligned" in L.gvd_relattn_last_error()
    odd, far = (ctypes.c_int * 4)(0, 2, 1, 9), (ctypes.c_int * 4)(0, 1, 2, 5000)
    for kw, word in ((dict(B=0), b"sizes"), (dict(Nk=0), b"sizes"), (dict(D=32), b"head dim"), (dict(buckets=7), b"even"), (dict(buckets=0), b"buckets"),
                     (dict(buckets=258), b"too many buckets"), (dict(first=odd), b"descend"), (dict(first=far), b"far"), (dict(scale=0.0), b"scale"),
                     (dict(scale=float("nan")), b"scale"), (dict(q_rs=100), b"strides"), (dict(table_type=3), b"type"), (dict(is_bf16=2), b"type"),
                     (dict(q_start=1 << 30), b"q_start"), (dict(B=1 << 20, H=1 << 12), b"too many"), (dict(Nq=1 << 25), b"too many")):
        bad, _keep = problem(**kw)
        assert L.gvd_relattn_fwd_workspace(ctypes.byref(bad)) == -1 and word in L.gvd_relattn_last_error(), (kw, L.gvd_relattn_last_error())
        assert L.gvd_relattn_bwd_workspace(ctypes.byref(bad)) == -1
        assert L.gvd_relattn_fwd(ctypes.byref(bad), *[ctypes.c_void_p(16)] * 8) == -1 and L.gvd_relattn_bwd(ctypes.byref(bad), *[ctypes.c_void_p(16)] * 13) == -1
    long, _ = problem(Nq=600, Nk=3000)            # its keys are walked in parts, which need room
    assert L.gvd_relattn_fwd_workspace(ctypes.byref(long)) > 0
    assert L.gvd_relattn_fwd(ctypes.byref(long), *[ctypes.c_void_p(16)] * 5, None, None, None) == -1 and b"workspace" in L.gvd_relattn_last_error()
    many, _ = problem(B=1 << 21, H=8, Nq=1, Nk=40)
    assert L.gvd_relattn_fwd(ctypes.byref(many), *[ctypes.c_void_p(16)] * 8) == -1 and b"workgroups" in L.gvd_relattn_last_error()
    starts, _ = problem(q_starts=16)
    assert L.gvd_relattn_bwd(ctypes.byref(starts), *[ctypes.c_void_p(16)] * 13) == -1 and b"q_start" in L.gvd_relattn_last_error()
    shared, _ = problem(B=2, kv_bs=0)
    assert L.gvd_relattn_bwd(ctypes.byref(shared), *[ctypes.c_void_p(16)] * 13) == -1 and b"shared" in L.gvd_relattn_last_error()


@pytest.fixture
def reference_math():
    ops.use_reference_math(True)
    yield
    ops.use_reference_math(False)


def test_refusals_on_the_host(reference_math):
    q, k, v, t, _ = inputs(2, 3, 5, 7, device="cpu", dtype=torch.float32)
    call = ops.relative_bias_attention
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    for args, kw in (((q[0], k, v, t, 3), {}), ((q, k, v[:, :6], t, 3), {}), ((q, k, v, t, 5), {}), ((q, k, v, t, 0), {}), ((q, k[..., :64], v[..., :64], t, 3), {}),
                     ((q, k, v, t[:, :2], 3), {}), ((q, k, v, t[:7], 3), {}), ((q, k, v, t.double(), 3), {}), ((q, k, v, t, 3), dict(max_distance=8)),
                     ((q, k, v, t, 3), dict(max_distance=2000)), ((q, k, v, t, 3), dict(scale=0.0)), ((q, k, v, t, 3), dict(scale=float("nan"))),
                     ((q, k, v, t, 3), dict(kv_lens=i32(1))), ((q, k, v, t, 3), dict(kv_lens=torch.tensor([1, 2]))), ((q, k, v, t, 3), dict(q_start=i32(1, 2, 3))),
                     ((q, k, v, t, 3), dict(q_start=1 << 30)), ((q, k.expand(3, 2, 7, 192)[0], v, t, 3), dict(frame_major=True)), ((q, k, v, t[:0], 3), {})):
        with pytest.raises(ValueError):
            call(*args, **kw)


def test_cpu_tensors_raise_outside_the_tests():
    q, k, v, t, _ = inputs(1, 1, 2, 2, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.relative_bias_attention(q, k, v, t, 1)


@pytest.mark.parametrize("kw", [dict(), dict(causal=True, bidirectional=False), dict(causal=True, q_start=-2), dict(frame_major=True, scale=0.3)])
def test_the_explicit_form_and_its_gradients(reference_math, kw):
    q, k, v, t, g = inputs(2, 3, 5, 5, device="cpu", dtype=torch.float32, frame_major=kw.get("frame_major", False))
    kw = dict(kw, kv_lens=torch.tensor([4, 0], dtype=torch.int32))
    if not kw.get("frame_major"):
        k[0, 4], v[0, 4], k[1], v[1] = float("nan"), float("inf"), float("nan"), float("nan")
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, t)]
    out = ops.relative_bias_attention(*leaves, 3, **kw)
    want, _ = formula(q, k, v, t, 3, g, **kw)
    got = dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, g)), out=out.detach())
    for n, y in want.items():
        torch.testing.assert_close(got[n].double(), y, rtol=1e-5, atol=1e-5, msg=n)
    # the formula's own gradients against differences (64 bits, central, h = 1e-5: error ~ h^2)
    qd, kd, vd, td = (x.double() for x in (q, k, v, t))
    f = lambda table: float((formula(q, k, v, table, 3, None, **kw)[0]["out"] * g.double()).sum())  # noqa: E731
    for b, h in ((0, 0), (1, 2), (17, 1)):
        e = torch.zeros_like(td)
        e[b, h] = 1e-5
        assert abs((f(td + e) - f(td - e)) / 2e-5 - float(want["dtable"][b, h])) < 1e-6


def test_lengths_of_zero_on_the_host(reference_math):
    t = torch.zeros(8, 1)
    for nq, nk in ((0, 3), (3, 0), (0, 0)):
        q, k = torch.randn(2, nq, 64), torch.randn(2, nk, 64)
        assert ops.relative_bias_attention(q, k, k, t, 1).shape == (2, nq, 64)


# ---- on the device: forms and sizes ------------------------------------------------------------------------------------------------
DTYPES = [torch.float16, torch.bfloat16]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 16, 25, 31, 32])
def test_frames(n, dtype):
    """The frames of a pixel, frames outermost: the wave-an-item form, more items than waves at the larger batch."""
    for B, H in ((1, 1), (3, 5), (700, 3)):
        q, k, v, t, g = inputs(B, H, n, n, dtype, frame_major=True, seed=n)
        check(q, k, v, t, g, H, frame_major=True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk", [(33, 33), (64, 64), (65, 63), (1, 40), (5, 300), (130, 1), (127, 129), (200, 77), (300, 300)])
def test_rows(nq, nk, dtype):
    q, k, v, t, g = inputs(2, 3, nq, nk, dtype, seed=nq)
    check(q, k, v, t, g, 3)
    check(q, k, v, t, g, 3, causal=True, bidirectional=False, q_start=nk - nq)


@gpu
@pytest.mark.parametrize("table_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("buckets,max_distance", [(2, 2), (8, 64), (32, 128), (64, 500), (256, 1024)])
def test_tables(buckets, max_distance, table_dtype):
    q, k, v, t, g = inputs(1, 2, 700, 650, torch.bfloat16, table_dtype, buckets, seed=buckets)
    check(q, k, v, t, g, 2, max_distance=max_distance)
    if buckets <= 128:
        check(q, k, v, t, g, 2, max_distance=max_distance, bidirectional=False)
    q, k, v, t, g = inputs(5, 2, 20, 30, torch.float16, table_dtype, buckets, seed=buckets)
    check(q, k, v, t, g, 2, max_distance=max_distance)


@gpu
@pytest.mark.parametrize("nq,nk", [(1, 5000), (2, 3000), (3, 1111), (4, 257), (7, 2000), (600, 3000)])
def test_keys_in_parts(nq, nk):
    """Few rows against many keys: the keys are cut and joined."""
    for dtype in DTYPES:
        q, k, v, t, g = inputs(2, 5, nq, nk, dtype, seed=nk)
        check(q, k, v, t, g, 5, train=False)
        check(q, k, v, t, g, 5, train=False, causal=True, bidirectional=False, q_start=torch.tensor([nk - nq, 3], dtype=torch.int32, device=DEV),
              kv_lens=torch.tensor([nk, 2], dtype=torch.int32, device=DEV))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,nq,nk", [(2, 3, 140, 200), (1, 2, 300, 700), (1, 2, 70, 1100), (1, 5, 333, 3001), (3, 8, 129, 1001), (8, 20, 130, 75), (1, 20, 5, 4000)])
def test_every_division_of_the_work(B, H, nq, nk, dtype):
    """128 or 256 rows a workgroup, four waves or eight, the keys whole or in parts: with and without what the backward keeps, whole and ragged, causal from the middle."""
    q, k, v, t, g = inputs(B, H, nq, nk, dtype, seed=nq)
    check(q, k, v, t, g, H)
    lens = torch.tensor([nk - 1, nk // 2, 1, 0, nk, 64, 65, 2][:B], dtype=torch.int32, device=DEV)
    check(q, k, v, t, g, H, causal=True, q_start=nk // 2, kv_lens=lens)


@gpu
def test_a_table_of_32_bits_has_a_gradient_of_32_bits():
    """Sums that cancel: with delta from the rounded output the error would be about 2^-10; independent errors of 32 bits leave below 1e-5 of the norm."""
    for kw, shape in ((dict(), (1, 4, 500, 500)), (dict(causal=True), (2, 2, 301, 301)), (dict(frame_major=True), (300, 4, 25, 25))):
        q, k, v, t, g = inputs(*shape, torch.bfloat16, seed=1, frame_major=kw.get("frame_major", False))
        want, _ = formula(q, k, v, t, shape[1], g, **kw)
        t.requires_grad_(True)
        (dt,) = torch.autograd.grad(ops.relative_bias_attention(q, k, v, t, shape[1], **kw), t, g)
        assert float((dt.double() - want["dtable"]).norm() / want["dtable"].norm()) < 1e-5


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_with_a_mean(dtype):
    """dS is a difference of numbers of the mean's size.  Two roundings to the type lie between exact sums and each gradient (dS or P as a factor, the result):
    2 x eps / 2 of the norm, where a delta from the rounded output alone would leave about ten times that."""
    q, k, v, t, g = inputs(1, 3, 300, 300, dtype, seed=3)
    k, v = (k.float() + 0.5).to(dtype), (v.float() + 3.0).to(dtype)
    want, _ = formula(q, k, v, t, 3, g)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
    got = dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(ops.relative_bias_attention(*leaves, 3), leaves, g)))
    for n in ("dq", "dk", "dv"):
        assert float((got[n].double() - want[n]).norm() / want[n].norm()) < torch.finfo(dtype).eps, n


# ---- masks -----------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n,frame_major", [(25, True), (25, False), (100, False), (333, False)])
@pytest.mark.parametrize("causal,q_start", [(False, 0), (True, 0), (True, -3), (True, 5), (True, -1000)])
def test_lengths_and_rows_that_see_nothing(n, frame_major, causal, q_start):
    q, k, v, t, g = inputs(6, 2, n, n, torch.bfloat16, seed=n, frame_major=frame_major)
    lens = torch.tensor([n, 0, 1, n - 1, n + 7, -4], dtype=torch.int32, device=DEV)
    for b, m in enumerate(lens.tolist()):
        m = max(m, 0)
        for x in (k, v):
            (x[m:, b] if frame_major else x[b, m:]).fill_(float("nan"))
        if m < n:
            (v[m:, b] if frame_major else v[b, m:])[:1].fill_(float("inf"))
    check(q, k, v, t, g, 2, causal=causal, q_start=q_start, kv_lens=lens, frame_major=frame_major)


@gpu
@pytest.mark.parametrize("n", [20, 90, 700])
def test_entries_of_minus_infinity_and_of_the_lowest_value(n):
    q, k, v, t, g = inputs(2, 3, n, n, torch.float16, torch.float32, seed=5)
    t[3:5] = float("-inf")                       # buckets that are masked
    check(q, k, v, t, g, 3)
    t[:, 1] = float("-inf")                      # a head that sees nothing
    check(q, k, v, t, g, 3)
    for low in (torch.finfo(torch.float32).min, -65504.0, -1e9):   # a mask by a large number
        for both in (True, False):
            t = torch.full((32, 3), low, device=DEV)
            check(q, k, v, t, g, 3, bidirectional=both)
            t[0] = 0.5
            check(q, k, v, t, g, 3, bidirectional=both)


@gpu
def test_large_scores():
    """Scores up to a few hundred: the running maximum moves and weights stay finite."""
    q, k, v, t, g = inputs(1, 2, 300, 400, torch.bfloat16, seed=6)
    t[7] += 200.0
    want, err = formula(q, k, v, t, 2, scale=4.0)
    out = ops.relative_bias_attention(q, k, v, t, 2, scale=4.0)
    assert bool(torch.isfinite(out).all())
    close(dict(out=out), want, dict(out=33 * err["out"]), ["out"])   # scores are 32 times as large as the bound of 16 counts with, and so are their errors


# ---- memory: strides, alignment, sharing, offsets -------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n", [25, 150])
def test_strides(n):
    B, H = 3, 2
    C = H * D
    gen = torch.Generator().manual_seed(0)
    t = torch.randn(32, H, generator=gen).to(DEV)
    packed = torch.randn(B, n, 3 * C, generator=gen).half().to(DEV)
    q, k, v = packed[..., :C], packed[..., C:2 * C], packed[..., 2 * C:]
    want, err = formula(q, k, v, t, H)
    close(dict(out=ops.relative_bias_attention(q, k, v, t, H)), want, err, ["out"])
    wide = torch.randn(B, n + 5, C + 8, generator=gen).half().to(DEV)
    v2 = wide[:, 2:n + 2, 8:]                    # other strides than k's, a row and a channel offset
    want, err = formula(q, k, v2, t, H)
    close(dict(out=ops.relative_bias_attention(q, k, v2, t, H)), want, err, ["out"])
    odd = torch.randn(B * n * C + 1, generator=gen).half().to(DEV)[1:].view(B, n, C)   # 2 bytes off every alignment
    want, err = formula(odd, k, odd, t, H)
    close(dict(out=ops.relative_bias_attention(odd, k, odd, t, H)), want, err, ["out"])
    turned = q.contiguous().transpose(0, 1)      # [n, B, C] view: frame-major of the same memory
    want, err = formula(turned, turned, turned, t, H, frame_major=True)
    close(dict(out=ops.relative_bias_attention(turned, turned, turned, t, H, frame_major=True)), want, err, ["out"])
    tt = torch.randn(H, 32, generator=gen).to(DEV).t()
    leaves = [x.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for x in (q, k, v, tt)]
    g = torch.randn(n, B, C, generator=gen).half().to(DEV).transpose(0, 1)
    out = ops.relative_bias_attention(*leaves, H)
    want, err = formula(q, k, v, tt, H, g)
    got = dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, g)), out=out.detach())
    close(got, want, err)


@gpu
@pytest.mark.parametrize("n", [25, 150])
def test_keys_and_values_shared_by_the_batch(n):
    q, k, v, t, g = inputs(4, 2, n, n, torch.bfloat16, seed=2)
    k, v = k[:1].clone(), v[:1].clone()
    want, err = formula(q, k, v, t, 2, g)
    for args in ((q, k, v), (q, k.expand(4, -1, -1), v.expand(4, -1, -1))):
        close(dict(out=ops.relative_bias_attention(*args, t, 2)), want, err, ["out"])
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
    got = dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(ops.relative_bias_attention(*leaves, 2), leaves, g)))
    for x in ("dk", "dv"):   # summed over the batch from gradients of 16 bits: each rounded (in err), the sum once more per addition
        want[x], err[x] = want[x].sum(0, keepdim=True), err[x].sum(0, keepdim=True) + 4 * 2.0 ** -8 * want[x].abs().sum(0, keepdim=True)
    close(got, want, err, ["dq", "dk", "dv", "dtable"])


@gpu
def test_offsets_beyond_32_bits():
    """A cache of 8.6e9 bytes and rows of it behind 2^32 bytes: the last batch entry alone is compared."""
    B, H, n = 2, 1, 40
    big = torch.zeros(B, 1 << 25, 64, dtype=torch.float16, device=DEV)[:, -n:]
    q, k, v, t, _ = inputs(B, H, 3, n, seed=3)
    big.copy_(k)
    assert big.stride(0) * 2 >= 1 << 32
    want, err = formula(q, k, v, t, H)
    full = torch.zeros(B, 1 << 25, 64, dtype=torch.float16, device=DEV)[:, -n:]
    full.copy_(v)
    close(dict(out=ops.relative_bias_attention(q, big, full, t, H)), want, err, ["out"])
    q2, _, _, _, _ = inputs(B, H, 50, n, seed=4)
    want, err = formula(q2, k, v, t, H)
    close(dict(out=ops.relative_bias_attention(q2, big, full, t, H)), want, err, ["out"])


@gpu
def test_lengths_of_zero():
    t = torch.zeros(8, 1, device=DEV, requires_grad=True)
    for B, nq, nk in ((2, 0, 3), (2, 3, 0), (0, 3, 3)):
        q = torch.randn(B, nq, 64, device=DEV).half().requires_grad_(True)
        k = torch.randn(B, nk, 64, device=DEV).half().requires_grad_(True)
        out = ops.relative_bias_attention(q, k, k, t, 1)
        assert out.shape == q.shape and bool((out == 0).all())
        for x, y in zip(torch.autograd.grad(out, (q, k, t), torch.ones_like(out)), (q, k, t)):
            assert x.shape == y.shape and bool((x == 0).all())


@gpu
def test_refusals_on_the_device():
    q, k, v, t, g = inputs(2, 1, 40, 40)
    with pytest.raises(NotImplementedError, match="q_start"):
        ops.relative_bias_attention(q.requires_grad_(True), k, v, t, 1, q_start=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="kv_lens"):
        ops.relative_bias_attention(q, k, v, t, 1, kv_lens=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="table"):
        ops.relative_bias_attention(q, k, v, t.cpu(), 1)
    import lvdm_amd
    with lvdm_amd.allow_torch_fallback(False), pytest.raises(RuntimeError, match="no hand-written kernel"):
        ops.relative_bias_attention(q.detach().float(), k.float(), v.float(), t, 1)


# ---- repeats, streams, graphs ------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n", [25, 400])
def test_the_same_call_gives_the_same_bits(n):
    q, k, v, t, g = inputs(3, 2, n, n, torch.bfloat16)
    leaves = [x.requires_grad_(True) for x in (q, k, v, t)]
    runs = []
    for _ in range(3):
        out = ops.relative_bias_attention(*leaves, 2)
        runs.append([out.detach(), *torch.autograd.grad(out, leaves, g)])
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


@gpu
def test_runs_on_the_current_stream():
    q, k, v, t, g = inputs(2, 2, 600, 600)
    want, err = formula(q, k, v, t, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k2 = (k * 2) * 0.5                       # made on the side stream
        out = ops.relative_bias_attention(q, k2, v, t, 2)
    torch.cuda.current_stream().wait_stream(side)
    close(dict(out=out), want, err, ["out"])


@gpu
@pytest.mark.parametrize("shape", [(4, 3, 25, 25), (2, 2, 200, 200), (3, 2, 1, 3000)])
def test_replays_equal_eager_calls(shape):
    """Two captured graphs of different sizes in one program, replayed in turn with eager calls between them."""
    lens = torch.tensor([shape[3]] * shape[0], dtype=torch.int32, device=DEV)
    graphs = []
    for seed, cut in ((0, 0), (1, 1)):
        q, k, v, t, _ = inputs(shape[0], shape[1], shape[2], shape[3] - cut, seed=seed)
        with torch.no_grad():
            for _ in range(2):
                ops.relative_bias_attention(q, k, v, t, shape[1], kv_lens=lens)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = ops.relative_bias_attention(q, k, v, t, shape[1], kv_lens=lens)
        graphs.append((graph, q, k, v, t, out))
    for rep in range(4):
        for graph, q, k, v, t, out in graphs:
            q.copy_(torch.randn(q.shape, device=DEV))
            lens.fill_(max(1, shape[3] - 7 * rep))
            graph.replay()
            with torch.no_grad():
                eager = ops.relative_bias_attention(q, k, v, t, shape[1], kv_lens=lens)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), rep


@gpu
@pytest.mark.parametrize("n", [25, 300])
def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(n):
    """Refused in the forward, before there is a backward to capture; the capture goes on without it, and works once the eager graph is gone."""
    H = 3
    q, k, v = (torch.randn(2, n, H * D, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    table = torch.randn(32, H, device=DEV, requires_grad=True)
    g = torch.randn_like(q)
    eager = ops.relative_bias_attention(q, k, v, table, H)          # lives on
    want, = torch.autograd.grad(eager, [table], g, retain_graph=True)
    side = torch.cuda.Stream()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph, stream=side):
        x += 1
        with pytest.raises(RuntimeError, match="eager graph"):
            ops.relative_bias_attention(q, k, v, table, H)
        with torch.no_grad():
            y = ops.relative_bias_attention(q, k, v, table, H)      # inference is no concern
    graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(y, ops.relative_bias_attention(q, k, v, table, H)) and float(x[0]) == 1
    del eager
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2, stream=side):
        got, = torch.autograd.grad(ops.relative_bias_attention(q, k, v, table, H), [table], g)
    for _ in range(3):
        got.zero_()
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@gpu
def test_a_captured_pass_of_two_layers_that_share_a_table_replays():
    """The second use of the table meets its accumulating node, made in the same capture."""
    H, n = 3, 70
    q, k, v = (torch.randn(2, n, H * D, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    table = torch.randn(32, H, device=DEV, requires_grad=True)

    def one():
        x = ops.relative_bias_attention(q, k, v, table, H)
        y = ops.relative_bias_attention(x, k, v, table, H, causal=True)
        got, = torch.autograd.grad(y, [table], torch.ones_like(y))
        return y.detach(), got
    one()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, got = one()
    for rep in range(4):
        q.copy_(torch.randn(q.shape, device=DEV))
        graph.replay()
        want = one()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(got, want[1]), rep


@gpu
@pytest.mark.parametrize("n", [25, 70])
def test_the_graph_is_an_ordinary_one(n):
    """A second pass over a kept graph, none over a freed one, none over inputs changed in place; gradients of some inputs only; no second derivatives."""
    H = 2
    q, k, v, t, g = inputs(2, H, n, n, torch.bfloat16)
    lens = torch.tensor([n, n // 2], dtype=torch.int32, device=DEV)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
    out = ops.relative_bias_attention(*leaves, H, kv_lens=lens)
    first = torch.autograd.grad(out, leaves, g, retain_graph=True)
    second = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(x, y) for x, y in zip(first, second))
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(out, leaves, g)
    for i in range(4):
        some = [x.detach().requires_grad_(j == i) for j, x in enumerate((q, k, v, t))]
        got, = torch.autograd.grad(ops.relative_bias_attention(*some, H, kv_lens=lens), [some[i]], g)
        assert torch.equal(got, first[i])
    for changed in (leaves[1], lens):
        out = ops.relative_bias_attention(*leaves, H, kv_lens=lens)
        with torch.no_grad():
            changed.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, leaves, g)
    out = ops.relative_bias_attention(*leaves, H)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out, leaves, g, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(leaves[0], torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.relative_bias_attention(dual, *leaves[1:], H)


@gpu
@pytest.mark.parametrize("n", [25, 200])
def test_a_captured_training_pass_replays(n):
    q, k, v, t, g = inputs(2, 2, n, n, torch.bfloat16)

    def one():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
        out = ops.relative_bias_attention(*leaves, 2, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = one()
    for rep in range(4):
        q.copy_(torch.randn(q.shape, device=DEV))
        t.copy_(torch.randn(t.shape, device=DEV))
        graph.replay()
        eager = one()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, eager)), rep


# ---- together -----------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n,frame_major", [(25, True), (130, False)])
def test_training_a_table_and_its_projection_with_the_optimizer(n, frame_major, bits):
    """A temporal layer's bias table and query projection: attention forward and backward, then the step; each step's gradients against the formula's, each
    update against AdamW's on those gradients."""
    H, B = 2, 6
    x, k, v, t, g = inputs(B, H, n, n, torch.bfloat16, frame_major=frame_major, seed=11)
    w = (torch.eye(H * D) + 0.05 * torch.randn(H * D, H * D, generator=torch.Generator().manual_seed(1))).bfloat16().to(DEV)
    table, weight = torch.nn.Parameter(t), torch.nn.Parameter(w)
    opt = FusedAdamW([dict(params=[table], lr=1e-2), dict(params=[weight], lr=1e-3)], weight_decay=0.0, state_bits=bits)
    for step in range(3):
        q = x @ weight
        out = ops.relative_bias_attention(q, k, v, table, H, frame_major=frame_major, max_distance=64)
        opt.zero_grad()
        out.backward(g)
        want, err = formula(q.detach(), k, v, table.detach(), H, g, frame_major=frame_major, max_distance=64)
        close(dict(out=out.detach(), dtable=table.grad), want, err, ["out", "dtable"])
        assert weight.grad.dtype == torch.bfloat16 and bool(torch.isfinite(weight.grad).all()) and float(weight.grad.abs().max()) > 0
        before = {p: (p.detach().double(), *[m.double() for m in opt.moments(p) or (torch.zeros_like(p, dtype=torch.float32),) * 2]) for p in (table, weight)}
        opt.step()
        for p, lr in ((table, 1e-2), (weight, 1e-3)):
            p0, m0, v0 = before[p]
            m1, v1 = 0.9 * m0 + 0.1 * p.grad.double(), 0.999 * v0 + 0.001 * p.grad.double() ** 2
            upd = lr / (1 - 0.9 ** (step + 1)) * m1 / ((v1 / (1 - 0.999 ** (step + 1))).sqrt() + 1e-8)
            half = torch.finfo(p.dtype).eps / 2
            # the step's own float32: 16 x 2^-24 of an update whose terms are at most ten times lr (m <= 0.9 m0 + 0.1 g each below its root's 32 times)
            assert bool(((p.detach().double() - (p0 - upd)).abs() <= half * (p0 - upd).abs() * 1.01 + 16 * 2.0 ** -24 * (p0.abs() + 32 * lr)).all()), (step, lr)
