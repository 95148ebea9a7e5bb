"""relative_bias_attention in the calls where it can answer wrongly without a word: tangents, entries brought to a limit, tensors that are made under another default
device, captures beside eager graphs, scores that grow along the keys, batches of many short rows; against its explicit form in 64 bits."""
import pytest
import torch

import test_relative_attention as plain
from lvdm_amd import ops, relative

gpu = pytest.mark.gpu
DEV = "cuda:0"
D = 64


def inputs(B, H, Nq, Nk, dtype=torch.float16, table_dtype=torch.float32, buckets=32, frame_major=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rows = (lambda n: (n, B, H * D)) if frame_major else (lambda n: (B, n, H * D))
    mk = lambda n: torch.randn(*rows(n), generator=gen).to(dtype).to(DEV)  # noqa: E731
    return mk(Nq), mk(Nk), mk(Nk), (0.8 * torch.randn(buckets, H, generator=gen)).to(table_dtype).to(DEV), mk(Nq)


def formula(q, k, v, t, H, g, d32, **kw):
    """Results in 64 bits, by the explicit form and autograd, and how far a kernel may be: d32 is the relative error of a weight before it is rounded; weights and dS are
    rounded to the rows' type (u), results once more.  dS = P (dP - delta): each factor d32 off, delta as a sum of weights times dP.  dQ forms dS from the delta that the
    rounded output gave, e_delta off at most, and takes (that) P K off again: the roundings of both see it."""
    u, u_t = torch.finfo(q.dtype).eps / 2, torch.finfo(t.dtype).eps / 2
    small = 2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -126
    leaves = [x.detach().double().requires_grad_(True) for x in (q, k, v, t)]
    out = relative.relative_bias_attention_math(*leaves, H, **kw)
    want = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *torch.autograd.grad(out, leaves, g.double()))))
    scale = kw.get("scale") or D ** -0.5
    heads = lambda x: x.detach().double().reshape(*x.shape[:2], H, D).transpose(1, 2)  # noqa: E731
    rows = lambda x: x.transpose(1, 2).reshape(x.shape[0], x.shape[2], H * D)  # noqa: E731
    Q, K, V, G = (heads(x) for x in (q, k, v, g))
    dist = torch.arange(K.shape[2], device=DEV)[None] - torch.arange(Q.shape[2], device=DEV)[:, None]
    bucket = relative.relative_buckets(dist, t.shape[0], kw.get("max_distance", 128), kw.get("bidirectional", True))
    T = t.detach().double().clamp(max=10000.0)
    a = Q @ K.transpose(-1, -2) * scale + T.masked_fill(T <= -10000.0, float("-inf"))[bucket].permute(2, 0, 1)
    if kw.get("causal"):
        a = a.masked_fill(dist > 0, float("-inf"))
    p = a.softmax(-1)
    dp = G @ V.transpose(-1, -2)
    spread = (p * dp.abs()).sum(-1, keepdim=True)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    e_p = (u + d32) * p + small
    e_delta = 2 * (u + d32) * (G.abs() * (p @ V.abs())).sum(-1, keepdim=True)
    e_ds = u * (ds.abs() + 2 * p * e_delta) + 3 * d32 * p * (dp.abs() + spread) + small
    e_t = torch.zeros_like(want["dtable"]).index_add_(0, bucket.reshape(-1), (3 * d32 * p * (dp.abs() + spread)).sum(0).permute(1, 2, 0).reshape(-1, H))
    err = dict(out=rows(e_p @ V.abs()), dq=rows(e_ds @ K.abs()) * scale, dk=rows(e_ds.transpose(-1, -2) @ Q.abs()) * scale, dv=rows(e_p.transpose(-1, -2) @ G.abs()), dtable=e_t)
    return want, {n: 1.01 * e + (u_t if n == "dtable" else u) * want[n].abs() + 2.0 ** -24 for n, e in err.items()}


def kernels(q, k, v, t, H, g, **kw):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
    out = ops.relative_bias_attention(*leaves, H, **kw)
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *torch.autograd.grad(out, leaves, g))))


def close(got, want, err):
    for n, y in want.items():
        off = (got[n].double() - y).abs()
        assert bool((off <= err[n]).all()), (n, float((off / err[n]).max()))


# ---- entries that are brought to a limit -----------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n", [25, 70, 200])
@pytest.mark.parametrize("table_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_an_entry_above_the_limit_counts_as_the_limit_and_has_no_gradient(table_dtype, n):
    """Scores start from 10000 / scale = 80000, whose half step is 2^-8: 64 additions leave a score at most 64 x 2^-8 / 8 = 2^-5 off, a weight (over a sum of
    weights) exp(2^-4) - 1 < 0.065."""
    H = 2
    q, k, v, t, g = inputs(2, H, n, n, table_dtype=table_dtype, seed=n)
    for entry in (1e4, 2e4, 6e4, float("inf")):
        t[3], t[6] = entry, entry                 # keys three and six behind: the softmax is between the two
        if table_dtype == torch.bfloat16 and entry == 1e4:
            t[3], t[6] = 9984.0, 9984.0           # (the value below 10000)
        want, err = formula(q, k, v, t, H, g, 0.065)
        got = kernels(q, k, v, t, H, g)
        close(got, want, err)
        if entry == 1e4:
            first = got
            assert bool((want["dtable"][[3, 6]] != 0).all()) and bool((got["dtable"][[3, 6]] != 0).all())     # at the limit itself there is one
            continue
        assert bool((want["dtable"][[3, 6]] == 0).all()) and bool((got["dtable"][[3, 6]] == 0).all())
        if table_dtype != torch.bfloat16:
            assert all(torch.equal(got[x], first[x]) for x in ("out", "dq", "dk", "dv"))   # whatever the entry: the same results


@gpu
@pytest.mark.parametrize("n", [25, 70])
def test_an_entry_that_masks_has_no_gradient(n):
    q, k, v, t, g = inputs(2, 2, n, n, seed=n)
    for entry in (-1e4, -6e4, float("-inf")):
        t[3] = entry
        want, err = formula(q, k, v, t, 2, g, 2.0 ** -15)
        got = kernels(q, k, v, t, 2, g)
        close(got, want, err)
        assert bool((got["dtable"][3] == 0).all()) and bool((got["dtable"][4] != 0).all())


# ---- other default devices ---------------------------------------------------------------------------------------------------------
@pytest.fixture
def nothing_kept():
    relative._first_tensor.cache_clear()
    yield
    relative._first_tensor.cache_clear()


def test_the_first_distances_lie_on_the_host_whatever_the_default_device(nothing_kept):
    with torch.device("meta"):
        kept = relative._first_tensor(16, 128)
    assert kept.device.type == "cpu" and kept.tolist() == list(relative.first_distances(16, 128)) and relative._first_tensor(16, 128) is kept


def test_first_distances_that_the_host_cannot_read_are_refused():
    q, t = torch.zeros(1, 2, D), torch.zeros(8, 1)
    row = torch.arange(4, dtype=torch.int32)
    call = lambda first: relative.ext().attend(q, q, q, t, 1, first, True, False, 0, None, None, False)  # noqa: E731
    assert call(row) is None                            # (rows on the CPU: left to the caller)
    for first in (row.to("meta"), row.long(), row.view(2, 2), row[::2], row[:0]):
        with pytest.raises(RuntimeError, match="read by the host"):
            call(first)


@gpu
def test_a_call_under_another_default_device(nothing_kept):
    q, k, v, t, g = inputs(2, 2, 25, 25)
    want = kernels(q, k, v, t, 2, g)
    relative._first_tensor.cache_clear()
    with torch.device(DEV):
        got = kernels(q, k, v, t, 2, g)
    assert all(torch.equal(got[n], x) for n, x in want.items())


# ---- forward-mode derivatives ----------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n", [1, 25, 70])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_a_tangent_is_refused_whether_or_not_anything_needs_a_gradient(which, n):
    q, k, v, t, _ = inputs(2, 2, n, n)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        args = [q, k, v, t]
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        assert not args[which].requires_grad
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.relative_bias_attention(*args, 2)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            ops.relative_bias_attention(*args, 2)
        args[(which + 1) % 4] = args[(which + 1) % 4].clone().requires_grad_(True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.relative_bias_attention(*args, 2)
        with torch.inference_mode():      # tangents are not propagated here, by any operator
            out = ops.relative_bias_attention(*args, 2)
    assert torch.equal(out, ops.relative_bias_attention(q, k, v, t, 2))


# ---- captures beside eager graphs -------------------------------------------------------------------------------------------------
def leaves_behind(which, n, H=2):
    """Inputs that reach a leaf through other nodes: () -> (q, k, v, table) made anew from the same leaves, and the leaf."""
    q, k, v, t, _ = inputs(2, H, n, n, torch.bfloat16, seed=n)
    if which == "a table of another memory order":       # (a copy is made of it)
        leaf = t.t().contiguous().t().requires_grad_(True)
        assert not leaf.is_contiguous()
        return lambda: (q, k, v, leaf), leaf
    if which == "keys shared by the batch":              # (expanded)
        leaf = k[:1].clone().requires_grad_(True)
        return lambda: (q, leaf, v[:1], t), leaf
    if which == "a table behind a cast":
        leaf = t.requires_grad_(True)
        return lambda: (q, k, v, leaf.bfloat16()), leaf
    leaf = torch.ones(H * D, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    return lambda: (torch.relu(q * leaf) + q, k, v, t), leaf        # queries behind three nodes


WAYS = ["a table of another memory order", "keys shared by the batch", "a table behind a cast", "queries behind three nodes"]


@gpu
@pytest.mark.parametrize("n", [25, 70])
@pytest.mark.parametrize("which", WAYS)
def test_a_capture_is_refused_where_a_leaf_behind_other_nodes_has_an_eager_graph(which, n):
    make, leaf = leaves_behind(which, n)
    eager = ops.relative_bias_attention(*make(), 2)                 # lives on
    trained = eager.detach().clone()                                # (summed from unrounded weights, inference from rounded ones: other last bits)
    with torch.no_grad():
        inferred = ops.relative_bias_attention(*make(), 2)
    side, graph, x = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph, stream=side):
        x += 1
        with pytest.raises(RuntimeError, match="eager graph"):
            ops.relative_bias_attention(*make(), 2)
        with torch.no_grad():
            y = ops.relative_bias_attention(*make(), 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, inferred) and float(x[0]) == 1
    del eager
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second, stream=side):                     # nothing lives: taken
        out = ops.relative_bias_attention(*make(), 2)
    for _ in range(3):
        out.detach().zero_()
        second.replay()
        torch.cuda.synchronize()
        assert out.requires_grad and torch.equal(out.detach(), trained)


@gpu
def test_a_capture_does_not_go_on_from_an_eager_graph():
    q, k, v, t, _ = inputs(2, 2, 25, 25)
    q = q.requires_grad_(True) * 1.0                                # made before the capture, on another stream
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="eager graph"):
            ops.relative_bias_attention(q, k, v, t, 2)
        y = ops.relative_bias_attention(q.detach(), k, v, t, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.relative_bias_attention(q.detach(), k, v, t, 2))


@gpu
def test_two_streams_of_one_capture_share_a_leaf():
    """The second call meets the table's accumulating node on the other stream, which is captured as well."""
    q, k, v, t, _ = inputs(2, 2, 70, 70, torch.bfloat16)
    t.requires_grad_(True)
    one, two, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=one):
        a = ops.relative_bias_attention(q, k, v, t, 2)
        two.wait_stream(one)
        with torch.cuda.stream(two):
            b = ops.relative_bias_attention(q, k, v, t, 2, causal=True)
        one.wait_stream(two)
    for rep in range(3):
        q.copy_(torch.randn(q.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.relative_bias_attention(q, k, v, t, 2)) and torch.equal(b, ops.relative_bias_attention(q, k, v, t, 2, causal=True)), rep


# ---- sizes beyond 32 bits ------------------------------------------------------------------------------------------------------------
@gpu
def test_sizes_that_an_int_does_not_hold_are_refused():
    """Expanded tensors take no memory: 2^32 + 5 keys would be 5 in 32 bits."""
    q, k, v, t, _ = inputs(1, 1, 3, 1)
    for n in (2 ** 31, 2 ** 32 + 5, 2 ** 25):
        with pytest.raises(RuntimeError, match="too many"):
            ops.relative_bias_attention(q, k.expand(1, n, D), v.expand(1, n, D), t, 1)


# ---- scores that are large, or grow along the keys ---------------------------------------------------------------------------------------
SHAPES = [(1, 2, 25, 30), (1, 2, 3, 700), (1, 2, 140, 700), (2, 3, 300, 400), (1, 2, 70, 1100), (3, 8, 600, 640)]      # every form: short, few, rows whole and in parts


@gpu
@pytest.mark.parametrize("B,H,nq,nk", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_scores_and_their_gradients(B, H, nq, nk, dtype):
    """Scores of several hundred.  64 products of sum |q k| < 128 at a scale of 4 leave a score 64 x 2^-24 x 512 = 2^-9 off at most, a weight (over their sum) 2^-8; the type's
    roundings are no larger than elsewhere."""
    q, k, v, t, g = inputs(B, H, nq, nk, dtype, seed=6)
    heads = lambda x: x.double().reshape(*x.shape[:2], H, D).transpose(1, 2)  # noqa: E731
    assert float((heads(q).abs() @ heads(k).abs().transpose(-1, -2)).max()) < 128
    t[7] += 200.0
    want, err = formula(q, k, v, t, H, g, 2.0 ** -8, scale=4.0)
    close(kernels(q, k, v, t, H, g, scale=4.0), want, err)
    with torch.no_grad():
        close(dict(out=ops.relative_bias_attention(q, k, v, t, H, scale=4.0)), dict(out=want["out"]), err)


@gpu
@pytest.mark.parametrize("B,H,nq,nk", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rise", [0.5, 3.0, 10.0, -5.0])
def test_scores_that_grow_or_fall_from_tile_to_tile(rise, dtype, B, H, nq, nk):
    """By `rise` every 64 keys, 0.5 and 3 below what moves the running maximum (a row's sum of a tile above 2^15) for some tiles, 10 above it at once.  Sums |q k| / 8 stay below
    17 x 10 + 16 < 192: a score is 64 x 2^-24 x 192 < 2^-10 off, a weight 2^-9."""
    q, k, v, t, g = inputs(B, H, nq, nk, dtype, seed=7)
    steps = (torch.arange(nk, device=DEV) // 64).float() * rise
    for h in range(H):
        q[:, :, h * D] = 8.0
        k[:, :, h * D] = steps.to(dtype)
    heads = lambda x: x.double().reshape(*x.shape[:2], H, D).transpose(1, 2)  # noqa: E731
    assert float((heads(q).abs() @ heads(k).abs().transpose(-1, -2)).max()) / 8 < 192
    want, err = formula(q, k, v, t, H, g, 2.0 ** -9)
    close(kernels(q, k, v, t, H, g), want, err)
    with torch.no_grad():
        close(dict(out=ops.relative_bias_attention(q, k, v, t, H)), dict(out=want["out"]), err)


# ---- many short rows ---------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [33, 48, 63, 64])
def test_more_than_32_frames_of_many_pixels(n, dtype):
    """Several workgroups a compute unit one after the other, each with a part of its rows in use."""
    q, k, v, t, g = plain.inputs(900, 3, n, n, dtype, frame_major=True, seed=n)
    plain.check(q, k, v, t, g, 3, frame_major=True)
    lens = torch.arange(900, device=DEV, dtype=torch.int32) % (n + 2)
    plain.check(q, k, v, t, g, 3, frame_major=True, causal=True, kv_lens=lens)


@gpu
@pytest.mark.parametrize("nq", [1, 2, 4])
def test_new_tokens_of_many_sequences(nq):
    q, k, v, t, _ = plain.inputs(1500, 2, nq, 70, torch.bfloat16, seed=nq)
    lens = torch.arange(1500, device=DEV, dtype=torch.int32) % 71
    plain.check(q, k, v, t, None, 2, train=False, causal=True, bidirectional=False, q_start=(lens - nq).to(torch.int32), kv_lens=lens)


# ---- values that are not finite -------------------------------------------------------------------------------------------------------
ALL_FORMS = [(25, 25), (32, 7), (1, 40), (3, 40), (2, 3000), (70, 70), (40, 3000), (300, 200)]


@gpu
@pytest.mark.parametrize("nq,nk", ALL_FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what,value", [("q", float("nan")), ("q", float("inf")), ("k", float("nan")), ("k", float("-inf")), ("v", float("nan"))])
def test_a_score_that_is_no_number_is_not_answered_with_zeros(what, value, dtype, nq, nk):
    """The rows that are NaN by the formula are NaN, with and without gradients, and so are the gradients (a loss scaler looks there); all others are as they were."""
    q, k, v, t, g = inputs(2, 2, nq, nk, dtype)
    want, err = formula(q, k, v, t, 2, g, 2.0 ** -14)
    n = min(nq, nk) - 1
    {"q": q, "k": k, "v": v}[what][1, n] = value
    leaves = [x.detach().double().requires_grad_(True) for x in (q, k, v, t)]
    out = relative.relative_bias_attention_math(*leaves, 2)
    bad = out.isnan()
    assert bool(bad[1].all() if what != "q" else bad[1, n].all()) and not bool(bad[0].any())
    got = kernels(q, k, v, t, 2, g)
    with torch.no_grad():
        plain_out = ops.relative_bias_attention(q, k, v, t, 2)
    for x in (got["out"], plain_out):
        assert torch.equal(x.isnan(), bad)
        assert bool(((x.double() - want["out"]).abs() <= err["out"])[~bad].all())
    for name, y in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, g.double())):
        assert bool(got[name].isnan()[y.isnan()].all()), name
    for name in ("dq", "dk", "dv"):
        assert bool(((got[name].double() - want[name]).abs() <= err[name])[0].all()), name


def nothing_seen(n, way, frame_major=False, device=DEV):
    """(arguments, which [batch, query] see nothing) of two batch entries."""
    none = torch.zeros(2, n, dtype=torch.bool, device=device)
    if way == "causal":
        none[:, :min(3, n)] = True
        return dict(causal=True, q_start=-3), none
    if way == "lengths":
        none[0] = True
        return dict(kv_lens=torch.tensor([0, n], dtype=torch.int32, device=device)), none
    return dict(causal=True, bidirectional=False, max_distance=33), none      # ("table": the entries of the nearest distances mask, so the first rows see nothing)


@pytest.mark.parametrize("way", ["causal", "lengths"])
def test_the_explicit_forms_rows_that_see_nothing_have_no_gradient(way):
    n, H = 7, 2
    gen = torch.Generator().manual_seed(0)
    q, k, v, g = (torch.randn(2, n, H * D, generator=gen) for _ in range(4))
    t = torch.randn(8, H, generator=gen)
    kw, none = nothing_seen(n, way, device="cpu")

    def grads(g):
        leaves = [x.clone().requires_grad_(True) for x in (q, k, v, t)]
        return torch.autograd.grad(relative.relative_bias_attention_math(*leaves, H, **kw), leaves, g)
    for value in (float("nan"), float("inf")):
        assert all(torch.equal(x, y) for x, y in zip(grads(g.masked_fill(none[..., None], value)), grads(g.masked_fill(none[..., None], 0.0))))


@gpu
@pytest.mark.parametrize("n,frame_major", [(1, False), (25, True), (32, False), (70, False), (333, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("way", ["causal", "lengths", "table"])
def test_rows_that_see_nothing_have_no_gradient_whatever_their_outputs_gradient_holds(way, dtype, n, frame_major):
    H = 2
    q, k, v, t, g = inputs(2, H, n, n, dtype, frame_major=frame_major, seed=n)
    kw, none = nothing_seen(n, way)
    if way == "table":
        t[:5] = float("-inf")
        none[:, :min(5, n)] = True
    kw["frame_major"] = frame_major
    rows = (none.t() if frame_major else none)[..., None]
    want = kernels(q, k, v, t, H, g.masked_fill(rows, 0.0), **kw)
    assert all(bool(torch.isfinite(x).all()) for x in want.values()) and bool((want["dv"] != 0).any() if n > 5 else True)
    for value in (float("nan"), float("inf"), 1.0):
        got = kernels(q, k, v, t, H, g.masked_fill(rows, value), **kw)
        for name, x in want.items():
            assert torch.equal(got[name], x), (name, value)
    if way == "lengths":                     # queries of an empty entry are whatever was there
        q2 = q.clone()
        (q2[:, 0] if frame_major else q2[0]).fill_(float("nan"))
        got = kernels(q2, k, v, t, H, g, **kw)
        for name, x in kernels(q, k, v, t, H, g, **kw).items():
            assert torch.equal(got[name], x), name
