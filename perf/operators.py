"""Cases of the training operators that stand next to the rasterizer's and the diffusion path's kernels:

* an AdamW step over many tensors at once (`fused_optim.FusedAdamW`), moments in 32 bits or in 8;
* attention with a learned relative position bias by buckets (`lvdm_amd.ops.relative_bias_attention`): inference, one new token against a
  cache, and a training pass with the gradients of queries, keys, values and the bias table.

With `own` false `run` computes the plain form: elementary torch operations in 32 bits."""
import math
import os
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
D = 64          # channels of a head, as everywhere in the U-Net
BLOCK = 256     # elements that share a scale where moments are held in 8 bits


def _package():
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "guidedvd-3dgs_amd")
    if p not in sys.path:
        sys.path.insert(0, p)


# ---- cases ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the bias tables of four temporal layers: what is trained when only the tables are adapted; all latency
        dict(name="adamw_tables", op="adamw", bits=32, dtype="fp32", model="tables", size=32, wd=0.01, eps=1e-8, step=7),
        # the Gaussians of the default rasterizer benchmark (five tensors: positions, opacities, scales, rotations, SH)
        dict(name="adamw_gaussians_200k", op="adamw", bits=32, dtype="fp32", model="gaussians", size=200000, wd=0.0, eps=1e-15, step=1000),
        # a dense scene: ten times as many, memory-bound throughout
        dict(name="adamw_gaussians_2m", op="adamw", bits=32, dtype="fp32", model="gaussians", size=2000000, wd=0.0, eps=1e-15, step=1000),
        # the default scene with its moments in 8 bits
        dict(name="adamw8_gaussians_200k", op="adamw", bits=8, dtype="fp32", model="gaussians", size=200000, wd=0.0, eps=1e-15, step=1000),
        # a temporal transformer block of the U-Net in 16 bits with 8-bit moments: matrices and vectors mixed
        dict(name="adamw8_block_bf16", op="adamw", bits=8, dtype="bf16", model="block", size=640, wd=0.01, eps=1e-8, step=50),
        # temporal attention at the U-Net's bottleneck for 320x448 video (5 x 7 pixels, 20 heads): small, latency counts
        dict(name="relbias_infer_small", op="infer", dtype="fp16", table="fp16", B=35, H=20, Nq=25, Nk=25, frame_major=True, causal=False,
             ragged=False, buckets=32, max_distance=128),
        # temporal attention of the first level at 576x1024 (72 x 128 pixels, 5 heads, 25 frames), frames outermost
        dict(name="relbias_infer_frames", op="infer", dtype="fp16", table="fp16", B=9216, H=5, Nq=25, Nk=25, frame_major=True, causal=False,
             ragged=False, buckets=32, max_distance=128),
        # the same layer at 320x448 (40 x 56 pixels) in training, the table in 32 bits
        dict(name="relbias_train_frames", op="train", dtype="fp16", table="fp32", B=2240, H=5, Nq=25, Nk=25, frame_major=True, causal=False,
             ragged=False, buckets=32, max_distance=128),
        # a long self-attention row in training: the 36 x 64 tokens of the second level, 10 heads
        dict(name="relbias_train_tokens", op="train", dtype="bf16", table="fp32", B=1, H=10, Nq=2304, Nk=2304, frame_major=False, causal=False,
             ragged=False, buckets=32, max_distance=128),
        # a padded causal batch of odd length in training, the table in 16 bits; one entry of the batch is empty
        dict(name="relbias_train_ragged", op="train", dtype="bf16", table="bf16", B=3, H=8, Nq=1111, Nk=1111, frame_major=False, causal=True,
             ragged=True, buckets=32, max_distance=128),
        # all 9216 tokens of the first level in one row, 5 heads
        dict(name="relbias_infer_tokens", op="infer", dtype="fp16", table="fp16", B=1, H=5, Nq=9216, Nk=9216, frame_major=False, causal=False,
             ragged=False, buckets=32, max_distance=128),
        # one new token each for 16 sequences against their caches of up to 8192 tokens
        dict(name="relbias_serve_one", op="infer", dtype="bf16", table="bf16", B=16, H=10, Nq=1, Nk=8192, frame_major=False, causal=True,
             ragged=True, buckets=32, max_distance=128),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["adamw", "adamw", "infer", "infer", "serve", "train", "train"])
    if kind == "adamw":
        model = rng.choice(["tables", "gaussians", "gaussians", "block"])
        size = {"tables": _log(rng, 4, 256), "gaussians": _log(rng, 100, 1500000), "block": 8 * _log(rng, 4, 160)}[model]
        return dict(op="adamw", bits=rng.choice([32, 8]), dtype="fp32" if model != "block" else rng.choice(["bf16", "fp16", "fp32"]), model=model,
                    size=size, wd=rng.choice([0.0, 0.01]), eps=rng.choice([1e-8, 1e-15]), step=_log(rng, 1, 10000))
    c = dict(op="train" if kind == "train" else "infer", dtype=rng.choice(["fp16", "bf16"]), table=rng.choice(["fp32", "fp16", "bf16"]))
    if kind == "serve":
        c |= dict(B=_log(rng, 1, 64), H=rng.choice([5, 8, 10, 20]), Nq=rng.choice([1, 1, 2, 7]), Nk=_log(rng, 8, 8192), frame_major=False,
                  causal=True, ragged=True)
    elif rng.random() < 0.5:   # the frames of many pixels
        n = rng.randint(1, 32)
        c |= dict(B=_log(rng, 1, 8000 if kind == "infer" else 4000), H=rng.choice([5, 8, 10]), Nq=n, Nk=n, frame_major=True,
                  causal=rng.random() < 0.3, ragged=False)
    else:                      # long rows
        n = _log(rng, 33, 6000 if kind == "infer" else 2300)
        c |= dict(B=rng.choice([1, 2, 3]) if n < 1500 else 1, H=rng.choice([5, 8, 10]), Nq=n, Nk=n, frame_major=False,
                  causal=rng.random() < 0.4, ragged=rng.random() < 0.3)
        if kind == "infer" and n > 4000:
            c["H"] = 5
    c |= dict(buckets=rng.choice([8, 32, 64]), max_distance=rng.choice([64, 128, 500]))
    return c


def _shapes(case):
    n, model = case["size"], case["model"]
    if model == "gaussians":
        return [(n, 3), (n, 1), (n, 3), (n, 4), (n, 16, 3)]
    if model == "tables":
        return [(n, 5), (n, 10), (n, 20), (n, 8)]
    return [(n,), (n,), (3 * n, n), (n, n), (n,), (8 * n, n), (8 * n,), (n, 4 * n), (n,), (32, max(1, n // 64))]


# ---- what a program has in hand ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    if case["op"] != "adamw":
        return _prepare_attention(case, rand, gen)
    dt = _DT[case["dtype"]]
    s = dict(case=case, lr=1e-4, betas=(0.9, 0.999), step=case["step"], seed=seed & 0xffff, p=[], g=[], m=[], v=[], ms=[], vs=[])
    for shape in _shapes(case):
        n = math.prod(shape)
        size = 10.0 ** (torch.rand(1, device="cuda", generator=gen) * 3 - 5)     # gradients of different tensors differ by orders of magnitude
        own_size = size * torch.exp(rand(*shape))                                # ... and within one
        s["p"].append(rand(*shape).to(dt))
        s["g"].append((own_size * rand(*shape)).to(dt))
        m = 0.3 * own_size * rand(*shape)
        v = (own_size * (0.5 + torch.rand(*shape, device="cuda", generator=gen))) ** 2
        if case["bits"] == 32:
            s["m"].append(m)
            s["v"].append(v)
            continue
        for codes, scales, x in (("m", "ms", m), ("v", "vs", v.sqrt())):         # 8 bits: the second moment's root is held
            blocks = _blocks(x.reshape(-1))
            scale = blocks.abs().amax(1) / 448.0
            q = (blocks / scale[:, None]).to(torch.float8_e4m3fn).reshape(-1)[:n].reshape(shape)
            s[codes].append(q.contiguous())
            s[scales].append(scale)
    if own:
        _package()
        from fused_optim import FusedAdamW
        params = [torch.nn.Parameter(p) for p in s["p"]]
        opt = FusedAdamW(params, lr=s["lr"], betas=s["betas"], eps=case["eps"], weight_decay=case["wd"], state_bits=case["bits"], seed=s["seed"])
        for i, p in enumerate(params):
            p.grad = s["g"][i]
            st = opt.state[p]
            st["step"] = torch.tensor(float(case["step"]))
            st["exp_avg"], st["exp_avg_sq" if case["bits"] == 32 else "exp_avg_rms"] = s["m"][i], s["v"][i]
            if case["bits"] == 8:
                st["exp_avg_scale"], st["exp_avg_rms_scale"] = s["ms"][i], s["vs"][i]
        s["opt"], s["params"] = opt, params
    return s


def _prepare_attention(case, rand, gen):
    B, H, Nq, Nk, dt = case["B"], case["H"], case["Nq"], case["Nk"], _DT[case["dtype"]]
    rows = (lambda n: (n, B, H * D)) if case["frame_major"] else (lambda n: (B, n, H * D))
    s = dict(case=case, q=rand(*rows(Nq)).to(dt), k=rand(*rows(Nk)).to(dt), v=rand(*rows(Nk)).to(dt),
             table=(0.7 * rand(case["buckets"], H)).to(_DT[case["table"]]), lens=None, start=0)
    if case["ragged"]:
        lens = torch.randint(Nq if Nq < Nk else 0, Nk + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
        lens[0] = Nk
        if case["op"] == "train" and B > 1:
            lens[B - 1] = 0                                        # nothing to attend to: zeros, and no gradient
        s["lens"] = lens
        if case["op"] == "infer" and Nq < Nk:
            s["start"] = lens - Nq                                 # the new tokens are the last of each sequence
        behind = torch.arange(Nk, device="cuda")[None, :, None] >= lens[:, None, None]
        s["k"].masked_fill_(behind, float("nan"))                  # what lies behind a sequence is whatever was there
        s["v"].masked_fill_(behind, float("nan"))
    if case["op"] == "train":
        s["dout"] = rand(*rows(Nq)).to(dt)
        if own:
            for n in ("q", "k", "v", "table"):
                s[n].requires_grad_(True)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        if own:
            state["opt"].step()
            return _moments(state)
        return _adamw(state) if case["bits"] == 32 else _adamw8(state)
    if own:
        _package()
        from lvdm_amd import ops
        args = dict(max_distance=case["max_distance"], bidirectional=not case["causal"], causal=case["causal"], q_start=state["start"],
                    kv_lens=state["lens"], frame_major=case["frame_major"])
        out = ops.relative_bias_attention(state["q"], state["k"], state["v"], state["table"], case["H"], **args)
        if case["op"] == "infer":
            return out
        dq, dk, dv, dtable = torch.autograd.grad(out, [state["q"], state["k"], state["v"], state["table"]], state["dout"])
        return dict(out=out, dq=dq, dk=dk, dv=dv, dtable=dtable)
    return _attention(state, torch.float32)


def _moments(s):
    if s["case"]["bits"] == 32:
        return dict(p=s["p"], m=s["m"], v=s["v"])
    return dict(p=s["p"], m=s["m"], v=s["v"], ms=s["ms"], vs=s["vs"])


def _update(s, i, g, m, v):
    """The new moments and parameter of tensor i from its gradient and old moments, all in the type of g."""
    case, (b1, b2), t = s["case"], s["betas"], s["step"]
    m = m + (1 - b1) * (g - m)
    v = b2 * v + (1 - b2) * (g * g)
    p = s["p"][i].to(g.dtype) * (1 - s["lr"] * case["wd"])
    p = p - (s["lr"] / (1 - b1 ** t)) * (m / (v.sqrt() / math.sqrt(1 - b2 ** t) + case["eps"]))
    return p, m, v


def _adamw(s):
    s["step"] += 1
    for i in range(len(s["p"])):
        p, m, v = _update(s, i, s["g"][i].float(), s["m"][i], s["v"][i])
        s["p"][i].copy_(p)
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
    return _moments(s)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).reshape(-1, BLOCK)


def _mix(h):
    h = ((h ^ (h >> 16)) * 0x7A2D4F2D) & 0xffffffff
    h = ((h ^ (h >> 15)) * 0x5C8B3B55) & 0xffffffff
    return h ^ (h >> 16)


def _random(s, i, n):
    """32 given bits for each element of tensor i at this step: a hash of (seed, tensor, step, element)."""
    key = _mix(_mix(_mix((s["seed"] + 0x3D1C27A5) & 0xffffffff) ^ i) ^ (s["step"] & 0xffffffff))
    return _mix(torch.arange(n, device="cuda", dtype=torch.int64) * 0x9D2C5681 + key & 0xffffffff)


def _to_8_bits(x, bits16, least):
    """x >= 0 (at most 448) as e4m3, rounded up with the probability of its distance from the lower neighbour; `bits16` are the draw's 16 bits.
    Scaled by 2^-120 a float's own exponent and upper mantissa bits are the code's, its subnormals among them."""
    b = (x.clamp(max=448.0) * 2.0 ** -120).view(torch.int32) + (bits16.to(torch.int32) << 4) >> 20
    return torch.where(least, b.clamp(min=1), b).clamp(max=0x7e)


def _adamw8(s):
    s["step"] += 1
    for i in range(len(s["p"])):
        n, shape = s["p"][i].numel(), s["p"][i].shape
        m = (_blocks(s["m"][i].float().reshape(-1)) * s["ms"][i][:, None]).reshape(-1)[:n].reshape(shape)
        r = (_blocks(s["v"][i].float().reshape(-1)) * s["vs"][i][:, None]).reshape(-1)[:n].reshape(shape)
        p, m, v = _update(s, i, s["g"][i].float(), m, r * r)
        h = _blocks(_random(s, i, n))
        m, r = _blocks(m.reshape(-1)), _blocks(v.sqrt().reshape(-1))
        big_m, big_r = m.abs().amax(1, keepdim=True), r.amax(1, keepdim=True)
        cm = _to_8_bits(torch.where(big_m > 0, m.abs() * (448.0 / big_m), 0.0), h & 0xffff, torch.zeros_like(m, dtype=torch.bool))
        cm = cm | torch.where(m < 0, 0x80, 0)
        cr = _to_8_bits(torch.where(big_r > 0, r * (448.0 / big_r), 0.0), h >> 16, r > 0)
        for name, c in (("m", cm), ("v", cr)):
            s[name][i].copy_(c.to(torch.uint8).reshape(-1)[:n].reshape(shape).view(torch.float8_e4m3fn))
        s["p"][i].copy_(p)
        s["ms"][i].copy_(big_m[:, 0] / 448.0)
        s["vs"][i].copy_(big_r[:, 0] / 448.0)
    return _moments(s)


def _thresholds(side, max_distance):
    """The least distance of each bucket of one side: the first half one by one, the others by equal ratios up to max_distance."""
    exact = side // 2
    rest = side - exact
    got, n = list(range(exact + 1)), exact
    for k in range(1, rest):
        while n ** rest * exact ** k < exact ** rest * max_distance ** k:      # n < exact * (max_distance / exact) ** (k / rest), in whole numbers
            n += 1
        got.append(n)
    return got[:side]


def _bucket(d, buckets, max_distance, both):
    """The bucket of each distance d (key position less query position)."""
    side = buckets // 2 if both else buckets
    t = torch.tensor(_thresholds(side, max_distance), device=d.device)
    n = d.abs() if both else (-d).clamp(min=0)
    b = torch.bucketize(n, t, right=True) - 1
    return b + torch.where(d > 0, side, 0) if both else b


def _heads(x, frame_major, H, dt):
    x = x.detach().transpose(0, 1) if frame_major else x.detach()
    return x.to(dt).reshape(x.shape[0], x.shape[1], H, D).transpose(1, 2).contiguous()


def _attention(s, dt):
    """Forward, and for a training pass the gradients, by the formulas, in `dt`; rounded once at the end."""
    c, H, fm = s["case"], s["case"]["H"], s["case"]["frame_major"]
    q, k, v = (_heads(s[n], fm, H, dt) for n in ("q", "k", "v"))
    table, scale = s["table"].detach().to(dt), D ** -0.5
    j = torch.arange(c["Nk"], device="cuda")
    start = s["start"][:, None, None].long() if torch.is_tensor(s["start"]) else s["start"]
    d = j[None, None, :] - (torch.arange(c["Nq"], device="cuda")[None, :, None] + start)
    bucket = _bucket(d, c["buckets"], c["max_distance"], not c["causal"])          # [B or 1, Nq, Nk]
    seen = torch.ones_like(d, dtype=torch.bool) if not c["causal"] else d <= 0
    if s["lens"] is not None:
        there = j[None, :] < s["lens"][:, None]
        seen = seen & there[:, None, :]
        k, v = (torch.where(there[:, None, :, None], x, 0.0) for x in (k, v))
    a = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale + table[bucket].permute(0, 3, 1, 2)
    a = a.masked_fill(~seen[:, None], -math.inf)
    top = a.amax(-1, keepdim=True)
    a = torch.exp(a - torch.where(top == -math.inf, 0.0, top))
    total = a.sum(-1, keepdim=True)
    p = a / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, v)
    del a, top, total

    def back(x, like):
        x = x.transpose(1, 2).reshape(x.shape[0], x.shape[2], H * D)
        x = x.transpose(0, 1).contiguous() if fm else x
        return x.to(like.dtype) if dt == torch.float32 else x

    if c["op"] == "infer":
        return back(out, s["q"])
    g = _heads(s["dout"], fm, H, dt)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), g)
    ds = torch.matmul(g, v.transpose(-1, -2).contiguous())
    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
    del p
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q) * scale
    ds = ds.sum(0)                                                                 # training batches share their distances
    rows = torch.zeros(H, c["Nq"], c["buckets"], device="cuda", dtype=dt)
    dtable = rows.scatter_add_(2, bucket.expand(H, -1, -1), ds).double().sum(1).t().to(dt)
    if dt == torch.float32:
        dtable = dtable.to(s["table"].dtype)
    return dict(out=back(out, s["q"]), dq=back(dq, s["q"]), dk=back(dk, s["q"]), dv=back(dv, s["q"]), dtable=dtable)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(x) for x in _shapes(case))
        e = 4 if case["dtype"] == "fp32" else 2
        return dict(bytes=n * (3 * e + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)), flops=n * 15)
    B, H, Nq, Nk = case["B"], case["H"], case["Nq"], case["Nk"]
    pairs = Nq * Nk
    if case["causal"]:
        pairs = sum(min(Nk, max(0, i + 1)) for i in range(Nq)) if Nq == Nk else pairs
    if case["ragged"]:
        B = B * 0.5 + 0.5                                          # lengths are uniform; the first is full
    seq = 2 * B * H * D
    if case["op"] == "infer":
        return dict(bytes=seq * (2 * Nq + 2 * Nk), flops=4 * B * H * pairs * D)
    return dict(bytes=seq * (4 * Nq + 4 * Nk), flops=14 * B * H * pairs * D)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    return _exact_attention(s)


def _exact_adamw(s):
    case, (b1, b2), t = s["case"], s["betas"], s["step"] + 1
    s["step"] = t
    res = dict(p=[], m=[], v=[], ms=[], vs=[])
    for i, p in enumerate(s["p"]):
        n, shape = p.numel(), p.shape
        g, m, v = s["g"][i].double(), s["m"][i].double(), s["v"][i].double()
        if case["bits"] == 8:
            wide = lambda scale: scale.double().repeat_interleave(BLOCK)[:n].reshape(shape)  # noqa: E731
            m, v = m * wide(s["ms"][i]), (v * wide(s["vs"][i])) ** 2
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        mean, root = m / (1 - b1 ** t), torch.sqrt(v / (1 - b2 ** t))
        res["p"].append(p.double() - s["lr"] * (mean / (root + case["eps"]) + case["wd"] * p.double()))
        if case["bits"] == 32:
            res["m"].append(m)
            res["v"].append(v)
            continue
        h = _random(s, i, n)
        for name, scales, x, u in (("m", "ms", m, h % 65536), ("v", "vs", torch.sqrt(v), h // 65536)):
            x = x.reshape(-1)
            scale = _blocks(x).abs().amax(1) / 448
            y = x.abs() / scale.clamp(min=1e-300).repeat_interleave(BLOCK)[:n]
            step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)   # the distance of e4m3's values around y
            y = torch.floor(y / step + u / 65536) * step
            if name == "v":
                y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
            res[name].append((y.clamp(max=448) * torch.sign(x)).reshape(shape))
            res[scales].append(scale)
    return {k: x for k, x in res.items() if x}


def _exact_attention(s):
    """Every (batch entry, head) by itself where rows are long; the formulas as written down, softmax by its log-sum-exp."""
    c, H, fm = s["case"], s["case"]["H"], s["case"]["frame_major"]
    if c["B"] * H * c["Nq"] * c["Nk"] * (3 if c["op"] == "train" else 1) > 4e9:
        return None
    rows = lambda x: (x.detach().permute(1, 0, 2) if fm else x.detach()).double()  # noqa: E731
    q, k, v = rows(s["q"]), rows(s["k"]), rows(s["v"])
    both, nb = not c["causal"], c["buckets"]
    side = nb // 2 if both else nb
    one_by_one = side // 2

    def which(n):
        if n < one_by_one:
            return n
        ratio = math.log(n / one_by_one) / math.log(c["max_distance"] / one_by_one)
        return min(side - 1, one_by_one + int(ratio * (side - one_by_one) + 1e-9))
    far = c["Nk"] + c["Nq"]
    by_distance = torch.tensor([which(abs(x)) + (side if x > 0 else 0) if both else which(max(-x, 0)) for x in range(-far, far + 1)], device="cuda")
    train = c["op"] == "train"
    g = rows(s["dout"]) if train else None
    res = dict(out=torch.zeros_like(q))
    if train:
        res |= dict(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v),
                    dtable=torch.zeros(nb, H, device="cuda", dtype=torch.float64))
    many = max(1, int(2e8 // (c["Nq"] * c["Nk"]))) if s["lens"] is None else 1    # batch entries at once where none is shorter
    for h in range(H):
        ch = slice(h * D, h * D + D)
        for b in range(0, c["B"], many):
            bs = slice(b, b + many)
            n = c["Nk"] if s["lens"] is None else int(s["lens"][b])
            if n == 0:
                continue
            i = torch.arange(c["Nq"], device="cuda") + (int(s["start"][b]) if torch.is_tensor(s["start"]) else s["start"])
            dist = torch.arange(n, device="cuda")[None] - i[:, None]
            buck = by_distance[dist.clamp(-far, far) + far]
            a = q[bs, :, ch] @ k[bs, :n, ch].transpose(1, 2) / math.sqrt(D) + s["table"].detach().double()[:, h][buck]
            if c["causal"]:
                a = torch.where(dist > 0, -math.inf, a)
            p = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
            p = torch.where(torch.isnan(p), 0.0, p)                               # a row that sees nothing
            res["out"][bs, :, ch] = o = p @ v[bs, :n, ch]
            if train:
                do = g[bs, :, ch]
                ds = p * (do @ v[bs, :n, ch].transpose(1, 2) - (do * o).sum(-1, keepdim=True))
                res["dv"][bs, :n, ch] = p.transpose(1, 2) @ do
                res["dq"][bs, :, ch] = ds @ k[bs, :n, ch] / math.sqrt(D)
                res["dk"][bs, :n, ch] = ds.transpose(1, 2) @ q[bs, :, ch] / math.sqrt(D)
                res["dtable"][:, h].index_add_(0, buck.reshape(-1), ds.sum(0).reshape(-1))
    res = {n: (x.permute(1, 0, 2) if fm and n != "dtable" else x) for n, x in res.items()}
    return res if train else res["out"]
