"""Attention with a learned relative position bias by buckets: the hand-written kernels of csrc/relattn_forward.hip and relattn_backward.hip through the
C-ABI library lib/libgvd_relattn.so (include/gvd_relattn.h).  The entry point is `ops.relative_bias_attention`, beside `ops.attention`.
"""
import ctypes
import functools
import importlib.util
import os

import torch

from . import ops

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.environ.get("GVD_RELATTN_LIB") or os.path.join(os.path.dirname(_HERE), "lib", "libgvd_relattn.so")  # env: A/B builds
_EXT_PATH = os.path.join(os.path.dirname(_HERE), "lib", "_gvd_relattn_torch.so")
_LIB = _EXT = None
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_SIDE, MAX_DISTANCE = 128, 1024      # GVD_RELATTN_MAX_SIDE, GVD_RELATTN_MAX_REACH


def lib():
    global _LIB
    if _LIB is None:
        if not os.path.exists(_LIB_PATH):
            raise RuntimeError(f"{_LIB_PATH} is missing: build the HIP extensions first "
                               f"(python -c 'import __graft_entry__ as g; g.build()')")
        L = ctypes.CDLL(_LIB_PATH)
        L.gvd_relattn_last_error.restype = ctypes.c_char_p
        for f in (L.gvd_relattn_fwd_workspace, L.gvd_relattn_bwd_workspace):
            f.restype = ctypes.c_longlong
        _LIB = L
    return _LIB


def ext():
    """The compiled operator (csrc/relattn_torch_ext.cpp: forward and backward as one node of the graph) over the same library instance."""
    global _EXT
    if _EXT is None:
        lib()
        if not os.path.exists(_EXT_PATH):
            raise RuntimeError(f"{_EXT_PATH} is missing: build the extensions first (python -c 'import __graft_entry__ as g; g.build()')")
        spec = importlib.util.spec_from_file_location("_gvd_relattn_torch", _EXT_PATH)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.init(_LIB_PATH)
        _EXT = mod
    return _EXT


@functools.lru_cache(maxsize=64)
def first_distances(side, max_distance):
    """The least distance of each of one side's buckets: the first half of them one distance each, the others by equal ratios up to max_distance, from which on
    all share the last.  Whole-number arithmetic: bucket exact + k begins at the least n with n >= exact (max_distance / exact)^(k / rest)."""
    exact = side // 2
    rest = side - exact
    if not 1 <= side <= MAX_SIDE:
        raise ValueError(f"relative_bias_attention: {side} buckets a side (1 .. {MAX_SIDE})")
    if not exact < max_distance <= MAX_DISTANCE:
        raise ValueError(f"relative_bias_attention: max_distance {max_distance} (above {exact}, the buckets of one distance, and at most {MAX_DISTANCE})")
    got, n = list(range(exact + 1)), exact
    for k in range(1, rest):
        while n ** rest * exact ** k < exact ** rest * max_distance ** k:
            n += 1
        got.append(n)
    return tuple(got[:side])


@functools.lru_cache(maxsize=64)
def _first_tensor(side, max_distance):
    return torch.tensor(first_distances(side, max_distance), dtype=torch.int32, device="cpu")     # (kept, and read by the host: whatever the default device is)


def relative_buckets(distance, buckets, max_distance=128, bidirectional=True):
    """The bucket (int64) of each distance (key position less query position, an integer tensor): `buckets` is even where bidirectional, and keys ahead of
    the query have the upper half; otherwise keys ahead share the bucket of distance 0."""
    side = buckets // 2 if bidirectional else buckets
    first = torch.tensor(first_distances(side, max_distance), device=distance.device)
    n = distance.abs() if bidirectional else (-distance).clamp(min=0)
    b = torch.searchsorted(first, n.contiguous(), right=True) - 1
    return b + side * (distance > 0) if bidirectional else b


def relative_bias_attention_math(q, k, v, table, heads, *, max_distance=128, bidirectional=True, causal=False, q_start=0, kv_lens=None, scale=None,
                                 frame_major=False):
    """Explicit form in torch operations (differentiable by autograd), softmax in the inputs' type or float32."""
    if frame_major:
        q, k, v = (t.transpose(0, 1) for t in (q, k, v))
    B, Nq, C = q.shape
    Nk, d = k.shape[1], C // heads
    wide = lambda t: t.to(torch.promote_types(t.dtype, torch.float32)).reshape(t.shape[0], t.shape[1], heads, d).permute(0, 2, 1, 3)  # noqa: E731
    qh, kh, vh = wide(q), wide(k.expand(B, -1, -1)), wide(v.expand(B, -1, -1))
    j = torch.arange(Nk, device=q.device)
    start = q_start.view(-1, 1, 1).long() if torch.is_tensor(q_start) else q_start
    dist = j - (torch.arange(Nq, device=q.device)[None, :, None] + start)
    seen = dist <= 0 if causal else torch.ones_like(dist, dtype=torch.bool)
    if kv_lens is not None:
        there = j[None] < kv_lens.view(-1, 1)
        seen = seen & there[:, None]
        kh, vh = (t.masked_fill(~there[:, None, :, None], 0.0) for t in (kh, vh))
    entries = table.to(qh.dtype).clamp(max=10000.0)
    bias = entries.masked_fill(entries <= -10000.0, float("-inf"))[relative_buckets(dist, table.shape[0], max_distance, bidirectional)].permute(0, 3, 1, 2)
    s = torch.matmul(qh, kh.transpose(-1, -2).contiguous()) * (d ** -0.5 if scale is None else scale) + bias
    s = s.masked_fill(~seen[:, None], float("-inf"))
    empty = (s == float("-inf")).all(-1, keepdim=True)
    p = s.masked_fill(empty, 0.0).softmax(-1).masked_fill(empty, 0.0)
    out = torch.matmul(p, vh).masked_fill(empty, 0.0).permute(0, 2, 1, 3).reshape(B, Nq, C).to(q.dtype)     # (no gradient passes there, whatever it holds)
    return out.transpose(0, 1).contiguous() if frame_major else out


def _check_arguments(q, k, v, table, heads, bidirectional, q_start, kv_lens, scale, frame_major, max_distance):
    bad = lambda what: ValueError(f"relative_bias_attention: {what}")  # noqa: E731
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape:
        raise bad(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: three dimensions each, k and v of one shape")
    bd = 1 if frame_major else 0
    B, C = q.shape[bd], q.shape[2]
    if heads <= 0 or C % heads or k.shape[2] != C or k.shape[bd] not in (1, B):
        raise bad(f"q {tuple(q.shape)}, k {tuple(k.shape)} with {heads} heads: channels heads * d on either side, and one batch size (or one K / V for the whole batch)")
    if table.dim() != 2 or table.shape[1] != heads or table.shape[0] < 1 or table.dtype not in _TYPES:
        raise bad(f"table {table.dtype} {tuple(table.shape)}: [buckets, heads] of float32, float16 or bfloat16")
    if bidirectional and table.shape[0] % 2:
        raise bad("an even number of buckets where both directions have their own")
    first_distances(table.shape[0] // 2 if bidirectional else table.shape[0], max_distance)
    if not 1e-30 < scale < 1e30:
        raise bad(f"scale {scale}")
    for name, t in (("k", k), ("v", v), ("table", table)):
        if t.device != q.device:
            raise bad(f"{name} is on {t.device}, q on {q.device}")
    for name, t in (("kv_lens", kv_lens), ("q_start", q_start if torch.is_tensor(q_start) else None)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (B,) or t.device != q.device or not t.is_contiguous()):
            raise bad(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}; a contiguous int32 [{B}] on {q.device} is wanted")
    if not torch.is_tensor(q_start) and not -2 ** 29 <= int(q_start) <= 2 ** 29:
        raise bad(f"q_start {q_start}")


def relative_bias_attention(q, k, v, table, heads, *, max_distance=128, bidirectional=True, causal=False, q_start=0, kv_lens=None, scale=None,
                            frame_major=False):
    """See ops.relative_bias_attention."""
    on_dev = ops._require_device(q, "relative_bias_attention")
    if on_dev:
        buckets = table.shape[0]
        out = (_EXT or ext()).attend(q, k, v, table, heads, _first_tensor(buckets // 2 if bidirectional else buckets, max_distance), bidirectional, causal, q_start,
                                     kv_lens, scale, frame_major)
        if out is not None:
            return out
    scale = (q.shape[-1] // max(heads, 1)) ** -0.5 if scale is None else float(scale)
    _check_arguments(q, k, v, table, heads, bidirectional, q_start, kv_lens, scale, frame_major, max_distance)
    if on_dev:
        ops._torch_form("relative_bias_attention", f"dtypes {q.dtype}, {k.dtype}, {v.dtype}, head dim {q.shape[-1] // heads} (the MFMA kernels cover 16-bit heads of 64)")
    return relative_bias_attention_math(q, k, v, table, heads, max_distance=max_distance, bidirectional=bidirectional, causal=causal, q_start=q_start,
                                        kv_lens=kv_lens, scale=scale, frame_major=frame_major)
