"""relative_bias_attention in the calls where it can answer wrongly without a word: tangents, entries brought to a limit, tensors that are made under another default
device, captures beside eager graphs, scores that grow along the keys, batches of many short rows; against its explicit form in 64 bits."""
import pytest
import torch

from lvdm_amd import ops, relative

gpu = pytest.mark.gpu
DEV = "cuda:0"
D = 64


def inputs(B, H, Nq, Nk, dtype=torch.float16, table_dtype=torch.float32, buckets=32, frame_major=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rows = (lambda n: (n, B, H * D)) if frame_major else (lambda n: (B, n, H * D))
    mk = lambda n: torch.randn(*rows(n), generator=gen).to(dtype).to(DEV)  # noqa: E731
    return mk(Nq), mk(Nk), mk(Nk), (0.8 * torch.randn(buckets, H, generator=gen)).to(table_dtype).to(DEV), mk(Nq)


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
