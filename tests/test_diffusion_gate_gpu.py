"""The feed-forward's gate under autograd, in the U-Net of the reference's goldens: once in the epilogues of its two GEMMs (the way that runs where weights are frozen), once
as a row kernel of its own.  Either way every feed-forward is counted, and outputs and input gradients meet the goldens (openaimodel3d.py:548-603, attention.py:415-450) within
the bars that tests/test_diffusion_goldens_gpu.py derives."""
import pytest
import torch

import test_diffusion_goldens_gpu as goldens
from fill_by_name import fill_by_name

pytestmark = pytest.mark.gpu
DEV = goldens.DEV


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("tag", ["shared", "perframe"])
def test_unet_golden_and_the_launches_of_its_gates(tag, fused, monkeypatch):
    from lvdm_amd import gemm
    from lvdm_amd.unet import FeedForward, UNetModel
    if not fused:
        monkeypatch.setenv("GVD_NO_FUSED_FF", "1")
    modes, launch = [], gemm._gate_gemm
    monkeypatch.setattr(gemm, "_gate_gemm", lambda x, w, y, aux, mode, **kw: (modes.append(mode), launch(x, w, y, aux, mode, **kw))[1])
    unet = fill_by_name(UNetModel(**goldens.UNET64)).half().eval().to(DEV).to_token_major().requires_grad_(False)
    blocks = sum(isinstance(m, FeedForward) for m in unet.modules())
    assert blocks > 0
    G = goldens.G
    x = torch.tensor(G[f"unet64_{tag}_x"], device=DEV).half().requires_grad_(True)
    ctx = torch.tensor(G[f"unet64_{tag}_ctx"], device=DEV).half()
    with goldens._Counters() as c:
        y = unet(x, torch.tensor([250], device=DEV), context=ctx, fs=torch.tensor([10], device=DEV))
        (gx,) = torch.autograd.grad(y, x, torch.tensor(G[f"unet64_{tag}_gy"], device=DEV).half())
    assert y.dtype == torch.float16
    assert c.n["conv"] >= 2 * 40 and c.n["attn"] > 10 and c.n["attn_bwd"] > 10 and c.n["gn_bwd"] > 10 and c.n["gemm"] > 100 and c.n["ln"] == 0, c.n
    assert (modes.count(2), modes.count(3), c.n["geglu"]) == ((blocks, blocks, 0) if fused else (0, 0, blocks)), (modes, c.n, blocks)
    e_y, e_g = goldens._rel(y, G[f"unet64_{tag}_y"]), goldens._rel(gx, G[f"unet64_{tag}_gx"])
    assert e_y < 2e-2 and e_g < 4e-2, (e_y, e_g)
