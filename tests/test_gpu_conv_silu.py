"""SiLU of far negative sums: small, but as exact as any other result down to the type's smallest normal value."""
import pytest
import torch

from genllm_amd import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C", [8, 7])
def test_far_negative_sums(C):
    """One tap of weight 1, so that the sum is x: -60 to -91 in quarters and halves, which bf16 holds, and the largest ones.
    x / (1 + exp(-x)) has the error of exp's argument, |x| log2(e) half steps of fp32 (130 at most, 2^-17 relative), and
    a few of its own: 2^-16 of the value beside bf16's own half step."""
    x = torch.cat([torch.arange(-91, -59, 0.5), torch.tensor([-3.0, -0.25, 0.0, 0.25, 3.0, 88.0, 91.0, 1e4, 1e30])]).bfloat16()
    S = x.numel()
    x = x[None, :, None].expand(1, S, C).contiguous().cuda()
    w = torch.zeros(C, 2, dtype=torch.bfloat16, device="cuda")
    w[:, 1] = 1.0
    out = torch.zeros_like(x)
    paged.causal_conv(x, w, out)
    torch.cuda.synchronize()
    d = x.double().cpu()
    want = d / (1 + torch.exp(-d))
    assert float(want[want < 0].max()) < -1.2e-38  # all normal
    bound = (2.0 ** -8 + 2.0 ** -16) * want.abs()
    off = (out.double().cpu() - want).abs()
    worst = (off - bound).amax()
    assert bool((off <= bound).all()), (float(worst), d[off > bound][:4].tolist())
