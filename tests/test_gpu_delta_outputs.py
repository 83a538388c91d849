"""Outputs of the delta rule's chunked form hold the bits of 32-bit arithmetic before their one rounding.

All terms of the sums below are positive, so that a sum is as large as its terms' absolute values and the error of each part
shows relative to the result.  Half steps of fp32 (2^-24, relative) between the inputs and an output, at most:

  q's norm: sum of squares 5, root and reciprocal 2, scale and product 2                                 9
  the same for k's, where it is normalised                                                               9
  decay: its rate and softplus 5 and the running difference's rounding 1, of |G| <= 1; 2^x 2; product 1  9
  u: beta 4, its product 1, the sums of parts (six products, three accumulators) 8                      13
  S or P: parts' sums (six products of two steps, or three of four) 12, products and their sum 2        14

which is 54: 2^-18 is 64 of them.  Two bf16 parts leave up to 2^-16 of each term."""
import math

import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, delta_rule

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
SLACK = 2.0 ** -18


def assert_one_rounding(got, want, label, scale=None):
    """|got - want| within half a step of want's own binade and SLACK of the terms' size (want's own where all are positive).
    Below the smallest normal value the steps get no smaller: tiny eps / 2 is half of one (fp16 2^-14 2^-10 / 2 = 2^-25)."""
    g, w = got.detach().cpu().double(), want
    bits = {BF16: 8, F16: 11}[got.dtype]
    half = torch.ldexp(torch.ones_like(w), torch.frexp(w)[1] - 1 - bits)
    half = half.clamp(min=torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps / 2)
    bound = half + SLACK * (w.abs() if scale is None else scale)
    worst = ((g - w).abs() / bound).max().item()
    over = ((g - w).abs() > bound).double().mean().item()
    print(f"[{label}] worst {worst:.4f} of its bound, {over:.2e} of the elements above", flush=True)
    assert worst <= 1.0, f"{label}: {worst} times the bound"


def call(x, out, l2_eps=1e-6):
    paged.gated_delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], x["state"], out, x["scale"], l2_eps=l2_eps)
    torch.cuda.synchronize()


def positive(g, *shape):
    return torch.rand(shape, generator=g) + 0.25


SHAPES = [(1, 70, 1, 2, 128, 128), (2, 200, 2, 4, 64, 64), (1, 130, 3, 3, 64, 128), (1, 100, 2, 2, 128, 64),
          (2, 140, 12, 24, 128, 128), (3, 90, 24, 24, 64, 64)]  # the last two: two chains per workgroup


@pytest.mark.parametrize("B,S,Hk,Hv,Dk,Dv", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_state_read(B, S, Hk, Hv, Dk, Dv, dtype):
    """beta 0: out is the decayed state beside q."""
    g = torch.Generator().manual_seed(S + Dk)
    x = {"q": positive(g, B, S, Hk, Dk).to(dtype).cuda(), "k": positive(g, B, S, Hk, Dk).to(dtype).cuda(),
         "v": positive(g, B, S, Hv, Dv).to(dtype).cuda(), "a": (-torch.rand(B, S, Hv, generator=g) / S).cuda(),
         "b": torch.zeros(B, S, Hv).cuda(), "state": positive(g, B, Hv, Dk, Dv).cuda(), "scale": 0.37}
    want, new = delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], x["state"], x["scale"], l2_eps=1e-6)
    out = torch.zeros(B, S, Hv, Dv, dtype=dtype, device="cuda")
    call(x, out)
    assert_one_rounding(out, want, f"state read {dtype} {Dk}x{Dv}")


@pytest.mark.parametrize("B,S,Hk,Hv,Dk,Dv", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_writes_read(B, S, Hk, Hv, Dk, Dv, dtype):
    """Keys along the axes, no two alike in a chunk, and nothing left from one chunk to the next: u = beta v, and out is
    the chunk's own writes beside q."""
    g = torch.Generator().manual_seed(S + Dk)
    k = torch.zeros(B, S, Hk, Dk)
    k[:, torch.arange(S), :, torch.arange(S) % 64] = 1.0
    a = -torch.rand(B, S, Hv, generator=g) / 64
    a[:, ::64] = -math.inf
    x = {"q": positive(g, B, S, Hk, Dk).to(dtype).cuda(), "k": k.to(dtype).cuda(),
         "v": positive(g, B, S, Hv, Dv).to(dtype).cuda(), "a": a.cuda(),
         "b": positive(g, B, S, Hv).cuda(), "state": positive(g, B, Hv, Dk, Dv).cuda(), "scale": 0.37}
    want, new = delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], x["state"], x["scale"], l2_eps=1e-6)
    out = torch.zeros(B, S, Hv, Dv, dtype=dtype, device="cuda")
    call(x, out)
    assert_one_rounding(out, want, f"writes read {dtype} {Dk}x{Dv}")


@pytest.mark.parametrize("S", [33, 70, 500])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt(S, dtype):
    """Usual values: errors against the sums of the terms' absolute values, of which the row's largest output is a
    part at least."""
    g = torch.Generator().manual_seed(S)
    B, Hk, Hv, D = 1, 2, 4, 128
    x = {c: torch.nn.functional.silu(torch.randn(B, S, H, D, generator=g) * 1.5).to(dtype).cuda()
         for c, H in (("q", Hk), ("k", Hk), ("v", Hv))}
    x["a"] = (-torch.rand(B, S, Hv, generator=g)).cuda()
    x["b"] = torch.rand(B, S, Hv, generator=g).cuda()
    x["state"], x["scale"] = (torch.randn(B, Hv, D, D, generator=g) * 0.3).cuda(), D ** -0.5
    want, new = delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], x["state"], x["scale"], l2_eps=1e-6)
    out = torch.zeros(B, S, Hv, D, dtype=dtype, device="cuda")
    call(x, out)
    assert_one_rounding(out, want, f"prompt of {S} {dtype}", want.abs().amax(-1, keepdim=True))


@pytest.mark.parametrize("squared,v,S", [(5, 8.0, 64), (4, 1.0, 128), (4, 1.0, 79), (17, 2.0, 90)])
@pytest.mark.parametrize("heads", [1, 40])  # 40: two chains per workgroup
def test_tokens_before_an_overflow(squared, v, S, heads):
    """Equal keys with beta |k|^2 above 2: every token's u is 1 - |k|^2 times the last one's, until it leaves fp32.
    Outputs up to there are the rule's.  Each token adds at most eight half steps of fp32 to what it multiplies,
    relative, and 2^-14 is 1024 of them."""
    k = torch.zeros(1, S, heads, 64)
    k[..., 0], k[..., 1] = {4: (2, 0), 5: (2, 1), 17: (4, 1)}[squared]
    x = {"q": torch.zeros(1, S, heads, 64), "k": k, "v": torch.full((1, S, heads, 128), v)}
    x["q"][..., :2] = torch.tensor([0.5, 1.0])
    x = {c: t.to(BF16).cuda() for c, t in x.items()}
    x["a"], x["b"] = torch.zeros(1, S, heads).cuda(), torch.ones(1, S, heads).cuda()
    x["state"], x["scale"] = torch.zeros(1, heads, 64, 128).cuda(), 0.125
    want, _ = delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], x["state"], x["scale"])
    # u and the products that form it are at most 64 times out here
    n = int((want.abs().amax((0, 2, 3)) < 2.0 ** 121).sum())
    assert 0 < n <= S
    out = torch.zeros(1, S, heads, 128, dtype=BF16, device="cuda")
    call(x, out, l2_eps=None)
    assert_rounded(out[:, :n], want[:, :n], f"|k|^2 {squared}, {n} tokens of {S}")
    if n < S:
        assert not bool(torch.isfinite(out[:, -1]).any()) or bool((out[:, -1].abs() > 2.0 ** 100).any())


@pytest.mark.parametrize("S", [3, 80])
@pytest.mark.parametrize("order", ["token", "head"])
def test_one_buffer_for_all(S, order):
    """q, k, v and out in one buffer, beside each other in every row or head by head: nothing is shared, and nothing else
    in the buffer is written."""
    g = torch.Generator().manual_seed(S)
    B, Hk, Hv, D = 2, 2, 4, 64
    H = 2 * Hk + 2 * Hv + 1  # the last head is nobody's
    if order == "token":
        buf = torch.randn(B, S, H, D, generator=g).bfloat16().cuda()
    else:
        buf = torch.randn(B, H, S, D, generator=g).bfloat16().cuda().transpose(1, 2)
    first = buf.clone()
    q, k, v, out, _ = torch.split(buf, [Hk, Hk, Hv, Hv, 1], 2)
    x = {"q": q, "k": k, "v": v, "a": (-torch.rand(B, S, Hv, generator=g)).cuda(), "b": torch.rand(B, S, Hv, generator=g).cuda(),
         "state": torch.randn(B, Hv, D, D, generator=g).cuda(), "scale": 0.125}
    want, _ = delta_rule(q, k, v, x["a"], x["b"], x["state"], x["scale"], l2_eps=1e-6)
    call(x, out)
    assert_rounded(out, want, f"one buffer, {order}")
    keep = [h for h in range(H) if not 2 * Hk + Hv <= h < 2 * Hk + 2 * Hv]
    assert torch.equal(buf[:, :, keep], first[:, :, keep])
