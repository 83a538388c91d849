"""The causal convolution on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, causal_conv

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def inputs(seed, B, S, C, W, dtype=BF16, n=None, wide=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, C + wide, generator=g).to(dtype).cuda()[..., wide // 2 : wide // 2 + C]
    return {"x": x, "w": (torch.randn(C, W, generator=g) * 0.5).to(dtype).cuda(),
            "bias": (torch.randn(C, generator=g) * 0.3).to(dtype).cuda(),
            "state": torch.randn(n or B, W - 1, C, generator=g).to(dtype).cuda()}


def slack(x):
    """Sums of W products and a bias in fp32, each off by at most 2^-24 of the terms' sum, which the row's largest
    output bounds only up to cancellation: 2^-16 of it leaves a factor of 2^8."""
    return 2.0 ** -16


@pytest.mark.parametrize("S", [1, 2, 3, 4, 5, 15, 16, 17, 31, 33, 100])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("C", [1, 7, 64, 1003])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sizes(S, W, C, dtype):
    x = inputs(S + 10 * W + C, 2, S, C, W, dtype)
    want, new = causal_conv(x["x"], x["w"], x["state"], x["bias"])
    out = torch.zeros(2, S, C, dtype=dtype, device="cuda")
    paged.causal_conv(x["x"], x["w"], out, x["state"], bias=x["bias"])
    torch.cuda.synchronize()
    assert_rounded(out, want, f"S={S} W={W} C={C}", slack(x))
    assert torch.equal(x["state"].cpu().double(), new)


@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("state", [True, False])
def test_forms(silu, bias, state):
    x = inputs(5, 2, 21, 96, 4)
    b, s = (x["bias"] if bias else None), (x["state"] if state else None)
    want, new = causal_conv(x["x"], x["w"], s, b, silu)
    out = torch.zeros(2, 21, 96, dtype=BF16, device="cuda")
    paged.causal_conv(x["x"], x["w"], out, s, bias=b, silu=silu)
    torch.cuda.synchronize()
    assert_rounded(out, want, f"{silu} {bias} {state}", slack(x))
    if state:
        assert torch.equal(s.cpu().double(), new)


@pytest.mark.parametrize("wide", [16, 6])
@pytest.mark.parametrize("S", [1, 40])
def test_strides(wide, S):
    """Channels of a wider tensor, at offsets that allow 16-byte accesses and that do not."""
    x = inputs(6, 3, S, 200, 4, wide=wide)
    want, new = causal_conv(x["x"], x["w"], x["state"], x["bias"])
    out = torch.zeros(S, 3, 200 + wide, dtype=BF16, device="cuda").transpose(0, 1)[..., wide // 2 : wide // 2 + 200]
    paged.causal_conv(x["x"], x["w"], out, x["state"], bias=x["bias"])
    torch.cuda.synchronize()
    assert_rounded(out, want, "strides", slack(x))
    assert torch.equal(x["state"].cpu().double(), new)


@pytest.mark.parametrize("S", [1, 2, 50])
@pytest.mark.parametrize("C", [24, 25])
def test_padded_batch_over_a_pool(S, C):
    x = inputs(7, 7, S, C, 4, n=9)
    ids = torch.tensor([5, 0, -3, 8, 5, 9, 2], dtype=torch.int32)
    lens = torch.tensor([S, max(1, S - 1), S, 0, S, S, 2 * S], dtype=torch.int32)
    before = x["state"].clone()
    want, new = causal_conv(x["x"], x["w"], before[ids.long().clamp(0, 8).cuda()], None, True, lens)
    out = torch.full((7, S, C), 2.5, dtype=BF16, device="cuda")
    paged.causal_conv(x["x"], x["w"], out, x["state"], seq_lens=lens.cuda(), state_ids=ids.cuda())
    torch.cuda.synchronize()
    for i in (0, 1, 6):
        n = min(int(lens[i]), S)
        assert_rounded(out[i, :n], want[i, :n], f"entry {i}", slack(x))
        assert bool((out[i, n:] == 2.5).all())
        assert torch.equal(x["state"][ids[i]].cpu().double(), new[i])
    for i in (2, 3):
        assert bool((out[i] == 2.5).all())
    for i in (4, 5):  # an earlier entry's state; no such state
        assert bool(torch.isnan(out[i]).all())
    for j in (1, 3, 4, 6, 7, 8):
        assert torch.equal(x["state"][j], before[j])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_special_values_stay_in_their_window(bad):
    x = inputs(8, 1, 40, 16, 4)
    x["x"][0, 20, 3] = bad
    want, new = causal_conv(x["x"], x["w"], x["state"], None)
    out = torch.zeros(1, 40, 16, dtype=BF16, device="cuda")
    paged.causal_conv(x["x"], x["w"], out, x["state"])
    torch.cuda.synchronize()
    clean = torch.ones(40, 16, dtype=torch.bool)
    clean[20:24, 3] = False
    assert bool(torch.isfinite(out[0].cpu()[clean]).all())
    got, exp = out[0, 20:24, 3].cpu().double(), want[0, 20:24, 3]
    assert torch.equal(torch.isnan(got), torch.isnan(exp)) and torch.equal(got[~torch.isnan(exp)], exp[~torch.isnan(exp)])


def test_large_arguments_of_silu():
    x = inputs(9, 1, 8, 8, 2)
    x["x"][:] = torch.tensor([1e4, -1e4, 300.0, -300.0, 88.0, -88.0, 1e30, -1e30], device="cuda").to(BF16)
    x["w"][:] = 1.0
    want, _ = causal_conv(x["x"], x["w"], x["state"], None)
    out = torch.zeros(1, 8, 8, dtype=BF16, device="cuda")
    paged.causal_conv(x["x"], x["w"], out, x["state"])
    torch.cuda.synchronize()
    g, w = out.cpu().double(), want
    # where exp(88) is near the end of fp32 the result is below 1e-30: it may be flushed
    assert bool(((g - w).abs() <= 2.0 ** -8 * 1.02 * w.abs() + 1e-30).all())


def test_turns_add_up_and_graph():
    x = inputs(10, 2, 90, 64, 4)
    first = x["state"].clone()
    whole = torch.zeros(2, 90, 64, dtype=BF16, device="cuda")
    paged.causal_conv(x["x"], x["w"], whole, x["state"])
    end = x["state"].clone()
    x["state"].copy_(first)
    parts = torch.zeros_like(whole)
    at = 0
    for n in (1, 1, 2, 30, 3, 53):
        paged.causal_conv(x["x"][:, at : at + n], x["w"], parts[:, at : at + n], x["state"])
        at += n
    torch.cuda.synchronize()
    assert torch.equal(whole, parts) and torch.equal(end, x["state"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.causal_conv(x["x"], x["w"], parts, x["state"])
    for _ in range(3):
        x["state"].copy_(first)
        parts.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(whole, parts) and torch.equal(end, x["state"])


def test_other_stream_and_channels_beside_each_other():
    """On a stream of the caller's, from one half of a tensor's channels into the other."""
    x = inputs(12, 2, 30, 64, 4)
    both = torch.cat([x["x"], torch.zeros_like(x["x"])], -1)
    want, new = causal_conv(x["x"], x["w"], x["state"], x["bias"])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    paged.causal_conv(both[..., :64], x["w"], both[..., 64:], x["state"], bias=x["bias"], stream=stream)
    stream.synchronize()
    assert_rounded(both[..., 64:], want, "beside", slack(x))
    assert torch.equal(both[..., :64], x["x"]) and torch.equal(x["state"].cpu().double(), new)


def test_nothing_to_do():
    x = inputs(13, 2, 4, 16, 4)
    before = x["state"].clone()
    out = torch.full((2, 4, 16), 3.0, dtype=BF16, device="cuda")
    paged.causal_conv(x["x"][:, :0], x["w"], out[:, :0], x["state"])
    paged.causal_conv(x["x"][:0], x["w"], out[:0], x["state"])
    paged.causal_conv(x["x"], x["w"], out, x["state"], seq_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(before, x["state"]) and bool((out == 3.0).all())


def test_python_refusals():
    x = inputs(11, 1, 8, 16, 4)
    out = torch.zeros(1, 8, 16, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        paged.causal_conv(x["x"], x["w"].half(), out, x["state"])
    with pytest.raises(ValueError):
        paged.causal_conv(x["x"], x["w"], out[:, :7], x["state"])
    with pytest.raises(ValueError):
        paged.causal_conv(x["x"], x["w"], out, x["state"][:, :2])
    with pytest.raises(paged.GenllmError):
        paged.causal_conv(x["x"], x["w"], x["x"], x["state"])  # in place
    with pytest.raises(paged.GenllmError):
        paged.causal_conv(out[:, 1:], x["w"], out[:, :7], x["state"])  # rows of one buffer, one apart
