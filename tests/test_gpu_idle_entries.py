"""Entries of a batch without tokens keep the ids that they had: they claim no state from the entries behind them."""
import math

import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, assert_state, causal_conv, delta_rule

pytestmark = pytest.mark.gpu

IDS = [2, 0, 2, 4, 0, 4, 9, 2, -1]
LIVE = {2: 2, 3: 4, 4: 0}  # entry: state


def lens_of(S):
    return [0, -3, S, S, S, max(1, S - 1), 0, S, S]


@pytest.mark.parametrize("S,H", [(1, 2), (20, 2), (80, 2), (80, 16)])  # 16 heads: two chains per workgroup
def test_delta_rule(S, H):
    g = torch.Generator().manual_seed(S)
    B = len(IDS)
    x = [torch.randn(B, S, H, 64, generator=g).bfloat16().cuda() for _ in "qkv"]
    a, b = (-torch.rand(B, S, H, generator=g)).cuda(), torch.rand(B, S, H, generator=g).cuda()
    for t in (*x, a, b):
        t[0], t[1], t[6] = math.nan, math.nan, math.nan
    state = torch.randn(6, H, 64, 64, generator=g).cuda()
    first, lens = state.clone(), torch.tensor(lens_of(S), dtype=torch.int32)
    out = torch.full((B, S, H, 64), 2.5, dtype=torch.bfloat16, device="cuda")
    paged.gated_delta_rule(*x, a, b, state, out, 0.125, l2_eps=1e-6, seq_lens=lens.cuda(),
                           state_ids=torch.tensor(IDS, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    for i, slot in LIVE.items():
        row = [t[i : i + 1] for t in (*x, a, b)]
        want, new = delta_rule(*row, first[slot : slot + 1], 0.125, l2_eps=1e-6)
        assert_rounded(out[i : i + 1], want, f"entry {i}")
        assert_state(state[slot : slot + 1], new, S, f"entry {i}")
    for i in (0, 1, 6, 8):
        assert bool((out[i] == 2.5).all()), f"idle entry {i}"
    for i in (5, 7):  # states of entries 3 and 2
        n = int(lens[i])
        assert bool(torch.isnan(out[i, :n]).all()) and bool((out[i, n:] == 2.5).all()), f"entry {i}"
    for j in (1, 3, 5):
        assert torch.equal(state[j], first[j])


@pytest.mark.parametrize("S", [1, 2, 50])
@pytest.mark.parametrize("C", [24, 25])
def test_convolution(S, C):
    g = torch.Generator().manual_seed(S)
    B = len(IDS)
    x, w = torch.randn(B, S, C, generator=g).bfloat16().cuda(), torch.randn(C, 4, generator=g).bfloat16().cuda()
    x[0], x[1], x[6] = math.nan, math.nan, math.nan
    state = torch.randn(6, 3, C, generator=g).bfloat16().cuda()
    first, lens = state.clone(), torch.tensor(lens_of(S), dtype=torch.int32)
    out = torch.full((B, S, C), 2.5, dtype=torch.bfloat16, device="cuda")
    paged.causal_conv(x, w, out, state, seq_lens=lens.cuda(), state_ids=torch.tensor(IDS, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    for i, slot in LIVE.items():
        want, new = causal_conv(x[i : i + 1], w, first[slot : slot + 1])
        assert_rounded(out[i : i + 1], want, f"entry {i}", 2.0 ** -16)
        assert torch.equal(state[slot : slot + 1].cpu().double(), new)
    for i in (0, 1, 6, 8):
        assert bool((out[i] == 2.5).all()), f"idle entry {i}"
    for i in (5, 7):
        assert bool(torch.isnan(out[i, : int(lens[i])]).all()), f"entry {i}"
    for j in (1, 3, 5):
        assert torch.equal(state[j], first[j])
