"""Batches of unlike entries: single tokens and chunks in one call, more units than a wave has lanes, and the forms of the
kernel for more than 16 rows in fp16."""
import pytest
import torch

from genllm_amd import paged
from test_gpu_attention_batch import BF, HF, Case

pytestmark = pytest.mark.gpu


def workspace(c):
    return paged.paged_attention_batch_workspace_bytes(c.q.shape[0], c.S, c.Hq, c.H, c.D, c.ids[0].shape[1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tiles_of_64_rows(D, f8, dtype):
    """17 to 64 rows for a kv head, split and not: eight waves in two key groups."""
    for Hq, H, S, n in ((2, 1, 20, [20, 700, 300]), (8, 2, 13, [50, 13, 90]), (5, 5, 64, [64, 400, 65])):
        c = Case(Hq, H, D, dtype, f8, n, S, [S, S, S - 1], seed=Hq)
        assert S * Hq // H <= 64
        c.run()
        c.check(f"tiles of 64, {Hq} heads")
        c.run(window=70, sinks=3)
        c.check(f"tiles of 64, {Hq} heads, windows", window=70, sinks=3)


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("Hq,H,D", [(6, 3, 64), (8, 8, 128)])
def test_whole_prompts_in_fp16(Hq, H, D, f8):
    """Prompts of a thousand tokens whose tiles are all there at once."""
    S, B = 1030, {64: 4, 128: 3}[D]
    c = Case(Hq, H, D, HF, f8, [S, S + 900, 700, S - 1][:B], S, [S, S, 650, S - 1][:B])
    assert workspace(c) == 0
    c.run()
    c.check("whole prompts")


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("B,Hq,H,S", [(100, 16, 1, 2), (70, 8, 2, 5), (9, 4, 1, 300)])
def test_more_units_than_lanes(B, Hq, H, S, f8):
    """More row tiles of more than 16 rows than a wave has lanes, whose contexts are split."""
    n = [(37 * i) % 90 for i in range(B)]
    n[B // 2], n[B - 1] = 1500, 900
    ql = [min(S, 1 + i % 3) for i in range(B)]
    ql[B // 2] = ql[0] = S
    c = Case(Hq, H, 128, BF, f8, n, S, ql)
    assert workspace(c) > 0 and B * -(-S * Hq // H // 128) > 64
    c.run()
    c.check("more units")
    c.run(window=400, sinks=20)
    c.check("more units, windows", window=400, sinks=20)


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("B,Hq,H,S", [(64, 8, 2, 200), (12, 8, 2, 200), (200, 8, 2, 4)])
def test_a_chunk_among_tokens(B, Hq, H, S, f8):
    """A chunk, a single token at the end of a long context and single tokens of short ones, in one call: with tiles that
    are split, and with so many padded ones that they are not."""
    n = [1 + (29 * i) % 200 for i in range(B)]
    n[1], n[B - 2] = S + 300, 2500
    ql = [1] * B
    ql[1], ql[5] = S, 0
    c = Case(Hq, H, 64, BF, f8, n, S, ql)
    c.q[5] = float("nan")
    c.run()
    c.check("mixed")
