"""K's and V's 8-bit pages in one pool."""
import math

import pytest
import torch

from genllm_amd import paged
from test_batch_refusals import INV, pages, refused
from test_gpu_pages_f8 import BF, HF, Pages, rows


def one_pool(B, P, H, D, layout, scales):
    """Pages whose tables name different blocks of one pool, with one array of scales or two."""
    p = Pages(B, 2 * P, H, D, layout, seed=D)
    both = p.ids[0]
    p.ids = [both[:, :P], both[:, P:]]
    p.dev = [both.cuda()[:, :P], both.cuda()[:, P:]]
    p.pools[1], p.want[1] = p.pools[0], p.want[0]
    if scales == 1:
        p.scales[1], p.exps[1] = p.scales[0], p.exps[0]
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scales", [1, 2])
@pytest.mark.parametrize("H,D,layout", [(3, 128, "head"), (2, 64, "token"), (2, 256, "head")])
def test_prompts_and_tokens(H, D, layout, scales, dtype):
    p = one_pool(3, 5, H, D, layout, scales)
    start, lens = [0, 16, 5], [40, 33, 17]
    p.write(rows(3, 40, H, D, dtype, 1), rows(3, 40, H, D, dtype, 2, 0.1), start, lens)
    p.check("prompts")
    at = [a + n for a, n in zip(start, lens)]
    for step in range(18):
        p.write(rows(3, 1, H, D, dtype, 10 + step), rows(3, 1, H, D, dtype, 40 + step, 0.1), at)
        p.check(f"token {step}")
        at = [a + 1 for a in at]
    p.read([0, 3, 16], 37, dtype, [37, 20, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 30])
def test_attention(S):
    """The same rows in one pool and in two are attended alike."""
    H, D, n = 2, 128, [70, 45]
    k, v = rows(2, 70, H, D, BF, 1), rows(2, 70, H, D, BF, 2)
    q = rows(2, S, 8, D, BF, 3)
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(lens)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(S)).view(2, 10).int().cuda()
    got = []
    for shared in (True, False):
        kp, ks = paged.f8_pool(20, H, D)
        vp, vs = (kp, ks) if shared else paged.f8_pool(20, H, D)
        ids = table[:, :5], table[:, 5:]
        paged.kv_scatter_f8(k, v, kp, vp, ks, vs, *ids, zero, seq_lens=lens)
        out = torch.zeros_like(q)
        paged.paged_attention_batch(q, out, kp, vp, *ids, lens, 1 / math.sqrt(D), k_scales=ks, v_scales=vs)
        torch.cuda.synchronize()
        got.append(out)
    assert bool(got[0].any()) and torch.equal(*got)


@pytest.mark.parametrize("kw,msg", [
    (dict(vp=3 << 30, vpb=16384), b"v_pool overlaps k_pool"), (dict(vp=(3 << 30) + 8192), b"v_pool overlaps k_pool"),
    (dict(vp=3 << 30, vs=(5 << 30) + 20), b"v_scales overlaps k_scales"), (dict(vs=5 << 30), b"v_scales overlaps k_scales"),
    (dict(vp=3 << 30, vs=3 << 30), b"v_scales overlaps k_pool")])
def test_other_overlaps_are_refused(kw, msg):
    refused(pages(**kw), INV, msg)
